// tok_common.h -- shared helpers of the token-transformer kernels (tok_*.hip).
#pragma once
#include "common.h"
#include "../../include/musev_tokens.h"

typedef __bf16 bf16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// eight 16-bit elements of either type
template <typename T> struct Vec8;
template <> struct Vec8<half_t> { typedef half8v type; };
template <> struct Vec8<bf16_t> { typedef bf16x8 type; };

// calls body(T{}) with the element type of a descriptor
#define MV_DISPATCH_TYPE(dtype, ...)                         \
    do {                                                     \
        if ((dtype) == MV_F16) { typedef half_t T; __VA_ARGS__; } \
        else { typedef bf16_t T; __VA_ARGS__; }              \
    } while (0)
