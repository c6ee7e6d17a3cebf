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

// eight elements at any element address: one 16-byte access (global memory takes it unaligned), or the `n` (1 .. 7) elements a row ends with
template <typename T> struct Loose8 {
    typedef unsigned short raw __attribute__((ext_vector_type(8)));
    struct __attribute__((packed, aligned(2))) bytes { raw v; };
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float* out) {
    typedef typename Vec8<T>::type V;
    V v;
    if (n >= 8) v = __builtin_bit_cast(V, ((const typename Loose8<T>::bytes*)p)->v);
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
        for (int e = 0; e < 7; ++e)
            if (e < n) v[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = (float)v[e];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float* in) {
    typedef typename Vec8<T>::type V;
    V v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)in[e];
    if (n >= 8) ((typename Loose8<T>::bytes*)p)->v = __builtin_bit_cast(typename Loose8<T>::raw, v);
    else
        for (int e = 0; e < 7; ++e)
            if (e < n) p[e] = v[e];
}

// calls body(T{}) with the element type of a descriptor
#define MV_DISPATCH_TYPE(dtype, ...)                         \
    do {                                                     \
        if ((dtype) == MV_F16) { typedef half_t T; __VA_ARGS__; } \
        else { typedef bf16_t T; __VA_ARGS__; }              \
    } while (0)
