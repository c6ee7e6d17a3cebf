// tokens.h -- shared helpers of the token-transformer kernels.
#pragma once
#include "../common.h"
#include "../../../include/musev_tokens.h"

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
    typedef raw anywhere __attribute__((aligned(2)));
};
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type load8_raw(const T* p, int n) {
    typedef typename Vec8<T>::type V;
    V v;
    if (n >= 8) v = __builtin_bit_cast(V, ((const typename Loose8<T>::bytes*)p)->v);
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
        for (int e = 0; e < 7; ++e)
            if (e < n) v[e] = p[e];
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float* out) {
    const typename Vec8<T>::type v = load8_raw(p, n);
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

// load8 past the caches: for inputs that they cannot hold (`cold`, uniform)
template <typename T>
__device__ __forceinline__ void load8_from(const T* p, int n, float* out, bool cold) {
    if (cold && n >= 8) {
        const typename Vec8<T>::type v = __builtin_bit_cast(typename Vec8<T>::type, __builtin_nontemporal_load((const typename Loose8<T>::anywhere*)p));
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = (float)v[e];
    } else load8(p, n, out);
}
constexpr int64_t COLD_BYTES = 256ll << 20;   // the last-level cache

// store8 of a result that the caches need not keep for this kernel (non-temporal: the gated norm of 53 248 x 1280 130 -> 112 us)
template <typename T>
__device__ __forceinline__ void store8_stream(T* p, int n, const float* in) {
    typedef typename Vec8<T>::type V;
    if (n >= 8) {
        V v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)in[e];
        __builtin_nontemporal_store(__builtin_bit_cast(typename Loose8<T>::raw, v), (typename Loose8<T>::anywhere*)p);
    } else store8(p, n, in);
}

// sums over 16 lanes (cross-lane moves of the VALU) and over a wave (two exchanges more)
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lanes16_sum(float v) {
    v += lane_move<0xB1>(v);    // lanes 1 0 3 2 of a quad
    v += lane_move<0x4E>(v);    // lanes 2 3 0 1
    v += lane_move<0x141>(v);   // mirrored within 8
    v += lane_move<0x140>(v);   // mirrored within 16
    return v;
}
__device__ __forceinline__ float wave_sum_fast(float v) {
    v = lanes16_sum(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}

// a launch has fewer than 2^32 work items
#define MV_REQUIRE_GRID(name, blocks, threads) \
    MV_REQUIRE((int64_t)(blocks) * (threads) < (1ll << 32), "%s: %ld blocks of %d threads (a launch has fewer than 2^32 work items)", name, (long)(blocks), (int)(threads))

// calls body(T{}) with the element type of a descriptor
#define MV_DISPATCH_TYPE(dtype, ...)                         \
    do {                                                     \
        if ((dtype) == MV_F16) { typedef half_t T; __VA_ARGS__; } \
        else { typedef bf16_t T; __VA_ARGS__; }              \
    } while (0)
