// tok_linear.hip -- the int8 projection (include/musev_tokens.h: mv_quantize_rows_i8, mv_gemm_i8).
#include "tok_common.h"

// ---- activations to int8, one scale per row ------------------------------------------------------------------------------------
// code = rne(127 x / top) with top = max |x|: 127 x is exact in fp32 for 16-bit inputs and a correctly rounded quotient of an 18-bit and
// an 11-bit number is never rounded ONTO a tie (a value that is no tie is at least 2^-12 away from one, the quotient's half step is
// 2^-18), so the code is that of the exact quotient.  f (a power of two) keeps 127 x of bf16's largest and smallest values in range.
struct RowScale {
    float f, den, scale;
    bool finite;
};
__device__ __forceinline__ RowScale row_scale(unsigned top_bits) {
    RowScale r;
    const float top = __uint_as_float(top_bits);
    r.finite = top_bits < 0x7f800000u;
    r.f = top > 0x1p100f ? 0x1p-32f : top < 0x1p-80f ? 0x1p64f : 1.0f;
    r.den = top > 0.f && r.finite ? top * r.f : 1.0f;
    r.scale = top / 127.0f;
    return r;
}
__device__ __forceinline__ int row_code(float x, const RowScale& r) { return r.finite ? (int)rintf(127.0f * (x * r.f) / r.den) : 0; }

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int64_t ldx, int k, int8_t* codes, int64_t ldc, float* scale) {
    __shared__ unsigned red[4];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    unsigned top = 0;   // |x| as bits: ordered like the values, NaN above infinity
    for (int i = threadIdx.x; i < k; i += 256) top = max(top, __float_as_uint((float)xr[i]) & 0x7fffffffu);
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    const RowScale r = row_scale(top);
    if (threadIdx.x == 0) scale[row] = r.scale;
    for (int i = threadIdx.x; i < ldc; i += 256) codes[row * ldc + i] = i < k ? (int8_t)row_code((float)xr[i], r) : (int8_t)0;
}

extern "C" int mv_quantize_rows_i8(const void* x, int64_t ldx, int64_t rows, int32_t k, int32_t dtype, int8_t* codes, int64_t ldc, float* scale,
                                   void* stream) {
    MV_REQUIRE(dtype == MV_F16 || dtype == MV_BF16, "mv_quantize_rows_i8: element type %d", dtype);
    MV_REQUIRE(rows >= 0 && rows < (1ll << 31) && k >= 1 && k <= 131072, "mv_quantize_rows_i8: %ld rows of %d (1 .. 131072)", (long)rows, k);
    MV_REQUIRE(ldc % 128 == 0 && ldc >= k && ldc < k + 128, "mv_quantize_rows_i8: code rows of %ld for k = %d (k rounded up to 128)", (long)ldc, k);
    if (rows == 0) return MV_OK;
    MV_REQUIRE(x && codes && scale && ((uintptr_t)codes & 15) == 0, "mv_quantize_rows_i8: null or unaligned pointer");
    MV_DISPATCH_TYPE(dtype, (quantize_rows_kernel<T><<<(unsigned)rows, 256, 0, (hipStream_t)stream>>>((const T*)x, ldx, k, codes, ldc, scale)));
    MV_CHECK_LAUNCH("mv_quantize_rows_i8");
    return MV_OK;
}

// ---- the product ---------------------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void store_i8_result(const mv_gemm_i8_desc& p, int64_t m, int n, int acc) {
    float v = p.a_scale[m] * p.w_scale[n] * (float)acc;
    if (p.bias) v += (float)((const T*)p.bias)[n];
    if (p.act == MV_ACT_SILU) v = mv_silu(v);
    if (p.residual) v += (float)((const T*)p.residual)[m * p.ldr + n];
    ((T*)p.out)[m * p.ldo + n] = (T)v;
}

template <typename T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const mv_gemm_i8_desc p) {
    const int n = blockIdx.x * 16 + (threadIdx.x & 15);
    for (int64_t m = (int64_t)blockIdx.y * 16 + (threadIdx.x >> 4); m < p.M; m += (int64_t)gridDim.y * 16) {
        if (n >= p.N) continue;
        const int4* a = (const int4*)(p.a + m * p.lda);
        const int4* w = (const int4*)(p.w + (int64_t)n * p.ldw);
        int acc = 0;
        for (int i = 0; i < p.kp / 16; ++i) {
            const int4 u = a[i], v = w[i];
            acc = __builtin_amdgcn_sdot4(u.x, v.x, acc, false);
            acc = __builtin_amdgcn_sdot4(u.y, v.y, acc, false);
            acc = __builtin_amdgcn_sdot4(u.z, v.z, acc, false);
            acc = __builtin_amdgcn_sdot4(u.w, v.w, acc, false);
        }
        store_i8_result<T>(p, m, n, acc);
    }
}

extern "C" int mv_gemm_i8(const mv_gemm_i8_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_gemm_i8: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_gemm_i8: element type %d", d->dtype);
    MV_REQUIRE(d->act == MV_ACT_NONE || d->act == MV_ACT_SILU, "mv_gemm_i8: activation %d", d->act);
    MV_REQUIRE(d->M >= 0 && d->M < (1ll << 31) && d->N >= 1 && d->kp >= 128 && d->kp % 128 == 0 && d->kp <= 131072,
               "mv_gemm_i8: M %ld, N %d, kp %d (a multiple of 128 up to 131072)", (long)d->M, d->N, d->kp);
    MV_REQUIRE(d->lda % 128 == 0 && d->ldw % 128 == 0 && d->lda >= d->kp && d->ldw >= d->kp, "mv_gemm_i8: lda %ld, ldw %ld for kp %d", (long)d->lda,
               (long)d->ldw, d->kp);
    if (d->M == 0) return MV_OK;
    MV_REQUIRE(d->a && d->w && d->a_scale && d->w_scale && d->out, "mv_gemm_i8: null pointer");
    MV_REQUIRE((((uintptr_t)d->a | (uintptr_t)d->w) & 15) == 0, "mv_gemm_i8: codes must be 16-byte aligned");
    const int64_t mt = (d->M + 15) / 16;
    const dim3 grid((d->N + 15) / 16, (unsigned)(mt < 32768 ? mt : 32768));
    MV_DISPATCH_TYPE(d->dtype, (gemm_i8_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(*d)));
    MV_CHECK_LAUNCH("mv_gemm_i8");
    return MV_OK;
}
