// tok_norm.hip -- the gated residual norm (include/musev_tokens.h: mv_gated_residual_norm).
#include "tok_common.h"

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// one block per row, the row's fp32 values in LDS
template <typename T>
__global__ __launch_bounds__(256) void gated_norm_kernel(const mv_gated_norm_desc p) {
    extern __shared__ __attribute__((aligned(16))) float row_s[];
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const int c = p.c, tid = threadIdx.x;
    const T* x = (const T*)p.x + row * p.ldx;
    const T* f = (const T*)p.f + row * p.ldf;
    T* so = (T*)p.stream_out + row * p.lds;
    T* ho = (T*)p.norm_out + row * p.ldh;
    const int64_t g = p.group_index ? (int64_t)p.group_index[row] : p.rows_per_group > 0 ? row / p.rows_per_group : 0;
    if (g < 0 || g >= p.groups) {
        for (int i = tid; i < c; i += 256) {
            so[i] = (T)NAN;
            if (p.norm_out) ho[i] = (T)NAN;
        }
        return;
    }
    const T* gate = p.gate ? (const T*)p.gate + g * p.ldg : nullptr;
    float mean = 0.f, rstd = 1.f;
    if (p.post) {
        if (p.layer) {
            float s = 0.f;
            for (int i = tid; i < c; i += 256) s += (float)f[i];
            mean = block_sum(s, red) / c;
        }
        float s = 0.f;
        for (int i = tid; i < c; i += 256) {
            const float v = (float)f[i] - mean;
            s += v * v;
        }
        rstd = rsqrtf(block_sum(s, red) / c + p.post_eps);
    }
    float sum = 0.f;
    for (int i = tid; i < c; i += 256) {
        float y = (float)f[i];
        if (p.post) {
            y = (y - mean) * rstd;
            if (p.post_gamma) y *= (float)((const T*)p.post_gamma)[i];
            if (p.post_beta) y += (float)((const T*)p.post_beta)[i];
        }
        const float s = p.alpha * (float)x[i] + (gate ? (float)gate[i] * y : y);
        row_s[i] = s;
        sum += s;
    }
    mean = 0.f;
    if (p.norm_out) {
        if (p.layer) mean = block_sum(sum, red) / c;
        float s = 0.f;
        for (int i = tid; i < c; i += 256) {
            const float v = row_s[i] - mean;
            s += v * v;
        }
        rstd = rsqrtf(block_sum(s, red) / c + p.pre_eps);
    }
    __syncthreads();   // (stream_out may be x or f: every read of the row is done)
    for (int i = tid; i < c; i += 256) {
        const float s = row_s[i];
        so[i] = (T)s;
        if (p.norm_out) {
            float h = (s - mean) * rstd;
            if (p.pre_gamma) h *= (float)((const T*)p.pre_gamma)[i];
            if (p.pre_beta) h += (float)((const T*)p.pre_beta)[i];
            if (p.scale) h *= 1.0f + (float)((const T*)p.scale)[g * p.ldsc + i];
            if (p.shift) h += (float)((const T*)p.shift)[g * p.ldsh + i];
            ho[i] = (T)h;
        }
    }
}

extern "C" int mv_gated_residual_norm(const mv_gated_norm_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_gated_residual_norm: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_gated_residual_norm: element type %d", d->dtype);
    MV_REQUIRE(d->c >= 1 && d->c <= 16384, "mv_gated_residual_norm: %d columns (1 .. 16384)", d->c);
    MV_REQUIRE(d->rows >= 0 && d->rows < (1ll << 31) && d->groups >= 1, "mv_gated_residual_norm: %ld rows, %ld groups", (long)d->rows, (long)d->groups);
    if (d->rows == 0) return MV_OK;
    MV_REQUIRE(d->x && d->f && d->stream_out, "mv_gated_residual_norm: null pointer");
    MV_DISPATCH_TYPE(d->dtype, (gated_norm_kernel<T><<<(unsigned)d->rows, 256, d->c * 4, (hipStream_t)stream>>>(*d)));
    MV_CHECK_LAUNCH("mv_gated_residual_norm");
    return MV_OK;
}
