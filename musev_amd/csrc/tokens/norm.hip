// tokens/norm.hip -- the gated residual norm (include/musev_tokens.h: mv_gated_residual_norm).
#include "tokens.h"

// sums over a row held by 16 or 32 lanes, a wave or four waves
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
    if constexpr (LANES == 16) v = lanes16_sum(v);
    else if constexpr (LANES == 32) {
        v = lanes16_sum(v);
        v += __shfl_xor(v, 16, 64);
    } else v = wave_sum_fast(v);
    if constexpr (LANES > 64) {
        __syncthreads();   // (the previous sum's readers are through)
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; ++w) v += red[w];
    }
    return v;
}

// A row stays in registers from its one read to its one write: NV chunks of 8 columns per lane, LANES lanes per row, 256 / LANES rows per
// block.  Both norms' statistics are formed in two passes over the registers (mean, then squared deviations), in fp32.  Bound by memory:
// x and f in, s and h out.
template <typename T, int NV, int LANES>
__global__ __launch_bounds__(256) void gated_norm_kernel(const mv_gated_norm_desc p, const bool cold) {
    __shared__ float red[4];
    const int lane = threadIdx.x % LANES, c = p.c;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= p.rows) return;   // (all lanes of a row; with four waves per row the grid is exact)
    T* so = (T*)p.stream_out + row * p.lds;
    T* ho = (T*)p.norm_out + row * p.ldh;
    const int64_t g = p.group_index ? (int64_t)p.group_index[row] : p.rows_per_group > 0 ? (int64_t)((unsigned)row / (unsigned)p.rows_per_group) : 0;
    if (g < 0 || g >= p.groups) {
        for (int i = lane; i < c; i += LANES) {
            so[i] = (T)NAN;
            if (p.norm_out) ho[i] = (T)NAN;
        }
        return;
    }
    const T* x = (const T*)p.x + row * p.ldx;
    const T* f = (const T*)p.f + row * p.ldf;
    float s[NV][8], y[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (j * LANES + lane) * 8;
        if (col < c) {
            load8_from(f + col, c - col, y[j], cold);
            load8_from(x + col, c - col, s[j], cold);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] = s[j][e] = 0.f;
        }
    }
    const float inv_c = 1.0f / (float)c;
    // mean and 1 / sqrt(mean square deviation + eps) of a row in registers (columns past c hold 0)
    auto statistics = [&](const float (&v)[NV][8], float eps, float& mean, float& rstd) __attribute__((always_inline)) {
        mean = 0.f;
        if (p.layer) {
            float t = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) t += v[j][e];
            mean = row_sum<LANES>(t, red) * inv_c;
        }
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (j * LANES + lane) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = col + e < c ? v[j][e] - mean : 0.f;
                t = __builtin_fmaf(d, d, t);
            }
        }
        rstd = 1.0f / sqrtf(row_sum<LANES>(t, red) * inv_c + eps);
    };
    float mean, rstd;
    if (p.post) statistics(y, p.post_eps, mean, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (j * LANES + lane) * 8;
        if (col >= c) continue;
        if (p.post) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] = (y[j][e] - mean) * rstd;
            if (p.post_gamma) {
                float w[8];
                load8((const T*)p.post_gamma + col, c - col, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[j][e] *= w[e];
            }
            if (p.post_beta) {
                float w[8];
                load8((const T*)p.post_beta + col, c - col, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[j][e] += w[e];
            }
        }
        if (p.gate) {
            float w[8];
            load8((const T*)p.gate + g * p.ldg + col, c - col, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] *= w[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = col + e < c ? __builtin_fmaf(p.alpha, s[j][e], y[j][e]) : 0.f;
        store8_stream(so + col, c - col, s[j]);
    }
    if (!p.norm_out) return;
    statistics(s, p.pre_eps, mean, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (j * LANES + lane) * 8;
        if (col >= c) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = (s[j][e] - mean) * rstd;
        float w[8];
        if (p.pre_gamma) {
            load8((const T*)p.pre_gamma + col, c - col, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[j][e] *= w[e];
        }
        if (p.pre_beta) {
            load8((const T*)p.pre_beta + col, c - col, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[j][e] += w[e];
        }
        if (p.scale) {
            load8((const T*)p.scale + g * p.ldsc + col, c - col, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[j][e] = __builtin_fmaf(s[j][e], w[e], s[j][e]);
        }
        if (p.shift) {
            load8((const T*)p.shift + g * p.ldsh + col, c - col, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[j][e] += w[e];
        }
        store8_stream(ho + col, c - col, s[j]);
    }
}

template <typename T, int NV, int LANES>
static int launch_norm(const mv_gated_norm_desc* d, hipStream_t st) {
    constexpr int R = 256 / LANES;
    const int64_t blocks = (d->rows + R - 1) / R;
    MV_REQUIRE_GRID("mv_gated_residual_norm", blocks, 256);
    // (53 248 x 1280, 273 MB of inputs: 123 -> 113 us where other work ran in between; 26 624 x 1280, half of that and still in the cache: 57 -> 65)
    const bool cold = d->rows * d->c * 4 > COLD_BYTES;
    gated_norm_kernel<T, NV, LANES><<<(unsigned)blocks, 256, 0, st>>>(*d, cold);
    MV_CHECK_LAUNCH("mv_gated_residual_norm");
    return MV_OK;
}

// A wave holds a row of up to 1536 columns where there are rows enough to fill the chip; the block's four waves share it otherwise.  Measured (us,
// rms, both norms, one / four waves per row): 1 x 1280 6.3 / 3.9; 1024 x 1280 7.9 / 5.6; 2048 x 640 6.5 / 6.8; 4099 x 1001 11.3 / 13.1; 16 000 x 1280
// 37 / 41; 16 000 x 2048 55 / 47.  Narrow rows share a wave (layer, indexed groups; a wave per row / shared): 37 590 x 44 40.4 / 14.7; 50 000 x 128 32.6 /
// 11.8; 1 x 128 3.7 / 3.6; 20 000 x 200 16.2 / 9.7; 200 x 256 4.3 / 4.2; with several chunks per lane only where rows are many: 20 000 x 320 17.5 / 13.8,
// 100 000 x 512 80 / 70, but 2000 x 320 5.2 / 7.7, 4000 x 512 6.5 / 7.3.
template <typename T>
static int launch_norm_width(const mv_gated_norm_desc* d, hipStream_t st) {
    const int c = d->c;
    if (c <= 128) return launch_norm<T, 1, 16>(d, st);
    if (c <= 256) return launch_norm<T, 1, 32>(d, st);
    if (c <= 384 && d->rows > 16384) return launch_norm<T, 3, 16>(d, st);
    if (c <= 512 && d->rows > 16384) return launch_norm<T, 2, 32>(d, st);
    if (c <= 512) return launch_norm<T, 1, 64>(d, st);
    if (c > 1536 ? c <= 2048 : d->rows <= 2048) return launch_norm<T, 1, 256>(d, st);
    if (c <= 1024) return launch_norm<T, 2, 64>(d, st);
    if (c <= 1536) return launch_norm<T, 3, 64>(d, st);
    if (c <= 4096) return launch_norm<T, 2, 256>(d, st);
    if (c <= 8192) return launch_norm<T, 4, 256>(d, st);
    return launch_norm<T, 8, 256>(d, st);
}

extern "C" int mv_gated_residual_norm(const mv_gated_norm_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_gated_residual_norm: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_gated_residual_norm: element type %d", d->dtype);
    MV_REQUIRE(d->c >= 1 && d->c <= 16384, "mv_gated_residual_norm: %d columns (1 .. 16384)", d->c);
    MV_REQUIRE(d->rows >= 0 && d->rows < (1ll << 31) && d->groups >= 1, "mv_gated_residual_norm: %ld rows, %ld groups", (long)d->rows, (long)d->groups);
    MV_REQUIRE(d->rows_per_group >= 0 && d->rows_per_group < (1ll << 31), "mv_gated_residual_norm: groups of %ld rows", (long)d->rows_per_group);
    if (d->rows == 0) return MV_OK;
    MV_REQUIRE(d->x && d->f && d->stream_out, "mv_gated_residual_norm: null pointer");
    MV_DISPATCH_TYPE(d->dtype, return launch_norm_width<T>(d, (hipStream_t)stream));
}
