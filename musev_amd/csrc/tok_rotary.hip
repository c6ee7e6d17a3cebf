// tok_rotary.hip -- rotary positions with several axes (include/musev_tokens.h: mv_rotary_axes).
#include "tok_common.h"

// The angle of a pair is position * turns full turns.  It is formed in fp64: at position 131072 an fp32 product of the two is off by
// up to 2^-7 turns, while the fp64 product keeps its fraction of a turn to 2^-35; only that fraction goes on in fp32.
__device__ __forceinline__ void turn_sincos(double pos, double turns, float* s, float* c) {
    const double t = pos * turns;
    sincospif(2.0f * (float)(t - rint(t)), s, c);
}

template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(const mv_rotary_desc p) {
    const int all = p.heads + (p.k ? p.kv_heads : 0);
    const int tail = p.d - 2 * p.pairs, per_head = p.pairs + tail;
    const int64_t total = p.tokens * all * per_head;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t tok = i / (all * per_head);
        const int r = (int)(i - tok * (all * per_head));
        const int head = r / per_head, e = r - head * per_head;
        const bool isk = head >= p.heads;
        const T* in = isk ? (const T*)p.k + tok * p.ldk + (head - p.heads) * p.d : (const T*)p.q + tok * p.ldq + head * p.d;
        T* out = isk ? (T*)p.out_k + tok * p.ldok + (head - p.heads) * p.d : (T*)p.out_q + tok * p.ldoq + head * p.d;
        if (e >= p.pairs) {
            out[p.pairs + e] = in[p.pairs + e];
            continue;
        }
        const int64_t at = tok * p.ldp + p.axis[e];
        const double pos = p.positions_f32 ? (double)((const float*)p.positions)[at] : (double)((const int32_t*)p.positions)[at];
        float sn, cs;
        turn_sincos(pos, p.turns[e], &sn, &cs);
        const int ia = p.halves ? e : 2 * e, ib = p.halves ? e + p.pairs : 2 * e + 1;
        const float a = (float)in[ia], b = (float)in[ib];
        out[ia] = (T)(a * cs - b * sn);
        out[ib] = (T)(a * sn + b * cs);
    }
}

extern "C" int mv_rotary_axes(const mv_rotary_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_rotary_axes: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_rotary_axes: element type %d", d->dtype);
    MV_REQUIRE(d->tokens >= 0 && d->heads >= 1 && d->d >= 2 && d->d <= 1024 && d->pairs >= 1 && 2 * d->pairs <= d->d && d->axes >= 1,
               "mv_rotary_axes: tokens %ld, heads %d, d %d, pairs %d, axes %d", (long)d->tokens, d->heads, d->d, d->pairs, d->axes);
    MV_REQUIRE(!d->k || d->kv_heads >= 1, "mv_rotary_axes: kv_heads %d", d->kv_heads);
    MV_REQUIRE((int64_t)(d->heads + (d->k ? d->kv_heads : 0)) * d->d <= (1 << 24), "mv_rotary_axes: more than 2^24 elements per token");
    if (d->tokens == 0) return MV_OK;
    MV_REQUIRE(d->q && d->out_q && d->positions && d->turns && d->axis && (!d->k || d->out_k), "mv_rotary_axes: null pointer");
    const int64_t work = d->tokens * (d->heads + (d->k ? d->kv_heads : 0)) * (d->d - d->pairs);
    const int64_t want = (work + 255) / 256;
    const int grid = (int)(want < 16384 ? want : 16384);
    MV_DISPATCH_TYPE(d->dtype, (rotary_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(*d)));
    MV_CHECK_LAUNCH("mv_rotary_axes");
    return MV_OK;
}
