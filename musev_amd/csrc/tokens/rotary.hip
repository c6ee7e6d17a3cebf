// tokens/rotary.hip -- rotary positions with several axes (include/musev_tokens.h: mv_rotary_axes).
#include "tokens.h"

// The angle of a pair is position * turns full turns.  It is formed in fp64: at position 131072 an fp32 product of the two is off by
// up to 2^-7 turns, while the fp64 product keeps its fraction of a turn to 2^-35; only that fraction goes on in fp32.
__device__ __forceinline__ void turn_sincos(double pos, double turns, float* s, float* c) {
    const double t = pos * turns;
    sincospif(2.0f * (float)(t - rint(t)), s, c);
}

// n / d for n * d < 2^32 as one high product, m = ceil(2^32 / d)
struct Div {
    unsigned d, m;
};
static Div make_div(unsigned d) { return Div{d, d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d)}; }
__device__ __forceinline__ unsigned div_of(unsigned n, Div v) { return v.d == 1 ? n : __umulhi(n, v.m); }

struct RotaryArgs {
    mv_rotary_desc p;
    Div per_token, per_head, pairs;   // work items of a token, of a head
    int rot_items, tokens_per_block;  // items of a head that turn (the others copy what passes through)
    bool large, cold;                 // results, inputs past the caches
};

// A block owns a few tokens: their sines and cosines go to LDS once, shared by all heads, then every thread takes work items of 8 elements
// (adjacent pairs: 4 pairs; halves: 8 + 8 elements) with 16-byte accesses.  Bound by memory: q and k in and out.
template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 turn[];   // [token][pair] {sin, cos}
    const mv_rotary_desc& p = a.p;
    const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int n_tok = (int)min((int64_t)a.tokens_per_block, p.tokens - tok0);
    for (unsigned i = threadIdx.x; i < (unsigned)(n_tok * p.pairs); i += 256) {
        const unsigned t = div_of(i, a.pairs), pr = i - t * p.pairs;
        const int64_t at = (tok0 + t) * p.ldp + p.axis[pr];
        const double pos = p.positions_f32 ? (double)((const float*)p.positions)[at] : (double)((const int32_t*)p.positions)[at];
        float sn, cs;
        turn_sincos(pos, p.turns[pr], &sn, &cs);
        turn[i] = float2{sn, cs};
    }
    __syncthreads();
    const unsigned total = n_tok * a.per_token.d;
    auto put = [&](T* to, int n, const float* v) __attribute__((always_inline)) {
        if (a.large) store8_stream(to, n, v);
        else store8(to, n, v);
    };
    for (unsigned i = threadIdx.x; i < total; i += 256) {
        const unsigned t = div_of(i, a.per_token), r = i - t * a.per_token.d;
        const unsigned head = div_of(r, a.per_head), e = r - head * a.per_head.d;
        const int64_t tok = tok0 + t;
        const bool isk = head >= (unsigned)p.heads;
        const T* in = isk ? (const T*)p.k + tok * p.ldk + (int)(head - p.heads) * p.d : (const T*)p.q + tok * p.ldq + (int)head * p.d;
        T* out = isk ? (T*)p.out_k + tok * p.ldok + (int)(head - p.heads) * p.d : (T*)p.out_q + tok * p.ldoq + (int)head * p.d;
        if (e >= (unsigned)a.rot_items) {   // what passes through
            const int at = 2 * p.pairs + (int)(e - a.rot_items) * 8, n = p.d - at;
            float v[8];
            load8(in + at, n, v);
            put(out + at, n, v);
            continue;
        }
        const float2* tr = turn + t * p.pairs;
        if constexpr (HALVES) {
            const int pr = (int)e * 8, n = p.pairs - pr;
            float u[8], w[8];
            load8_from(in + pr, n, u, a.cold);
            load8_from(in + p.pairs + pr, n, w, a.cold);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const float2 sc = tr[min(pr + x, p.pairs - 1)];
                const float x0 = u[x], y0 = w[x];
                u[x] = x0 * sc.y - y0 * sc.x;
                w[x] = x0 * sc.x + y0 * sc.y;
            }
            put(out + pr, n, u);
            put(out + p.pairs + pr, n, w);
        } else {
            const int pr = (int)e * 4, n = 2 * (p.pairs - pr);
            float u[8];
            load8_from(in + 2 * pr, n, u, a.cold);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 sc = tr[min(pr + x, p.pairs - 1)];
                const float x0 = u[2 * x], y0 = u[2 * x + 1];
                u[2 * x] = x0 * sc.y - y0 * sc.x;
                u[2 * x + 1] = x0 * sc.x + y0 * sc.y;
            }
            put(out + 2 * pr, n, u);
        }
    }
}

extern "C" int mv_rotary_axes(const mv_rotary_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_rotary_axes: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_rotary_axes: element type %d", d->dtype);
    MV_REQUIRE(d->tokens >= 0 && d->heads >= 1 && d->d >= 2 && d->d <= 1024 && d->pairs >= 1 && 2 * d->pairs <= d->d && d->axes >= 1,
               "mv_rotary_axes: tokens %ld, heads %d, d %d, pairs %d, axes %d", (long)d->tokens, d->heads, d->d, d->pairs, d->axes);
    MV_REQUIRE(!d->k || d->kv_heads >= 1, "mv_rotary_axes: kv_heads %d", d->kv_heads);
    MV_REQUIRE((int64_t)(d->heads + (d->k ? d->kv_heads : 0)) * d->d <= (1 << 17), "mv_rotary_axes: more than 2^17 elements per token");
    if (d->tokens == 0) return MV_OK;
    MV_REQUIRE(d->q && d->out_q && d->positions && d->turns && d->axis && (!d->k || d->out_k), "mv_rotary_axes: null pointer");
    RotaryArgs a;
    a.p = *d;
    const int heads = d->heads + (d->k ? d->kv_heads : 0), tail = d->d - 2 * d->pairs;
    a.rot_items = d->halves ? (d->pairs + 7) / 8 : (d->pairs + 3) / 4;
    a.per_head = make_div(a.rot_items + (tail + 7) / 8);
    a.per_token = make_div((unsigned)heads * a.per_head.d);
    a.pairs = make_div(d->pairs);
    MV_REQUIRE(a.per_token.d < 32768, "mv_rotary_axes: %u work items per token (below 32768)", a.per_token.d);   // (div_of's range)
    // As many tokens per block (up to 8) as give its 256 threads two work items each, but at least 1024 blocks.  Measured (us, 1 / 2 / 4 / 8 tokens):
    // 53 248 tokens of 512 items 147 / 153 / 161 / 165; 26 624 of 160 46.9 / 41.8 / 42.3 / 44.9; 16 384 of 16 10.7 / 6.9 / 5.2 / 4.4; 512 of 320 4.5 /
    // 5.0 / 6.5 / 10.2.
    a.tokens_per_block = 1;
    while (a.tokens_per_block < 8 && a.tokens_per_block * a.per_token.d < 512 && d->tokens >= 1024 * 2 * a.tokens_per_block) a.tokens_per_block *= 2;
    // non-temporal results from 64 MB on: 26 624 tokens x 20 heads x 128 (136 MB) 47.4 -> 42.4 us, 13 312 x 16 x 80 (34 MB) 15.5 -> 20.8
    a.large = d->tokens * heads * d->d * 2 > (64ll << 20);
    a.cold = d->tokens * heads * d->d * 2 > COLD_BYTES;   // (53 248 x 32 heads x 128: 146 -> 143 us)
    const int64_t grid = (d->tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    MV_REQUIRE_GRID("mv_rotary_axes", grid, 256);
    const size_t lds = (size_t)a.tokens_per_block * d->pairs * sizeof(float2);
    if (d->halves) MV_DISPATCH_TYPE(d->dtype, (rotary_kernel<T, true><<<(unsigned)grid, 256, lds, (hipStream_t)stream>>>(a)));
    else MV_DISPATCH_TYPE(d->dtype, (rotary_kernel<T, false><<<(unsigned)grid, 256, lds, (hipStream_t)stream>>>(a)));
    MV_CHECK_LAUNCH("mv_rotary_axes");
    return MV_OK;
}
