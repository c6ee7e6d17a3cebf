// tok_attention.hip -- packed attention (include/musev_tokens.h: mv_attention_packed).
#include "tok_common.h"

extern "C" int mv_tokens_abi_version(void) { return MV_TOKENS_ABI_VERSION; }

struct PackedItem {
    int q_row, q_len, k_row, kv_len, m0, key_begin, key_end, slot;
};

// one wave per packed row: 64 lanes hold the row's head dim two columns apart, the keys walk one after the other
template <typename T>
__global__ __launch_bounds__(256) void attention_rows_kernel(const mv_attn_packed_desc p) {
    const PackedItem it = ((const PackedItem*)p.items)[blockIdx.x / p.kv_heads];
    const int kvh = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads, lane = threadIdx.x & 63;
    for (int t = threadIdx.x >> 6; t < p.tile_rows; t += 4) {
        const int64_t r = (int64_t)it.m0 + t;
        if (r >= (int64_t)it.q_len * group) break;
        const int i = (int)(r / group), h = kvh * group + (int)(r % group);
        const T* q = (const T*)p.q + (int64_t)(it.q_row + i) * p.ldq + (int64_t)h * p.d;
        const int c0 = lane, c1 = lane + 64;
        const float q0 = c0 < p.d ? (float)q[c0] : 0.f, q1 = c1 < p.d ? (float)q[c1] : 0.f;
        const int64_t seen = p.causal ? (int64_t)i + it.kv_len - it.q_len + 1 : it.kv_len;
        const int end = (int)(seen < it.key_end ? seen : it.key_end);
        float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
        for (int j = it.key_begin; j < end; ++j) {
            const T* k = (const T*)p.k + (int64_t)(it.k_row + j) * p.ldk + (int64_t)kvh * p.d;
            const T* v = (const T*)p.v + (int64_t)(it.k_row + j) * p.ldv + (int64_t)kvh * p.d;
            const float s = p.scale * wave_sum((c0 < p.d ? q0 * (float)k[c0] : 0.f) + (c1 < p.d ? q1 * (float)k[c1] : 0.f));
            const float mn = fmaxf(m, s);
            const float a = m == -INFINITY ? 0.f : __expf(m - mn), e = __expf(s - mn);
            l = l * a + e;
            if (c0 < p.d) o0 = o0 * a + e * (float)v[c0];
            if (c1 < p.d) o1 = o1 * a + e * (float)v[c1];
            m = mn;
        }
        T* o = (T*)p.out + (int64_t)(it.q_row + i) * p.ldo + (int64_t)h * p.d;
        const float inv = seen > 0 ? 1.0f / l : 0.f;
        if (c0 < p.d) o[c0] = (T)(seen > 0 ? o0 * inv : 0.f);
        if (c1 < p.d) o[c1] = (T)(seen > 0 ? o1 * inv : 0.f);
    }
}

extern "C" int64_t mv_attention_packed_workspace_bytes(int32_t n_slots, int32_t kv_heads, int32_t d, int32_t tile_rows) {
    if (n_slots < 0 || kv_heads < 1 || d < 1 || tile_rows < 1) return -1;
    return (int64_t)n_slots * kv_heads * tile_rows * (d + 2) * 4;
}

extern "C" int mv_attention_packed(const mv_attn_packed_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_attention_packed: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_attention_packed: element type %d", d->dtype);
    MV_REQUIRE(d->d >= 8 && d->d <= 128 && d->d % 8 == 0, "mv_attention_packed: head dim %d (a multiple of 8 up to 128)", d->d);
    MV_REQUIRE(d->kv_heads >= 1 && d->heads >= d->kv_heads && d->heads % d->kv_heads == 0, "mv_attention_packed: %d heads over %d key / value heads",
               d->heads, d->kv_heads);
    MV_REQUIRE(d->n_items >= 0 && (int64_t)d->n_items * d->kv_heads < (1ll << 31), "mv_attention_packed: %d items", d->n_items);
    if (d->n_items == 0) return MV_OK;
    MV_REQUIRE(d->q && d->k && d->v && d->out && d->items, "mv_attention_packed: null pointer");
    MV_DISPATCH_TYPE(d->dtype, (attention_rows_kernel<T><<<(unsigned)(d->n_items * d->kv_heads), 256, 0, (hipStream_t)stream>>>(*d)));
    MV_CHECK_LAUNCH("mv_attention_packed");
    return MV_OK;
}
