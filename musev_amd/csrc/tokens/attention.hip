// tokens/attention.hip -- packed attention (include/musev_tokens.h: mv_attention_packed).
//
// One pass over the keys with a running maximum and sum.  A (sequence, key / value head) has q_len * group packed rows, row r = query
// r / group, head r % group of the group: the heads that share keys share the tile that holds them, and one token of a wide group is a
// tile of its own.  Scores are formed transposed, S^T = K Q^T with v_mfma_32x32x16: lane l then owns ONE packed row (column l & 31) and 16
// of every 32 keys (those with bit 2 = l >> 5), so maxima and sums are in-lane up to one exchange between the two half waves, and P^T
// already lies as the second operand of O^T += V^T P^T wants it: the contraction may walk its keys in any order, so step s takes the keys
// in the order the scores' registers hold them (16 s + 4 h + 0..3, 16 s + 8 + 4 h + 0..3 for half h) and V^T is read to match with the
// transposing LDS read (4 keys x 16 columns per 16 lanes).
// K and V tiles go global -> LDS directly (16 bytes per lane).  LDS rows are 128 or 256 bytes; the 16-byte slots of a row are permuted by
// an XOR with row bits, applied to the source column each lane fetches, so that both the 16-byte reads of K (16 rows, one column) and the
// transposing reads of V (4 rows x 64 bytes per half wave) touch every bank once.
// 4 waves x 32 packed rows share 64-key tiles, two stages, one barrier per tile, two blocks per CU: 64 KB on its way per CU, enough to stream the
// cache of a single token too, where one wave alone has rows (a form whose 4 waves walked tiles of their own for up to 32 rows was no faster:
// 16 requests over 86 k keys 82 against 77 us).
#include "tokens.h"

extern "C" int mv_tokens_abi_version(void) { return MV_TOKENS_ABI_VERSION; }

struct PackedItem {
    int q_row, q_len, k_row, kv_len, m0, key_begin, key_end, ws_row;
};
struct PackedJoin {
    int q_row, q_len, kv_len, m0, ws_row, parts, rows, pad;
};

__device__ __forceinline__ float16v mfma_32x32x16(half8v a, half8v b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float16v mfma_32x32x16(bf16x8 a, bf16x8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

template <typename T> struct ExpBits;   // both elements of a dword: exponent mask, and what lifts an all-ones exponent into the sign bit
template <> struct ExpBits<half_t> { static constexpr unsigned mask = 0x7c007c00u, one = 0x04000400u; };
template <> struct ExpBits<bf16_t> { static constexpr unsigned mask = 0x7f807f80u, one = 0x00800080u; };

// a score's factor to powers of two
__device__ __forceinline__ float score_factor(float scale) { return fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f); }

template <bool B> struct Masked { static constexpr bool value = B; };

// K16: 16-column steps of the head dim
template <int K16>
struct PackedCfg {
    static constexpr int RS = K16 <= 4 ? 64 : 128;     // elements per LDS row
    static constexpr int SLOTS = RS / 8;               // 16-byte slots per LDS row
    static constexpr int KT = 64;                      // keys per tile
    static constexpr int TILE = KT * RS;               // elements of a K (or V) tile
    static constexpr int PPW = TILE * 2 / 1024 / 4;    // 1-KiB pieces of it that one wave fetches
    static constexpr int LDS_BYTES = 2 * 2 * TILE * 2; // two stages of K, V
    static constexpr int NS = KT / 32, NB = (K16 + 1) / 2;   // 32-key score blocks of a tile, 32-column blocks of the output
};

// The slot permutation of a row.  K: 16 rows x one slot must fall on 16 different slots of a 256-byte line (two rows of 128 bytes share a
// line).  V: 4 rows x 64 bytes must fall on the 4 different quarters of a line.
template <int RS> __device__ __forceinline__ int swz_k(int row) { return RS == 128 ? (row & 15) : ((row >> 1) & 7); }
template <int RS> __device__ __forceinline__ int swz_v(int row) { return RS == 128 ? ((row & 3) << 2) : (((row >> 1) & 1) << 2); }

template <typename T, int K16>
__global__ __launch_bounds__(256, 2) void attention_packed_kernel(const mv_attn_packed_desc p) {
    using C = PackedCfg<K16>;
    typedef typename Vec8<T>::type V8;
    typedef __attribute__((address_space(3))) T lds_t;
    extern __shared__ __attribute__((aligned(256))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PackedItem it = ((const PackedItem*)p.items)[blockIdx.x / p.kv_heads];
    const int kvh = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
    const int rows = it.q_len * group;
    const int row0 = it.m0 + wave * 32;
    const bool active = row0 < rows;                       // (wave-uniform) the last tile's waves may have no row
    const int r = min(row0 + l31, rows - 1);               // this lane's packed row (padding lanes repeat the last one)
    const int qi = r / group, hq = kvh * group + (r - qi * group);
    const int seen = p.causal ? max(0, qi + it.kv_len - it.q_len + 1) : it.kv_len;
    const int lim = min(seen, it.key_end);                 // this row walks the keys [key_begin, lim)
    const int lim_hi = __builtin_amdgcn_readlane(lim, 31);

    // ---- Q (second operand of S^T): row in the lane, 8 columns per half wave and step; a negative scale turns its sign here ----
    const float c = score_factor(p.scale);
    V8 qf[K16];
    {
        const T* q = (const T*)p.q + (int64_t)(it.q_row + qi) * p.ldq + (int64_t)hq * p.d;
#pragma unroll
        for (int s = 0; s < K16; ++s) {
            const int col = 16 * s + 8 * h;
            u32x4 w = {0, 0, 0, 0};
            if (col < p.d) w = *(const u32x4*)(q + col);
            if (p.scale < 0.f) w ^= 0x80008000u;
            qf[s] = __builtin_bit_cast(V8, w);
        }
    }
    float16v acc[C::NB];
#pragma unroll
    for (int b = 0; b < C::NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
    float m = -3.0e38f / fmaxf(c, 1.0f), l = 0.f;    // reference of the exponents (score units; m * c stays finite), sum of this lane's own keys

    // ---- global -> LDS ----
    lds_t* ring = (lds_t*)((__attribute__((address_space(3))) char*)smem);
    unsigned ok[C::PPW], ov[C::PPW];   // byte offset of this lane's 16 bytes from the tile's first row; columns past d: out of range, read as 0
#pragma unroll
    for (int j = 0; j < C::PPW; ++j) {
        const int at = (wave * C::PPW + j) * 64 + lane;
        const int row = at / C::SLOTS, slot = at % C::SLOTS;
        const int sk = slot ^ swz_k<C::RS>(row), sv = slot ^ swz_v<C::RS>(row);
        ok[j] = sk * 8 < p.d ? (unsigned)((row * p.ldk + sk * 8) * 2) : 0x80000000u;
        ov[j] = sv * 8 < p.d ? (unsigned)((row * p.ldv + sv * 8) * 2) : 0x80000000u;
    }
    const char* kbase = (const char*)((const T*)p.k + (int64_t)it.k_row * p.ldk + (int64_t)kvh * p.d);
    const char* vbase = (const char*)((const T*)p.v + (int64_t)it.k_row * p.ldv + (int64_t)kvh * p.d);
    // tile at key `key` into stage `stage`: the descriptors start at the tile (64-bit address) and end with the sequence's last row, so rows
    // behind it read as 0
    auto issue = [&](int key, int stage) __attribute__((always_inline)) {
        const int left = min(it.kv_len - key, C::KT);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(kbase + (int64_t)key * p.ldk * 2), 0, (unsigned)(((left - 1) * p.ldk + p.d) * 2), 0x00020000);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(vbase + (int64_t)key * p.ldv * 2), 0, (unsigned)(((left - 1) * p.ldv + p.d) * 2), 0x00020000);
        lds_t* dst = ring + stage * 2 * C::TILE + wave * C::PPW * 512;
#pragma unroll
        for (int j = 0; j < C::PPW; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)(dst + j * 512), 16, (int)ok[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < C::PPW; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)(dst + C::TILE + j * 512), 16, (int)ov[j], 0, 0, 0);
    };

    // ---- one tile ----
    const int i16 = lane & 15;
    // A fragment's LDS address is one per lane and operand, its step or block an XOR (slots are permuted by XOR, rows are whole lines) and its
    // rows an immediate offset.  K fragment step k: row l31, slot 2 k + h; V^T fragment block b: keys 4 h + 0..3, columns 32 b.
    const unsigned ka = (unsigned)(l31 * C::RS + (h ^ swz_k<C::RS>(l31)) * 8) * 2;
    const int vrow = 4 * h + (i16 >> 2), vslot = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
    const unsigned va = (unsigned)(vrow * C::RS + (vslot ^ swz_v<C::RS>(vrow)) * 8 + (i16 & 1) * 4) * 2;
    auto compute = [&](int key, int stage, auto tag) __attribute__((always_inline)) {
        constexpr bool masked = decltype(tag)::value;   // some row may not see all of the tile
        // At two waves per SIMD (head dims from 65 on) fragments are read AHEAD matrix instructions before they are used and the order is pinned:
        // left to itself the compiler reads each just before its use and the matrix pipe waits out the LDS latency (d = 128, a causal prompt of 16384:
        // 1.04 -> 1.00 ms).  With more waves the others cover it and the compiler's own order is as good (d = 64, 8192 tokens: 166 against 171 us).
        constexpr bool PINNED = K16 > 4;
        const lds_t* sv = ring + stage * 2 * C::TILE + C::TILE;
        const unsigned kb = (unsigned)(uintptr_t)(ring + stage * 2 * C::TILE) + ka, vb = (unsigned)(uintptr_t)sv + va;
        constexpr int NK = K16 * C::NS, NV = 2 * C::NS * C::NB, AHEAD = PINNED ? 3 : 1;
        auto k_frag = [&](int f) __attribute__((always_inline)) {
            return *(const __attribute__((address_space(3))) V8*)(uintptr_t)((kb ^ (f / C::NS << 5)) + f % C::NS * 32 * C::RS * 2);
        };
        auto v_frag = [&](int f) __attribute__((always_inline)) {
            const unsigned at = (vb ^ (f % C::NB << 6)) + f / C::NB * 16 * C::RS * 2;
            const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(uintptr_t)at);
            const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(uintptr_t)(at + 8 * C::RS * 2));
            typedef short short8v __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(V8, short8v{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
        };
        float16v s[C::NS];
#pragma unroll
        for (int n = 0; n < C::NS; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = 0.f;
        V8 kf[NK], vf[NV];
#pragma unroll
        for (int f = 0; f < AHEAD && f < NK; ++f) kf[f] = k_frag(f);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < NK; ++f) {
            if constexpr (PINNED) __builtin_amdgcn_sched_barrier(0);
            s[f % C::NS] = mfma_32x32x16(kf[f], qf[f / C::NS], s[f % C::NS]);
            if (f + AHEAD < NK) kf[f + AHEAD] = k_frag(f + AHEAD);
        }
        if constexpr (PINNED) __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        if constexpr (masked) {
            const int left = lim - key - 4 * h;
#pragma unroll
            for (int n = 0; n < C::NS; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (32 * n + (e & 3) + 8 * (e >> 2) >= left) s[n][e] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < C::NS; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[n][e]);
        // The reference moves only when a score passes it by more than 2^6: P stays below 64 and the accumulators are rarely rescaled.
        // The exponent s c - m c is formed in one step with m c rounded: half a step of that is a factor common to the row, which the sum takes out
        // again.  Of references beyond 2^12 it could pass the type's range, so there the difference is formed first.
        float mc = m * c;
        if (__any((mx - m) * c > 6.0f || fabsf(mc) > 0x1p12f)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float mn = fmaxf(m, mx);
            const float a = __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            l *= a;
#pragma unroll
            for (int b = 0; b < C::NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][e] *= a;
            mc = m * c;
            if (__any(fabsf(mc) > 0x1p12f)) {
#pragma unroll
                for (int n = 0; n < C::NS; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[n][e] -= m;
                mc = 0.f;
            }
        }
        float t0 = 0.f, t1 = 0.f;
        if constexpr (!masked) {   // (beside the exponentials)
#pragma unroll
            for (int f = 0; f < AHEAD && f < NV; ++f) vf[f] = v_frag(f);
        }
        V8 pf[2 * C::NS];
#pragma unroll
        for (int n = 0; n < C::NS; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][e], c, -mc));
                if (e & 1) t1 += pe; else t0 += pe;
                s[n][e] = pe;
                pf[2 * n + (e >> 3)][e & 7] = (T)pe;   // P in the input type: half a step of it, relative, on each weight
            }
        l += t0 + t1;
        if constexpr (masked) {
            // a masked weight is 0, but 0 x infinity is not: where the tile's values are not all finite, the rows take their visible keys one
            // by one instead
            unsigned bad = 0;
#pragma unroll
            for (int j = 0; j < C::TILE / 512; ++j) {
                const u32x4 w = *(const __attribute__((address_space(3))) u32x4*)(sv + (j * 64 + lane) * 8);
                bad |= ((w.x & ExpBits<T>::mask) + ExpBits<T>::one) | ((w.y & ExpBits<T>::mask) + ExpBits<T>::one) |
                       ((w.z & ExpBits<T>::mask) + ExpBits<T>::one) | ((w.w & ExpBits<T>::mask) + ExpBits<T>::one);
            }
            if (__any((bad & 0x80008000u) != 0)) {
#pragma unroll 1
                for (int j = 0; j < C::KT; ++j) {
                    const int e = (j & 3) + 4 * ((j >> 3) & 3) + 16 * (j >> 5);
                    float pe = 0.f;
#pragma unroll
                    for (int x = 0; x < 16 * C::NS; ++x) pe = x == e ? s[x >> 4][x & 15] : pe;
                    pe = (float)(T)__shfl(pe, l31 + 32 * ((j >> 2) & 1), 64);
                    const bool vis = key + j < lim;
#pragma unroll
                    for (int b = 0; b < C::NB; ++b)
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const int col = 32 * b + (x & 3) + 8 * (x >> 2) + 4 * h;
                            const float v = (float)sv[j * C::RS + (((col >> 3) ^ swz_v<C::RS>(j)) << 3) + (col & 7)];
                            if (vis) acc[b][x] = __builtin_fmaf(pe, v, acc[b][x]);
                        }
                }
                return;
            }
        }
        if constexpr (masked) {
#pragma unroll
            for (int f = 0; f < AHEAD && f < NV; ++f) vf[f] = v_frag(f);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < NV; ++f) {
            if constexpr (PINNED) __builtin_amdgcn_sched_barrier(0);
            acc[f % C::NB] = mfma_32x32x16(vf[f], pf[f / C::NB], acc[f % C::NB]);
            if (f + AHEAD < NV) vf[f + AHEAD] = v_frag(f + AHEAD);
        }
        if constexpr (PINNED) __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
    };

    // The tiles that the item's first row sees whole -- all its rows do -- run without masks; at most (127 / group + 63) / 64 + 1 follow them.
    const int tiles = (it.key_end - it.key_begin + C::KT - 1) / C::KT;
    const int first_lim = p.causal ? min(it.m0 / group + it.kv_len - it.q_len + 1, it.key_end) : it.key_end;
    const int whole = max(0, first_lim - it.key_begin) / C::KT;
    auto walk = [&](int t, auto tag) __attribute__((always_inline)) {
        const int key = it.key_begin + t * C::KT;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // this wave's share of tile t has landed, its reads of tile t - 1 are over ...
        __builtin_amdgcn_s_barrier();                        // ... and everyone's; everyone has left tile t - 1 and its stage
        asm volatile("" ::: "memory");
        if (t + 1 < tiles) issue(key + C::KT, (t + 1) & 1);
        if (active && (!decltype(tag)::value || key < lim_hi)) compute(key, t & 1, tag);
    };
    if (tiles > 0) issue(it.key_begin, 0);
#pragma unroll 1
    for (int t = 0; t < whole; ++t) walk(t, Masked<false>{});
#pragma unroll 1
    for (int t = whole; t < tiles; ++t) walk(t, Masked<true>{});
    l += __shfl_xor(l, 32, 64);

    if (row0 + l31 >= rows) return;
    if (it.ws_row >= 0) {
        float* ws = (float*)p.workspace;
        // a part's sums as [4 columns][row][4]: what a half wave stores, and what the join reads, is contiguous
        const int part_rows = min(128, rows - it.m0);
        const int64_t first = (int64_t)kvh * p.ws_rows + it.ws_row, at = first + wave * 32 + l31;
#pragma unroll
        for (int b = 0; b < C::NB; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int quad = 8 * b + 2 * g + h;
                if (quad * 4 < p.d)
                    *(float4v*)(ws + first * p.d + (quad * part_rows + wave * 32 + l31) * 4) = float4v{acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]};
            }
        if (h == 0) {
            float* wml = ws + (int64_t)p.kv_heads * p.ws_rows * p.d + at * 2;
            wml[0] = m;
            wml[1] = l;
        }
        return;
    }
    const float inv = 1.0f / l;
    T* out = (T*)p.out + (int64_t)(it.q_row + qi) * p.ldo + (int64_t)hq * p.d;
#pragma unroll
    for (int b = 0; b < C::NB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = 32 * b + 8 * g + 4 * h;
            if (col >= p.d) continue;
            T w4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w4[e] = seen > 0 ? (T)(acc[b][4 * g + e] * inv) : (T)0.f;
            *(uint2*)(out + col) = *(const uint2*)w4;
        }
}

// Joins the parts of rows whose keys were split over several items: a thread takes four columns of a row.  G threads share its parts, in turn and four
// at a time: the parts were just written by other XCDs, and what the join of many parts costs is those loads' latency.  Attention and join (us, G = 1 /
// 8): 64 parts, one token over 8192 keys, 8 key / value heads 17.6 / 12.0; 52 parts, 2 x 4 tokens over 16 500 keys 22.5 / 18.0; 32 parts, 2 x 128
// tokens over 8192 29.8 / 28.9; 16 parts, 4 x 128 over 8192 39.9 / 39.4; 16 parts, one token over 2048 9.15 / 9.35; up to 9 parts of chunks 23.4 / 27.7.
template <typename T, int G>
__global__ __launch_bounds__(256) void attention_join_kernel(const mv_attn_packed_desc p, const int blocks) {
    constexpr int OWN = 256 / G;   // (row, four columns) of a block
    __shared__ float4v other_o[G > 1 ? G - 1 : 1][OWN];
    __shared__ float2v other_ml[G > 1 ? G - 1 : 1][OWN];
    const int join = blockIdx.x / (p.kv_heads * blocks), rest = blockIdx.x - join * (p.kv_heads * blocks);
    const int kvh = rest / blocks, own = threadIdx.x % OWN, part0 = threadIdx.x / OWN, group = p.heads / p.kv_heads;
    const PackedJoin jn = ((const PackedJoin*)p.joins)[join];
    const int x = (rest - kvh * blocks) * OWN + own;
    const int quad = x / jn.rows, row = x - quad * jn.rows;
    const bool valid = quad * 4 < p.d;   // (joins differ in their rows)
    const float* ws = (const float*)p.workspace;
    const int64_t first = (int64_t)kvh * p.ws_rows + jn.ws_row;
    const float* ml = ws + (int64_t)p.kv_heads * p.ws_rows * p.d + (first + row) * 2;
    const float* sums = ws + first * p.d + (int64_t)x * 4;
    // Weight of sums formed with reference m beside those with `top`: 2 to the difference of the references in the exponent.  Those are what the sums were
    // formed with: m c rounded, of references up to 2^12; m c itself beyond, where its rounding would be part of the weight (at 2^21 by up to 9 %), so the
    // difference is formed first.
    const float c = score_factor(p.scale);
    auto weight = [&](float m, float top) __attribute__((always_inline)) {
        float mc = m * c, tc = top * c;
        MV_KEEP_ONE_REGISTER(mc);   // (rounded products: the compiler would fuse one of them into the difference)
        MV_KEEP_ONE_REGISTER(tc);
        return __builtin_amdgcn_exp2f(fabsf(tc) > 0x1p12f ? (m - top) * c : mc - tc);
    };
    float mm = -3.0e38f, ll = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    if (valid)
        for (int s = part0; s < jn.parts; s += 4 * G) {
            float2v w[4];
            float4v v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = (int64_t)min(s + G * u, jn.parts - 1) * jn.rows;
                w[u] = *(const float2v*)(ml + at * 2);
                v[u] = *(const float4v*)(sums + at * p.d);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s + G * u >= jn.parts) w[u] = float2v{-3.0e38f, 0.f}, v[u] = float4v{0.f, 0.f, 0.f, 0.f};
            const float mn = fmaxf(fmaxf(mm, fmaxf(w[0].x, w[1].x)), fmaxf(w[2].x, w[3].x)), old = weight(mm, mn);
            mm = mn;
            ll *= old;
            o *= old;
            // (a part that saw no key holds zeros; one whose weight vanishes counts all the same: 0 x infinity is NaN, as it is where keys are not split)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float a = weight(w[u].x, mn);
                ll = __builtin_fmaf(a, w[u].y, ll);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a, v[u][e], o[e]);
            }
        }
    if constexpr (G > 1) {
        if (part0 > 0) {
            other_o[part0 - 1][own] = o;
            other_ml[part0 - 1][own] = float2v{mm, ll};
        }
        __syncthreads();
        if (part0 > 0) return;
        float mn = mm;
#pragma unroll
        for (int u = 0; u < G - 1; ++u) mn = fmaxf(mn, other_ml[u][own].x);
        const float a0 = weight(mm, mn);
        ll *= a0;
        o *= a0;
#pragma unroll
        for (int u = 0; u < G - 1; ++u) {
            const float2v w = other_ml[u][own];
            const float a = weight(w.x, mn);
            ll = __builtin_fmaf(a, w.y, ll);
            const float4v v = other_o[u][own];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a, v[e], o[e]);
        }
    }
    if (!valid) return;
    const int rr = jn.m0 + row, i = rr / group, head = kvh * group + (rr - i * group);
    const int see = p.causal ? i + jn.kv_len - jn.q_len + 1 : jn.kv_len;
    T w4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w4[e] = see > 0 ? (T)(o[e] / ll) : (T)0.f;
    *(uint2*)((T*)p.out + (int64_t)(jn.q_row + i) * p.ldo + (int64_t)head * p.d + quad * 4) = *(const uint2*)w4;
}

extern "C" int64_t mv_attention_packed_workspace_bytes(int64_t ws_rows, int32_t kv_heads, int32_t d) {
    if (ws_rows < 0 || kv_heads < 1 || d < 1) return -1;
    return ws_rows * kv_heads * (d + 2) * 4;
}

// threads that share a (row, four columns) of the join, by the parts of a join in the mean; blocks of a join
static int join_threads(const mv_attn_packed_desc* d) { return d->ws_rows > 16ll * d->n_joins * d->join_rows ? 8 : 1; }
static int join_blocks(const mv_attn_packed_desc* d) { return (d->join_rows * (d->d / 4) * join_threads(d) + 255) / 256; }

template <typename T, int K16>
static int launch_packed(const mv_attn_packed_desc* d, hipStream_t st) {
    static_assert(PackedCfg<K16>::LDS_BYTES <= 64 * 1024, "dynamic LDS without an attribute");
    attention_packed_kernel<T, K16><<<(unsigned)(d->n_items * d->kv_heads), 256, PackedCfg<K16>::LDS_BYTES, st>>>(*d);
    MV_CHECK_LAUNCH("mv_attention_packed");
    if (d->n_joins > 0) {
        const int blocks = join_blocks(d);
        const unsigned grid = (unsigned)(d->n_joins * d->kv_heads * blocks);
        if (join_threads(d) == 8) attention_join_kernel<T, 8><<<grid, 256, 0, st>>>(*d, blocks);
        else attention_join_kernel<T, 1><<<grid, 256, 0, st>>>(*d, blocks);
        MV_CHECK_LAUNCH("mv_attention_packed (join)");
    }
    return MV_OK;
}

template <typename T>
static int launch_head_dim(const mv_attn_packed_desc* d, hipStream_t st) {
    switch ((d->d + 15) / 16) {
        case 1: return launch_packed<T, 1>(d, st);
        case 2: return launch_packed<T, 2>(d, st);
        case 3: return launch_packed<T, 3>(d, st);
        case 4: return launch_packed<T, 4>(d, st);
        case 5: return launch_packed<T, 5>(d, st);
        case 6: return launch_packed<T, 6>(d, st);
        case 7: return launch_packed<T, 7>(d, st);
        default: return launch_packed<T, 8>(d, st);
    }
}

extern "C" int mv_attention_packed(const mv_attn_packed_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_attention_packed: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_attention_packed: element type %d", d->dtype);
    MV_REQUIRE(d->d >= 8 && d->d <= 128 && d->d % 8 == 0, "mv_attention_packed: head dim %d (a multiple of 8 up to 128)", d->d);
    MV_REQUIRE(d->kv_heads >= 1 && d->heads >= d->kv_heads && d->heads % d->kv_heads == 0, "mv_attention_packed: %d heads over %d key / value heads",
               d->heads, d->kv_heads);
    MV_REQUIRE(d->scale >= -1e6f && d->scale <= 1e6f, "mv_attention_packed: scale %g (at most 1e6 in size)", (double)d->scale);
    MV_REQUIRE(d->n_items >= 0 && d->n_joins >= 0 && (int64_t)d->n_items * d->kv_heads < (1ll << 31) && d->join_rows >= 0 && d->join_rows <= 128 &&
               (int64_t)d->n_joins * d->kv_heads * 128 < (1ll << 31), "mv_attention_packed: %d items, %d joins of up to %d rows", d->n_items, d->n_joins,
               d->join_rows);
    MV_REQUIRE_GRID("mv_attention_packed", (int64_t)d->n_items * d->kv_heads, 256);
    MV_REQUIRE_GRID("mv_attention_packed (join)", (int64_t)d->n_joins * d->kv_heads * join_blocks(d), 256);
    if (d->n_items == 0) return MV_OK;
    MV_REQUIRE(d->q && d->k && d->v && d->out && d->items, "mv_attention_packed: null pointer");
    MV_REQUIRE((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->out) & 15) == 0 && ((d->ldq | d->ldk | d->ldv | d->ldo) & 7) == 0,
               "mv_attention_packed: rows must be 16-byte aligned");
    MV_REQUIRE(d->ldk >= 0 && d->ldk <= (1 << 23) && d->ldv >= 0 && d->ldv <= (1 << 23), "mv_attention_packed: key / value row stride above 2^23");
    MV_REQUIRE(d->n_joins == 0 || (d->joins && d->workspace && ((uintptr_t)d->workspace & 15) == 0 &&
               d->workspace_bytes >= mv_attention_packed_workspace_bytes(d->ws_rows, d->kv_heads, d->d)),
               "mv_attention_packed: the workspace is missing, unaligned or too small");
    return d->dtype == MV_F16 ? launch_head_dim<half_t>(d, (hipStream_t)stream) : launch_head_dim<bf16_t>(d, (hipStream_t)stream);
}
