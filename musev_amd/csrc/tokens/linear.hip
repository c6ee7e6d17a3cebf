// tokens/linear.hip -- the int8 projection (include/musev_tokens.h: mv_quantize_rows_i8, mv_gemm_i8).
#include "tokens.h"

// ---- activations to int8, one scale per row ------------------------------------------------------------------------------------
// code = rne(127 x / top) with top = max |x|, of the exact quotient q: x = X 2^a and top = T 2^b with integers X, T < 2^11, so a q that is no
// half-integer is at least 1 / (2 T 2^(b - a)) = q / (2 * 127 X) > q 2^-19 away from every half-integer, and fp32 (2^-23 relative for the
// two roundings below) resolves that.  f (a power of two) keeps the factors of bf16's largest and smallest values in range.
struct RowScale {
    float f, inv, scale;
};
__device__ __forceinline__ RowScale row_scale(unsigned top_bits) {
    RowScale r;
    const float top = __uint_as_float(top_bits);
    const bool finite = top_bits < 0x7f800000u;
    r.f = !finite ? 0.0f : top > 0x1p100f ? 0x1p-32f : top < 0x1p-80f ? 0x1p64f : 1.0f;
    r.inv = top > 0.f && finite ? 127.0f / (top * r.f) : 0.0f;
    r.scale = top / 127.0f;
    return r;
}
// a product within q 2^-21 of a half-integer is that half-integer: the tie itself.  (A row that is not finite has f = inv = 0; its NaN and infinite elements become 0 in the last step.)
__device__ __forceinline__ int row_code(float x, const RowScale& r) {
    const float q = (x * r.f) * r.inv, twice = q + q, near = rintf(twice);
    const float v = rintf(fabsf(twice - near) < fabsf(twice) * 0x1p-21f ? 0.5f * near : q);
    return r.inv > 0.f ? (int)v : 0;
}

// |x| as bits: ordered like the values, NaN above infinity
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ unsigned lanes16_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));    // lanes 1 0 3 2 of a quad
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));    // lanes 2 3 0 1
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));   // mirrored within 8
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));   // mirrored within 16
}
template <int WAVES>
__device__ __forceinline__ unsigned row_top(unsigned v, unsigned* red) {
    v = lanes16_max(v);
    v = max(v, (unsigned)__shfl_xor((int)v, 16, 64));
    v = max(v, (unsigned)__shfl_xor((int)v, 32, 64));
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    return v;
}
__device__ __forceinline__ uint2 eight_codes(const float* v, const RowScale& r) {
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e >> 2] |= (unsigned)(row_code(v[e], r) & 255) << (8 * (e & 3));
    return uint2{w[0], w[1]};
}

// A row is read once and stays in registers between its maximum and its codes: NV chunks of 8 columns per lane, WAVES waves per row.  Rows
// wider than the registers hold (REREAD) are read a second time, from the caches.  Bound by memory: 2 bytes in, 1 out per element.
template <typename T, int NV, int WAVES, bool REREAD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int64_t ldx, int64_t rows, int k, int8_t* codes, int64_t ldc, float* scale) {
    __shared__ unsigned red[4];
    constexpr int LANES = 64 * WAVES;
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + threadIdx.x / LANES;
    if (row >= rows) return;
    const T* xr = x + row * ldx;
    int8_t* cr = codes + row * ldc;
    float v[NV][8];
    unsigned top = 0;
    const int step = NV * LANES * 8;
    for (int c0 = 0; c0 < (REREAD ? k : 1); c0 += step) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = c0 + (j * LANES + lane) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
            if (col < k) load8(xr + col, k - col, v[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[j][e]));
        }
    }
    const RowScale r = row_scale(row_top<WAVES>(top, red));
    if (lane == 0) scale[row] = r.scale;
    for (int c0 = 0; c0 < (REREAD ? (int)ldc : 1); c0 += step) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = c0 + (j * LANES + lane) * 8;
            if (REREAD) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
                if (col < k) load8(xr + col, k - col, v[j]);
            }
            if (col < ldc) *(uint2*)(cr + col) = eight_codes(v[j], r);   // (columns from k on: codes of 0)
        }
    }
}

template <typename T, int NV, int WAVES, bool REREAD>
static int launch_quantize(const void* x, int64_t ldx, int64_t rows, int k, int8_t* codes, int64_t ldc, float* scale, hipStream_t st) {
    constexpr int R = 4 / WAVES;
    const int64_t blocks = (rows + R - 1) / R;
    MV_REQUIRE_GRID("mv_quantize_rows_i8", blocks, 256);
    quantize_rows_kernel<T, NV, WAVES, REREAD><<<(unsigned)blocks, 256, 0, st>>>((const T*)x, ldx, rows, k, codes, ldc, scale);
    MV_CHECK_LAUNCH("mv_quantize_rows_i8");
    return MV_OK;
}
template <typename T>
static int launch_quantize_width(const void* x, int64_t ldx, int64_t rows, int k, int8_t* codes, int64_t ldc, float* scale, hipStream_t st) {
    if (ldc <= 512) return launch_quantize<T, 1, 1, false>(x, ldx, rows, k, codes, ldc, scale, st);
    if (ldc <= 1536) return launch_quantize<T, 3, 1, false>(x, ldx, rows, k, codes, ldc, scale, st);
    if (ldc <= 2048) return launch_quantize<T, 1, 4, false>(x, ldx, rows, k, codes, ldc, scale, st);
    if (ldc <= 6144) return launch_quantize<T, 3, 4, false>(x, ldx, rows, k, codes, ldc, scale, st);
    if (ldc <= 16384) return launch_quantize<T, 8, 4, false>(x, ldx, rows, k, codes, ldc, scale, st);
    return launch_quantize<T, 8, 4, true>(x, ldx, rows, k, codes, ldc, scale, st);
}

extern "C" int mv_quantize_rows_i8(const void* x, int64_t ldx, int64_t rows, int32_t k, int32_t dtype, int8_t* codes, int64_t ldc, float* scale,
                                   void* stream) {
    MV_REQUIRE(dtype == MV_F16 || dtype == MV_BF16, "mv_quantize_rows_i8: element type %d", dtype);
    MV_REQUIRE(rows >= 0 && rows < (1ll << 31) && k >= 1 && k <= 131071, "mv_quantize_rows_i8: %ld rows of %d (1 .. 131071)", (long)rows, k);
    MV_REQUIRE(ldc % 128 == 0 && ldc >= k && ldc < k + 128, "mv_quantize_rows_i8: code rows of %ld for k = %d (k rounded up to 128)", (long)ldc, k);
    if (rows == 0) return MV_OK;
    MV_REQUIRE(x && codes && scale && ((uintptr_t)codes & 15) == 0, "mv_quantize_rows_i8: null or unaligned pointer");
    MV_DISPATCH_TYPE(dtype, return launch_quantize_width<T>(x, ldx, rows, k, codes, ldc, scale, (hipStream_t)stream));
}

// ---- the product ---------------------------------------------------------------------------------------------------------------
typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

// Tiles through LDS: BM rows of activations x BN rows of weights, 128 bytes of K per step, two stages (one computed on, one on its way; three
// or four stages of 64 or 128 bytes were no faster), every wave WM x WN of the result in v_mfma_i32_32x32x32_i8 blocks (weights as the first
// operand: a lane holds 4 consecutive outputs of one row).  LDS rows are 128 bytes = 8 slots of 16 and two rows share a 256-byte line of banks, so
// the slots of a row are permuted by the line's number and a fragment read (16 rows, one slot) touches every bank once.  The permutation is
// applied to the column each lane fetches (global -> LDS directly).
// KS groups of waves share a block's tile and take the steps of K in turn, each with stages of its own: where a product has fewer tiles than
// there are CUs and a long K, the latency of its steps is what it costs.  The groups' sums meet in LDS.
constexpr int BK = 128;

template <int BM, int BN, int WM, int WN, int KS>
struct GemmI8Cfg {
    static constexpr int WAVES = (BM / WM) * (BN / WN), THREADS = 64 * WAVES * KS;
    static constexpr int SLOTS = BK / 16, PROWS = 1024 / BK;            // slots of a row; rows of a 1-KiB piece
    static constexpr int STAGE = (BM + BN) * BK;
    static constexpr int PA = BM / PROWS / WAVES, PW = BN / PROWS / WAVES;   // pieces a wave fetches of each tile
    static constexpr int SROW = WN + 4;                                 // floats per row of the result staging
    static constexpr int STAGING = WAVES * 32 * SROW * 4, SUMS = WM * WN * 4;   // bytes; of a wave's sums
    static constexpr int AFTER = STAGING + (KS - 1) * WAVES * SUMS;
    static constexpr int LDS = KS * 2 * STAGE > AFTER ? KS * 2 * STAGE : AFTER;
    static_assert(BM % (PROWS * WAVES) == 0 && BN % (PROWS * WAVES) == 0, "every wave fetches whole pieces");
    static __device__ __forceinline__ int swz(int row) { return (row / (256 / BK)) % SLOTS; }
};

template <typename T, int BM, int BN, int WM, int WN, int KS, bool COLD>
__global__ __launch_bounds__((GemmI8Cfg<BM, BN, WM, WN, KS>::THREADS), 2) void gemm_i8_kernel(const mv_gemm_i8_desc p, const int tiles_m, const int tiles_n) {
    using C = GemmI8Cfg<BM, BN, WM, WN, KS>;
    typedef __attribute__((address_space(3))) char lds_c;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    lds_c* const lds = (lds_c*)smem;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave_id / C::WAVES, wave = wave_id - kg * C::WAVES;
    int tm, tn;
    mv_tile_order(mv_xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, MV_TILE_GROUP, &tm, &tn);
    const int64_t m0 = (int64_t)tm * BM;
    const int n0 = tn * BN;
    const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;

    // descriptors end with the matrices' last rows: rows behind them read as 0
    const int ma = (int)min((int64_t)BM, p.M - m0), na = min(BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + m0 * p.lda), 0, (unsigned)(ma * p.lda), 0x00020000);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + n0 * p.ldw), 0, (unsigned)(na * p.ldw), 0x00020000);
    unsigned oa[C::PA], ow[C::PW];
    const int prow = lane / C::SLOTS, pslot = lane % C::SLOTS;
#pragma unroll
    for (int j = 0; j < C::PA; ++j) {
        const int row = (wave * C::PA + j) * C::PROWS + prow;
        oa[j] = (unsigned)(row * p.lda + ((pslot ^ C::swz(row)) << 4));
    }
#pragma unroll
    for (int j = 0; j < C::PW; ++j) {
        const int row = (wave * C::PW + j) * C::PROWS + prow;
        ow[j] = (unsigned)(row * p.ldw + ((pslot ^ C::swz(row)) << 4));
    }
    auto issue = [&](int k, int stage) __attribute__((always_inline)) {
        lds_c* dst = lds + (kg * 2 + stage) * C::STAGE;
#pragma unroll
        for (int j = 0; j < C::PA; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(dst + (wave * C::PA + j) * 1024), 16, (int)oa[j], k, 0, 0);
#pragma unroll
        for (int j = 0; j < C::PW; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(dst + BM * BK + (wave * C::PW + j) * 1024), 16, (int)ow[j], k, 0, 0);
    };
    int16v acc[WM / 32][WN / 32];
#pragma unroll
    for (int i = 0; i < WM / 32; ++i)
#pragma unroll
        for (int j = 0; j < WN / 32; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    int fo[BK / 32];   // byte offset of fragment step s in a 32-row block (row l31)
#pragma unroll
    for (int s = 0; s < BK / 32; ++s) fo[s] = l31 * BK + (((2 * s + h) ^ C::swz(l31)) << 4);

    // what the result needs besides the sums.  A lane holds row l31 of every 32 while it multiplies, and finishes columns n .. n + 7 of the rows
    // lane / LPR + RPP x of every 32.
    typedef typename Vec8<T>::type V8;
    constexpr int LPR = WN / 8, RPP = 64 / LPR, PASSES = 32 / RPP, NRES = WM / 32 * PASSES;   // lanes per row, rows per pass
    constexpr int FIRST = NRES > 8 ? NRES / 2 : NRES;   // residual loads the registers have room for beside the fragments; the others follow the last step
    const int c8 = (lane % LPR) * 8, n = n0 + wn + c8, left = p.N - n, frow = lane / LPR;
    float as[WM / 32];
#pragma unroll
    for (int i = 0; i < WM / 32; ++i) as[i] = p.a_scale[min(m0 + wm + 32 * i + l31, p.M - 1)];
    // The residual is fetched beside the last two steps: as long as the sums take, its loads are hidden (26 624 x 1280 -> 5120: one block per CU,
    // nothing else would hide them).  Every lane makes all its loads, whole ones of 16 bytes, so that at least FIRST of them are younger than the
    // last stage's when the wait below counts: rows past the end fetch the last one, columns past the end (and the fewer than 8 that end a row,
    // which are read where they are added) the row's last 8.
    V8 res[NRES];
    auto residual_at = [&](int x) __attribute__((always_inline)) {
        const T* r = (const T*)p.residual + min(m0 + wm + 32 * (x / PASSES) + (x % PASSES) * RPP + frow, p.M - 1) * p.ldr + min(n, p.N - 8);
        if constexpr (COLD)   // (a residual that the last-level cache cannot hold)
            return __builtin_bit_cast(V8, __builtin_nontemporal_load((const typename Loose8<T>::anywhere*)r));
        return __builtin_bit_cast(V8, ((const typename Loose8<T>::bytes*)r)->v);
    };
    const bool early = p.residual && kg == 0 && p.kp > KS * BK && p.N >= 8;

    const int steps = p.kp / BK, turns = (steps + KS - 1) / KS;   // this group's steps: kg, kg + KS, ...; the first group has one every turn
    if (kg < steps) issue(kg * BK, 0);
#pragma unroll 1
    for (int t = 0; t < turns; ++t) {
        // this wave's share of the step has landed ...
        if (t + 1 == turns && early) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(FIRST) : "memory");   // (the residual's loads are the youngest)
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                      // ... and everyone's; everyone has left the stage of the step before
        asm volatile("" ::: "memory");
        if ((t + 1) * KS + kg < steps) issue(((t + 1) * KS + kg) * BK, (t + 1) & 1);
        if (t + 2 == turns && early) {
            asm volatile("" ::: "memory");   // (behind the last stage's loads)
#pragma unroll
            for (int x = 0; x < FIRST; ++x) res[x] = residual_at(x);
            asm volatile("" ::: "memory");
        }
        if (KS > 1 && t * KS + kg >= steps) break;   // (the last turn: this group has no step left, nor a barrier)
        const lds_c* sa = lds + (kg * 2 + (t & 1)) * C::STAGE + wm * BK;
        const lds_c* sw = lds + (kg * 2 + (t & 1)) * C::STAGE + BM * BK + wn * BK;
        // the next quarter's fragments (small tiles: the whole step's) are read before this quarter's matrix instructions, in pinned order: left to
        // itself the compiler reads them just before their use and the matrix pipe waits out the LDS latency
        int4v fa[4][WM / 32], fw[4][WN / 32];
        auto read = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < WM / 32; ++i) fa[s][i] = *(const __attribute__((address_space(3))) int4v*)(sa + i * 32 * BK + fo[s]);
#pragma unroll
            for (int j = 0; j < WN / 32; ++j) fw[s][j] = *(const __attribute__((address_space(3))) int4v*)(sw + j * 32 * BK + fo[s]);
        };
        constexpr int AHEAD = WM * WN > 64 * 32 ? 1 : 3;
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) read(s);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s + AHEAD < 4) read(s + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < WM / 32; ++i)
#pragma unroll
                for (int j = 0; j < WN / 32; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s][j], fa[s][i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (early) {
#pragma unroll
        for (int x = FIRST; x < NRES; ++x) res[x] = residual_at(x);
    }
    __syncthreads();   // the stages become the groups' sums and the waves' result staging
    if constexpr (KS > 1) {
        int4v* sums = (int4v*)(smem + C::STAGING) + lane;   // [group - 1][wave][block][quad of registers][lane]
        if (kg > 0) {
            sums += ((kg - 1) * C::WAVES + wave) * (C::SUMS / 16);
#pragma unroll
            for (int i = 0; i < WM / 32; ++i)
#pragma unroll
                for (int j = 0; j < WN / 32; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        sums[((i * (WN / 32) + j) * 4 + g) * 64] = int4v{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int o = 0; o < KS - 1; ++o)
#pragma unroll
            for (int i = 0; i < WM / 32; ++i)
#pragma unroll
                for (int j = 0; j < WN / 32; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int4v v = sums[(o * C::WAVES + wave) * (C::SUMS / 16) + ((i * (WN / 32) + j) * 4 + g) * 64];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * g + e] += v[e];
                    }
    }

    // 32 rows at a time through this wave's own LDS, so that rows are read (residual) and written 16 bytes per lane
    float* st = (float*)smem + wave * 32 * C::SROW;
    float ws[8], bs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        ws[e] = e < left ? p.w_scale[n + e] : 0.f;
        bs[e] = p.bias && e < left ? (float)((const T*)p.bias)[n + e] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < WM / 32; ++i) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int j = 0; j < WN / 32; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float4v v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][4 * g + e] * as[i];
                *(float4v*)(st + l31 * C::SROW + 32 * j + 8 * g + 4 * h) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int x = 0; x < PASSES; ++x) {
            const int row = x * RPP + frow;
            const int64_t m = m0 + wm + 32 * i + row;
            if (m >= p.M || left <= 0) continue;
            const float4v u = *(const float4v*)(st + row * C::SROW + c8), w = *(const float4v*)(st + row * C::SROW + c8 + 4);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(e < 4 ? u[e & 3] : w[e & 3], ws[e], bs[e]);
            if (p.act == MV_ACT_SILU)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = mv_silu(v[e]);
            if (early && left >= 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += (float)res[i * PASSES + x][e];
            } else if (p.residual) {
                float r[8];
                load8((const T*)p.residual + m * p.ldr + n, left, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += r[e];
            }
            // (the small tile's results are small: the next kernel may find them in the caches)
            if constexpr (BM > 64) store8_stream((T*)p.out + m * p.ldo + n, left, v);
            else store8((T*)p.out + m * p.ldo + n, left, v);
        }
    }
}

// Few rows of activations (M <= 16 MT): the weights are streamed once, straight from memory into fragments.  A block owns 16 weight rows, its
// 8 waves take 128-byte units of K in turn; in a unit, lane group g = lane / 16 holds bytes 32 g .. 32 g + 31 of its row as the fragments of two
// v_mfma_i32_16x16x64_i8 (weights and activations in the same order of K: the sum does not care which).  The waves' sums meet in LDS.
template <typename T, int MT>
__global__ __launch_bounds__(512) void gemm_i8_few_kernel(const mv_gemm_i8_desc p) {
    __shared__ int part[8][MT * 256];
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16;
    const int8_t* w = p.w + (int64_t)min(n0 + l15, p.N - 1) * p.ldw + 32 * g;
    const int8_t* a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = p.a + min((int64_t)(16 * t + l15), p.M - 1) * p.lda + 32 * g;
    int4v acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = int4v{0, 0, 0, 0};
    for (int k = wave * 128; k < p.kp; k += 8 * 128) {
        const int4v w0 = *(const int4v*)(w + k), w1 = *(const int4v*)(w + k + 16);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int4v a0 = *(const int4v*)(a[t] + k), a1 = *(const int4v*)(a[t] + k + 16);
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, a0, acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, a1, acc[t], 0, 0, 0);
        }
    }
    // lane l holds weight rows 4 g .. 4 g + 3 of activation row l15
#pragma unroll
    for (int t = 0; t < MT; ++t) *(int4v*)(&part[wave][t * 256 + l15 * 16 + 4 * g]) = acc[t];
    __syncthreads();
    for (int x = tid; x < MT * 256; x += 512) {
        const int64_t m = x >> 4;
        const int n = n0 + (x & 15);
        if (m >= p.M || n >= p.N) continue;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < 8; ++v) sum += part[v][x];
        float v = __builtin_fmaf((float)sum * p.a_scale[m], p.w_scale[n], p.bias ? (float)((const T*)p.bias)[n] : 0.f);
        if (p.act == MV_ACT_SILU) v = mv_silu(v);
        if (p.residual) v += (float)((const T*)p.residual)[m * p.ldr + n];
        ((T*)p.out)[m * p.ldo + n] = (T)v;
    }
}

// Quantisation and product in one launch, for so few activations that every block can quantise them for itself: up to 16384 codes of up to 4 rows,
// 8192 of up to 16.  Measured (us of GPU time, one launch / two; a second launch also costs the host 4): 1 x 1280 -> 5120 4.9 / 6.4; 4 x 4096 -> 1280
// 7.6 / 10.8; 8 x 1024 -> 1280 5.0 / 5.8; 16 x 512 -> 5120 6.8 / 5.5; 16 x 1024 -> 5120 10.2 / 6.8.  All 512 threads read x (each keeps its elements in registers between the row's maximum and the codes), the codes go to LDS
// and the weights stream as above, their first two units already on their way meanwhile.
constexpr int ONE_LAUNCH = 16384;
static bool one_launch(int64_t m, int64_t kp) { return m <= 16 && m * kp <= (m <= 4 ? ONE_LAUNCH : ONE_LAUNCH / 2); }

template <typename T>
__global__ __launch_bounds__(512) void linear_i8_few_kernel(const mv_linear_i8_desc p) {
    __shared__ int part[8][256];
    __shared__ unsigned tops[16];
    __shared__ __attribute__((aligned(16))) int8_t codes[ONE_LAUNCH + 16 * 16];   // rows kp + 16 bytes apart: 16 rows' fragments on different banks
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16, m_rows = (int)p.M, kp = (int)p.kp, stride = kp + 16;
    const int8_t* w = p.w + (int64_t)min(n0 + l15, p.N - 1) * p.ldw + 32 * g;
    int4v w0[2], w1[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int k = min((wave + 8 * u) * 128, kp - 128);
        w0[u] = *(const int4v*)(w + k);
        w1[u] = *(const int4v*)(w + k + 16);
    }
    if (tid < 16) tops[tid] = 0;
    __syncthreads();
    constexpr int NC = ONE_LAUNCH / 8 / 512;   // chunks of 8 codes per thread
    const int per_row = kp / 8, total = m_rows * per_row;
    float v[NC][8];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int ch = tid + 512 * j, m = ch / per_row, col = (ch - m * per_row) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
        if (ch < total && col < p.K) load8((const T*)p.x + m * p.ldx + col, p.K - col, v[j]);
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[j][e]));
        top = lanes16_max(top);   // (16 lanes are of one row: kp is a multiple of 128)
        if (l15 == 0 && ch < total) atomicMax(&tops[m], top);   // (a maximum does not depend on the order)
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int ch = tid + 512 * j, m = ch / per_row, col = (ch - m * per_row) * 8;
        if (ch < total) *(uint2*)(codes + m * stride + col) = eight_codes(v[j], row_scale(tops[m]));
    }
    __syncthreads();
    int4v acc = {0, 0, 0, 0};
    const int8_t* a = codes + min(l15, m_rows - 1) * stride + 32 * g;
    int u = 0;
    for (int k = wave * 128; k < kp; k += 8 * 128, ++u) {
        const int4v b0 = u == 0 ? w0[0] : u == 1 ? w0[1] : *(const int4v*)(w + k), b1 = u == 0 ? w1[0] : u == 1 ? w1[1] : *(const int4v*)(w + k + 16);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b0, *(const int4v*)(a + k), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b1, *(const int4v*)(a + k + 16), acc, 0, 0, 0);
    }
    *(int4v*)(&part[wave][l15 * 16 + 4 * g]) = acc;
    __syncthreads();
    const int m = tid >> 4, n = n0 + (tid & 15);
    if (m >= m_rows || n >= p.N) return;
    int sum = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) sum += part[x][tid];
    float r = __builtin_fmaf((float)sum * row_scale(tops[m]).scale, p.w_scale[n], p.bias ? (float)((const T*)p.bias)[n] : 0.f);
    if (p.act == MV_ACT_SILU) r = mv_silu(r);
    if (p.residual) r += (float)((const T*)p.residual)[m * p.ldr + n];
    ((T*)p.out)[m * p.ldo + n] = (T)r;
}

template <typename T, int BM, int BN, int WM, int WN, int KS, bool COLD = false>
static int launch_gemm_i8(const mv_gemm_i8_desc* d, hipStream_t st) {
    using C = GemmI8Cfg<BM, BN, WM, WN, KS>;
    const auto kernel = gemm_i8_kernel<T, BM, BN, WM, WN, KS, COLD>;
    const int64_t tm = (d->M + BM - 1) / BM, tn = ((int64_t)d->N + BN - 1) / BN;
    MV_REQUIRE_GRID("mv_gemm_i8", tm * tn, C::THREADS);
    if (C::LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
        if (e != hipSuccess) {
            mv_set_error("mv_gemm_i8: %s", hipGetErrorString(e));
            return MV_ERR_LAUNCH;
        }
    }
    kernel<<<(unsigned)(tm * tn), C::THREADS, C::LDS, st>>>(*d, (int)tm, (int)tn);
    MV_CHECK_LAUNCH("mv_gemm_i8");
    return MV_OK;
}

template <typename T>
static int launch_gemm_i8_shape(const mv_gemm_i8_desc* d, hipStream_t st) {
    // Up to 32 rows of a short K: the weight stream (us, stream / 32 x 32 tiles: 16 x 1280 x 5120 4.5 / 4.9; 20 x 640 x 640 3.1 / 4.6; 32 x 2048 x 2048
    // 5.0 / 5.5; beyond, its waves' turns add up: 32 x 5120 x 5120 16.4 / 8.2).
    if (d->M <= 32 && d->kp <= 2048) {
        const int64_t grid = ((int64_t)d->N + 15) / 16;
        MV_REQUIRE_GRID("mv_gemm_i8", grid, 512);
        if (d->M <= 16) gemm_i8_few_kernel<T, 1><<<(unsigned)grid, 512, 0, st>>>(*d);
        else gemm_i8_few_kernel<T, 2><<<(unsigned)grid, 512, 0, st>>>(*d);
        MV_CHECK_LAUNCH("mv_gemm_i8");
        return MV_OK;
    }
    // The largest tile that fills the chip: 256 x 256 (one block per CU) from three quarters of a round on, 128 x 128 where one round holds them, 128 x 64
    // (three per CU) from two blocks per CU, 64 x 64 below, where K is long and tiles are few in two or four groups, and 32 x 32 in four groups up to two per CU.
    // Measured (us, M x K x N; 256 / 128 x 64 / 64 / 64 in groups / 32 in groups): 8192^3 472 / 655 / 799 / - / -; 26 624 x 1280 x 5120 249 / 315 /
    // 380 / 792 / -; 4096 x 1280 x 2560 27.2 / 25.1 / 32.8 / 62 / -; 2048 x 1280 x 1280 22.9 / 10.3 / 10.8 / 18.4 / 22.6; 512 x 5120 x 1280 60 / 23.0 /
    // 19.8 / 13.9 / 16.3; 512 x 1280 x 1280 22.5 / 8.4 / 6.6 / 7.1 / 9.1; 300 x 5120 x 1280 61 / 19.3 / 14.0 / 11.8 / 10.8; 64 x 1280 x 1280 20 / 8.2 /
    // 6.4 / 6.8 / 5.1.
    const auto tiles = [&](int64_t bm, int64_t bn) { return ((d->M + bm - 1) / bm) * ((d->N + bn - 1) / bn); };
    // A residual past the last-level cache is read non-temporally (272 MB, 26 624 x 1280 -> 5120 with the quantisation: 280 -> 272 us; 136 MB, 6656 x 1280
    // -> 10240 and still in the cache: 129.5 -> 132).  The 256 x 256 tiles run in rounds of one per CU: where the last round would hold at most half of
    // one, the rows of its tiles go to the smaller tiles, which spread them over the chip.  Measured with a residual (us; 128 x 64 alone / 256 alone /
    // 256 and the rest apart), K = 1280, N = 4096: 160 tiles 23.6 / 25.3 / -; 208 31.2 / 26.4 / -; 272 38.4 / 48.2 / 37.3; 352 47.3 / 48.9 / 41.4; 384 51.4 /
    // 48.9 / 43.3; 416 56.5 / 50.5 / 51.4; 640 86.3 / 76.6 / 71.5; 672 89.8 / 75.1 / 80.6.  K = 4096: 160 54.7 / 52.4 / -; 272 95.8 / 109.2 / 76.8; 384 130.6 /
    // 112.6 / 103.1; 400 - / 115.9 / 121.2.  K = 640: 160 16.9 / 18.1 / -; 272 26.4 / 34.1 / 26.8; 384 34.2 / 36.3 / 33.2; 416 37.4 / 36.5 / 37.3.
    // They are taken where more than three quarters of their area is result: a tile costs the same however few of its columns or rows there are.
    // Measured (us; 256 / the smaller tiles), 53 248 rows, K = 320 and 1280: N = 64 (a quarter) 12.4 / 6.5, 22.6 / 14.8; 128 13.8 / 9.4, 24.2 / 16.6; 264
    // 26.5 / 23.0, 45.9 / 38.6; 320 24.6 / 18.9, 44.5 / 37.2; 192 and 384 (three quarters) 13.6 / 12.4, 23.5 / 23.0 and 24.9 / 21.7, 45.1 / 44.3; 416 24.8 / 24.5,
    // 45.0 / 48.4; 224 13.2 / 15.7, 23.8 / 32.3; few rows, K = 1280, N = 51 200: 64 21.1 / 15.6; 300 43.0 / 41.7; 448 44.6 / 52.6.
    if (const int64_t all = tiles(256, 256); all >= 192 && d->M * d->N > all * (256 * 256 / 4 * 3)) {
        constexpr int64_t CUS = 256;
        const int64_t cols = ((int64_t)d->N + 255) / 256, whole = all / CUS * CUS / cols, left = all - whole * cols;
        mv_gemm_i8_desc head = *d, tail = *d;
        const bool split = whole > 0 && left > 0 && left <= CUS / 2;
        if (split) {
            head.M = whole * 256;
            tail.M -= head.M;
            tail.a += head.M * d->lda;
            tail.a_scale += head.M;
            if (d->residual) tail.residual = (const T*)d->residual + head.M * d->ldr;
            tail.out = (T*)d->out + head.M * d->ldo;
        }
        const int rc = d->residual && d->M * d->N * 2 > COLD_BYTES ? launch_gemm_i8<T, 256, 256, 128, 64, 1, true>(&head, st)
                                                                   : launch_gemm_i8<T, 256, 256, 128, 64, 1>(&head, st);
        return rc == MV_OK && split ? launch_gemm_i8_shape<T>(&tail, st) : rc;
    }
    // 128 x 128 tiles (two blocks per CU) where one round holds them all and they fill more than half of it.  Measured with a residual, N = 4096 (us; the
    // rules below / 128 x 128): K = 1280, 288 tiles 14.5 / 14.3, 448 19.9 / 15.2, 512 21.1 / 16.1, 544 22.2 / 24.3; K = 4096, 288 31.2 / 28.5, 384 35.0 / 31.8,
    // 512 52.2 / 38.1, 544 52.3 / 56.3; K = 640, 288 10.3 / 10.6, 384 10.7 / 10.7, 448 13.7 / 11.1; 256 tiles of K = 2048 14.6 / 15.0.
    if (const int64_t t = tiles(128, 128); t <= 512 && (t > 384 || (t > 256 && d->kp >= 1280))) return launch_gemm_i8<T, 128, 128, 64, 32, 1>(d, st);
    if (tiles(128, 64) >= 512) return launch_gemm_i8<T, 128, 64, 64, 32, 1>(d, st);
    if (tiles(32, 32) <= 512) return launch_gemm_i8<T, 32, 32, 32, 32, 4>(d, st);
    // 64 x 64 in groups (us, N = 1280; one / two / four): K = 2048, 240 tiles 7.8 / 7.7 / 7.7, 300 8.6 / 10.0 / 13.5; K = 2560, 260 10.1 / 10.6 / 14.8, 400
    // 13.1 / 11.9 / 16.7; K = 4096, 240 17.7 / 13.9 / 12.1, 260 17.0 / 13.6 / 20.0, 500 19.1 / 18.3 / 23.1, 520 19.7 / 27.6 / 31.2.
    if (tiles(64, 64) <= 256 && d->kp >= 2048) return launch_gemm_i8<T, 64, 64, 32, 32, 4>(d, st);
    if (tiles(64, 64) <= 512 && d->kp >= 2560) return launch_gemm_i8<T, 64, 64, 32, 32, 2>(d, st);
    return launch_gemm_i8<T, 64, 64, 32, 32, 1>(d, st);
}

extern "C" int mv_gemm_i8(const mv_gemm_i8_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_gemm_i8: null descriptor");
    MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_gemm_i8: element type %d", d->dtype);
    MV_REQUIRE(d->act == MV_ACT_NONE || d->act == MV_ACT_SILU, "mv_gemm_i8: activation %d", d->act);
    MV_REQUIRE(d->M >= 0 && d->M < (1ll << 31) && d->N >= 1 && d->kp >= 128 && d->kp % 128 == 0 && d->kp <= 131072,
               "mv_gemm_i8: M %ld, N %d, kp %d (a multiple of 128 up to 131072)", (long)d->M, d->N, d->kp);
    MV_REQUIRE(d->lda % 128 == 0 && d->ldw % 128 == 0 && d->lda >= d->kp && d->ldw >= d->kp && d->lda <= (1 << 22) && d->ldw <= (1 << 22),
               "mv_gemm_i8: lda %ld, ldw %ld for kp %d", (long)d->lda,
               (long)d->ldw, d->kp);
    if (d->M == 0) return MV_OK;
    MV_REQUIRE(d->a && d->w && d->a_scale && d->w_scale && d->out, "mv_gemm_i8: null pointer");
    MV_REQUIRE((((uintptr_t)d->a | (uintptr_t)d->w) & 15) == 0, "mv_gemm_i8: codes must be 16-byte aligned");
    return d->dtype == MV_F16 ? launch_gemm_i8_shape<half_t>(d, (hipStream_t)stream) : launch_gemm_i8_shape<bf16_t>(d, (hipStream_t)stream);
}

extern "C" int mv_linear_i8(const mv_linear_i8_desc* d, void* stream) {
    MV_REQUIRE(d, "mv_linear_i8: null descriptor");
    MV_REQUIRE(d->M >= 0 && d->K >= 1 && d->K <= 131071 && d->kp >= d->K && d->kp < d->K + 128 && d->kp % 128 == 0, "mv_linear_i8: M %ld, K %d (1 .. 131071: the sums fit 32 bits), kp %ld", (long)d->M, d->K, (long)d->kp);
    if (d->M == 0) return MV_OK;
    if (one_launch(d->M, d->kp)) {
        MV_REQUIRE(d->dtype == MV_F16 || d->dtype == MV_BF16, "mv_linear_i8: element type %d", d->dtype);
        MV_REQUIRE(d->act == MV_ACT_NONE || d->act == MV_ACT_SILU, "mv_linear_i8: activation %d", d->act);
        MV_REQUIRE(d->N >= 1 && d->ldw % 128 == 0 && d->ldw >= d->kp, "mv_linear_i8: N %d, ldw %ld for kp %ld", d->N, (long)d->ldw, (long)d->kp);
        MV_REQUIRE(d->x && d->w && d->w_scale && d->out && ((uintptr_t)d->w & 15) == 0, "mv_linear_i8: null or unaligned pointer");
        const int64_t grid = ((int64_t)d->N + 15) / 16;
        MV_REQUIRE_GRID("mv_linear_i8", grid, 512);
        MV_DISPATCH_TYPE(d->dtype, (linear_i8_few_kernel<T><<<(unsigned)grid, 512, 0, (hipStream_t)stream>>>(*d)));
        MV_CHECK_LAUNCH("mv_linear_i8");
        return MV_OK;
    }
    MV_REQUIRE(d->workspace, "mv_linear_i8: null workspace");
    mv_gemm_i8_desc g;
    g.a = (const int8_t*)d->workspace;
    g.a_scale = (const float*)(g.a + d->M * d->kp);
    g.w = d->w;
    g.w_scale = d->w_scale;
    g.bias = d->bias;
    g.residual = d->residual;
    g.out = d->out;
    g.M = d->M;
    g.N = d->N;
    g.kp = (int32_t)d->kp;
    g.lda = d->kp;
    g.ldw = d->ldw;
    g.ldr = d->ldr;
    g.ldo = d->ldo;
    g.act = d->act;
    g.dtype = d->dtype;
    const int rc = mv_quantize_rows_i8(d->x, d->ldx, d->M, d->K, d->dtype, (int8_t*)d->workspace, d->kp, (float*)g.a_scale, stream);
    return rc == MV_OK ? mv_gemm_i8(&g, stream) : rc;
}
