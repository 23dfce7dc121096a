// Paged multi-query attention with score modifiers on tcgen05: prompt chunks
// and chains of 64 packed query rows or more (row = query token x head of the
// GQA group), bf16 or fp16 pools of 16-token blocks, head_dim 64 or 128.
//
// One CTA owns (sequence b, KV head h), two query tiles w = 0, 1 of up to 128
// packed rows (whole tokens: tpt = 128 / G of them, so any group size works)
// and a run of 128-key tiles, nearest keys first, so that the running maximum
// is set early and O is rarely rescaled.  Three roles:
//
//   warps 16-18: producers.  K and V tiles arrive as 16-token block boxes of 64
//                columns (TMA, 128-byte swizzle) in a 160 KB ring, in the order
//                the MMAs read them.  Blocks past the sequence and ids outside
//                the pool are loaded from a coordinate outside the tensor map,
//                which fills zeros: what another block holds cannot reach the
//                result.
//   warp 19    : one thread issues S_w(i) = Q_w K(i)^T into TMEM columns
//                [128 w, 128 w + 128) and O_w += P_w(i) V(i) into [256 + D w, ..)
//                with P_w read from TMEM, the two tiles in turn: while the tensor
//                pipe works on one tile, the softmax of the other runs.
//   warps 0-15 : softmax of tile w = warp / 8; thread (c, r) owns keys
//                [64 c, 64 c + 64) of row r (TMEM lane r), 32 at a time, so that
//                four warps an SM sub-partition fit.  Half c's P goes over its own
//                S columns, [64 c, 64 c + 32).  Both halves of a row use one
//                reference maximum, which follows only when a half's maximum is far
//                above the last one (Half16; exact after the final division), so that
//                nearly all tiles need one pass and a vote of the two warps that
//                share the rows.
//
// Scores: the capped score is a polynomial on the FMA pipe (packed pairs,
// fma.rn.f32x2) of four coefficients while every z of a warp is in its range —
// with a cap of 50 that is |score| <= 25 —, then of five (40), and
// 1 - 2 / (1 + 2^(2 z log2 e)) beyond: the special function unit is left to the
// exponentials, which fill it.  Tiles that some row of a warp sees only in part
// take a path with per-key tests.
//
// Measured, 4 sequences x 1024 rows behind 4k to 8k keys, 32 / 8 heads of 128,
// bf16: 530 us uncapped (805 TFLOP/s), 649 us capped (660), 567 us with the
// distance bias, 682 us with both, 1016 us when nearly all scores are beyond the
// polynomials; the MMAs at cuBLAS's rate would take 263 us.  The tensor pipe is
// active 35 % of the time and the issue slots are 56 % taken: each tile is a chain
// S -> softmax -> P -> PV -> next S, and for heads of 128 two S and two O fill the
// 512 TMEM columns, so that no whole third S runs ahead (two half-width S a tile
// were not tried; heads of 64 leave 128 columns).  6 ragged prompts of up to 700
// rows, 16 heads of 64, fp16, prefix and bias: 90 us for 6.3 us of MMAs; 288 CTAs,
// one an SM, are two waves, with the tensor pipe active 10 % of the time.
//
// V rows that no row of the CTA sees (past the context, past the last row's
// position, left of the first row's window, all past the prefix) are zeroed in
// shared memory before the MMAs read them: 0 * NaN is NaN.
//
// With fewer CTAs than SMs the key tiles of each are split over several CTAs
// (n_split), which write unnormalised partial rows to the workspace;
// scored_tc_join_kernel joins them.  Every wait is bounded, as in the kernels
// beside this one; tcgen05.ld / st are warp-collective, so every branch around
// them is decided warp-uniformly.
#pragma once

#include "attn_prefill_tc.cuh"

namespace cx {

constexpr int kScKeys = 128;     // keys per tile

struct ScoredTcParams {
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* ctx_lens;
    const int32_t* q_start;      // NULL: one query row per sequence
    const float* slopes;
    const int32_t* prefix;
    TreeMask tree;               // TREE instantiations
    const void* q;
    void* out;
    float* part;                 // n_split > 1: [CTA][split][256][D + 2]
    int64_t q_stride;
    int32_t batch, hk, hq, group, tpt, n_ctiles, n_blocks, layer, window, n_split;
    int32_t q_dtype, out_dtype;
    float scale_log2;            // |scale| * log2(e)
    float z_scale;               // |scale| / cap
    float cap_log2;              // cap * log2(e)
    float c4[4], c5[5];          // the polynomials in the raw score (ScPoly), base 2
    float s4_max, s5_max;        // |score| up to which each holds
    int32_t neg;                 // scale < 0: Q is negated (tanh is odd)
    uint64_t wait_ns;            // limit of every pipeline wait (cx_set_wait_limit_ns)
};

template <int D_>
struct ScCfg {
    static constexpr int D = D_;
    static constexpr int HALVES = D / 64;
    static constexpr int Q_HALF = kTcRows * 128;
    static constexpr int Q_BYTES = HALVES * Q_HALF;
    static constexpr int KV_HALF = kScKeys * 128;
    static constexpr int SLOT = HALVES * KV_HALF;
    static constexpr int SLOTS = 160 * 1024 / SLOT;
    static constexpr int OFF_RING = 2 * Q_BYTES;
    static constexpr int OFF_BAR = OFF_RING + SLOTS * SLOT;
    static constexpr int OFF_GEOM = OFF_BAR + 256;
    static constexpr int OFF_RED = OFF_BAR + 320;       // one float a row of both tiles
    static constexpr int SMEM = OFF_RED + 1024 + 1024;  // + 1 KB alignment slack
    static constexpr int TMEM_COLS = 512;
    static constexpr int N_PROD = 3;
    static constexpr int SOFTMAX = 512;                 // softmax threads
    static constexpr int THREADS = SOFTMAX + 128;
    static constexpr int PROD_WARP = 16, MMA_WARP = 19;
    // setmaxnreg split of the 640 x 96 registers the block is launched with
    static constexpr int REG_SOFTMAX = 104, REG_OTHER = 64;
    static_assert(REG_SOFTMAX * SOFTMAX + REG_OTHER * 128 <= THREADS * 96, "register split");
    static_assert(SMEM <= 232448 && SMEM > 232448 / 2, "one CTA per SM");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The capped score as a polynomial in the raw product s: cap log2(e) tanh(z),
// z = s z_scale, is s times a polynomial in s^2 whose coefficients have
// z_scale^(2k + 1) multiplied in on the host.  Four coefficients hold for
// |z| <= 0.5 (absolute error of tanh 1.3e-7, least squares reweighted as for the
// five up to 0.8): the fewer, the less the FMA pipe, which the tensor pipe waits
// for here, has to do.
constexpr float kTanh4Max = 0.5f;
constexpr float kTanh4[4] = {0.9999976761901168f, -0.33320655207747635f, 0.1314514555556039f,
                             -0.043372480976138675f};
constexpr float kTanh5[5] = {kTanhC0, kTanhC1, kTanhC2, kTanhC3, kTanhC4};

// cap * log2(e) * tanh(z) for any z.
__device__ __forceinline__ float cap_any(float z, float cap_log2) {
    return fmaf(-2.f * cap_log2, rcp_approx(1.f + ex2_sfu(z * 2.8853900817779268f)), cap_log2);
}

// tcgen05.mma with A (M x 16, 16-bit pairs per 32-bit column, row i in lane i)
// read from TMEM.
__device__ __forceinline__ void sc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b,
                                          uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Ring item q of n key tiles, in the order the MMA thread reads them: K(0),
// then K(i + 1), V(i) for i = 0 .., and V(n - 1) last.
__device__ __forceinline__ void sc_item(int q, int n, bool& is_v, int& i) {
    is_v = q > 0 && ((q & 1) == 0 || q == 2 * n - 1);
    i = q == 0 ? 0 : q == 2 * n - 1 ? n - 1 : is_v ? q / 2 - 1 : (q + 1) / 2;
}
__device__ __forceinline__ int sc_pos_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int sc_pos_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

// The same where the two query tiles' places work on one tile's keys in turn (TREE):
// K(0), K(1), then K(i + 2), V(i), and the last two V.
__device__ __forceinline__ void sc_item2(int q, int n, bool& is_v, int& i) {
    const bool tail = q >= 2 * n - 2;
    is_v = q >= min(2, n) && (tail || (q & 1));
    i = q < min(2, n) ? q : tail ? q - n : is_v ? (q - 3) / 2 : q / 2 + 1;
}
__device__ __forceinline__ int sc_pos_k2(int i) { return i < 2 ? i : 2 * i - 2; }
__device__ __forceinline__ int sc_pos_v2(int i, int n) { return i >= n - 2 ? i + n : 2 * i + 3; }

// The key tiles of a CTA: n_pre tiles from block 0 (the prefix left of the
// window), then tiles from block kb0 on.
struct ScTiles {
    int n_pre, kb0, n;           // n: all of them
    __device__ __forceinline__ int block(int t) const {
        constexpr int BPT = kScKeys / kBlockTok;
        return t < n_pre ? t * BPT : kb0 + (t - n_pre) * BPT;
    }
};

// The `n` lowest bits, 0 <= n <= 32.
__device__ __forceinline__ uint32_t sc_below(int n) { return n >= 32 ? ~0u : (1u << n) - 1; }

// What the softmax warps need of a CTA's geometry, in shared memory and read
// there where it is used: their registers are all taken (two more values kept
// through the key loop, and the spills inside it, took 650 instead of 509 us for
// 4 x 1024 uncapped rows).
struct ScGeom {
    int n_pre, kb0, first, n_tiles, pre, win, ctx, run_hi, run_lo, nblk, pos0, t0, t_end;
};

// Which sequence, KV head and pair of query tiles CTA `cta` has: the longest
// contexts first (batches of up to 32; beyond, in order), within a sequence the
// latest tiles first, so that the last CTAs to start are short (without it the
// SMs idled 15 % of 512 CTAs' time).  Every lane of a warp calls it.  (WIDE: batches of
// up to 128, the same way.)
template <bool WIDE>
__device__ __forceinline__ void sc_place(const ScoredTcParams& p, int cta, int lane, int& b,
                                         int& h, int& ctile) {
    const int per_seq = p.hk * p.n_ctiles;
    const int place = cta / per_seq, rem = cta - place * per_seq;
    h = rem % p.hk;
    ctile = p.n_ctiles - 1 - rem / p.hk;
    b = place;
    if constexpr (WIDE) {
        if (p.batch > 128 || p.batch == 1) return;
        int ctx[4], before[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ctx[k] = lane + 32 * k < p.batch ? p.ctx_lens[lane + 32 * k] : INT32_MIN;
            before[k] = 0;
        }
#pragma unroll
        for (int k0 = 0; k0 < 4; ++k0) {
            for (int j = 32 * k0; j < min(p.batch, 32 * k0 + 32); ++j) {
                const int o = __shfl_sync(0xffffffffu, ctx[k0], j & 31);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    before[k] += o > ctx[k] || (o == ctx[k] && j < lane + 32 * k);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned at = __ballot_sync(
                0xffffffffu, lane + 32 * k < p.batch && before[k] == place);
            if (at) b = 32 * k + __ffs((int)at) - 1;
        }
        return;
    }
    if (p.batch > 32 || p.batch == 1) return;
    const int ctx = lane < p.batch ? p.ctx_lens[lane] : INT32_MIN;
    int before = 0;
    for (int j = 0; j < p.batch; ++j) {
        const int o = __shfl_sync(0xffffffffu, ctx, j);
        before += o > ctx || (o == ctx && j < lane);
    }
    const unsigned at = __ballot_sync(0xffffffffu, lane < p.batch && before == place);
    b = __ffs((int)at) - 1;
}

// TREE: the query rows are the nodes of a drafted tree; tiles that hold drafted keys
// are masked by 32 bits of a row's word at a time.  A tree whose rows fill one query
// tile would run as one chain S -> softmax -> P -> PV -> next S, with half of the
// softmax warps idle: both query tiles then hold its rows and take the key tiles in
// turn (`turns`), each with its own maxima, sums and O, which are joined at the end.  64
// trees of 26 nodes (104 rows) behind 1k to 8k keys, 8 KV heads of 128: 377 us as a chain, 371 in two places with the
// loads and MMAs issued as by the kernel without trees, 294 with elected threads.
template <int DH, typename E, bool CAP, bool ALIBI, bool TREE = false>
__global__ void __launch_bounds__(ScCfg<DH>::THREADS, 1)
    scored_tc_kernel(const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const ScoredTcParams p) {
    using C = ScCfg<DH>;
    constexpr int D = C::D, SLOTS = C::SLOTS, BPT = kScKeys / kBlockTok;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = sm + C::OFF_RING;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* empty = full + SLOTS;
    uint64_t* s_full = empty + SLOTS;      // [2] S_w ready
    uint64_t* p_full = s_full + 2;         // [2] P_w written, O_w rescaled
    uint64_t* o_done = p_full + 2;         // [2] PV_w complete
    uint64_t* mma_drain = o_done + 2;      // last commit of the MMA thread
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(mma_drain + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile int* s_issued = s_abort + 1;  // ring items whose loads were issued (TREE: by warp)

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = TREE ? (int)warp_uniform(tid >> 5) : tid >> 5;
    const int cta = (int)blockIdx.x;
    int b, h, ctile;
    sc_place<TREE>(p, cta, lane, b, h, ctile);
    const int G = p.group, tpt = p.tpt;
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T = p.q_start ? p.q_start[b + 1] - qs : 1;
    const int cap_tok = (int)(p.table_stride * kBlockTok);
    const int ctx = min(max(p.ctx_lens[b], 0), cap_tok);
    if (ctile == 0 && h == 0 && blockIdx.y == 0 && tid == 0) {
        if (p.ctx_lens[b] > cap_tok) raise_flag(CX_DEV_TABLE_OVERRUN);
        if (T < 0 || (ctx > 0 && T > ctx) || T > (int64_t)p.n_ctiles * 2 * tpt)
            raise_flag(CX_DEV_BAD_QLEN);
    }
    const int t0 = ctile * 2 * tpt;                          // first token of tile 0
    if (t0 >= T) return;
    const int nq = t0 + tpt < T ? 2 : 1;
    const bool turns = TREE && nq == 1;
    const int t_end = min(T, t0 + nq * tpt);
    const int pos0 = ctx - T;                                // position of token 0
    const int win = p.window;
    const int pre = p.prefix ? min(max(p.prefix[b], 0), TREE ? max(pos0, 0) : ctx) : 0;
    const int run_hi = min(pos0 + t_end - 1, ctx - 1);       // last key past the prefix
    const int run_lo = win > 0 ? max(0, pos0 + (TREE ? 0 : t0) - win + 1) : 0;
    ScTiles tiles;
    {
        const int hi = max(run_hi, pre - 1);
        tiles.kb0 = run_lo / kBlockTok;
        tiles.n_pre = pre > 0 ? (pre + kScKeys - 1) / kScKeys : 0;
        if (tiles.n_pre * BPT >= tiles.kb0 && tiles.n_pre > 0) tiles.n_pre = tiles.kb0 = 0;
        const int lo_tok = tiles.kb0 * kBlockTok;
        tiles.n = tiles.n_pre + (hi >= lo_tok ? (hi - lo_tok) / kScKeys + 1 : 0);
    }
    const int nblk_seq = (ctx + kBlockTok - 1) / kBlockTok;
    // this CTA's tiles, in order: first, first - 1, ...
    const int per = (tiles.n + p.n_split - 1) / p.n_split;
    const int i_lo = min(tiles.n, (int)blockIdx.y * per);
    const int n_tiles = min(tiles.n, i_lo + per) - i_lo;
    const int first = tiles.n - 1 - i_lo;

    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&full[s], C::N_PROD);
            mbar_init(&empty[s], 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&s_full[w], 1);
            mbar_init(&p_full[w], 256);
            mbar_init(&o_done[w], 1);
        }
        mbar_init(mma_drain, 1);
        *s_abort = 0;
        *s_issued = 0;
        if (TREE) s_issued[1] = s_issued[2] = 0;
        *reinterpret_cast<ScGeom*>(sm + C::OFF_GEOM) =
            ScGeom{tiles.n_pre, tiles.kb0, first, n_tiles, pre,  win,  ctx,
                   run_hi,      run_lo,    nblk_seq, pos0, t0, t_end};
        fence_mbar_init();
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(s_tmem)),
                     "r"(C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp < C::PROD_WARP) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFTMAX));
        const int w = warp >> 3, c = (warp >> 2) & 1, r = tid & 127;
        const int pair_bar = 4 + w * 4 + (warp & 3);         // the two warps of these 32 rows
        const int tw = turns ? 0 : w;                        // the query tile of its rows
        const int t = t0 + tw * tpt + r / G;                 // this row's token
        const int head = h * G + r % G;
        // ---- half a row of Q_w -> shared memory: 16-bit, K-major, swizzled, zero
        // padding rows.  Only the MMA warp waits for it (named barrier 3).
        {
            unsigned char* qdst = sm + w * C::Q_BYTES;
            const bool row_ok = t < min(t_end, t0 + (tw + 1) * tpt) && r < tpt * G;
            const int64_t row = (int64_t)(qs + t) * p.q_stride + (int64_t)head * D;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const int d = c * (D / 2) + k * 8;
                uint4 w4 = make_uint4(0, 0, 0, 0);
                if (row_ok) {
                    if (p.q_dtype == CX_F32) {
                        const float4* s4 = reinterpret_cast<const float4*>(
                            static_cast<const float*>(p.q) + row + d);
                        const float4 a = __ldg(s4), e = __ldg(s4 + 1);
                        w4 = make_uint4(Half16<E>::pack(a.x, a.y), Half16<E>::pack(a.z, a.w),
                                        Half16<E>::pack(e.x, e.y), Half16<E>::pack(e.z, e.w));
                    } else {
                        w4 = __ldg(
                            reinterpret_cast<const uint4*>(static_cast<const E*>(p.q) + row + d));
                    }
                    if (p.neg) {
                        w4.x ^= 0x80008000u;
                        w4.y ^= 0x80008000u;
                        w4.z ^= 0x80008000u;
                        w4.w ^= 0x80008000u;
                    }
                }
                *reinterpret_cast<uint4*>(qdst + tc_swz(r, d, kTcRows)) = w4;
            }
            fence_async_smem();
            named_bar_arrive(3, C::SOFTMAX + 32);
        }
        if (w < nq || turns) {
            const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tm_s = tmem + w * kScKeys + c * 64 + lane_off;
            const uint32_t tm_o = tmem + 2 * kScKeys + w * D + c * (D / 2) + lane_off;
            volatile const ScGeom& g = *reinterpret_cast<const ScGeom*>(sm + C::OFF_GEOM);
            int pos = pos0 + t;
            const float slope = ALIBI ? p.slopes[head] * 1.4426950408889634f : 0.f;
            const float cl = p.cap_log2;
            const f2 sl2 = f2_of(p.scale_log2, p.scale_log2);
            auto dup = [](float x) { return f2_of(x, x); };
            // s P(s^2) + add, by four or five coefficients
            auto poly4 = [&](f2 s, f2 add) {
                const f2 y = f2_mul(s, s);
                f2 q = f2_fma(dup(p.c4[3]), y, dup(p.c4[2]));
                q = f2_fma(q, y, dup(p.c4[1]));
                return f2_fma(s, f2_fma(q, y, dup(p.c4[0])), add);
            };
            auto poly5 = [&](f2 s) {
                const f2 y = f2_mul(s, s);
                f2 q = f2_fma(dup(p.c5[4]), y, dup(p.c5[3]));
                q = f2_fma(q, y, dup(p.c5[2]));
                q = f2_fma(q, y, dup(p.c5[1]));
                return f2_mul(s, f2_fma(q, y, dup(p.c5[0])));
            };
            bool wide = false;     // some score was beyond four coefficients
            bool any_bad = false;
            for (int blk = lane; blk < nblk_seq; blk += 32) {
                const int id = p.tables[(int64_t)b * p.table_stride + blk];
                any_bad |= id < 0 || id >= p.n_blocks;
            }
            any_bad = __any_sync(0xffffffffu, any_bad);
            // positions of this warp's first and last row (TREE: of the last key that
            // every node sees, and behind every node)
            const int w_lo = TREE ? pos0 - 1 : __shfl_sync(0xffffffffu, pos, 0);
            const int w_hi = __shfl_sync(0xffffffffu, pos, 31);
            if constexpr (TREE) {
                if (t < t_end) pos = pos0 + p.tree.depths[qs + t];
            }
            // the reference of a row (base 2): kLead above the maximum it is set to, and
            // following a maximum that is kRescale above it (Half16)
            constexpr float kRescale = Half16<E>::kGrowLog2, kLead = Half16<E>::kLeadLog2;
            float m = -INFINITY, l = 0.f;
            // `ok` turns false (warp-uniformly) when a bounded wait gives up; the warp
            // then skips its waits and TMEM work but keeps meeting the other half's
            // barrier, so that warp never waits forever.
            bool ok = true;
            float* red = reinterpret_cast<float*>(sm + C::OFF_RED) + w * 128 + r;
            // the larger (sum: the total) of both halves' values of this row; every
            // thread of the two warps calls it
            auto both = [&](float x, bool sum) {
                if (c == 1) *red = x;
                named_bar_sync(pair_bar, 64);
                if (c == 0) {
                    x = sum ? x + *red : fmaxf(x, *red);
                    *red = x;
                }
                named_bar_sync(pair_bar, 64);
                return c == 0 ? x : *red;    // (c == 1 alone reads it now: it writes it next)
            };
            for (int i = 0; i < (turns ? (g.n_tiles + 1 - w) >> 1 : g.n_tiles); ++i) {
                if (ok)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[w], i & 1, s_abort,
                                                                   p.wait_ns));
                const int tile = g.first - (turns ? 2 * i + w : i);
                const int b0 = tile < g.n_pre ? tile * BPT : g.kb0 + (tile - g.n_pre) * BPT;
                const int kb = b0 * kBlockTok + c * 64;      // this half's first key
                unsigned bad4 = 0;                           // its bad blocks
                if (any_bad) {
                    const int blk = b0 + c * 4 + lane;
                    const int id = lane < 4 && blk < g.nblk
                                       ? p.tables[(int64_t)b * p.table_stride + blk]
                                       : 0;
                    bad4 = __ballot_sync(0xffffffffu, id < 0 || id >= p.n_blocks);
                }
                // of this warp's 32 rows: some key is ahead of some row; some row does not
                // see some key
                const bool ahead = kb + 63 > w_lo;
                const bool edge =
                    bad4 != 0 || !(kb + 64 <= g.pre ||
                                   (!ahead && (g.win <= 0 || kb > w_hi - g.win)));
                // the final scores (base 2) of keys kb + j0 .. kb + j0 + 31
                auto score = [&](float (&v)[32], int j0) {
                    bool small = true;
                    if constexpr (CAP) {
                        float a0 = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            a0 = max3(a0, fabsf(v[j]), fabsf(v[j + 1]));
                        small = !__any_sync(0xffffffffu, a0 > p.s5_max);
                    }
                    if (CAP && !small) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = cap_any(v[j] * p.z_scale, cl);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            f2 x = f2_of(v[j], v[j + 1]);
                            x = CAP ? poly5(x) : f2_mul(x, sl2);
                            f2_get(x, v[j], v[j + 1]);
                        }
                    }
                    const int k0j = kb + j0;
                    if constexpr (ALIBI) {
                        // slope * -|pos - key|: the distance is exact, so near keys, whose
                        // weights count, lose nothing in long contexts
                        const float d0 = (float)(k0j - pos);
                        if (TREE && ahead) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                int key = k0j + j;
                                if (key >= pos0)
                                    key = tree_key_pos(p.tree, qs, T, pos0, key - pos0);
                                v[j] = fmaf(-slope, fabsf((float)(key - pos)), v[j]);
                            }
                        } else if (ahead) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                v[j] = fmaf(-slope, fabsf(d0 + (float)j), v[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                v[j] = fmaf(slope, d0 + (float)j, v[j]);
                        }
                    }
                    if (edge) {
                        const int jp = g.pre - k0j, hi = pos - k0j, win = g.win;
                        const int lo = win > 0 ? hi - win : INT32_MIN;
                        if constexpr (TREE) {
                            // bits of the committed keys that the row sees, then of its kin
                            const int jb = min(max(pos0 - k0j, 0), 32);
                            const int first = min(max(lo + 1, 0), 32);
                            uint32_t keep = sc_below(jb) & (~sc_below(first) | sc_below(min(max(jp, 0), 32)));
                            if (jb < 32 && t < t_end)
                                keep |= tree_bits(p.tree, qs + t, t, k0j - pos0);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                v[j] = (keep >> j) & 1u ? v[j] : -INFINITY;
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const bool keep = j < jp || (j <= hi && j > lo);
                                v[j] = keep ? v[j] : -INFINITY;
                            }
                        }
                        if (bad4 != 0) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                v[j] = (bad4 >> ((j0 + j) >> 4)) & 1u ? -INFINITY : v[j];
                        }
                    }
                };
                // ---- p = 2^(x - m) as 16-bit pairs, and this half's row maximum, in one
                // pass against the reference maximum so far; again, against a new one,
                // when the maximum is kRescale above it, or key by key when a score
                // was beyond the polynomial.  Both are rare past the first tile, and the
                // exponentials need not wait for a maximum.  (A growth of 2^8 alone, as the
                // kernels beside this one have, took 712 instead of 548 us here: some of
                // 32 rows grows by that in every few tiles.) ----
                // one packed expression scores a pair: all keys seen, none ahead of its
                // row, and no score of a tile before was beyond the polynomial
                bool plain = !edge && !(ALIBI && ahead) && !wide;
                if (ok) tc_fence_after();
                uint32_t pk[32];
                float psum = 0.f;
                for (;;) {
                    float mt = -INFINITY, largest = 0.f;
                    const float m_use = m == -INFINITY ? 0.f : m;
                    const f2 negm = f2_of(-m_use, -m_use);
                    f2 sum0 = 0, sum1 = 0;     // two fp32 zeros each
                    if (ok) {
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch) {
                            float v[32];
                            tc_ld32(tm_s + ch * 32, v);
                            tc_wait_ld();
                            const float base = slope * (float)(kb + ch * 32 - pos) - m_use;
                            auto emit = [&](auto plain_tag) {
                                constexpr bool PLAIN = decltype(plain_tag)::value;
                                // maxima: of raw scores, of x with a bias, of |raw| for the cap
                                float a0 = -INFINITY, a1 = -INFINITY, n0 = 0.f, n1 = 0.f;
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    const float v0 = v[2 * k], v1 = v[2 * k + 1];
                                    if (!(PLAIN && ALIBI)) {
                                        if (k & 1)
                                            a1 = max3(a1, v0, v1);
                                        else
                                            a0 = max3(a0, v0, v1);
                                    }
                                    if (PLAIN && CAP) {
                                        if (k & 1)
                                            n1 = max3(n1, fabsf(v0), fabsf(v1));
                                        else
                                            n0 = max3(n0, fabsf(v0), fabsf(v1));
                                    }
                                    f2 x = f2_of(v0, v1);
                                    if constexpr (!PLAIN) {
                                        x = f2_add(x, negm);           // v holds the scores
                                    } else {
                                        // bias slope * (key - pos): exact near the query
                                        const f2 add =
                                            ALIBI ? f2_of(fmaf(slope, (float)(2 * k), base),
                                                          fmaf(slope, (float)(2 * k + 1), base))
                                                  : negm;
                                        x = CAP ? poly4(x, add) : f2_fma(x, sl2, add);
                                    }
                                    float e0, e1;
                                    f2_get(x, e0, e1);
                                    if (PLAIN && ALIBI) {
                                        if (k & 1)
                                            a1 = max3(a1, e0, e1);
                                        else
                                            a0 = max3(a0, e0, e1);
                                    }
                                    e0 = ex2_sfu(e0);
                                    e1 = ex2_sfu(e1);
                                    // (the sum of what the PV product gets: numerator and
                                    // denominator round alike)
                                    const uint32_t u = Half16<E>::pack(e0, e1);
                                    if (k & 1)
                                        sum1 = f2_add(sum1, Half16<E>::unpack(u));
                                    else
                                        sum0 = f2_add(sum0, Half16<E>::unpack(u));
                                    pk[ch * 16 + k] = u;
                                }
                                mt = max3(mt, a0, a1);
                                if (PLAIN && CAP) largest = max3(largest, n0, n1);
                            };
                            if (plain) {
                                emit(std::true_type{});
                            } else {
                                score(v, ch * 32);
                                emit(std::false_type{});
                            }
                        }
                    }
                    bool large = false;
                    if (plain) {
                        if (CAP) large = __any_sync(0xffffffffu, largest > p.s4_max);
                        // (beyond its range the polynomial may be far above the cap: no
                        // maximum of such scores becomes a reference)
                        if (ALIBI)
                            mt = large ? -INFINITY : mt + m_use;
                        else
                            mt = CAP ? cap_any(mt * p.z_scale, cl) : mt * p.scale_log2;
                    }
                    const bool grow =
                        mt > m + kRescale || (m == -INFINITY && mt > -INFINITY);
                    float s0, s1, s2, s3;
                    f2_get(sum0, s0, s1);
                    f2_get(sum1, s2, s3);
                    psum = (s0 + s1) + (s2 + s3);
                    if (bar_red_and(pair_bar, 64, !(ok && (grow || large)))) break;
                    const float mr = both(mt, false);
                    float alpha = 1.f;
                    if (mr > m + kRescale || (m == -INFINITY && mr > -INFINITY)) {
                        alpha = exp2f(m - (mr + kLead));
                        m = mr + kLead;
                    }
                    l *= alpha;
                    // O_w holds PV_w(0 .. i-1): S_w(i) was issued after PV_w(i-1)
                    if (ok && i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                        for (int k = 0; k < D / 32; ++k) {
                            float o[16];
                            sc_ld16(tm_o + k * 16, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= alpha;
                            sc_st16(tm_o + k * 16, reinterpret_cast<const uint32_t(&)[16]>(o));
                        }
                        tc_wait_st();
                    }
                    wide = wide || large;
                    plain = plain && !large;
                }
                if (!ok) continue;
                // zero the V rows that no row of the CTA sees
                if (w == 0 || turns) {
                    const int pre = g.pre, ctx = g.ctx, run_hi = g.run_hi, run_lo = g.run_lo;
                    const int kbase = kb - c * 64;
                    auto dead = [&](int key) {
                        return key >= ctx || (key >= pre && (key > run_hi || key < run_lo));
                    };
                    const bool any_dead = kbase + kScKeys > ctx ||
                                          (kbase + kScKeys > pre &&
                                           (kbase + kScKeys - 1 > run_hi || kbase < run_lo));
                    if (any_dead) {
                        const int q = turns ? sc_pos_v2(2 * i + w, g.n_tiles)
                                            : sc_pos_v(i, g.n_tiles);
                        ok = __all_sync(0xffffffffu,
                                        mbar_wait_bounded(&full[q % SLOTS], (q / SLOTS) & 1,
                                                          s_abort, p.wait_ns));
                        if (!ok) continue;
                        if (dead(kbase + r)) {
                            // half c of the row's 16-byte chunks
                            uint4* z = reinterpret_cast<uint4*>(ring + (q % SLOTS) * C::SLOT +
                                                                r * 128);
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                const int ch = c * (D / 16) + k;
                                z[(ch >> 3) * (C::KV_HALF / 16) + (ch & 7)] =
                                    make_uint4(0, 0, 0, 0);
                            }
                        }
                        fence_async_smem();
                    }
                }
                // P over this half's first 32 S columns (keys 2k, 2k + 1 of the half in
                // column k)
                tc_st32(tm_s, reinterpret_cast<const float*>(pk));
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[w]);
                l += psum;
            }
            // ---- epilogue: the row's denominator over both halves, then this half's
            // columns to the output, or to this split's part ----
            const int n_tiles = turns ? (g.n_tiles + 1 - w) >> 1 : g.n_tiles;
            if (n_tiles > 0 && ok) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[w], (n_tiles - 1) & 1,
                                                                s_abort, p.wait_ns));
                if (ok) tc_fence_after();
            }
            l = both(l, true);
            // where the row goes, worked out again rather than kept through the key loop
            int tid_e;
            asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid_e));
            const int r_e = tid_e & 127, t_e = g.t0 + w * tpt + r_e / G, head_e = h * G + r_e % G;
            const bool row_ok = t_e < min((int)g.t_end, (int)g.t0 + (w + 1) * tpt) && r_e < tpt * G;
            float* part = nullptr;
            if (TREE && turns) {
                // both places' rows: references and sums through the ring, which nothing
                // reads any more behind the barrier
                float* x = reinterpret_cast<float*>(ring);
                named_bar_sync(2, C::SOFTMAX);
                if (c == 0) {
                    x[w * 128 + r] = m;
                    x[256 + w * 128 + r] = l;
                }
                if (!ok) *s_abort = 1;
                // (the other place's O as well is read below: its warps saw its last product
                // finish and met these here)
                tc_fence_before();
                named_bar_sync(2, C::SOFTMAX);
                tc_fence_after();
                ok = __all_sync(0xffffffffu, !*s_abort);
                const float m0 = x[r], m1 = x[128 + r], M = fmaxf(m0, m1);
                const float f0 = exp2f(m0 - ref_base(M)), f1 = exp2f(m1 - ref_base(M));
                const float L = x[256 + r] * f0 + x[384 + r] * f1;
                const bool two = g.n_tiles > 1;              // (the second has an O)
                const int64_t o_row = ((int64_t)(qs + (g.t0 + r / G)) * p.hq + h * G + r % G) * D;
                const bool in = (g.t0 + r / G) < min((int)g.t_end, (int)g.t0 + tpt) && r < tpt * G;
                float* to = nullptr;
                if (p.n_split > 1) {
                    to = p.part + (((int64_t)cta * p.n_split + blockIdx.y) * 256 + r) * (D + 2);
                    if (c == 0 && w == 0) {
                        to[D] = ok ? M : -INFINITY;
                        to[D + 1] = L;
                    }
                }
                const float inv = to ? 1.f : sum_inv(L);
                // a quarter of the columns a thread: 16 at a time
                const uint32_t tm_c = tmem + 2 * kScKeys + lane_off;
#pragma unroll 1
                for (int k = 0; ok && k < D / 64; ++k) {
                    const int col = c * (D / 2) + w * (D / 4) + k * 16;
                    float a[16], b[16];
                    __syncwarp();
                    if (g.n_tiles > 0) {
                        sc_ld16(tm_c + col, a);
                        if (two) sc_ld16(tm_c + D + col, b);
                        tc_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float y = g.n_tiles > 0 ? a[e] * f0 : 0.f;
                        a[e] = (two ? fmaf(b[e], f1, y) : y) * inv;
                    }
                    if (!in) continue;
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        if (to)
                            *reinterpret_cast<float2*>(to + col + e) = make_float2(a[e], a[e + 1]);
                        else
                            store2_as(p.out, p.out_dtype, o_row + col + e, a[e], a[e + 1]);
                    }
                }
                if (!ok) raise_flag(CX_DEV_WAIT_TIMEOUT);
            } else {
            if (p.n_split > 1) {
                part = p.part + (((int64_t)cta * p.n_split + blockIdx.y) * 256 + w * 128 + r_e) *
                                    (D + 2);
                if (c == 0) {
                    part[D] = ok ? m : -INFINITY;
                    part[D + 1] = l;
                }
            }
            if (ok) {
                const float inv = part ? 1.f : sum_inv(l);
                const int64_t o_row = ((int64_t)(qs + t_e) * p.hq + head_e) * D + c * (D / 2);
#pragma unroll 1
                for (int k = 0; k < D / 64; ++k) {
                    float ov[32];
                    __syncwarp();          // padding rows have skipped the stores
                    if (n_tiles > 0) {
                        tc_ld32(tm_o + k * 32, ov);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = 0.f;
                    }
                    if (!row_ok) continue;
                    if (part) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            *reinterpret_cast<float2*>(part + c * (D / 2) + k * 32 + e) =
                                make_float2(ov[e], ov[e + 1]);
                    } else if (p.out_dtype == CX_F32) {
                        float* dst = static_cast<float*>(p.out) + o_row + k * 32;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(dst + e) = make_float4(
                                ov[e] * inv, ov[e + 1] * inv, ov[e + 2] * inv, ov[e + 3] * inv);
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                                                              o_row + k * 32);
                        const bool bf = p.out_dtype == CX_BF16;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t u[4];
#pragma unroll
                            for (int k2 = 0; k2 < 4; ++k2) {
                                const float x = ov[e + 2 * k2] * inv, y = ov[e + 2 * k2 + 1] * inv;
                                u[k2] = bf ? Half16<__nv_bfloat16>::pack(x, y)
                                           : Half16<__half>::pack(x, y);
                            }
                            dst[e / 8] = make_uint4(u[0], u[1], u[2], u[3]);
                        }
                    }
                }
            } else {
                *s_abort = 1;
                raise_flag(CX_DEV_WAIT_TIMEOUT);
            }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_OTHER));
        if constexpr (TREE) {
            // Whole warps that elect a thread for every MMA and box (as latent_tc_kernel's).
            const uint32_t tries =
                (uint32_t)min((unsigned long long)p.wait_ns / 500 + 1, 1ull << 30);
            const int n = (int)warp_uniform(n_tiles);
            const bool tn = warp_uniform(turns) != 0;
            bool ok = true;
            if (warp < C::MMA_WARP) {
                const int pw = warp - C::PROD_WARP;
                const int32_t* tab = p.tables + (int64_t)b * p.table_stride;
                auto id_of = [&](int q) {             // this lane's block of item q; INT32_MIN: none
                    bool is_v;
                    int i;
                    if (tn)
                        sc_item2(q, n, is_v, i);
                    else
                        sc_item(q, n, is_v, i);
                    const int blk = tiles.block(first - i) + lane;
                    return q < 2 * n && lane < BPT && blk < nblk_seq ? tab[blk] : INT32_MIN;
                };
                int id = id_of(0), id_next = id_of(1), s = 0;
                uint32_t use = 0;                     // parity of the fill before, of slot s
                for (int q = 0; q < 2 * n; ++q) {
                    bool is_v;
                    int i;
                    if (tn)
                        sc_item2(q, n, is_v, i);
                    else
                        sc_item(q, n, is_v, i);
                    int z = -1;                       // outside the map: the copy fills zeros
                    if (id >= 0 && id < p.n_blocks)
                        z = (p.layer * p.n_blocks + id) * p.hk + h;
                    else if (id != INT32_MIN)
                        raise_flag(CX_DEV_BAD_BLOCK);
                    int z3[3];
#pragma unroll
                    for (int k = 0; k < 3; ++k) z3[k] = __shfl_sync(0xffffffffu, z, pw + 3 * k);
                    id = id_next;
                    id_next = id_of(q + 2);
                    if (q >= SLOTS && !(ok = el_wait(&empty[s], use ^ 1, s_abort, tries))) break;
                    const uint32_t bar = warp_uniform(smem_addr(&full[s]));
                    const uint32_t dst = warp_uniform(smem_addr(ring + s * C::SLOT + pw * 2048));
                    const bool v = warp_uniform(is_v) != 0;
                    el_expect(bar, (pw < 2 ? 3 : 2) * (C::SLOT / BPT));
                    auto boxes = [&](const CUtensorMap* m, auto count) {
#pragma unroll
                        for (int k = 0; k < decltype(count)::value; ++k)
#pragma unroll
                            for (int hf = 0; hf < C::HALVES; ++hf)
                                el_tma(dst + hf * C::KV_HALF + k * 3 * 2048, m, bar, hf * 64, 0,
                                       z3[k]);
                    };
                    if (pw < 2) {
                        if (v)
                            boxes(&tmv, std::integral_constant<int, 3>{});
                        else
                            boxes(&tmk, std::integral_constant<int, 3>{});
                    } else {
                        if (v)
                            boxes(&tmv, std::integral_constant<int, 2>{});
                        else
                            boxes(&tmk, std::integral_constant<int, 2>{});
                    }
                    if (lane == 0) s_issued[pw] = q + 1;
                    if (++s == SLOTS) {
                        s = 0;
                        use ^= 1;
                    }
                }
            } else {
                constexpr uint32_t idesc_s = sc_idesc<E>(kTcRows, kScKeys, 0);
                constexpr uint32_t idesc_o = sc_idesc<E>(kTcRows, D, 1);
                named_bar_sync(3, C::SOFTMAX + 32);    // Q_0, Q_1 are in shared memory
                const uint32_t tm = warp_uniform(tmem);
                const uint32_t q_lo = warp_uniform(el_desc_lo(sm, 16));
                const uint32_t k_lo = warp_uniform(el_desc_lo(ring, 16));
                const uint32_t v_lo = warp_uniform(el_desc_lo(ring, C::KV_HALF));
                auto wait = [&](uint64_t* bar, int parity) {
                    const bool r = el_wait(bar, parity & 1, s_abort, tries);
                    if (r) tc_fence_after();
                    return r;
                };
                auto issue_s = [&](int w, int slot) {
                    const uint32_t kd = warp_uniform(k_lo + (uint32_t)(slot * (C::SLOT >> 4)));
                    const uint32_t qd = warp_uniform(q_lo + (uint32_t)(w * (C::Q_BYTES >> 4)));
                    const uint32_t d = warp_uniform(tm + w * kScKeys);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        el_mma(d, qd + (((kk >> 2) * C::Q_HALF + (kk & 3) * 32) >> 4),
                               kd + (((kk >> 2) * C::KV_HALF + (kk & 3) * 32) >> 4), idesc_s,
                               kk > 0 ? 1u : 0u);
                    el_commit(&s_full[w]);
                };
                auto issue_pv = [&](int w, int slot, bool acc) {
                    const uint32_t vd = warp_uniform(v_lo + (uint32_t)(slot * (C::SLOT >> 4)));
                    const uint32_t o_t = warp_uniform(tm + 2 * kScKeys + w * D);
                    const uint32_t p_t = warp_uniform(tm + w * kScKeys), a0 = warp_uniform(acc);
#pragma unroll
                    for (int kk = 0; kk < kScKeys / 16; ++kk)
                        el_mma_ts(o_t, p_t + (kk >> 2) * 64 + (kk & 3) * 8, vd + kk * (2048 >> 4),
                                  idesc_o, kk > 0 ? 1u : a0);
                };
                // key tiles ahead: one for both query tiles, or one for either place
                const int ahead = tn ? 2 : 1, nqw = tn ? 1 : nq;
                auto pos_k = [&](int i) { return tn ? sc_pos_k2(i) : sc_pos_k(i); };
                auto pos_v = [&](int i) { return tn ? sc_pos_v2(i, n) : sc_pos_v(i, n); };
                for (int i = 0; ok && i < min(ahead, n); ++i) {
                    if (!(ok = wait(&full[i], 0))) break;
                    issue_s(i, i);
                    if (nqw == 2) issue_s(1, i);
                    el_commit(&empty[i]);
                }
                for (int i = 0; ok && i < n; ++i) {
                    const bool next = i + ahead < n;
                    const int kp = pos_k(i + ahead), vp = pos_v(i);
                    if (next && !(ok = wait(&full[kp % SLOTS], kp / SLOTS))) break;
                    if (!(ok = wait(&full[vp % SLOTS], vp / SLOTS))) break;
                    for (int k = 0; ok && k < nqw; ++k) {
                        const int w = tn ? i & 1 : k, j = tn ? i >> 1 : i;
                        if (!(ok = wait(&p_full[w], j))) break;
                        issue_pv(w, vp % SLOTS, j > 0);
                        el_commit(&o_done[w]);
                        if (next) issue_s(w, kp % SLOTS);
                    }
                    if (!ok) break;
                    el_commit(&empty[vp % SLOTS]);
                    if (next) el_commit(&empty[kp % SLOTS]);
                }
                el_commit(mma_drain);
            }
            if (!ok && lane == 0) {
                *s_abort = 1;
                raise_flag(CX_DEV_WAIT_TIMEOUT);
            }
        } else if (warp < C::MMA_WARP) {
            // ---------------- producers: blocks pw, pw + 3, .. of each item ----------------
            const int pw = warp - C::PROD_WARP;
            const int32_t* tab = p.tables + (int64_t)b * p.table_stride;
            int my_blocks = 0;
            for (int k = pw; k < BPT; k += C::N_PROD) ++my_blocks;
            // block id of this lane's block (lane < 8) of item q; -1: load zeros
            auto item_ids = [&](int q) {
                bool is_v;
                int i;
                sc_item(q, n_tiles, is_v, i);
                int id = -1;
                if (lane < BPT) {
                    const int blk = tiles.block(first - i) + lane;
                    if (blk < nblk_seq) {
                        id = tab[blk];
                        if (id < 0 || id >= p.n_blocks) {
                            raise_flag(CX_DEV_BAD_BLOCK);
                            id = -1;
                        }
                    }
                }
                return id;
            };
            int ids = n_tiles > 0 ? item_ids(0) : -1;
            for (int q = 0; q < 2 * n_tiles; ++q) {
                bool is_v;
                int i;
                sc_item(q, n_tiles, is_v, i);
                const int next = q + 1 < 2 * n_tiles ? item_ids(q + 1) : -1;
                const int s = q % SLOTS, use = q / SLOTS;
                bool go = true;
                if (lane == 0 && use > 0 &&
                    !mbar_wait_bounded(&empty[s], (use - 1) & 1, s_abort, p.wait_ns))
                    go = false;
                go = __shfl_sync(0xffffffffu, go, 0) && !*s_abort;
                // all three warps issue an item or none does: s_issued stays exact
                if (!bar_red_and(1, 32 * C::N_PROD, go)) {
                    if (lane == 0) {
                        *s_abort = 1;
                        raise_flag(CX_DEV_WAIT_TIMEOUT);
                    }
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&full[s], my_blocks * (C::SLOT / BPT));
                unsigned char* dst = ring + s * C::SLOT;
                for (int k = pw; k < BPT; k += C::N_PROD) {
                    const int id = __shfl_sync(0xffffffffu, ids, k);
                    if (lane == 0) {
                        // outside the map: the copy fills zeros
                        const int z = id >= 0 ? (p.layer * p.n_blocks + id) * p.hk + h : -1;
#pragma unroll
                        for (int hf = 0; hf < C::HALVES; ++hf)
                            tma_load_3d(dst + hf * C::KV_HALF + k * 2048, is_v ? &tmv : &tmk,
                                        &full[s], hf * 64, 0, z);
                    }
                }
                if (pw == 0 && lane == 0) *s_issued = q + 1;
                ids = next;
            }
        } else {
            // ---------------- MMA issuer ----------------
            named_bar_sync(3, C::SOFTMAX + 32);        // Q_0, Q_1 are in shared memory
            if (lane == 0) {
                constexpr uint32_t idesc_s = sc_idesc<E>(kTcRows, kScKeys, 0);
                constexpr uint32_t idesc_o = sc_idesc<E>(kTcRows, D, 1);
                // Descriptors of the first k-step; the others are constants further (16-byte
                // units; shared memory ends below 2^18, so the address field never
                // carries).  Built anew for every MMA they kept this thread busy for
                // longer than the MMAs run.
                const uint64_t q_desc = tc_sdesc(smem_addr(sm), 16, 1024);
                const uint64_t k_desc = tc_sdesc(smem_addr(ring), 16, 1024);
                const uint64_t v_desc = tc_sdesc(smem_addr(ring), C::KV_HALF, 1024);
                bool ok = true;
                auto wait = [&](uint64_t* bar, int parity) {
                    const bool r = mbar_wait_bounded(bar, parity & 1, s_abort, p.wait_ns);
                    if (r) tc_fence_after();
                    return r;
                };
                auto issue_s = [&](int w, int slot) {
                    const uint64_t kd = k_desc + (uint32_t)(slot * (C::SLOT >> 4));
                    const uint64_t qd = q_desc + (uint32_t)(w * (C::Q_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        tc_mma(tmem + w * kScKeys,
                               qd + (((kk >> 2) * C::Q_HALF + (kk & 3) * 32) >> 4),
                               kd + (((kk >> 2) * C::KV_HALF + (kk & 3) * 32) >> 4), idesc_s,
                               kk > 0);
                    tc_commit(&s_full[w]);
                };
                // O_w += P_w V: 128 keys in steps of 16
                auto issue_pv = [&](int w, int slot, bool acc) {
                    const uint64_t vd = v_desc + (uint32_t)(slot * (C::SLOT >> 4));
                    const uint32_t o_t = tmem + 2 * kScKeys + w * D, p_t = tmem + w * kScKeys;
#pragma unroll
                    for (int kk = 0; kk < kScKeys / 16; ++kk)
                        sc_mma_ts(o_t, p_t + (kk >> 2) * 64 + (kk & 3) * 8, vd + kk * (2048 >> 4),
                                  idesc_o, (acc || kk > 0) ? 1u : 0u);
                };
                if (n_tiles > 0) {
                    ok = wait(&full[0], 0);
                    if (ok) {
                        issue_s(0, 0);
                        if (nq == 2) issue_s(1, 0);
                        tc_commit(&empty[0]);
                    }
                }
                for (int i = 0; ok && i < n_tiles; ++i) {
                    const bool next = i + 1 < n_tiles;
                    const int kp = sc_pos_k(i + 1), vp = sc_pos_v(i, n_tiles);
                    if (next && !(ok = wait(&full[kp % SLOTS], kp / SLOTS))) break;
                    if (!(ok = wait(&full[vp % SLOTS], vp / SLOTS))) break;
                    for (int w = 0; ok && w < nq; ++w) {
                        if (!(ok = wait(&p_full[w], i))) break;
                        issue_pv(w, vp % SLOTS, i > 0);
                        tc_commit(&o_done[w]);
                        if (next) issue_s(w, kp % SLOTS);   // after PV_w(i)
                    }
                    if (!ok) break;
                    tc_commit(&empty[vp % SLOTS]);
                    if (next) tc_commit(&empty[kp % SLOTS]);
                }
                if (!ok) {
                    *s_abort = 1;
                    raise_flag(CX_DEV_WAIT_TIMEOUT);
                }
                tc_commit(mma_drain);   // completes once every MMA issued above has
            }
        }
    }

    // ---- teardown: drain this CTA's own copies and MMAs, then free TMEM ----
    tc_fence_before();
    __syncthreads();
    if (*s_abort && tid == 0) {
        int issued = *s_issued;
        if (TREE) issued = max(issued, max(s_issued[1], s_issued[2]));
        for (int s = 0; s < SLOTS; ++s) {
            const int uses = issued > s ? (issued - 1 - s) / SLOTS + 1 : 0;
            // (TREE: a slot that not all producers came to never completes; what the others
            // loaded into it ends well within the wait)
            if (uses > 0)
                mbar_wait_bounded(&full[s], (uses - 1) & 1, nullptr,
                                  TREE ? 20000000ull : kWaitLimitNs);
        }
    }
    if (tid == C::MMA_WARP * 32) mbar_wait_bounded(mma_drain, 0, nullptr, kWaitLimitNs);
    __syncthreads();
    tc_fence_after();
    if (warp == C::MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(C::TMEM_COLS)
                     : "memory");
}

// Joins the parts of split rows: one warp per (CTA, row); part rows hold the
// unnormalised O, its reference maximum (base 2) and the denominator.
template <int D, bool TREE = false>      // (TREE: the one of its translation unit)
__global__ void __launch_bounds__(256) scored_tc_join_kernel(const ScoredTcParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t job = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int cta = (int)(job >> 8), wr = (int)(job & 255), w = wr >> 7, r = wr & 127;
    if (cta >= p.batch * p.hk * p.n_ctiles) return;
    int b, h, ctile;
    sc_place<TREE>(p, cta, lane, b, h, ctile);
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T = p.q_start ? p.q_start[b + 1] - qs : 1;
    const int t = (ctile * 2 + w) * p.tpt + r / p.group;
    if (r >= p.tpt * p.group || t >= T) return;
    const float* src = p.part + ((int64_t)cta * p.n_split * 256 + wr) * (D + 2);
    constexpr int64_t STEP = 256 * (D + 2);
    float M = -INFINITY;
    for (int s = 0; s < p.n_split; ++s) M = fmaxf(M, src[s * STEP + D]);
    float L = 0.f, o[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
    for (int s = 0; s < p.n_split; ++s) {
        const float m = src[s * STEP + D], f = exp2f(m - ref_base(M));
        L = fmaf(src[s * STEP + D + 1], f, L);  // (of a part of NaN: NaN)
        if (m == -INFINITY) continue;           // a part that saw no key
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = fmaf(src[s * STEP + e * 32 + lane], f, o[e]);
    }
    const float inv = sum_inv(L);
    const int64_t row = ((int64_t)(qs + t) * p.hq + h * p.group + r % p.group) * D;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) store_as(p.out, p.out_dtype, row + e * 32 + lane, o[e] * inv);
}

template <int DH, typename E, bool TREE>
static int launch_scored_tc(const CUtensorMap& tk, const CUtensorMap& tv, const ScoredTcParams& p,
                            cudaStream_t st) {
    using C = ScCfg<DH>;
    const int64_t grid = (int64_t)p.n_ctiles * p.batch * p.hk;
    if (grid <= 0) return CX_OK;
    if (grid > INT32_MAX / 256)
        return fail(CX_ERR_UNSUPPORTED, "cx_paged_attend: grid too large");
    auto go = [&](auto kern) {
        CX_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           C::SMEM));
        kern<<<dim3((unsigned)grid, (unsigned)p.n_split), C::THREADS, C::SMEM, st>>>(tk, tv, p);
        return check_launch("scored_tc_kernel");
    };
    int rc = p.cap_log2 > 0.f ? (p.slopes ? go(scored_tc_kernel<DH, E, true, true, TREE>)
                                          : go(scored_tc_kernel<DH, E, true, false, TREE>))
                              : (p.slopes ? go(scored_tc_kernel<DH, E, false, true, TREE>)
                                          : go(scored_tc_kernel<DH, E, false, false, TREE>));
    if (rc != CX_OK || p.n_split == 1) return rc;
    scored_tc_join_kernel<DH, TREE><<<(unsigned)(grid * 32), 256, 0, st>>>(p);
    return check_launch("scored_tc_join_kernel");
}

}  // namespace cx
