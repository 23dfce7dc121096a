// Paged multi-query attention with score modifiers on tcgen05: prompt chunks
// and chains of 64 packed query rows or more (row = query token x head of the
// GQA group), bf16 or fp16 pools of 16-token blocks, head_dim 64 or 128.
//
// One CTA owns (sequence b, KV head h), two query tiles w = 0, 1 of up to 128
// packed rows (whole tokens: tpt = 128 / G of them, so any group size works)
// and a run of 128-key tiles, nearest keys first, so that the running maximum
// is set early and O is rarely rescaled.  Three roles:
//
//   warps 8-10 : producers.  K and V tiles arrive as 16-token block boxes of 64
//                columns (TMA, 128-byte swizzle) in a 160 KB ring, in the order
//                the MMAs read them.  Blocks past the sequence and ids outside
//                the pool are loaded from a coordinate outside the tensor map,
//                which fills zeros: what another block holds cannot reach the
//                result.
//   warp 11    : one thread issues S_w(i) = Q_w K(i)^T into TMEM columns
//                [128 w, 128 w + 128) and O_w += P_w(i) V(i) into [256 + D w, ..)
//                with P_w read from TMEM, PV_w in two halves of 64 keys, so that
//                the first starts while the second half's exponentials run.
//   warps 0-7  : softmax of tile w = warp / 4, thread r owning row r.  The row's
//                128 scores are read from TMEM once and stay in registers
//                (setmaxnreg: 216 of them for these warps, 72 for the others).
//
// Scores: tanh(z) is z P(z^2), P of degree 4 fitted to tanh over |z| <= 0.8
// (least squares, reweighted to an even error; absolute error 4e-7 in fp32)
// while every z of a warp's tile is that small — with a cap of 30 that is
// |score| <= 24 — and 1 - 2 / (1 + 2^(2 z log2 e)) otherwise.  The polynomial
// runs as packed pairs on the FMA pipe (fma.rn.f32x2) and leaves the special
// function unit, which the exponentials fill, alone.  Tiles that some row sees
// only in part take a general path with per-key tests.
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
    const void* q;
    void* out;
    float* part;                 // n_split > 1: [CTA][split][256][D + 2]
    int64_t q_stride;
    int32_t batch, hk, hq, group, tpt, n_ctiles, n_blocks, layer, window, n_split;
    int32_t q_dtype, out_dtype;
    float scale_log2;            // |scale| * log2(e)
    float z_scale;               // |scale| / cap
    float cap_log2;              // cap * log2(e)
    int32_t neg;                 // scale < 0: Q is negated (tanh is odd)
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
    static constexpr int SMEM = OFF_BAR + 320 + 1024;   // + 1 KB alignment slack
    static constexpr int TMEM_COLS = 512;
    static constexpr int N_PROD = 3;
    static constexpr int THREADS = 384;
    static constexpr int PROD_WARP = 8, MMA_WARP = 11;
    // setmaxnreg split of the 384 x 168 registers the block is launched with
    static constexpr int REG_SOFTMAX = 216, REG_OTHER = 72;
    static_assert(REG_SOFTMAX * 256 + REG_OTHER * 128 <= THREADS * 168, "register split");
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

// cap * log2(e) * tanh(z) for any z.
__device__ __forceinline__ float cap_any(float z, float cap_log2) {
    return fmaf(-2.f * cap_log2, rcp_approx(1.f + ex2_sfu(z * 2.8853900817779268f)), cap_log2);
}

template <typename E>
__host__ __device__ constexpr uint32_t sc_idesc(int m, int n, int b_mn) {
    // operand types: 1 bf16, 0 fp16
    const uint32_t ty = std::is_same<E, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (ty << 7) | (ty << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
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

// The key tiles of a CTA: n_pre tiles from block 0 (the prefix left of the
// window), then tiles from block kb0 on.
struct ScTiles {
    int n_pre, kb0, n;           // n: all of them
    __device__ __forceinline__ int block(int t) const {
        constexpr int BPT = kScKeys / kBlockTok;
        return t < n_pre ? t * BPT : kb0 + (t - n_pre) * BPT;
    }
};

template <int DH, typename E, bool CAP, bool ALIBI>
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
    uint64_t* p_half = s_full + 2;         // [2] P_w of the first 64 keys written, O_w rescaled
    uint64_t* p_full = p_half + 2;         // [2] P_w of the other 64 keys written
    uint64_t* o_done = p_full + 2;         // [2] PV_w complete
    uint64_t* mma_drain = o_done + 2;      // last commit of the MMA thread
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(mma_drain + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile int* s_issued = s_abort + 1;  // ring items whose loads were issued

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta = (int)blockIdx.x;
    const int bh = cta / p.n_ctiles;
    const int ctile = p.n_ctiles - 1 - cta % p.n_ctiles;     // longest first
    const int b = bh / p.hk, h = bh % p.hk;
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
    const int t_end = min(T, t0 + nq * tpt);
    const int pos0 = ctx - T;                                // position of token 0
    const int win = p.window;
    const int pre = p.prefix ? min(max(p.prefix[b], 0), ctx) : 0;
    const int run_hi = min(pos0 + t_end - 1, ctx - 1);       // last key past the prefix
    const int run_lo = win > 0 ? max(0, pos0 + t0 - win + 1) : 0;
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
            mbar_init(&p_half[w], 128);
            mbar_init(&p_full[w], 128);
            mbar_init(&o_done[w], 1);
        }
        mbar_init(mma_drain, 1);
        *s_abort = 0;
        *s_issued = 0;
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

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFTMAX));
        const int w = warp >> 2, r = tid & 127;
        const int tw0 = t0 + w * tpt;                        // first token of this tile
        const int tw1 = min(t_end, tw0 + tpt);
        const int t = tw0 + r / G;
        const bool row_ok = t < tw1 && r < tpt * G;
        const int head = h * G + r % G;
        // ---- Q_w -> shared memory: 16-bit, K-major, swizzled, zero padding rows.
        // Only the MMA warp waits for it (named barrier 3).
        {
            unsigned char* qdst = sm + w * C::Q_BYTES;
            const int64_t row = (int64_t)(qs + t) * p.q_stride + (int64_t)head * D;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint4 w4 = make_uint4(0, 0, 0, 0);
                if (row_ok) {
                    if (p.q_dtype == CX_F32) {
                        const float4* s4 = reinterpret_cast<const float4*>(
                            static_cast<const float*>(p.q) + row + c * 8);
                        const float4 a = __ldg(s4), e = __ldg(s4 + 1);
                        w4 = make_uint4(Half16<E>::pack(a.x, a.y), Half16<E>::pack(a.z, a.w),
                                        Half16<E>::pack(e.x, e.y), Half16<E>::pack(e.z, e.w));
                    } else {
                        w4 = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(p.q) +
                                                                  row + c * 8));
                    }
                    if (p.neg) {
                        w4.x ^= 0x80008000u;
                        w4.y ^= 0x80008000u;
                        w4.z ^= 0x80008000u;
                        w4.w ^= 0x80008000u;
                    }
                }
                *reinterpret_cast<uint4*>(qdst + tc_swz(r, c * 8, kTcRows)) = w4;
            }
            fence_async_smem();
            named_bar_arrive(3, 256 + 32);
        }
        if (w < nq) {
            const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tm_s = tmem + w * kScKeys + lane_off;
            const uint32_t tm_o = tmem + 2 * kScKeys + w * D + lane_off;
            const int pos = pos0 + t;
            const int pos_lo = pos0 + tw0, pos_hi = pos0 + tw1 - 1;
            const float slope =
                ALIBI ? p.slopes[min(head, p.hq - 1)] * 1.4426950408889634f : 0.f;
            const float cl = p.cap_log2;
            const f2 zs2 = f2_of(p.z_scale, p.z_scale);
            const f2 k0 = f2_of(cl * kTanhC0, cl * kTanhC0), k1 = f2_of(cl * kTanhC1, cl * kTanhC1),
                     k2 = f2_of(cl * kTanhC2, cl * kTanhC2), k3 = f2_of(cl * kTanhC3, cl * kTanhC3),
                     k4 = f2_of(cl * kTanhC4, cl * kTanhC4);
            const f2 sl2 = f2_of(p.scale_log2, p.scale_log2);
            const int32_t* tab = p.tables + (int64_t)b * p.table_stride;
            bool any_bad = false;
            for (int blk = lane; blk < nblk_seq; blk += 32) {
                const int id = tab[blk];
                any_bad |= id < 0 || id >= p.n_blocks;
            }
            any_bad = __any_sync(0xffffffffu, any_bad);
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int i = 0; i < n_tiles; ++i) {
                if (!__all_sync(0xffffffffu,
                                mbar_wait_bounded(&s_full[w], i & 1, s_abort, kWaitLimitNs))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                float v[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc_ld32(tm_s + c * 32, &v[c * 32]);
                const int b0 = tiles.block(first - i), kbase = b0 * kBlockTok;
                unsigned bad8 = 0;
                if (any_bad) {
                    const int blk = b0 + lane;
                    const int id = lane < BPT && blk < nblk_seq ? tab[blk] : 0;
                    bad8 = __ballot_sync(0xffffffffu, id < 0 || id >= p.n_blocks);
                }
                bool general = bad8 != 0 ||
                               !(kbase + kScKeys <= pre ||
                                 (kbase + kScKeys - 1 <= pos_lo && (win <= 0 || kbase > pos_hi - win)));
                tc_wait_ld();
                float mt;                      // this tile's row maximum (base 2)
                if (!general) {
                    if constexpr (ALIBI) {
                        // bias slope * (kbase + j - pos), exact near the query
                        const float c0 = slope * (float)(kbase - pos);
                        const bool fwd = kbase + kScKeys - 1 > pos_lo;   // all of it prefix
                        if constexpr (CAP) {
                            float mx = -INFINITY, mn = INFINITY;
#pragma unroll
                            for (int j = 0; j < 128; j += 2) {
                                mx = max3(mx, v[j], v[j + 1]);
                                mn = min3(mn, v[j], v[j + 1]);
                            }
                            general = fwd || __any_sync(0xffffffffu,
                                                        fmaxf(mx, -mn) * p.z_scale > kTanhMax);
                        } else {
                            general = __any_sync(0xffffffffu, fwd);
                        }
                        if (!general) {
#pragma unroll
                            for (int j = 0; j < 128; j += 2) {
                                const f2 bias = f2_of(fmaf(slope, (float)j, c0),
                                                      fmaf(slope, (float)(j + 1), c0));
                                f2 x = f2_of(v[j], v[j + 1]);
                                if constexpr (CAP) {
                                    x = f2_mul(x, zs2);
                                    const f2 y = f2_mul(x, x);
                                    x = f2_fma(x, f2_fma(f2_fma(f2_fma(f2_fma(k4, y, k3), y, k2), y,
                                                               k1), y, k0), bias);
                                } else {
                                    x = f2_fma(x, sl2, bias);
                                }
                                f2_get(x, v[j], v[j + 1]);
                            }
                            float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 128; j += 4) {
                                a0 = max3(a0, v[j], v[j + 1]);
                                a1 = max3(a1, v[j + 2], v[j + 3]);
                            }
                            mt = fmaxf(a0, a1);
                        }
                    } else {
                        float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 128; j += 4) {
                            a0 = max3(a0, v[j], v[j + 1]);
                            a1 = max3(a1, v[j + 2], v[j + 3]);
                        }
                        const float mx = fmaxf(a0, a1);
                        if constexpr (CAP) {
                            float n0 = INFINITY, n1 = INFINITY;
#pragma unroll
                            for (int j = 0; j < 128; j += 4) {
                                n0 = min3(n0, v[j], v[j + 1]);
                                n1 = min3(n1, v[j + 2], v[j + 3]);
                            }
                            const float big = fmaxf(mx, -fminf(n0, n1)) * p.z_scale;
                            general = __any_sync(0xffffffffu, big > kTanhMax);
                            mt = cap_any(mx * p.z_scale, cl);
                        } else {
                            mt = mx * p.scale_log2;
                        }
                    }
                }
                if (general) {
                    // some row sees only part of the tile, or a score is beyond
                    // the polynomial: key by key
                    float a = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 128; ++j) {
                        const int key = kbase + j;
                        float x = CAP ? cap_any(v[j] * p.z_scale, cl) : v[j] * p.scale_log2;
                        if constexpr (ALIBI) x = fmaf(-slope, (float)abs(pos - key), x);
                        const bool keep = (key < pre || (key <= pos && (win <= 0 || key > pos - win))) &&
                                          !((bad8 >> (j >> 4)) & 1u);
                        v[j] = keep ? x : -INFINITY;
                        a = fmaxf(a, v[j]);
                    }
                    mt = a;
                }
                // lazy rescale: the reference maximum stays until a row's grows by
                // more than 2^8 (exact after the final division)
                const bool grow = mt > m + kTcRescaleLog2 || (m == -INFINITY && mt > -INFINITY);
                const float m_new = grow ? mt : m;
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = grow ? exp2f(m - m_use) : 1.f;
                m = m_new;
                // O_w holds PV_w(0 .. i-1): S_w(i) was issued after PV_w(i-1)
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        asm volatile(
                            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                            "%15}, [%16];"
                            : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]),
                              "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]), "=r"(o[9]),
                              "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]),
                              "=r"(o[15])
                            : "r"(tm_o + c * 16));
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        asm volatile(
                            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                            "%16};" ::"r"(tm_o + c * 16),
                            "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]),
                            "r"(o[6]), "r"(o[7]), "r"(o[8]), "r"(o[9]), "r"(o[10]), "r"(o[11]),
                            "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15])
                            : "memory");
                    }
                    tc_wait_st();
                }
                // zero the V rows that no row of the CTA sees
                if (w == 0) {
                    auto dead = [&](int key) {
                        return key >= ctx || (key >= pre && (key > run_hi || key < run_lo));
                    };
                    const bool any_dead = kbase + kScKeys > ctx ||
                                          (kbase + kScKeys > pre &&
                                           (kbase + kScKeys - 1 > run_hi || kbase < run_lo));
                    if (any_dead) {
                        const int q = sc_pos_v(i, n_tiles);
                        if (!__all_sync(0xffffffffu,
                                        mbar_wait_bounded(&full[q % SLOTS], (q / SLOTS) & 1,
                                                          s_abort, kWaitLimitNs))) {
                            ok = false;
                            break;
                        }
                        if (dead(kbase + r)) {
                            uint4* z = reinterpret_cast<uint4*>(ring + (q % SLOTS) * C::SLOT +
                                                                r * 128);
#pragma unroll
                            for (int hf = 0; hf < C::HALVES; ++hf)
#pragma unroll
                                for (int c = 0; c < 8; ++c)
                                    z[hf * (C::KV_HALF / 16) + c] = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_smem();
                    }
                }
                // p = 2^(x - m), 16-bit pairs over S_w's first 64 columns (keys 2c,
                // 2c + 1 in column c), 64 keys at a time
                f2 sum0 = 0, sum1 = 0;         // two fp32 zeros each
                const f2 negm = f2_of(-m_use, -m_use);
                auto emit = [&](auto done_tag) {
                constexpr bool DONE = decltype(done_tag)::value;   // v holds x already
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float pk[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        const int j = hf * 64 + 2 * c;
                        f2 x = f2_of(v[j], v[j + 1]);
                        if constexpr (DONE) {
                            x = f2_add(x, negm);
                        } else if constexpr (CAP) {
                            x = f2_mul(x, zs2);
                            const f2 y = f2_mul(x, x);
                            x = f2_fma(x, f2_fma(f2_fma(f2_fma(f2_fma(k4, y, k3), y, k2), y, k1),
                                                 y, k0), negm);
                        } else {
                            x = f2_fma(x, sl2, negm);
                        }
                        float e0, e1;
                        f2_get(x, e0, e1);
                        e0 = ex2_sfu(e0);
                        e1 = ex2_sfu(e1);
                        if (c & 1)
                            sum1 = f2_add(sum1, f2_of(e0, e1));
                        else
                            sum0 = f2_add(sum0, f2_of(e0, e1));
                        pk[c] = __uint_as_float(Half16<E>::pack(e0, e1));
                    }
                    tc_st32(tm_s + hf * 32, pk);
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive(hf ? &p_full[w] : &p_half[w]);
                }
                };
                if (ALIBI || general)
                    emit(std::true_type{});
                else
                    emit(std::bool_constant<ALIBI>{});
                float s0, s1, s2, s3;
                f2_get(sum0, s0, s1);
                f2_get(sum1, s2, s3);
                l = l * alpha + ((s0 + s1) + (s2 + s3));
            }
            // ---- epilogue: rows to the output, or to this split's part ----
            if (n_tiles > 0 && ok) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[w], (n_tiles - 1) & 1,
                                                                s_abort, kWaitLimitNs));
                if (ok) tc_fence_after();
            }
            float* part = nullptr;
            if (p.n_split > 1) {
                part = p.part + (((int64_t)cta * p.n_split + blockIdx.y) * 256 + w * 128 + r) *
                                    (D + 2);
                part[D] = ok ? m : -INFINITY;
                part[D + 1] = l;
            }
            if (ok) {
                const float inv = part ? 1.f : l > 0.f ? 1.f / l : 0.f;
                const int64_t o_row = ((int64_t)(qs + t) * p.hq + head) * D;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    float ov[32];
                    if (n_tiles > 0) {
                        tc_ld32(tm_o + c * 32, ov);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = 0.f;
                    }
                    if (!row_ok) continue;
                    if (part) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            *reinterpret_cast<float2*>(part + c * 32 + e) =
                                make_float2(ov[e], ov[e + 1]);
                    } else if (p.out_dtype == CX_F32) {
                        float* dst = static_cast<float*>(p.out) + o_row + c * 32;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(dst + e) = make_float4(
                                ov[e] * inv, ov[e + 1] * inv, ov[e + 2] * inv, ov[e + 3] * inv);
                    } else {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                                                              o_row + c * 32);
                        const bool bf = p.out_dtype == CX_BF16;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t u[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float x = ov[e + 2 * k] * inv, y = ov[e + 2 * k + 1] * inv;
                                u[k] = bf ? Half16<__nv_bfloat16>::pack(x, y)
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
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_OTHER));
        if (warp < C::MMA_WARP) {
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
                    !mbar_wait_bounded(&empty[s], (use - 1) & 1, s_abort, kWaitLimitNs))
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
            named_bar_sync(3, 256 + 32);               // Q_0, Q_1 are in shared memory
            if (lane == 0) {
                constexpr uint32_t idesc_s = sc_idesc<E>(kTcRows, kScKeys, 0);
                constexpr uint32_t idesc_o = sc_idesc<E>(kTcRows, D, 1);
                const uint32_t q_base = smem_addr(sm), r_base = smem_addr(ring);
                bool ok = true;
                auto wait = [&](uint64_t* bar, int parity) {
                    const bool r = mbar_wait_bounded(bar, parity & 1, s_abort, kWaitLimitNs);
                    if (r) tc_fence_after();
                    return r;
                };
                auto issue_s = [&](int w, int slot) {
                    const uint32_t kb = r_base + slot * C::SLOT, qw = q_base + w * C::Q_BYTES;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        tc_mma(tmem + w * kScKeys,
                               tc_sdesc(qw + (kk >> 2) * C::Q_HALF + (kk & 3) * 32, 16, 1024),
                               tc_sdesc(kb + (kk >> 2) * C::KV_HALF + (kk & 3) * 32, 16, 1024),
                               idesc_s, kk > 0);
                    tc_commit(&s_full[w]);
                };
                // half hf of O_w += P_w V: 64 keys in steps of 16
                auto issue_pv = [&](int w, int slot, int hf, bool acc) {
                    const uint32_t vb = r_base + slot * C::SLOT;
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const int kk = hf * 4 + k4;
                        sc_mma_ts(tmem + 2 * kScKeys + w * D, tmem + w * kScKeys + kk * 8,
                                  tc_sdesc(vb + kk * 2048, C::KV_HALF, 1024), idesc_o,
                                  (acc || kk > 0) ? 1u : 0u);
                    }
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
                        if (!(ok = wait(&p_half[w], i))) break;
                        issue_pv(w, vp % SLOTS, 0, i > 0);
                        if (!(ok = wait(&p_full[w], i))) break;
                        issue_pv(w, vp % SLOTS, 1, true);
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
        const int issued = *s_issued;
        for (int s = 0; s < SLOTS; ++s) {
            const int uses = issued > s ? (issued - 1 - s) / SLOTS + 1 : 0;
            if (uses > 0) mbar_wait_bounded(&full[s], (uses - 1) & 1, nullptr, kWaitLimitNs);
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
template <int D>
__global__ void __launch_bounds__(256) scored_tc_join_kernel(const ScoredTcParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t job = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int cta = (int)(job >> 8), wr = (int)(job & 255), w = wr >> 7, r = wr & 127;
    const int bh = cta / p.n_ctiles, ctile = p.n_ctiles - 1 - cta % p.n_ctiles;
    const int b = bh / p.hk, h = bh % p.hk;
    if (b >= p.batch) return;
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
        const float m = src[s * STEP + D];
        if (m == -INFINITY) continue;          // a part that saw no key
        const float f = exp2f(m - M);
        L = fmaf(src[s * STEP + D + 1], f, L);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = fmaf(src[s * STEP + e * 32 + lane], f, o[e]);
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const int64_t row = ((int64_t)(qs + t) * p.hq + h * p.group + r % p.group) * D;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) store_as(p.out, p.out_dtype, row + e * 32 + lane, o[e] * inv);
}

template <int DH, typename E>
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
    int rc = p.cap_log2 > 0.f ? (p.slopes ? go(scored_tc_kernel<DH, E, true, true>)
                                          : go(scored_tc_kernel<DH, E, true, false>))
                              : (p.slopes ? go(scored_tc_kernel<DH, E, false, true>)
                                          : go(scored_tc_kernel<DH, E, false, false>));
    if (rc != CX_OK || p.n_split == 1) return rc;
    scored_tc_join_kernel<DH><<<(unsigned)(grid * 32), 256, 0, st>>>(p);
    return check_launch("scored_tc_join_kernel");
}

}  // namespace cx
