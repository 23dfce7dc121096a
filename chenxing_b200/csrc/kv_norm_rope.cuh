// RMS norm of query and key heads, rotation of their leading dims and the
// slot-mapped append, in one pass over the step's rows:
//     y = x * rsqrt(mean(x^2) + eps) * w          (per head, fp32)
//     (y_a, y_b) -> (y_a c - y_b s, y_b c' + y_a s')   for the pairs of y[0, rot)
// K rows go to their pool slots, V rows are copied, Q rows go to q_out; each
// value is rounded once, to its destination's type.
#pragma once

#include <algorithm>

#include "cx_common.cuh"  // unity build: included from cxkv.cu after kv_ops.cuh

namespace cx {

struct NormRopeParams {
    PoolGeom g;
    int64_t layer;
    cx_qkv rows;
    cx_norm_rope how;
    const int64_t* slots;
    const int64_t* positions;
    void* kp;
    void* vp;
    void* q_out;
    int32_t pool_dtype, q_out_dtype;
    uint64_t wait_ns;          // limit of the staged form's waits (cx_set_wait_limit_ns)
};

template <typename S>
__device__ __forceinline__ float norm_weight(const void* w, bool f32, int d) {
    return f32 ? static_cast<const float*>(w)[d] : Conv<S>::to_f(static_cast<const S*>(w)[d]);
}

// One warp per row of a token ([Q heads | K heads | V heads]): the sum of
// squares in a first sweep, then pairs and the unrotated rest, re-read from L1.
template <typename S>
__global__ void __launch_bounds__(256) kv_append_norm_rope_kernel(const NormRopeParams p) {
    const int lane = threadIdx.x & 31;
    const int H = (int)p.g.n_kv_heads, D = (int)p.g.head_dim, hq = (int)p.rows.n_q_heads;
    const int rot = (int)p.how.rot_dim, half = rot / 2;
    const int64_t per_tok = hq + 2 * H, jobs = p.rows.n_tokens * per_tok;
    const int64_t cap = p.g.n_blocks * p.g.block_size;
    for (int64_t job = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); job < jobs;
         job += (int64_t)gridDim.x * (blockDim.x >> 5)) {
        const int64_t t = job / per_tok;
        const int row = (int)(job - t * per_tok);
        const int64_t pos = p.positions[t];
        if (pos < 0 || pos >= p.how.table_rows) {
            if (lane == 0) raise_flag(CX_DEV_BAD_POSITION);
            continue;
        }
        const bool is_q = row < hq, is_v = row >= hq + H;
        const int h = is_q ? row : is_v ? row - hq - H : row - hq;
        int64_t dst;
        if (is_q) {
            dst = (t * hq + h) * D;
        } else {
            const int64_t slot = p.slots[t];
            if (slot < 0) continue;                       // stored nowhere
            if (slot >= cap) {
                if (lane == 0) raise_flag(CX_DEV_BAD_SLOT);
                continue;
            }
            dst = p.g.tile(p.layer, slot / p.g.block_size, h) + (slot % p.g.block_size) * D;
        }
        const S* x = is_q ? static_cast<const S*>(p.rows.q) + t * p.rows.q_token_stride +
                                h * p.rows.q_head_stride
                   : is_v ? static_cast<const S*>(p.rows.v) + t * p.rows.v_token_stride +
                                h * p.rows.v_head_stride
                          : static_cast<const S*>(p.rows.k) + t * p.rows.k_token_stride +
                                h * p.rows.k_head_stride;
        auto put = [&](int d, float y) {
            store_as(is_q ? p.q_out : is_v ? p.vp : p.kp, is_q ? p.q_out_dtype : p.pool_dtype,
                     dst + d, y);
        };
        if (is_v) {
            for (int d = lane; d < D; d += 32) put(d, Conv<S>::to_f(x[d]));
            continue;
        }
        const void* w = is_q ? p.how.q_weight : p.how.k_weight;
        const bool wf32 = (is_q ? p.how.q_weight_dtype : p.how.k_weight_dtype) == CX_F32;
        float inv = 1.f;
        if (w) {
            float ss = 0.f;
            for (int d = lane; d < D; d += 32) {
                const float v = Conv<S>::to_f(x[d]);
                ss = fmaf(v, v, ss);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(ss / (float)D + p.how.eps);
        }
        auto get = [&](int d) {
            const float v = Conv<S>::to_f(x[d]);
            return w ? v * inv * norm_weight<S>(w, wf32, d) : v;
        };
        const float* c = p.how.cos_table + pos * rot;
        const float* s = p.how.sin_table + pos * rot;
        for (int j = lane; j < half; j += 32) {
            const bool inter = p.how.interleaved != 0;
            const int ia = inter ? 2 * j : j, ib = inter ? 2 * j + 1 : j + half;
            const int jb = inter ? j : j + half;
            const float a = get(ia), b = get(ib);
            put(ia, a * c[j] - b * s[j]);
            put(ib, b * c[jb] + a * s[jb]);
        }
        for (int d = rot + lane; d < D; d += 32) put(d, get(d));
    }
}

// N elements of T as one access of N * sizeof(T) bytes (two of 16 for 32).
template <typename T, int N>
struct Chunk {
    static constexpr int BYTES = N * (int)sizeof(T);
    using W = typename std::conditional<
        BYTES >= 16, uint4, typename std::conditional<BYTES == 8, uint2, uint32_t>::type>::type;
    static constexpr int NW = BYTES / (int)sizeof(W);
    W w[NW];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = __ldg(reinterpret_cast<const W*>(p) + i);
    }
    __device__ __forceinline__ void load_shared(const T* p) {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = reinterpret_cast<const W*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < NW; ++i) reinterpret_cast<W*>(p)[i] = w[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) reinterpret_cast<uint32_t*>(w)[i] = 0u;
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Conv<T>::to_f(e[i]);
    }
    __device__ __forceinline__ void set(const float (&x)[N]) {
        if constexpr (sizeof(T) == 2) {
            uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) u[i] = Half16<T>::pack(x[2 * i], x[2 * i + 1]);
        } else {
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (int i = 0; i < N; ++i) e[i] = x[i];
        }
    }
};

// One row in registers: norm, rotation, store.  `xa`, `xb`: the lane's two chunks
// of V elements at ea and eb (neighbours of a V row: 2 V li and 2 V li + V);
// ca .. sb: cos / sin of the lane's pairs (half-split: of both halves).  Every
// lane of the warp must call it (shuffles over the L lanes of a row); only
// `store` lanes write.
template <typename S, typename O, int V>
__device__ __forceinline__ void norm_rope_row(const NormRopeParams& p, float (&xa)[V],
                                              float (&xb)[V], const float (&ca)[V],
                                              const float (&sa)[V], const float (&cb)[V],
                                              const float (&sb)[V], int L, int li, int ea, int eb,
                                              bool turn, bool is_q, bool is_v, bool store,
                                              O* dst) {
    // rows of a warp's groups may differ in kind: all reduce, some use it
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
    for (int o = L >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!store) return;
    Chunk<O, V> c;
    if (is_v) {
        c.set(xa);
        c.store(dst + li * 2 * V);
        c.set(xb);
        c.store(dst + li * 2 * V + V);
        return;
    }
    const void* w = is_q ? p.how.q_weight : p.how.k_weight;
    if (w) {
        const float inv = rsqrtf(ss / (float)(int)p.g.head_dim + p.how.eps);
        float wa[V], wb[V];
        if ((is_q ? p.how.q_weight_dtype : p.how.k_weight_dtype) == CX_F32) {
            Chunk<float, V> k;
            k.load(static_cast<const float*>(w) + ea);
            k.get(wa);
            k.load(static_cast<const float*>(w) + eb);
            k.get(wb);
        } else {
            Chunk<S, V> k;
            k.load(static_cast<const S*>(w) + ea);
            k.get(wa);
            k.load(static_cast<const S*>(w) + eb);
            k.get(wb);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            xa[i] = xa[i] * inv * wa[i];
            xb[i] = xb[i] * inv * wb[i];
        }
    }
    if (turn && p.how.interleaved) {
        // pairs (2 i, 2 i + 1) of the 2 V neighbours
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float& x0 = 2 * i < V ? xa[2 * i] : xb[2 * i - V];
            float& x1 = 2 * i < V ? xa[2 * i + 1] : xb[2 * i + 1 - V];
            const float y0 = x0 * ca[i] - x1 * sa[i];
            x1 = x1 * ca[i] + x0 * sa[i];
            x0 = y0;
        }
    } else if (turn) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float y0 = xa[i] * ca[i] - xb[i] * sa[i];
            xb[i] = xb[i] * cb[i] + xa[i] * sb[i];
            xa[i] = y0;
        }
    }
    c.set(xa);
    c.store(dst + ea);
    c.set(xb);
    c.store(dst + eb);
}

// Address of row `row` ([Q heads | K heads | V heads]) of token t.
template <typename S>
__device__ __forceinline__ const S* norm_rope_src(const NormRopeParams& p, int64_t t, int row,
                                                  int hq, int H) {
    if (row < hq)
        return static_cast<const S*>(p.rows.q) + t * p.rows.q_token_stride +
               row * p.rows.q_head_stride;
    if (row < hq + H)
        return static_cast<const S*>(p.rows.k) + t * p.rows.k_token_stride +
               (row - hq) * p.rows.k_head_stride;
    return static_cast<const S*>(p.rows.v) + t * p.rows.v_token_stride +
           (row - hq - H) * p.rows.v_head_stride;
}

// What a token's position and slot allow, flags raised by `report`.
struct TokenFate {
    bool q_ok, kv_ok;
    int64_t kv_dst;     // pool element of the token's row of head 0
};
__device__ __forceinline__ TokenFate token_fate(const NormRopeParams& p, int64_t pos, int64_t slot,
                                                bool live, bool report) {
    TokenFate f;
    const bool pos_ok = pos >= 0 && pos < p.how.table_rows;
    const bool slot_bad = slot >= p.g.n_blocks * p.g.block_size;
    if (live && report) {
        if (!pos_ok)
            raise_flag(CX_DEV_BAD_POSITION);
        else if (slot_bad)
            raise_flag(CX_DEV_BAD_SLOT);
    }
    f.q_ok = live && pos_ok;
    f.kv_ok = f.q_ok && slot >= 0 && !slot_bad;
    const uint32_t bs = (uint32_t)p.g.block_size;
    const uint32_t blk = f.kv_ok ? (uint32_t)slot / bs : 0u;
    f.kv_dst = p.g.tile(p.layer, blk, 0) +
               (int64_t)((uint32_t)(f.kv_ok ? slot : 0) - blk * bs) * p.g.head_dim;
    return f;
}

// Vector form for few tokens.  A row is read once, by `L` lanes (a power of
// two, at most a warp) that hold two chunks of V elements each: both halves of V
// pairs in the rotated part (half-split), 2 V neighbours elsewhere and for
// interleaved pairs.  One row per group of L lanes; the row's loads are issued
// before the position and the slot are known (a skipped token's rows are still
// valid memory).  The host guarantees: head_dim and rot_dim multiples of 2 V,
// accesses aligned, n_tokens * rows * L < 2^31, n_blocks * block_size < 2^31.
template <typename S, typename O, int V>
__global__ void __launch_bounds__(256)
    kv_append_norm_rope_vec_kernel(const NormRopeParams p, int L) {
    const int H = (int)p.g.n_kv_heads, D = (int)p.g.head_dim, hq = (int)p.rows.n_q_heads;
    const int rot = (int)p.how.rot_dim, R = hq + 2 * H;
    const uint32_t gid = (blockIdx.x * 256u + threadIdx.x) / (uint32_t)L;
    const int li = (int)(threadIdx.x & (unsigned)(L - 1));
    const int64_t t = gid / (uint32_t)R;
    const int row = (int)(gid - (uint32_t)t * (uint32_t)R);
    const bool inter = p.how.interleaved != 0;
    const bool live = t < p.rows.n_tokens && li * 2 * V < D;
    const bool turn = li < rot / (2 * V);             // lanes of the rotated part
    const int ea = !inter && turn ? li * V : li * 2 * V;
    const int eb = !inter && turn ? li * V + rot / 2 : ea + V;
    const bool is_q = row < hq, is_v = row >= hq + H;
    const int h = is_q ? row : is_v ? row - hq - H : row - hq;
    int64_t pos = -1, slot = -1;
    float xa[V], xb[V], ca[V], sa[V], cb[V], sb[V];
    Chunk<S, V> a, b;
    a.zero();
    b.zero();
    if (live) {
        pos = p.positions[t];
        slot = p.slots[t];
        const S* x = norm_rope_src<S>(p, t, row, hq, H);
        a.load(x + (is_v ? li * 2 * V : ea));         // V rows: plain neighbours
        b.load(x + (is_v ? li * 2 * V + V : eb));
    }
    const TokenFate f = token_fate(p, pos, slot, live, row == 0 && li == 0);
    if (f.q_ok && turn && !is_v) {
        const int64_t at = pos * rot + li * V;
        Chunk<float, V> c;
        c.load(p.how.cos_table + at);
        c.get(ca);
        c.load(p.how.sin_table + at);
        c.get(sa);
        if (!inter) {
            c.load(p.how.cos_table + at + rot / 2);
            c.get(cb);
            c.load(p.how.sin_table + at + rot / 2);
            c.get(sb);
        }
    }
    a.get(xa);
    b.get(xb);
    O* dst = is_q ? static_cast<O*>(p.q_out) + (t * hq + h) * D
                  : static_cast<O*>(is_v ? p.vp : p.kp) + f.kv_dst +
                        (int64_t)h * p.g.block_size * D;
    norm_rope_row<S, O, V>(p, xa, xb, ca, sa, cb, sb, L, li, ea, eb, turn, is_q, is_v,
                           is_q ? f.q_ok : f.kv_ok, dst);
}

// Untiled bulk copy into this CTA's shared memory, completing on `bar`; both
// addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

// V fp32 values of shared memory as pairs.
template <int V>
__device__ __forceinline__ void load_pairs(f2 (&x)[V / 2], const float* p) {
#pragma unroll
    for (int i = 0; i < V / 2; i += 2) {
        if constexpr (V >= 4) {
            const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p + 2 * i);
            x[i] = u.x;
            x[i + 1] = u.y;
        } else {
            x[i] = *reinterpret_cast<const f2*>(p + 2 * i);
        }
    }
}

// A chunk of V elements as fp32 pairs, and back with one rounding.
template <typename T, int V>
__device__ __forceinline__ void chunk_pairs(const Chunk<T, V>& c, f2 (&x)[V / 2]) {
    if constexpr (sizeof(T) == 4) {
        const float* e = reinterpret_cast<const float*>(c.w);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) x[i] = f2_of(e[2 * i], e[2 * i + 1]);
    } else {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(c.w);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) x[i] = Half16<T>::unpack(u[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void pairs_chunk(const f2 (&x)[V / 2], Chunk<T, V>& c) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        float lo, hi;
        f2_get(x[i], lo, hi);
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float*>(c.w)[2 * i] = lo;
            reinterpret_cast<float*>(c.w)[2 * i + 1] = hi;
        } else {
            reinterpret_cast<uint32_t*>(c.w)[i] = Half16<T>::pack(lo, hi);
        }
    }
}

// Vector form for many tokens: a CTA walks tokens blockIdx.x, + gridDim.x, ...
// Its last warp copies each token's rows and cos / sin values into one of
// kTokStages shared-memory stages (five bulk copies) ahead of the other warps,
// and leaves there what the token's position and slot allow.  Each group of L
// lanes takes about three rows of the token, with its cos / sin pairs in
// registers and the arithmetic on packed pairs; chunks of four elements, so that
// fp32 loads from shared memory are contiguous across lanes.
// 8192 tokens of 48 rows of 128 bf16 (210 MB, 32 us at the HBM copy rate) take
// 45 us.  Issue slots are 69 % taken, DRAM 42 % busy; warps wait in about equal
// parts for fixed latencies, shared memory and their turn to issue.  The same
// arithmetic on scalars took 48 where this took 46; what was tried before, at the
// same time: the register form, 68 us (a thread
// waits for the position, then for cos / sin, with 32 bytes of its row in
// flight) and 121 us with four rows a thread (one block an SM); per-thread
// copies and one CTA barrier a token, 76 us; chunks of eight, where cos / sin and
// weights are read again for every row with two-way bank conflicts (84 % of the
// shared-memory wavefronts), 47 us; six rows a group, too few warps, 82 us.
// The host guarantees what the other form needs, the heads of a token
// contiguous, rows and table rows multiples of 16 bytes at 16-byte addresses,
// and room for the stages.
constexpr int kTokStages = 3;
constexpr int kTokRows = 3;        // rows a group takes, about
constexpr int kTokThreads = 288;   // at most: 8 warps and the producer
constexpr uint64_t kDrainLimitNs = 2000000000ull;   // of the producer's last wait

struct TokStage {          // beside the rows of a stage
    int64_t kv_dst;        // pool element of the token's row of head 0
    int32_t q_ok, kv_ok;
};

template <typename S, typename O, int V>
__global__ void __launch_bounds__(kTokThreads, 3)
    kv_append_norm_rope_tok_kernel(const NormRopeParams p, int L, int n_groups, int stage_bytes) {
    extern __shared__ __align__(16) unsigned char tok_sm[];
    __shared__ uint64_t full[kTokStages], empty[kTokStages];
    __shared__ TokStage info[kTokStages];
    __shared__ int s_abort;
    const int H = (int)p.g.n_kv_heads, D = (int)p.g.head_dim, hq = (int)p.rows.n_q_heads;
    const int rot = (int)p.how.rot_dim, R = hq + 2 * H;
    const int tid = threadIdx.x, lane = tid & 31, n_warps = (int)(blockDim.x >> 5) - 1;
    const int64_t T = p.rows.n_tokens, step = gridDim.x;
    float* s_w = reinterpret_cast<float*>(tok_sm + kTokStages * stage_bytes);   // [2][D]
    if (tid == 0) {
        for (int s = 0; s < kTokStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], n_warps);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    for (int d = tid; d < 2 * D; d += blockDim.x) {
        const void* w = d < D ? p.how.q_weight : p.how.k_weight;
        const bool f32 = (d < D ? p.how.q_weight_dtype : p.how.k_weight_dtype) == CX_F32;
        s_w[d] = w ? norm_weight<S>(w, f32, d < D ? d : d - D) : 1.f;
    }
    __syncthreads();
    volatile int* abort = &s_abort;

    if (tid >= n_warps * 32) {
        // ---- producer: lane 0; the position and slot of the next token are loaded
        // while this one's copies are issued ----
        if (lane != 0) return;
        const uint32_t qb = (uint32_t)(hq * D * (int)sizeof(S)),
                       kb = (uint32_t)(H * D * (int)sizeof(S)), cb = (uint32_t)rot * 4u;
        int64_t pos = p.positions[blockIdx.x], slot = p.slots[blockIdx.x];
        int s = 0, phase = 1, issued = 0;             // phase 1: the first round waits for nothing
        for (int64_t t = blockIdx.x; t < T; t += step) {
            const int64_t pos_t = pos, slot_t = slot;
            if (t + step < T) {
                pos = p.positions[t + step];
                slot = p.slots[t + step];
            }
            if (!mbar_wait_bounded<1>(&empty[s], phase, abort, p.wait_ns)) {
                *abort = 1;
                raise_flag(CX_DEV_WAIT_TIMEOUT);
                break;
            }
            const TokenFate f = token_fate(p, pos_t, slot_t, true, true);
            info[s].kv_dst = f.kv_dst;
            info[s].q_ok = f.q_ok;
            info[s].kv_ok = f.kv_ok;
            uint32_t dst = smem_addr(tok_sm) + s * stage_bytes;
            mbar_arrive_expect_tx(&full[s], qb + 2 * kb + (f.q_ok ? 2 * cb : 0u));
            if (qb)
                bulk_load(dst, static_cast<const S*>(p.rows.q) + t * p.rows.q_token_stride, qb,
                          &full[s]);
            bulk_load(dst + qb, static_cast<const S*>(p.rows.k) + t * p.rows.k_token_stride, kb,
                      &full[s]);
            bulk_load(dst + qb + kb, static_cast<const S*>(p.rows.v) + t * p.rows.v_token_stride,
                      kb, &full[s]);
            dst += qb + 2 * kb;
            if (f.q_ok) {
                bulk_load(dst, p.how.cos_table + pos_t * rot, cb, &full[s]);
                bulk_load(dst + cb, p.how.sin_table + pos_t * rot, cb, &full[s]);
            }
            ++issued;
            if (++s == kTokStages) {
                s = 0;
                phase ^= 1;
            }
        }
        // the CTA's shared memory stays until its copies have landed
        for (int i = issued > kTokStages ? issued - kTokStages : 0; i < issued; ++i)
            mbar_wait_bounded<1>(&full[i % kTokStages], (i / kTokStages) & 1, nullptr,
                              kDrainLimitNs);
        return;
    }

    // ---- the other warps: rows ----
    const int grp = tid / L, li = tid & (L - 1);
    const bool inter = p.how.interleaved != 0;
    const bool turn = li < rot / (2 * V);
    // (lanes past the row read its start and store nothing)
    const int ea = li * 2 * V >= D ? 0 : !inter && turn ? li * V : li * 2 * V;
    const int eb = !inter && turn ? ea + rot / 2 : ea + V;
    const bool lane_ok = grp < n_groups && li * 2 * V < D;
    const float inv_d = 1.f / (float)D;
    const float* wq = p.how.q_weight ? s_w : nullptr;
    const float* wk = p.how.k_weight ? s_w + D : nullptr;
    const int64_t head_step = p.g.block_size * D;
    int s = 0, phase = 0;
    for (int64_t t = blockIdx.x; t < T; t += step) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded<1>(&full[s], phase, abort, p.wait_ns))) {
            if (lane == 0 && !*abort) {
                *abort = 1;
                raise_flag(CX_DEV_WAIT_TIMEOUT);
            }
            break;
        }
        const bool q_ok = info[s].q_ok != 0, kv_ok = info[s].kv_ok != 0;
        O* q_dst = static_cast<O*>(p.q_out) + t * hq * D;
        O* k_dst = static_cast<O*>(p.kp) + info[s].kv_dst;
        O* v_dst = static_cast<O*>(p.vp) + info[s].kv_dst;
        const S* rows = reinterpret_cast<const S*>(tok_sm + s * stage_bytes);
        const float* cs = reinterpret_cast<const float*>(rows + R * D);
        f2 c[V / 2], n[V / 2], c2[V / 2], n2[V / 2];
        if (turn && !inter) {
            load_pairs<V>(c, cs + li * V);
            load_pairs<V>(n, cs + rot + li * V);
            load_pairs<V>(c2, cs + rot / 2 + li * V);
            load_pairs<V>(n2, cs + rot + rot / 2 + li * V);
        }
        // one query or key row: `live` lanes hold it, `ok` says whether it is stored
        auto turned_row = [&](const S* src, const float* w, bool live, bool ok, O* dst) {
            Chunk<S, V> a, b;
            a.zero();
            b.zero();
            if (live) {
                a.load_shared(src + ea);
                b.load_shared(src + eb);
            }
            f2 pa[V / 2], pb[V / 2];
            chunk_pairs<S, V>(a, pa);
            chunk_pairs<S, V>(b, pb);
            if (w) {
                f2 s0 = 0, s1 = 0;
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    s0 = f2_fma(pa[i], pa[i], s0);
                    s1 = f2_fma(pb[i], pb[i], s1);
                }
                float lo, hi;
                f2_get(f2_add(s0, s1), lo, hi);
                float ss = lo + hi;
                for (int o = L >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float inv = rsqrtf(fmaf(ss, inv_d, p.how.eps));
                const f2 inv2 = f2_of(inv, inv);
                f2 wa[V / 2], wb[V / 2];
                load_pairs<V>(wa, w + ea);
                load_pairs<V>(wb, w + eb);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    pa[i] = f2_mul(f2_mul(pa[i], inv2), wa[i]);
                    pb[i] = f2_mul(f2_mul(pb[i], inv2), wb[i]);
                }
            }
            if (turn && !inter) {
                const f2 minus = f2_of(-1.f, -1.f);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const f2 ra = f2_fma(pa[i], c[i], f2_mul(f2_mul(pb[i], minus), n[i]));
                    pb[i] = f2_fma(pb[i], c2[i], f2_mul(pa[i], n2[i]));
                    pa[i] = ra;
                }
            } else if (turn) {
                // pairs (2 i, 2 i + 1) of the 2 V neighbours
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float cc = cs[li * V + i], nn = cs[rot + li * V + i];
                    f2& x = i < V / 2 ? pa[i] : pb[i - V / 2];
                    float x0, x1;
                    f2_get(x, x0, x1);
                    x = f2_of(x0 * cc - x1 * nn, x1 * cc + x0 * nn);
                }
            }
            if (live && ok) {
                Chunk<O, V> ya, yb;
                pairs_chunk<O, V>(pa, ya);
                pairs_chunk<O, V>(pb, yb);
                ya.store(dst + ea);
                yb.store(dst + eb);
            }
        };
        // the same number of rounds for every group: the shuffles need whole warps
        for (int r0 = 0; r0 < hq; r0 += n_groups)
            turned_row(rows + (r0 + grp) * D, wq, lane_ok && r0 + grp < hq, q_ok,
                       q_dst + (r0 + grp) * D);
        for (int r0 = 0; r0 < H; r0 += n_groups)
            turned_row(rows + (hq + r0 + grp) * D, wk, lane_ok && r0 + grp < H, kv_ok,
                       k_dst + (r0 + grp) * head_step);
        for (int h = grp; h < H && lane_ok && kv_ok; h += n_groups) {
            Chunk<S, 2 * V> x;
            x.load_shared(rows + (hq + H + h) * D + li * 2 * V);
            O* dst = v_dst + h * head_step + li * 2 * V;
            if constexpr (std::is_same<S, O>::value) {
                x.store(dst);
            } else {
                f2 px[V];
                chunk_pairs<S, 2 * V>(x, px);
                Chunk<O, 2 * V> y;
                pairs_chunk<O, 2 * V>(px, y);
                y.store(dst);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == kTokStages) {
            s = 0;
            phase ^= 1;
        }
    }
}

// Whether the heads of a token are not contiguous, or a bulk copy of a token's
// rows or of a table row would be unaligned.
static bool not_bulk(const NormRopeParams& p, int size) {
    const uintptr_t a =
        reinterpret_cast<uintptr_t>(p.rows.q) | reinterpret_cast<uintptr_t>(p.rows.k) |
        reinterpret_cast<uintptr_t>(p.rows.v) | reinterpret_cast<uintptr_t>(p.how.cos_table) |
        reinterpret_cast<uintptr_t>(p.how.sin_table);
    const int64_t st = (p.rows.q_token_stride | p.rows.k_token_stride | p.rows.v_token_stride) *
                       size;
    const int64_t D = p.g.head_dim;
    auto apart = [&](int64_t head_stride, int64_t heads) { return heads > 1 && head_stride != D; };
    return ((a | (uintptr_t)st) & 15) != 0 || apart(p.rows.q_head_stride, p.rows.n_q_heads) ||
           apart(p.rows.k_head_stride, p.g.n_kv_heads) ||
           apart(p.rows.v_head_stride, p.g.n_kv_heads);
}

// Launches the vector kernel with V elements a chunk, if the sizes, strides and
// addresses allow it; `done` says whether they did.
template <typename S, typename O, int V>
static int try_norm_rope_vec(const NormRopeParams& p, cudaStream_t st, bool staged, bool* done) {
    const int64_t D = p.g.head_dim, rot = p.how.rot_dim;
    auto off = [](const void* ptr, int64_t stride0, int64_t stride1, int size) {
        const uintptr_t a = (uintptr_t)(V * size < 16 ? V * size : 16);
        return (reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(stride0 * size) |
                (uintptr_t)(stride1 * size)) & (a - 1);
    };
    const int s = (int)sizeof(S), o = (int)sizeof(O);
    if (D % (2 * V) != 0 || rot % (2 * V) != 0 || D > 64 * V ||
        off(p.rows.q, p.rows.q_token_stride, p.rows.q_head_stride, s) ||
        off(p.rows.k, p.rows.k_token_stride, p.rows.k_head_stride, s) ||
        off(p.rows.v, p.rows.v_token_stride, p.rows.v_head_stride, s) ||
        off(p.kp, 0, 0, o) || off(p.vp, 0, 0, o) || off(p.q_out, 0, 0, o) ||
        off(p.how.cos_table, 0, 0, 4) || off(p.how.sin_table, 0, 0, 4) ||
        off(p.how.q_weight, 0, 0, p.how.q_weight_dtype == CX_F32 ? 4 : s) ||
        off(p.how.k_weight, 0, 0, p.how.k_weight_dtype == CX_F32 ? 4 : s) ||
        p.g.n_blocks * p.g.block_size >= (1ll << 31))
        return CX_OK;
    int L = 1;
    while (L * 2 * V < D) L *= 2;
    const int64_t R = p.rows.n_q_heads + 2 * p.g.n_kv_heads, T = p.rows.n_tokens;
    if (T * R * L >= (1ll << 31)) return CX_OK;
    // much data: the staged form.  48 rows of 128 bf16: 1024 tokens (12.6 MB) take
    // 9.8 us in either form, 1500 14.4 us in the register form and 11.6 us staged,
    // 512 5.9 and 9.0; rows of 3 KB a token (12 of 64 fp32) are faster in the
    // register form at 4096 tokens still (6.5 against 9.2 us)
    if constexpr (V == 4) {
        const int64_t row_warps = (R * L + 31) / 32;
        const int warps = (int)std::min<int64_t>((row_warps + kTokRows - 1) / kTokRows,
                                                 kTokThreads / 32 - 1);
        const int n_groups = warps * 32 / L, threads = warps * 32 + 32;  // + producer
        const int64_t stage = R * D * s + 2 * rot * 4, smem = kTokStages * stage + 2 * D * 4;
        // CTAs an SM holds by shared memory and by registers (at most 72 a thread)
        const int64_t per_sm =
            std::min<int64_t>(std::min(16, 65536 / (72 * threads)), 224 * 1024 / (smem + 1536));
        // (V rows leave the stage in chunks of 2 V elements, 16 bytes at a time)
        const bool v_off = (reinterpret_cast<uintptr_t>(p.vp) & 15) != 0;
        if (staged && D * s % 16 == 0 && rot % 4 == 0 && per_sm >= 2 && !not_bulk(p, s) &&
            !v_off && R * D * s >= 4096 && T * R * D * s >= (14ll << 20) &&
            T >= 3ll * num_sms()) {
            *done = true;
            auto kern = kv_append_norm_rope_tok_kernel<S, O, V>;
            CX_CUDA_CHECK(cudaFuncSetAttribute(
                kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            const unsigned grid = (unsigned)std::min<int64_t>(per_sm * num_sms(), T / 3);
            kern<<<grid, threads, smem, st>>>(p, L, n_groups, (int)stage);
            return check_launch("kv_append_norm_rope_tok_kernel");
        }
    }
    if (staged) return CX_OK;
    *done = true;
    kv_append_norm_rope_vec_kernel<S, O, V>
        <<<(unsigned)((T * R * L + 255) / 256), 256, 0, st>>>(p, L);
    return check_launch("kv_append_norm_rope_vec_kernel");
}

template <typename S, typename O>
static int launch_norm_rope_vec(const NormRopeParams& p, cudaStream_t st, bool* done) {
    int rc = try_norm_rope_vec<S, O, 4>(p, st, true, done);
    if (rc == CX_OK && !*done) rc = try_norm_rope_vec<S, O, 8>(p, st, false, done);
    if (rc == CX_OK && !*done) rc = try_norm_rope_vec<S, O, 4>(p, st, false, done);
    if (rc == CX_OK && !*done) rc = try_norm_rope_vec<S, O, 2>(p, st, false, done);
    return rc;
}

template <typename S>
static int launch_norm_rope(const NormRopeParams& p, cudaStream_t st) {
    // one destination type: the rows' own, or a 16-bit one under fp32 rows
    bool done = false;
    int rc = CX_OK;
    if (p.rows.n_q_heads == 0 || p.q_out_dtype == p.pool_dtype) {
        if (p.pool_dtype == p.rows.dtype)
            rc = launch_norm_rope_vec<S, S>(p, st, &done);
        else if constexpr (std::is_same<S, float>::value) {
            rc = p.pool_dtype == CX_BF16 ? launch_norm_rope_vec<S, __nv_bfloat16>(p, st, &done)
                                         : launch_norm_rope_vec<S, __half>(p, st, &done);
        }
    }
    if (rc != CX_OK || done) return rc;
    const int64_t jobs = p.rows.n_tokens * (p.rows.n_q_heads + 2 * p.g.n_kv_heads);
    kv_append_norm_rope_kernel<S><<<grid_for(jobs, 8), 256, 0, st>>>(p);
    return check_launch("kv_append_norm_rope_kernel");
}

}  // namespace cx

extern "C" int cx_kv_append_norm_rope(const cx_pool* pool, int64_t layer, const cx_qkv* rows,
                                      const int64_t* slot_mapping, const int64_t* positions,
                                      const cx_norm_rope* how, void* q_out, int32_t q_out_dtype,
                                      void* stream) {
    using namespace cx;
    int rc = check_pool(pool);
    if (rc) return rc;
    if (!rows || !how) return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: NULL rows or how");
    if (layer < 0 || layer >= pool->n_layers)
        return fail(CX_ERR_RANGE, "cx_kv_append_norm_rope: layer out of range");
    if (rows->n_tokens < 0 || rows->n_q_heads < 0 || how->table_rows < 0)
        return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: negative count");
    if (how->rot_dim < 2 || how->rot_dim % 2 != 0 || how->rot_dim > pool->head_dim)
        return fail(CX_ERR_SHAPE,
                    "cx_kv_append_norm_rope: rot_dim must be even, 2 .. head_dim");
    if (!(how->eps >= 0.f) || isinf(how->eps))
        return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: eps must be finite and >= 0");
    if ((how->q_weight && how->q_weight_dtype != CX_F32 && how->q_weight_dtype != rows->dtype) ||
        (how->k_weight && how->k_weight_dtype != CX_F32 && how->k_weight_dtype != rows->dtype))
        return fail(CX_ERR_DTYPE,
                    "cx_kv_append_norm_rope: weights must be CX_F32 or the rows' type");
    if (rows->n_tokens == 0) return CX_OK;
    if (!rows->k || !rows->v || !slot_mapping || !positions || !how->cos_table || !how->sin_table)
        return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: NULL array");
    if (rows->n_q_heads > 0 && (!rows->q || !q_out))
        return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: n_q_heads > 0 needs q and q_out");
    if (rows->n_q_heads > (1 << 20) || pool->n_kv_heads > (1 << 20) || pool->head_dim > (1 << 20))
        return fail(CX_ERR_UNSUPPORTED, "cx_kv_append_norm_rope: too many heads or dims");
    if (rows->q_token_stride < 0 || rows->q_head_stride < 0 || rows->k_token_stride < 0 ||
        rows->k_head_stride < 0 || rows->v_token_stride < 0 || rows->v_head_stride < 0)
        return fail(CX_ERR_SHAPE, "cx_kv_append_norm_rope: negative stride");
    if (rows->n_q_heads > 0 && elem_bytes(q_out_dtype) == 0)
        return fail(CX_ERR_DTYPE, "cx_kv_append_norm_rope: unknown q_out type");
    const NormRopeParams p{geom_of(pool), layer,    *rows,    *how,  slot_mapping, positions,
                           pool->k,       pool->v, q_out, pool->dtype, q_out_dtype,
                           wait_limit_ns()};
    cudaStream_t st = as_stream(stream);
    switch (rows->dtype) {
        case CX_F32: return launch_norm_rope<float>(p, st);
        case CX_BF16: return launch_norm_rope<__nv_bfloat16>(p, st);
        case CX_F16: return launch_norm_rope<__half>(p, st);
        default: return fail(CX_ERR_DTYPE, "cx_kv_append_norm_rope: unknown row type");
    }
}
