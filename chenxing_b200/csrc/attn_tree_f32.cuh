// Attention of drafted trees over fp32 pools, from kTrRows0 packed rows (node x GQA group)
// of a sequence on, in fp32 on CUDA cores.
//
//     s[r, j] = scale * q_r . k_j  (capped, biased by distance),   o_r = softmax(s_r) V
//
// 32 packed rows of a (sequence, KV head) share tiles of 32 keys in shared memory, two
// in turn, and a context is cut into parts over the grid, joined by their maxima.  A warp
// has 4 rows: a lane's key against them for the scores (a query element is one broadcast
// read), a lane's columns of every key for the outputs (heads of 64: half of the warp
// takes every other key).  Keys are counted through the visible ones alone, the prefix's
// and then the window's, so that parts are even whatever lies between.  It is bound by
// shared memory.  In passes of 128 bytes a warp: 8 for 16 products a lane of the scores (4 of
// the lanes' own keys, 4 broadcasts), 5 for 16 of the outputs of heads of 128 (4, and 1 of
// weights).
// 8 trees of 8 nodes, 8 / 2 heads of 64, behind up to 512 keys: 17 us where the split-K
// kernel for chains (which still has fewer rows: 32 trees of 4 behind up to 4,096 keys
// 86 us there, 143 here) took 35 to 52; 100 nodes of 4 heads behind 2,000 keys 66, the
// generic kernel 301.
#pragma once

#include "cx_common.cuh"

namespace cx {

constexpr int kTrRows = 32, kTrKeys = 32, kTrWarps = 8;
constexpr int64_t kTrRows0 = 9;   // packed rows of a sequence from which trees take it
// CTAs an SM that contexts are cut for (64 trees of 8 x 8 rows behind up to 4,000 keys: 2
// take 340 us, 4 285, 8 236, 12 238), and the most parts of one (one tree of 64 rows
// behind 16,000: 256 parts 92 us, 64 68)
constexpr int64_t kTrFill = 8, kTrParts = 64;

struct TreeRowsParams {
    const float* k;
    const float* v;
    const void* q;
    void* out;
    const int32_t* tables;
    const int32_t* ctx_lens;
    const int32_t* q_start;
    const int32_t* prefix;
    const float* slopes;
    TreeMask tree;
    int64_t table_stride, n_blocks, layer, q_stride;
    int32_t batch, hk, hq, group, max_q, row_tiles, n_split, block_size, window;
    int32_t q_dtype, out_dtype;
    float scale, softcap;
    float* part;              // [unit][split][kTrRows][D + 2]
};

// Rows of a unit (sequence, KV head, row tile).
struct TreeRowsUnit {
    int b, kh, qs, T, r0, nr;
    __device__ __forceinline__ TreeRowsUnit(const TreeRowsParams& p, int unit) {
        const int rt = unit % p.row_tiles, bh = unit / p.row_tiles;
        b = bh / p.hk;
        kh = bh - b * p.hk;
        qs = p.q_start[b];
        T = min(max(p.q_start[b + 1] - qs, 0), p.max_q);
        r0 = rt * kTrRows;
        nr = min(kTrRows, T * p.group - r0);
    }
};

template <int D>
struct TreeRowsCfg {
    // floats between rows: 4 modulo 32, so that eight lanes' 16-byte reads of their own
    // rows meet no bank twice
    static constexpr int SD = D + 4;
    static constexpr int BYTES = ((kTrRows + 4 * kTrKeys) * SD + kTrWarps * kTrKeys * 4) * 4;
};

template <int D>
__global__ void __launch_bounds__(kTrWarps * 32, 2) tree_rows_kernel(const TreeRowsParams p) {
    constexpr int SD = TreeRowsCfg<D>::SD;
    extern __shared__ float gsm[];                // queries, [2] K tiles, [2] V tiles, weights
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* s_q = gsm;
    float* s_k = s_q + kTrRows * SD;
    float* s_v = s_k + 2 * kTrKeys * SD;
    float4* s_p = reinterpret_cast<float4*>(s_v + 2 * kTrKeys * SD) + warp * kTrKeys;
    const TreeRowsUnit x(p, (int)blockIdx.x);
    const int raw = p.ctx_lens[x.b];
    const int64_t cap = p.table_stride * p.block_size;
    const int ctx = (int)min((int64_t)max(raw, 0), cap), base = ctx - x.T;
    if (x.r0 == 0 && x.kh == 0 && blockIdx.y == 0 && tid == 0) {
        if (raw > cap) raise_flag(CX_DEV_TABLE_OVERRUN);
        if (x.T != p.q_start[x.b + 1] - x.qs || (raw > 0 && x.T > ctx)) raise_flag(CX_DEV_BAD_QLEN);
    }
    if (x.nr <= 0) return;
    const int G = p.group;
    for (int i = tid; i < kTrRows * D; i += kTrWarps * 32) {
        const int r = i / D, d = i - r * D, R = x.r0 + r;
        s_q[r * SD + d] = r < x.nr ? load_as(p.q, p.q_dtype,
                                             (x.qs + R / G) * p.q_stride +
                                                 (int64_t)(x.kh * G + R % G) * D + d)
                                   : 0.f;
    }
    // keys [0, n_pre) and [lo, hi): the ones that some row may see
    const int pre = p.prefix ? min(max(p.prefix[x.b], 0), max(base, 0)) : 0;
    const int hi = max(0, min(base + (x.r0 + x.nr - 1) / G + 1, ctx));
    const int lo = min(hi, p.window > 0 ? max(0, base - p.window + 1) : 0);
    const int n_pre = min(pre, lo), n_keys = n_pre + hi - lo;
    const int per = ((n_keys + p.n_split - 1) / p.n_split + kTrKeys - 1) / kTrKeys * kTrKeys;
    const int v_lo = (int)blockIdx.y * per, v_hi = min(n_keys, v_lo + per);
    auto key_of = [&](int v) { return v < n_pre ? v : v - n_pre + lo; };

    const int R0 = 4 * warp;
    int at[4];                                    // where the row's node stands
    float slope[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int R = x.r0 + R0 + r;
        const bool in = R0 + r < x.nr;
        at[r] = in ? base + p.tree.depths[x.qs + R / G] : 0;
        slope[r] = in && p.slopes ? p.slopes[x.kh * G + R % G] : 0.f;
    }
    const int32_t* tab = p.tables + (int64_t)x.b * p.table_stride;
    bool bad = false;
    // virtual keys v0 .. v0 + 31 into buffer `buf`, four a warp; zeros for what is not there
    auto load = [&](int v0, int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = v0 + R0 + i;
            int64_t src = -1;
            if (v < v_hi) {
                const int k = key_of(v), blk = k / p.block_size;
                const int64_t id = tab[blk];
                if (id >= 0 && id < p.n_blocks)
                    src = (((p.layer * p.n_blocks + id) * p.hk + x.kh) * p.block_size +
                           (k - blk * p.block_size)) * D;
                else
                    bad = true;
            }
            const int row = (buf * kTrKeys + R0 + i) * SD;
            // (heads of 64: K by the lower lanes, V by the upper)
            const int c = 4 * (lane % (D / 4));
            const int64_t from = src < 0 ? 0 : src + c;
            if (D == 128 || lane < 16) cp_async16(s_k + row + c, p.k + from, src >= 0);
            if (D == 128 || lane >= 16) cp_async16(s_v + row + c, p.v + from, src >= 0);
        }
    };
    float o[4][4], m[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] = 0.f;
    }
    if (v_lo < v_hi) load(v_lo, 0);
    int buf = 0;
    for (int v0 = v_lo; v0 < v_hi; v0 += kTrKeys, buf ^= 1) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();                          // the tile is there; the other buffer was read
        if (v0 + kTrKeys < v_hi) load(v0 + kTrKeys, buf ^ 1);
        if (R0 >= x.nr) continue;
        // ---- scores of virtual key v0 + lane ----
        const float4* kr = reinterpret_cast<const float4*>(s_k + (buf * kTrKeys + lane) * SD);
        const float4* qr = reinterpret_cast<const float4*>(s_q + R0 * SD);
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int c = 0; c < D / 4; ++c) {
            const float4 kv = kr[c];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 qv = qr[r * (SD / 4) + c];
                a[r] = fmaf(qv.x, kv.x, a[r]);
                a[r] = fmaf(qv.y, kv.y, a[r]);
                a[r] = fmaf(qv.z, kv.z, a[r]);
                a[r] = fmaf(qv.w, kv.w, a[r]);
            }
        }
        const int k = key_of(v0 + lane);
        bool there = v0 + lane < v_hi;
        if (there) {
            const int64_t id = tab[k / p.block_size];
            there = id >= 0 && id < p.n_blocks;
        }
        const int to = p.slopes && there && k >= base
                           ? tree_key_pos(p.tree, x.qs, x.T, base, k - base)
                           : k;                   // where the key stands
        float pr[4], corr[4];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bool see = there && R0 + r < x.nr;
            if (see) {
                const int t = (x.r0 + R0 + r) / G;
                see = k < base ? k < pre || p.window <= 0 || k > at[r] - p.window
                               : tree_bits(p.tree, x.qs + t, t, k - base) & 1u;
            }
            float s = a[r] * p.scale;
            if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
            if (p.slopes) s -= slope[r] * (float)abs(at[r] - to);
            if (!see) s = -INFINITY;
            float top = s;
#pragma unroll
            for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            corr[r] = 1.f;
            if (top > m[r]) {
                corr[r] = expf(m[r] - top);
                m[r] = top;
                moved = true;
            }
            pr[r] = see ? expf(s - ref_base(m[r])) : 0.f;
            l[r] = fmaf(l[r], corr[r], pr[r]);
        }
        s_p[lane] = make_float4(pr[0], pr[1], pr[2], pr[3]);
        __syncwarp();
        if (moved) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][e] *= corr[r];
        }
        // ---- columns 4 (lane % (D / 4)) .. of every key, of heads of 64 every other ----
        const int first = D == 128 ? 0 : lane >> 4;
        const float* vt = s_v + (buf * kTrKeys + first) * SD + 4 * (lane % (D / 4));
#pragma unroll 4
        for (int j = 0; j < kTrKeys; j += 128 / D) {
            const float4 w = s_p[j + first];
            // (a key that none of the rows sees adds nothing, whatever it holds)
            if (w.x == 0.f && w.y == 0.f && w.z == 0.f && w.w == 0.f) continue;
            const float4 v = *reinterpret_cast<const float4*>(vt + j * SD);
            const float y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                o[r][0] = fmaf(y[r], v.x, o[r][0]);
                o[r][1] = fmaf(y[r], v.y, o[r][1]);
                o[r][2] = fmaf(y[r], v.z, o[r][2]);
                o[r][3] = fmaf(y[r], v.w, o[r][3]);
            }
        }
        __syncwarp();
    }
    asm volatile("griddepcontrol.launch_dependents;");
    if (bad && lane == 0) raise_flag(CX_DEV_BAD_BLOCK);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float L = l[r];
#pragma unroll
        for (int w = 16; w; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
        if constexpr (D == 64) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], 16);
        }
        if (R0 + r >= x.nr || lane >= D / 4) continue;
        if (p.n_split > 1) {
            float* dst = p.part + (((int64_t)blockIdx.x * p.n_split + blockIdx.y) * kTrRows + R0 + r) *
                                      (D + 2);
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                *reinterpret_cast<float2*>(dst + 4 * lane + e) = make_float2(o[r][e], o[r][e + 1]);
            if (lane == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[r], L);
        } else {
            const int R = x.r0 + R0 + r;
            const float inv = sum_inv(L);
            const int64_t row = (int64_t)(x.qs + R / G) * p.hq + x.kh * G + R % G;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                store_as(p.out, p.out_dtype, row * D + 4 * lane + e, o[r][e] * inv);
        }
    }
}

// Joins a row's parts: one CTA a row, a thread a column.
template <int D>
__global__ void __launch_bounds__(D) tree_rows_join(const TreeRowsParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRowsUnit x(p, (int)blockIdx.x);
    const int r = blockIdx.y, lane = threadIdx.x & 31;
    if (r >= x.nr) return;
    const float* src = p.part + ((int64_t)blockIdx.x * p.n_split * kTrRows + r) * (D + 2);
    constexpr int64_t STEP = kTrRows * (D + 2);
    __shared__ float s_f[kTrParts];
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < p.n_split; s += 32) M = fmaxf(M, src[s * STEP + D]);
#pragma unroll
    for (int w = 16; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    for (int s = lane; s < p.n_split; s += 32) {
        const float f = expf(src[s * STEP + D] - ref_base(M));
        L = fmaf(src[s * STEP + D + 1], f, L);
        if (threadIdx.x < 32) s_f[s] = f;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
    __syncthreads();
    float O = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.n_split; ++s) O = fmaf(src[s * STEP + threadIdx.x], s_f[s], O);
    const int R = x.r0 + r;
    store_as(p.out, p.out_dtype,
             ((int64_t)(x.qs + R / p.group) * p.hq + x.kh * p.group + R % p.group) * D + threadIdx.x,
             L == 0.f ? 0.f : O / L);
}

// fp32 pools with heads of 64 or 128 on 16-byte rows, blocks of any size.
static bool tree_rows_shape(const cx_pool* pool, const cx_attn_batch* b) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v);
    return pool->dtype == CX_F32 && (a & 15) == 0 && (pool->head_dim == 64 || pool->head_dim == 128) &&
           pool->block_size <= (1 << 24) && pool->n_kv_heads < (1 << 20) && b->batch < (1 << 24) &&
           b->n_q_heads / pool->n_kv_heads * b->max_q_len >= kTrRows0;
}

// Units, and the parts that each one's context is cut into.
static void tree_rows_grid(const cx_pool* pool, const cx_attn_batch* b, int64_t* row_tiles,
                           int64_t* units, int* n_split) {
    *row_tiles = (b->n_q_heads / pool->n_kv_heads * b->max_q_len + kTrRows - 1) / kTrRows;
    *units = b->batch * pool->n_kv_heads * *row_tiles;
    const int64_t keys = b->table_stride * pool->block_size;
    const int64_t want = kTrFill * std::max(num_sms(), 1) / std::max<int64_t>(*units, 1);
    *n_split = (int)std::max<int64_t>(
        1, std::min(std::min(want, (keys + kTrKeys - 1) / kTrKeys), kTrParts));
}

static size_t tree_rows_workspace(const cx_pool* pool, const cx_attn_batch* b) {
    int64_t row_tiles, units;
    int n_split;
    tree_rows_grid(pool, b, &row_tiles, &units, &n_split);
    return n_split == 1 ? 256 : (size_t)units * n_split * kTrRows * (pool->head_dim + 2) * 4;
}

template <bool TREE>
static int attend_tree_rows(const cx_pool* pool, int64_t layer, const cx_attn_batch& b,
                            const cx_attn_mods& m, const TreeMask& tree, float scale, const void* q,
                            int32_t q_dtype, void* out, void* ws, size_t ws_bytes,
                            cudaStream_t st) {
    int64_t row_tiles, units;
    TreeRowsParams p{};
    tree_rows_grid(pool, &b, &row_tiles, &units, &p.n_split);
    if (units > INT32_MAX || b.table_stride * pool->block_size > (1ll << 30))
        return fail(CX_ERR_UNSUPPORTED, "cx_paged_attend_tree: rows or tables too large");
    if (p.n_split > 1 && (!ws || ws_bytes < tree_rows_workspace(pool, &b) ||
                          (reinterpret_cast<uintptr_t>(ws) & 255) != 0))
        return fail(CX_ERR_WORKSPACE,
                    "cx_paged_attend_tree: workspace missing, too small or not 256-byte aligned");
    p.k = static_cast<const float*>(pool->k);
    p.v = static_cast<const float*>(pool->v);
    p.q = q;
    p.out = out;
    p.tables = b.block_tables;
    p.ctx_lens = b.ctx_lens;
    p.q_start = b.q_start;
    p.prefix = m.prefix_lens;
    p.slopes = m.alibi_slopes;
    p.tree = tree;
    p.table_stride = b.table_stride;
    p.n_blocks = pool->n_blocks;
    p.layer = layer;
    p.q_stride = m.q_stride;
    p.batch = (int)b.batch;
    p.hk = (int)pool->n_kv_heads;
    p.hq = (int)b.n_q_heads;
    p.group = p.hq / p.hk;
    p.max_q = (int)b.max_q_len;
    p.row_tiles = (int)row_tiles;
    p.block_size = (int)pool->block_size;
    p.window = b.window > 0 ? (int)b.window : 0;
    p.q_dtype = q_dtype;
    p.out_dtype = m.out_dtype;
    p.scale = scale;
    p.softcap = m.softcap;
    p.part = static_cast<float*>(ws);
    auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        CX_CUDA_CHECK(cudaFuncSetAttribute(tree_rows_kernel<D>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           TreeRowsCfg<D>::BYTES));
        tree_rows_kernel<D><<<dim3((unsigned)units, (unsigned)p.n_split), kTrWarps * 32,
                              TreeRowsCfg<D>::BYTES, st>>>(p);
        const int rc = check_launch("tree_rows_kernel");
        if (rc || p.n_split == 1) return rc;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)units, kTrRows);
        cfg.blockDim = D;
        cfg.stream = st;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        CX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tree_rows_join<D>, p));
        return check_launch("tree_rows_join");
    };
    return pool->head_dim == 128 ? go(std::integral_constant<int, 128>{})
                                 : go(std::integral_constant<int, 64>{});
}

}  // namespace cx
