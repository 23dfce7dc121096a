// Paged attention with score modifiers (cx_paged_attend): argument checks, the
// choice of the kernel and its launch.
#pragma once

#include <algorithm>

#include "cx_common.cuh"  // unity build: included from cxkv_scored.cu after the kernels
#include "attn_scored_tc.cuh"

namespace cx {

// What every TMA kernel needs of the pool and the batch: 16-token blocks, heads
// of 64 or 128, 16-byte alignment, indexes that fit 32 bits.
static bool tma_shape(const cx_pool* pool, const cx_attn_batch* b) {
    const int64_t tiles = pool->n_layers * pool->n_blocks * pool->n_kv_heads;
    const uintptr_t a = reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v);
    return (a & 15) == 0 && pool->block_size == kBlockTok && tiles < (1ll << 31) &&
           (pool->head_dim == 64 || pool->head_dim == 128) && b->batch < (1 << 24) &&
           pool->n_kv_heads * b->batch < (1 << 24);
}

// The tcgen05 kernel: 16-bit pools from 64 packed rows (query tokens x GQA
// group) of more than one token, and groups that the split-K kernels' 64 rows
// do not hold.
static bool tc_shape(const cx_pool* pool, const cx_attn_batch* b) {
    const int64_t G = b->n_q_heads / pool->n_kv_heads, rows = G * b->max_q_len;
    return pool->dtype != CX_F32 && tma_shape(pool, b) && G <= kTcRows &&
           (rows > 64 || (rows == 64 && b->max_q_len > 1));
}

// The split-K kernels: up to 64 packed rows.
static bool split_shape(const cx_pool* pool, const cx_attn_batch* b) {
    const int64_t rows = b->n_q_heads / pool->n_kv_heads * b->max_q_len;
    return tma_shape(pool, b) && rows >= 1 && rows <= 64 && !tc_shape(pool, b);
}

// The kernel of a call.  `vec`: q, its token stride and out are 16-byte aligned.
// 16-bit pools take queries of their own type or fp32, fp32 pools any type.
static int attend_kind(const cx_pool* pool, const cx_attn_batch* b, int32_t q_dtype, bool vec) {
    if (!vec) return CX_KERNEL_GENERIC;
    if (pool->dtype == CX_F32) return split_shape(pool, b) ? CX_KERNEL_FMA : CX_KERNEL_GENERIC;
    if (q_dtype != CX_F32 && q_dtype != pool->dtype) return CX_KERNEL_GENERIC;
    return tc_shape(pool, b)      ? CX_KERNEL_TCGEN05
           : split_shape(pool, b) ? CX_KERNEL_MMA
                                  : CX_KERNEL_GENERIC;
}

// CTAs of the tcgen05 kernel, and over how many the key tiles of each are split
// when they are fewer than half the SMs: at least 4 tiles (512 keys) a part.
// The host knows the contexts by the width of the tables only.
static void tc_grid(const cx_pool* pool, const cx_attn_batch* b, int* tpt, int64_t* n_ctiles,
                    int* n_split) {
    const int64_t G = b->n_q_heads / pool->n_kv_heads;
    *tpt = (int)(kTcRows / G);
    *n_ctiles = (b->max_q_len + 2 * *tpt - 1) / (2 * *tpt);
    const int64_t ctas = *n_ctiles * b->batch * pool->n_kv_heads, sms = grid_size();
    int64_t keys = b->table_stride * kBlockTok;
    if (b->window > 0) keys = std::min(keys, b->window + 2 * *tpt + kScKeys);
    const int64_t tiles = (keys + kScKeys - 1) / kScKeys;
    int64_t s = 1;
    if (ctas > 0 && 2 * ctas <= sms) s = std::min(sms / ctas, tiles / 4);
    *n_split = (int)std::max<int64_t>(1, s);
}

static size_t attend_workspace(const cx_pool* pool, const cx_attn_batch* b) {
    const int64_t rows = b->n_q_heads / pool->n_kv_heads * b->max_q_len;
    if (tc_shape(pool, b)) {
        int tpt, n_split;
        int64_t n_ctiles;
        tc_grid(pool, b, &tpt, &n_ctiles, &n_split);
        return n_split == 1 ? 256
                            : (size_t)(n_ctiles * b->batch * pool->n_kv_heads) * n_split * 256 *
                                  (pool->head_dim + 2) * 4;
    }
    if (!split_shape(pool, b)) return 256;
    return ws_layout(b->batch, unit_shape(pool, rows), rows, pool->head_dim, grid_size()).total;
}

// The split-K kernels (attn_paged_mma.cuh, attn_paged_f32.cuh) with MOD.
static int attend_split(const cx_pool* pool, int64_t layer, const cx_attn_batch& b,
                        const cx_attn_mods& m, float scale, const void* q, int32_t q_dtype,
                        void* out, void* ws, size_t ws_bytes, int32_t replan, bool plan_only,
                        cudaStream_t st) {
    const int64_t G = b.n_q_heads / pool->n_kv_heads, rows = G * b.max_q_len;
    const MmaShape sh = unit_shape(pool, rows);
    const int grid = grid_size();
    const WsLayout wl = ws_layout(b.batch, sh, rows, pool->head_dim, grid);
    if (!ws || ws_bytes < wl.total || (reinterpret_cast<uintptr_t>(ws) & 255) != 0)
        return fail(CX_ERR_WORKSPACE,
                    "cx_paged_attend: workspace missing, too small or not 256-byte aligned");
    char* w = static_cast<char*>(ws);
    MmaParams p{};
    p.tables = b.block_tables;
    p.table_stride = b.table_stride;
    p.ctx_lens = b.ctx_lens;
    p.q_start = b.q_start;
    p.batch = (int)b.batch;
    p.hk = (int)pool->n_kv_heads;
    p.hq = (int)b.n_q_heads;
    p.group = (int)G;
    p.max_q = (int)b.max_q_len;
    p.rows = (int)rows;
    p.hg = sh.hg;
    p.n_groups = sh.n_groups;
    p.mt = sh.mt;
    p.q_bf16 = q_dtype == CX_BF16;
    p.n_blocks = (int)pool->n_blocks;
    p.layer = (int)layer;
    p.window = b.window > 0 ? (int)b.window : 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.wait_ns = wait_limit_ns();
    p.q = q;
    p.plan = reinterpret_cast<int32_t*>(w + wl.plan);
    p.seq_start = reinterpret_cast<int32_t*>(w + wl.seq);
    p.blk_lo = reinterpret_cast<int32_t*>(w + wl.lo);
    p.counters = reinterpret_cast<int32_t*>(w + wl.cnt);
    p.partials = reinterpret_cast<float*>(w + wl.part);
    p.mod.slopes = m.alibi_slopes;
    p.mod.prefix = m.prefix_lens;
    p.plan_kind = m.prefix_lens ? 3 : 1;
    p.mod.q_stride = m.q_stride;
    p.mod.out = out;
    p.mod.out_dtype = m.out_dtype;
    p.mod.q_dtype = q_dtype;
    if (m.softcap > 0.f) {
        p.mod.cap_log2 = m.softcap * 1.4426950408889634f;
        p.mod.scale = scale / m.softcap;
        const float c[5] = {kTanhC0, kTanhC1, kTanhC2, kTanhC3, kTanhC4};
        for (int i = 0; i < 5; ++i) p.mod.c[i] = p.mod.cap_log2 * c[i];
    }
    if (replan) {
        paged_plan_kernel<<<1, 1024, 0, st>>>(p, grid);
        const int rc = check_launch("paged_plan_kernel");
        if (rc) return rc;
    }
    if (plan_only) return CX_OK;
    CUtensorMap tk, tv;
    int rc = make_pool_tmap(&tk, pool->k, pool, sh.hg);
    if (rc) return rc;
    rc = make_pool_tmap(&tv, pool->v, pool, sh.hg);
    if (rc) return rc;
    const bool d128 = pool->head_dim == 128;
    // Ranges cut into many partials are joined by a launch of their own where that
    // pays: with few ranges each is cut often (one chain of 6 rows over 15,000 bf16 keys
    // 505 -> 34 us, 8 fp32 chains of 4 over 600 48 -> 37; a call whose ranges are cut
    // less pays 2 us).  Chains of 16-bit types have many rows to join, so that one long
    // sequence among many short ones pays too: 128 chains of 5, one over 40,000 keys
    // and the rest over 400, 227 -> 150 us, against 4 us more for 128 even ones (173 ->
    // 178).  Single tokens and fp32 gain nothing there (141 -> 147 us).
    if (2 * b.batch * sh.n_groups <= grid)
        p.mod.join_min = 4;
    else if (b.max_q_len > 1 && pool->dtype != CX_F32)
        p.mod.join_min = 16;
    switch (pool->dtype) {
        case CX_F32:
            rc = d128 ? launch_f32_d<128, true>(sh, tk, tv, p, st, grid)
                      : launch_f32_d<64, true>(sh, tk, tv, p, st, grid);
            break;
        case CX_BF16: {
            using E = __nv_bfloat16;
            rc = d128 ? launch_mma_d<128, E, E, true>(sh, tk, tv, p, st, grid)
                      : launch_mma_d<64, E, E, true>(sh, tk, tv, p, st, grid);
            break;
        }
        default: {
            using E = __half;
            rc = d128 ? launch_mma_d<128, E, E, true>(sh, tk, tv, p, st, grid)
                      : launch_mma_d<64, E, E, true>(sh, tk, tv, p, st, grid);
        }
    }
    if (rc || !p.mod.join_min) return rc;
    const dim3 jg((grid - 1) / (p.mod.join_min - 1), sh.hg * p.rows);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = jg;
    cfg.blockDim = 256;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, d128 ? paged_join_kernel<128> : paged_join_kernel<64>,
                                     p));
    return check_launch("paged_join_kernel");
}

// The tcgen05 kernel (attn_scored_tc.cuh).
static int attend_tc(const cx_pool* pool, int64_t layer, const cx_attn_batch& b,
                     const cx_attn_mods& m, float scale, const void* q, int32_t q_dtype, void* out,
                     void* ws, size_t ws_bytes, cudaStream_t st) {
    ScoredTcParams p{};
    int64_t n_ctiles = 0;
    tc_grid(pool, &b, &p.tpt, &n_ctiles, &p.n_split);
    if (n_ctiles > (1 << 24)) return fail(CX_ERR_UNSUPPORTED, "cx_paged_attend: grid too large");
    if (p.n_split > 1 && (!ws || ws_bytes < attend_workspace(pool, &b) ||
                          (reinterpret_cast<uintptr_t>(ws) & 255) != 0))
        return fail(CX_ERR_WORKSPACE,
                    "cx_paged_attend: workspace missing, too small or not 256-byte aligned");
    p.tables = b.block_tables;
    p.table_stride = b.table_stride;
    p.ctx_lens = b.ctx_lens;
    p.q_start = b.q_start;
    p.slopes = m.alibi_slopes;
    p.prefix = m.prefix_lens;
    p.q = q;
    p.out = out;
    p.part = static_cast<float*>(ws);
    p.q_stride = m.q_stride;
    p.batch = (int)b.batch;
    p.hk = (int)pool->n_kv_heads;
    p.hq = (int)b.n_q_heads;
    p.group = p.hq / p.hk;
    p.n_ctiles = (int)n_ctiles;
    p.n_blocks = (int)pool->n_blocks;
    p.layer = (int)layer;
    p.window = b.window > 0 ? (int)b.window : 0;
    p.q_dtype = q_dtype;
    p.out_dtype = m.out_dtype;
    p.scale_log2 = fabsf(scale) * 1.4426950408889634f;
    p.z_scale = m.softcap > 0.f ? fabsf(scale) / m.softcap : 0.f;
    p.cap_log2 = m.softcap * 1.4426950408889634f;
    p.neg = scale < 0.f;
    p.wait_ns = wait_limit_ns();
    if (m.softcap > 0.f && p.z_scale > 0.f) {
        // In double: z_scale^9 may be small, but its product with the score is not.
        // Where a coefficient falls below fp32's normal range (caps beyond some
        // thousands), |z| <= 0.05, so that what it loses (the z^9 term is below 3e-14
        // there) does not count; where one is too large (caps below 1e-5) all are 0
        // and every score but 0 takes the other form.
        const double z1 = p.z_scale, z2 = z1 * z1;
        double zk = z1, least = 1, most = 0;
        for (int i = 0; i < 5; ++i, zk *= z2) {
            const double c = fabs(p.cap_log2 * kTanh5[i] * zk);
            least = std::min(least, c);
            most = std::max(most, c);
        }
        zk = most < 1e30 ? z1 : 0;
        for (int i = 0; i < 5; ++i, zk *= z2) {
            p.c5[i] = (float)(p.cap_log2 * kTanh5[i] * zk);
            if (i < 4) p.c4[i] = (float)(p.cap_log2 * kTanh4[i] * zk);
        }
        const bool small = least < 1e-36;
        p.s4_max = most >= 1e30 ? 0.f : (small ? 0.05f : kTanh4Max) / p.z_scale;
        p.s5_max = most >= 1e30 ? 0.f : (small ? 0.05f : kTanhMax) / p.z_scale;
    }
    CUtensorMap tk, tv;
    int rc = make_pool_tmap(&tk, pool->k, pool, 1);
    if (rc) return rc;
    rc = make_pool_tmap(&tv, pool->v, pool, 1);
    if (rc) return rc;
    if (pool->dtype == CX_BF16)
        return pool->head_dim == 128 ? launch_scored_tc<128, __nv_bfloat16>(tk, tv, p, st)
                                     : launch_scored_tc<64, __nv_bfloat16>(tk, tv, p, st);
    return pool->head_dim == 128 ? launch_scored_tc<128, __half>(tk, tv, p, st)
                                 : launch_scored_tc<64, __half>(tk, tv, p, st);
}

static int attend_scored(const cx_pool* pool, int64_t layer, const cx_attn_batch* bt,
                         const cx_attn_mods* mods, const void* q, int32_t q_dtype, void* out,
                         void* ws, size_t ws_bytes, int32_t replan, void* stream) {
    int rc = check_pool(pool);
    if (rc) return rc;
    if (!bt || !mods) return fail(CX_ERR_SHAPE, "cx_paged_attend: NULL batch or mods");
    if (layer < 0 || layer >= pool->n_layers)
        return fail(CX_ERR_RANGE, "cx_paged_attend: layer out of range");
    if (bt->batch < 0 || bt->n_q_heads <= 0 || bt->n_q_heads % pool->n_kv_heads != 0)
        return fail(CX_ERR_SHAPE,
                    "cx_paged_attend: n_q_heads must be a multiple of n_kv_heads");
    if (bt->q_start && bt->max_q_len < 1)
        return fail(CX_ERR_SHAPE, "cx_paged_attend: max_q_len must be at least 1");
    // (caps near the ends of fp32's range: their products and quotients overflow)
    if (!(mods->softcap == 0.f || (mods->softcap >= 1e-30f && mods->softcap <= 1e30f)))
        return fail(CX_ERR_SHAPE, "cx_paged_attend: softcap must be 0 or 1e-30 .. 1e30");
    if (elem_bytes(mods->out_dtype) == 0 || elem_bytes(q_dtype) == 0)
        return fail(CX_ERR_DTYPE, "cx_paged_attend: unknown query or output type");
    if (pool->head_dim > 256) return fail(CX_ERR_UNSUPPORTED, "cx_paged_attend: head_dim > 256");
    const int64_t row = bt->n_q_heads * pool->head_dim;
    if (mods->q_stride != 0 && mods->q_stride < row)
        return fail(CX_ERR_SHAPE, "cx_paged_attend: q_stride below n_q_heads * head_dim");
    if (bt->batch == 0) return CX_OK;
    if (!bt->block_tables || !bt->ctx_lens || !q || !out || bt->table_stride <= 0)
        return fail(CX_ERR_SHAPE, "cx_paged_attend: NULL array or empty table");
    const float scale = isnan(bt->scale) ? 1.0f / sqrtf((float)pool->head_dim) : bt->scale;
    if (mods->softcap > 0.f && !isfinite(scale / mods->softcap))
        return fail(CX_ERR_SHAPE, "cx_paged_attend: scale / softcap must be finite");
    cx_attn_mods m = *mods;
    if (m.q_stride == 0) m.q_stride = row;
    cx_attn_batch b = *bt;
    if (!b.q_start) b.max_q_len = 1;
    if (b.window > (1ll << 30)) b.window = 1ll << 30;    // above any context
    if (b.table_stride > (1ll << 26) || pool->n_blocks > INT32_MAX || b.max_q_len >= (1 << 24))
        return fail(CX_ERR_UNSUPPORTED, "cx_paged_attend: pool, table or max_q_len too large");
    const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                         static_cast<uintptr_t>(m.q_stride * elem_bytes(q_dtype));
    cudaStream_t st = as_stream(stream);
    const int kind = attend_kind(pool, &b, q_dtype, (al & 15) == 0);
    if (kind == CX_KERNEL_MMA || kind == CX_KERNEL_FMA)
        return attend_split(pool, layer, b, m, scale, q, q_dtype, out, ws, ws_bytes, replan,
                            false, st);
    if (kind == CX_KERNEL_TCGEN05)
        return attend_tc(pool, layer, b, m, scale, q, q_dtype, out, ws, ws_bytes, st);
    // a later layer of the step may have queries that the split-K kernels take:
    // the plan it then reads is made now
    if (replan && split_shape(pool, &b) && ws) {
        rc = attend_split(pool, layer, b, m, scale, q, q_dtype, out, ws, ws_bytes, 1, true, st);
        if (rc) return rc;
    }

    GenericParams g{};
    g.q = q;
    g.mod_out = out;
    g.mod = m;
    g.batch = b.batch;
    g.hq = b.n_q_heads;
    g.hk = pool->n_kv_heads;
    g.d = g.dv = pool->head_dim;
    g.max_q = b.max_q_len;
    g.scale = scale;
    g.mask_kind = 1;
    g.window = b.window;
    g.kp = pool->k;
    g.vp = pool->v;
    g.n_layers = pool->n_layers;
    g.n_blocks = pool->n_blocks;
    g.block_size = pool->block_size;
    g.layer = layer;
    g.tables = b.block_tables;
    g.table_stride = b.table_stride;
    g.ctx_lens = b.ctx_lens;
    g.q_start = b.q_start;
    return launch_generic<true, true>(q_dtype, pool->dtype, g, st);
}

}  // namespace cx

extern "C" {

int cx_paged_attend(const cx_pool* pool, int64_t layer, const cx_attn_batch* batch,
                    const cx_attn_mods* mods, const void* q, int32_t q_dtype, void* out,
                    void* workspace, size_t workspace_bytes, int32_t replan, void* stream) {
    return cx::attend_scored(pool, layer, batch, mods, q, q_dtype, out, workspace,
                             workspace_bytes, replan, stream);
}

size_t cx_paged_attend_workspace_bytes(const cx_pool* pool, const cx_attn_batch* batch) {
    if (!pool || !batch || pool->n_kv_heads <= 0 || batch->n_q_heads <= 0 || batch->batch < 0)
        return 0;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_workspace(pool, &b);
}

int cx_paged_attend_kind(const cx_pool* pool, const cx_attn_batch* batch, int32_t q_dtype) {
    if (!pool || !batch || pool->n_kv_heads <= 0) return CX_KERNEL_GENERIC;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_kind(pool, &b, q_dtype, true);
}

}  // extern "C"
