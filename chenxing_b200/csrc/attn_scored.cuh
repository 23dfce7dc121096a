// Paged attention with score modifiers (cx_paged_attend): argument checks and
// the choice of the kernel.
#pragma once

#include "cx_common.cuh"  // unity build: included from cxkv.cu after the kernels

namespace cx {

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
    if (!(mods->softcap >= 0.f) || isinf(mods->softcap))
        return fail(CX_ERR_SHAPE, "cx_paged_attend: softcap must be finite and >= 0");
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
    cx_attn_mods m = *mods;
    if (m.q_stride == 0) m.q_stride = row;

    GenericParams g{};
    g.q = q;
    g.mod_out = out;
    g.mod = m;
    g.batch = bt->batch;
    g.hq = bt->n_q_heads;
    g.hk = pool->n_kv_heads;
    g.d = g.dv = pool->head_dim;
    g.max_q = bt->q_start ? bt->max_q_len : 1;
    g.scale = scale;
    g.mask_kind = 1;
    g.window = bt->window;
    g.kp = pool->k;
    g.vp = pool->v;
    g.n_layers = pool->n_layers;
    g.n_blocks = pool->n_blocks;
    g.block_size = pool->block_size;
    g.layer = layer;
    g.tables = bt->block_tables;
    g.table_stride = bt->table_stride;
    g.ctx_lens = bt->ctx_lens;
    g.q_start = bt->q_start;
    return launch_generic<true, true>(q_dtype, pool->dtype, g, as_stream(stream));
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
    return cx_paged_workspace_bytes(pool, batch);
}

int cx_paged_attend_kind(const cx_pool*, const cx_attn_batch*, int32_t) {
    return CX_KERNEL_GENERIC;
}

}  // extern "C"
