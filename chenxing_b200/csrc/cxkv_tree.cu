// Translation unit of libcxkv.so with the attention of drafted trees
// (cx_paged_attend_tree): the TREE instantiations of the kernels with score
// modifiers.  It keeps a device flag word of its own, like the others.
#include "cx_common.cuh"
#include "attn_generic.cuh"
#include "attn_paged_mma.cuh"
#include "attn_scored.cuh"

namespace cx {

unsigned int* dev_flags_tree() { return dev_flags(); }

}  // namespace cx

extern "C" {

int cx_paged_attend_tree(const cx_pool* pool, int64_t layer, const cx_attn_batch* batch,
                         const cx_attn_mods* mods, const cx_tree* tree, const void* q,
                         int32_t q_dtype, void* out, void* workspace, size_t workspace_bytes,
                         int32_t replan, void* stream) {
    using namespace cx;
    if (!batch || !tree || !batch->q_start || !tree->masks || !tree->depths || tree->words < 1 ||
        tree->words > (1 << 20) || tree->words * 32 < batch->max_q_len)
        return fail(CX_ERR_SHAPE,
                    "cx_paged_attend_tree: a tree needs q_start, masks of max_q_len bits and depths");
    return attend_scored<true>(pool, layer, batch, mods, {tree->masks, tree->depths, tree->words},
                               q, q_dtype, out, workspace, workspace_bytes, replan, stream);
}

size_t cx_paged_attend_tree_workspace_bytes(const cx_pool* pool, const cx_attn_batch* batch) {
    if (!pool || !batch || pool->n_kv_heads <= 0 || batch->n_q_heads <= 0 || batch->batch < 0)
        return 0;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_workspace(pool, &b, true);
}

int cx_paged_attend_tree_kind(const cx_pool* pool, const cx_attn_batch* batch, int32_t q_dtype) {
    if (!pool || !batch || pool->n_kv_heads <= 0) return CX_KERNEL_GENERIC;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_kind(pool, &b, q_dtype, true, true);
}

}  // extern "C"
