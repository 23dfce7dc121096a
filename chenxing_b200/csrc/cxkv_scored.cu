// Second translation unit of libcxkv.so: attention with score modifiers
// (cx_paged_attend).  Apart from cxkv.cu so that the two compile side by side;
// each keeps its own device flag word.
#include "cx_common.cuh"
#include "attn_generic.cuh"
#include "attn_paged_mma.cuh"
#include "attn_scored.cuh"

namespace cx {

unsigned int* dev_flags_scored() { return dev_flags(); }

}  // namespace cx

extern "C" {

int cx_paged_attend(const cx_pool* pool, int64_t layer, const cx_attn_batch* batch,
                    const cx_attn_mods* mods, const void* q, int32_t q_dtype, void* out,
                    void* workspace, size_t workspace_bytes, int32_t replan, void* stream) {
    return cx::attend_scored<false>(pool, layer, batch, mods, {}, q, q_dtype, out, workspace,
                                    workspace_bytes, replan, stream);
}

size_t cx_paged_attend_workspace_bytes(const cx_pool* pool, const cx_attn_batch* batch) {
    if (!pool || !batch || pool->n_kv_heads <= 0 || batch->n_q_heads <= 0 || batch->batch < 0)
        return 0;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_workspace(pool, &b, false);
}

int cx_paged_attend_kind(const cx_pool* pool, const cx_attn_batch* batch, int32_t q_dtype) {
    if (!pool || !batch || pool->n_kv_heads <= 0) return CX_KERNEL_GENERIC;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    return cx::attend_kind(pool, &b, q_dtype, true, false);
}

}  // extern "C"
