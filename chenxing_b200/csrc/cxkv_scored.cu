// Second translation unit of libcxkv.so: attention with score modifiers
// (cx_paged_attend).  Apart from cxkv.cu so that the two compile side by side;
// each keeps its own device flag word.
#include "cx_common.cuh"
#include "attn_generic.cuh"
#include "attn_paged_mma.cuh"
#include "attn_scored.cuh"

namespace cx {

int copy_dev_flags_scored(cudaStream_t s, unsigned int* v) { return copy_dev_flags(s, v); }
int clear_dev_flags_scored(cudaStream_t s) { return clear_dev_flags(s); }

}  // namespace cx
