// Second translation unit of libcxkv.so: attention with score modifiers
// (cx_paged_attend).  Apart from cxkv.cu so that the two compile side by side;
// each keeps its own device flag word.
#include "cx_common.cuh"
#include "attn_generic.cuh"
#include "attn_paged_mma.cuh"
#include "attn_scored.cuh"

namespace cx {

int read_dev_flags_scored(cudaStream_t s, int clear, unsigned int* v) {
    return read_dev_flags(s, clear, v);
}

}  // namespace cx
