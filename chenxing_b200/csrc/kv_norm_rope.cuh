// RMS norm of query and key heads, rotation of their leading dims and the
// slot-mapped append, in one pass over the step's rows:
//     y = x * rsqrt(mean(x^2) + eps) * w          (per head, fp32)
//     (y_a, y_b) -> (y_a c - y_b s, y_b c' + y_a s')   for the pairs of y[0, rot)
// K rows go to their pool slots, V rows are copied, Q rows go to q_out; each
// value is rounded once, to its destination's type.
#pragma once

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

template <typename S>
static int launch_norm_rope(const NormRopeParams& p, cudaStream_t st) {
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
                           pool->k,       pool->v, q_out, pool->dtype, q_out_dtype};
    cudaStream_t st = as_stream(stream);
    switch (rows->dtype) {
        case CX_F32: return launch_norm_rope<float>(p, st);
        case CX_BF16: return launch_norm_rope<__nv_bfloat16>(p, st);
        case CX_F16: return launch_norm_rope<__half>(p, st);
        default: return fail(CX_ERR_DTYPE, "cx_kv_append_norm_rope: unknown row type");
    }
}
