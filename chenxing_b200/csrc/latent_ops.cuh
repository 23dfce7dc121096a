// Data movement of the latent cache (append, gather, block copy) and the move of
// accepted nodes in both kinds of cache.
#pragma once

#include "cx_common.cuh"

namespace cx {

// ---------------------------------------------------------------------------
// append: RMS norm of the latent, rotation of the shared key part and of the
// queries' rotary parts
// ---------------------------------------------------------------------------
struct LatAppendParams {
    const void* latent;
    const void* rope;
    const void* q;
    int64_t latent_tok, rope_tok, q_tok, q_head;
    const int64_t* slots;
    const int64_t* positions;       // NULL: no rotation
    const float* cos_table;
    const float* sin_table;
    int64_t table_rows, n_slots, layer_row0;   // layer_row0: first row of the layer
    const void* weight;             // NULL: no norm
    void* pool;
    void* q_out;
    int32_t n_tokens, heads, dc, dr, dtype, pool_dtype, weight_dtype, q_out_dtype, interleaved;
    float eps;
};

// 8 elements, 16-byte aligned, as they lie in memory: asked for at once, looked at
// when they are needed.
template <typename E> struct Raw8 {
    uint4 u;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        u = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(p) + i));
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) f2_get(Half16<E>::unpack(w[k]), x[2 * k], x[2 * k + 1]);
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        a = __ldg(s);
        b = __ldg(s + 1);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
};

__device__ __forceinline__ void store8_as(void* p, int32_t dtype, int64_t i, const float (&x)[8]) {
    if (dtype == CX_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = dtype == CX_BF16 ? Half16<__nv_bfloat16>::pack(x[2 * k], x[2 * k + 1])
                                : Half16<__half>::pack(x[2 * k], x[2 * k + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The rotation as in the kernels beside this one: a pair (x, y) at angle tables
// (c, s) of either element.
struct RopePair {
    float cx, sx, cy, sy;
    __device__ __forceinline__ void turn(float& x, float& y) const {
        const float a = x * cx - y * sx, b = y * cy + x * sy;
        x = a;
        y = b;
    }
};

// Where token t goes and its rotation; false: nothing of it is stored in the pool.
__device__ __forceinline__ bool lat_slot(const LatAppendParams& p, int64_t t, int64_t& row) {
    const int64_t s = p.slots[t];
    if (s < 0) return false;
    if (s >= p.n_slots) {
        if ((threadIdx.x & 31) == 0) raise_flag(CX_DEV_BAD_SLOT);
        return false;
    }
    row = p.layer_row0 + s;
    return true;
}

// One block per token.  Warp 0 has the pool row, the other warps 32 units of 8 pairs
// of the queries at a time: with rows of 16-byte multiples a lane holds 8 pairs, whose
// angles it loads once for all its heads.  All that a lane needs first (rows, slot,
// position) is asked for before any of it is looked at; then come the angles and the
// weights.  8,192 tokens, 32 heads, bf16, 90 MB: 23 us.  72 registers a lane: it still spills,
// 96 bytes in 16 bits and 172 in fp32.  With a head a lane, twice the warps and 56 registers,
// which spill more, 27 (64 tokens: 2.5 and 2.7); with loads that are converted where they are
// made, one after the other, 47.
constexpr int kLaHeads = 2;       // heads a lane asks for at once
constexpr int kLaWarps = 5;
template <typename E>
__global__ void __launch_bounds__(kLaWarps * 32, 5)
    latent_append_vec_kernel(const LatAppendParams p) {
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    const int units = p.dr / 16, half = p.dr / 2;     // units of 8 pairs a head
    const bool turn = p.positions != nullptr;
    const int64_t pos = turn ? p.positions[t] : 0;
    // first elements of unit u's two runs of 8
    auto run_a = [&](int u) { return p.interleaved ? 16 * u : 8 * u; };
    auto run_b = [&](int u) { return p.interleaved ? 16 * u + 8 : half + 8 * u; };
    // the angles of unit u's pairs: c[0 .. 1] and s[0 .. 1] of either pair element, or of
    // the first, c[2 .. 3] and s[2 .. 3] of the second
    struct Angles {
        float4 c[4], s[4];
    };
    auto angles = [&](int u) {
        Angles g;
        const float4* c = reinterpret_cast<const float4*>(p.cos_table + pos * p.dr + 8 * u);
        const float4* s = reinterpret_cast<const float4*>(p.sin_table + pos * p.dr + 8 * u);
        const int o = p.interleaved ? 0 : half / 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            g.c[k] = __ldg(c + k);
            g.s[k] = __ldg(s + k);
            g.c[2 + k] = __ldg(c + o + k);
            g.s[2 + k] = __ldg(s + o + k);
        }
        return g;
    };
    // the pairs turned: elements 2k, 2k + 1 of the 16, or k of either run
    auto rotate = [&](const Angles& g, float (&a)[8], float (&b)[8]) {
        if (p.interleaved) {
            const float4 c0 = g.c[0], c1 = g.c[1], s0 = g.s[0], s1 = g.s[1];
            RopePair{c0.x, s0.x, c0.x, s0.x}.turn(a[0], a[1]);
            RopePair{c0.y, s0.y, c0.y, s0.y}.turn(a[2], a[3]);
            RopePair{c0.z, s0.z, c0.z, s0.z}.turn(a[4], a[5]);
            RopePair{c0.w, s0.w, c0.w, s0.w}.turn(a[6], a[7]);
            RopePair{c1.x, s1.x, c1.x, s1.x}.turn(b[0], b[1]);
            RopePair{c1.y, s1.y, c1.y, s1.y}.turn(b[2], b[3]);
            RopePair{c1.z, s1.z, c1.z, s1.z}.turn(b[4], b[5]);
            RopePair{c1.w, s1.w, c1.w, s1.w}.turn(b[6], b[7]);
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 cx = g.c[k], sx = g.s[k], cy = g.c[2 + k], sy = g.s[2 + k];
                RopePair{cx.x, sx.x, cy.x, sy.x}.turn(a[4 * k], b[4 * k]);
                RopePair{cx.y, sx.y, cy.y, sy.y}.turn(a[4 * k + 1], b[4 * k + 1]);
                RopePair{cx.z, sx.z, cy.z, sy.z}.turn(a[4 * k + 2], b[4 * k + 2]);
                RopePair{cx.w, sx.w, cy.w, sy.w}.turn(a[4 * k + 3], b[4 * k + 3]);
            }
        }
    };
    const bool pool_row = warp == 0;
    if (pool_row) {
        const int64_t slot = p.slots[t], src = t * p.latent_tok;
        const int n8 = p.dc / 8;                      // (dc <= 512: up to 2 runs of 8 a lane)
        Raw8<E> lat[2], ra, rb;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (lane + 32 * k < n8) lat[k].load(p.latent, src + (lane + 32 * k) * 8);
        if (lane < units) {
            ra.load(p.rope, t * p.rope_tok + run_a(lane));
            rb.load(p.rope, t * p.rope_tok + run_b(lane));
        }
        const bool in_table = !turn || (pos >= 0 && pos < p.table_rows);
        if (lane == 0) {
            if (!in_table)
                raise_flag(CX_DEV_BAD_POSITION);
            else if (slot >= p.n_slots)
                raise_flag(CX_DEV_BAD_SLOT);
        }
        if (in_table && slot >= 0 && slot < p.n_slots) {
            const int64_t dst = (p.layer_row0 + slot) * (p.dc + p.dr);
            float x[2][8], sum = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (lane + 32 * k >= n8) continue;
                lat[k].get(x[k]);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(x[k][e], x[k][e], sum);
            }
            float f = 1.f;
            if (p.weight) {
#pragma unroll
                for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                f = rsqrtf(sum / (float)p.dc + p.eps);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int i = (lane + 32 * k) * 8;
                if (lane + 32 * k >= n8) continue;
                if (p.weight) {
                    float w[8];
                    if (p.weight_dtype == CX_F32) {
                        Raw8<float> r;
                        r.load(p.weight, i);
                        r.get(w);
                    } else {
                        Raw8<E> r;
                        r.load(p.weight, i);
                        r.get(w);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[k][e] = x[k][e] * f * w[e];
                }
                store8_as(p.pool, p.pool_dtype, dst + i, x[k]);
            }
            if (lane < units) {
                float a[8], b[8];
                ra.get(a);
                rb.get(b);
                if (turn) rotate(angles(lane), a, b);
                store8_as(p.pool, p.pool_dtype, dst + p.dc + run_a(lane), a);
                store8_as(p.pool, p.pool_dtype, dst + p.dc + run_b(lane), b);
            }
        }
    }
    if (!p.q || (pool_row && n_warps > 1)) return;
    // units of the queries: 32 % units == 0, so that a lane keeps one unit's angles
    const int w0 = n_warps > 1 ? warp - 1 : 0, nw = n_warps > 1 ? n_warps - 1 : 1;
    const int u = lane % units, step = nw * (32 / units);
    Angles g;
    for (int h0 = w0 * (32 / units) + lane / units, first = 1; h0 < p.heads;
         h0 += kLaHeads * step, first = 0) {
        Raw8<E> ra[kLaHeads], rb[kLaHeads];
#pragma unroll
        for (int k = 0; k < kLaHeads; ++k) {
            const int h = h0 + k * step;
            if (h >= p.heads) continue;
            const int64_t src = t * p.q_tok + h * p.q_head;
            ra[k].load(p.q, src + run_a(u));
            rb[k].load(p.q, src + run_b(u));
        }
        if (first && turn) {
            if (pos < 0 || pos >= p.table_rows) return;
            g = angles(u);
        }
#pragma unroll
        for (int k = 0; k < kLaHeads; ++k) {
            const int h = h0 + k * step;
            if (h >= p.heads) continue;
            float a[8], b[8];
            const int64_t dst = (t * p.heads + h) * p.dr;
            ra[k].get(a);
            rb[k].get(b);
            if (turn) rotate(g, a, b);
            store8_as(p.q_out, p.q_out_dtype, dst + run_a(u), a);
            store8_as(p.q_out, p.q_out_dtype, dst + run_b(u), b);
        }
    }
}

// Any alignment and widths: one block of 128 threads per token, element by element.
__global__ void __launch_bounds__(128) latent_append_kernel(const LatAppendParams p) {
    const int64_t t = blockIdx.x;
    int64_t pos = 0;
    const bool turn = p.positions != nullptr;
    if (turn) {
        pos = p.positions[t];
        if (pos < 0 || pos >= p.table_rows) {
            if (threadIdx.x == 0) raise_flag(CX_DEV_BAD_POSITION);
            return;
        }
    }
    const int half = p.dr / 2;
    auto pair = [&](const void* src, int64_t i0, void* dst, int32_t dst_type, int64_t o0, int k) {
        const int a = p.interleaved ? 2 * k : k, b = p.interleaved ? 2 * k + 1 : k + half;
        float x = load_as(src, p.dtype, i0 + a), y = load_as(src, p.dtype, i0 + b);
        if (turn) {
            const float* c = p.cos_table + pos * p.dr;
            const float* s = p.sin_table + pos * p.dr;
            const int o = p.interleaved ? k : k + half;
            const RopePair r{c[k], s[k], c[o], s[o]};
            r.turn(x, y);
        }
        store_as(dst, dst_type, o0 + a, x);
        store_as(dst, dst_type, o0 + b, y);
    };
    int64_t row;
    __shared__ float s_sum[4];
    if (lat_slot(p, t, row)) {                        // (the same for the whole block)
        const int64_t dst = row * (p.dc + p.dr), src = t * p.latent_tok;
        float f = 1.f;
        if (p.weight) {
            float sum = 0.f;
            for (int i = threadIdx.x; i < p.dc; i += 128) {
                const float x = load_as(p.latent, p.dtype, src + i);
                sum = fmaf(x, x, sum);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
            __syncthreads();
            f = rsqrtf((s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]) / (float)p.dc + p.eps);
        }
        for (int i = threadIdx.x; i < p.dc; i += 128) {
            float x = load_as(p.latent, p.dtype, src + i);
            if (p.weight) x = x * f * load_as(p.weight, p.weight_dtype, i);
            store_as(p.pool, p.pool_dtype, dst + i, x);
        }
        for (int k = threadIdx.x; k < half; k += 128)
            pair(p.rope, t * p.rope_tok, p.pool, p.pool_dtype, dst + p.dc, k);
    }
    if (!p.q) return;
    for (int i = threadIdx.x; i < p.heads * half; i += 128) {
        const int h = i / half;
        pair(p.q, t * p.q_tok + h * p.q_head, p.q_out, p.q_out_dtype,
             (t * p.heads + h) * p.dr, i - h * half);
    }
}

// ---------------------------------------------------------------------------
// gather and block copy
// ---------------------------------------------------------------------------
template <typename E>
__global__ void latent_gather_kernel(const E* pool, int64_t layer_row0, int64_t n_blocks,
                                     int block_size, const int32_t* table, int64_t n_tokens,
                                     int dc, int dr, E* latent, E* rope) {
    const int64_t t = blockIdx.x;
    if (t >= n_tokens) return;
    const int64_t id = table[t / block_size];
    if (id < 0 || id >= n_blocks) {
        if (threadIdx.x == 0) raise_flag(CX_DEV_BAD_BLOCK);
        return;
    }
    const E* src = pool + (layer_row0 + id * block_size + t % block_size) * (dc + dr);
    for (int i = threadIdx.x; i < dc + dr; i += blockDim.x) {
        if (i < dc)
            latent[t * dc + i] = src[i];
        else
            rope[t * dr + i - dc] = src[i];
    }
}

// Blocks src[i] -> dst[i] of layers [l0, l0 + gridDim.y): the first n_valid[i] (or
// n_slots) rows are one run of bytes, moved in words of V.
template <typename V>
__global__ void latent_copy_kernel(V* pool, int64_t layer_words, int64_t block_words,
                                   int64_t row_words, int64_t n_blocks, int64_t l0,
                                   const int32_t* src, const int32_t* dst,
                                   const int32_t* n_valid, int64_t n_slots, int64_t block_size) {
    const int64_t i = blockIdx.x;
    const int64_t a = src[i], b = dst[i];
    if (a < 0 || a >= n_blocks || b < 0 || b >= n_blocks) {
        if (threadIdx.x == 0) raise_flag(CX_DEV_BAD_BLOCK);
        return;
    }
    int64_t n = n_valid ? n_valid[i] : n_slots;
    n = (n < 0 ? 0 : n > block_size ? block_size : n) * row_words;
    V* base = pool + (l0 + blockIdx.y) * layer_words;
    for (int64_t k = threadIdx.x; k < n; k += blockDim.x)
        base[b * block_words + k] = base[a * block_words + k];
}

// ---------------------------------------------------------------------------
// accepted nodes: path[k] of sequence b moves to position base + k
// ---------------------------------------------------------------------------
struct AcceptParams {
    void* pool[2];                  // K and V, or one latent pool
    int32_t n_pools;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* ctx_lens;
    const int32_t* q_start;
    const int32_t* paths;
    int64_t path_stride, path_len;
    int64_t n_blocks, layer_words;  // words of V in a layer
    int32_t block_size, heads, row_words, planes;   // planes: layers * pools * heads
};

// A thread owns words (V) of the planes' rows (plane: layer, pool, head) of one sequence
// and moves each for every node in order, 8 at a time: a path ascends, so that its k-th
// node is at or behind position k, and what a group of 8 overwrites no later one
// reads.  No two threads share a word, so that rows which are both a source and a
// destination need no synchronisation.  Rows of 256 bytes are read where they lie: 64
// sequences x 5 nodes x 24 layers of 8 heads of 128, 28 MB, 12 us.
template <typename V>
__global__ void __launch_bounds__(256) accept_kernel(const AcceptParams p) {
    const int b = blockIdx.y;
    __shared__ int64_t s_from[32], s_to[32];
    __shared__ int s_n, s_more;
    const int lane = threadIdx.x & 31;
    const int32_t* path = p.paths + b * p.path_stride;
    const int32_t* tab = p.tables + b * p.table_stride;
    int n = lane < p.path_len ? path[lane] : -1;      // (beside the lengths, not behind them)
    const int q0 = p.q_start ? p.q_start[b] : b, T = p.q_start ? p.q_start[b + 1] - q0 : 1;
    const int64_t ctx = p.ctx_lens[b], cap = p.table_stride * p.block_size, base = ctx - T;
    if (T <= 0 || base < 0 || ctx > cap) {
        // (a row without nodes or context, as a padded batch has them: nothing to move, and
        // nothing wrong unless its path asks for some)
        if (threadIdx.x == 0 && blockIdx.x == 0 && n >= 0)
            raise_flag(T <= 0 ? CX_DEV_BAD_PATH : CX_DEV_BAD_QLEN);
        return;
    }
    const int64_t words = (int64_t)p.planes * p.row_words;
    int before = -1;                                  // the last node of the 32 before
    for (int64_t k0 = 0; k0 < p.path_len; k0 += 32) {
        if (threadIdx.x < 32) {
            const int64_t k = k0 + lane;
            if (k0 > 0) n = k < p.path_len ? path[k] : -1;
            int prev = __shfl_up_sync(0xffffffffu, n, 1);
            if (lane == 0) prev = before;
            before = __shfl_sync(0xffffffffu, n, 31);
            bool good = n >= 0 && n < T && n > prev && (k == 0 || prev >= 0);
            int64_t from = 0, to = 0;
            if (good) {
                const int64_t f = base + n, t = base + k;
                const int64_t fb = tab[f / p.block_size], tb = tab[t / p.block_size];
                if (fb < 0 || fb >= p.n_blocks || tb < 0 || tb >= p.n_blocks) {
                    if (blockIdx.x == 0) raise_flag(CX_DEV_BAD_BLOCK);
                    good = false;
                } else {
                    from = (fb * p.heads * p.block_size + f % p.block_size) * p.row_words;
                    to = (tb * p.heads * p.block_size + t % p.block_size) * p.row_words;
                }
            } else if (n >= 0 && blockIdx.x == 0) {
                raise_flag(CX_DEV_BAD_PATH);
            }
            s_from[lane] = from;
            s_to[lane] = to;
            const unsigned all = __ballot_sync(0xffffffffu, good);
            if (lane == 0) {
                s_n = all == 0xffffffffu ? 32 : __ffs((int)~all) - 1;   // up to the first that is not
                s_more = all == 0xffffffffu;
            }
        }
        __syncthreads();
        const int count = s_n;
        for (int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x; w < words;
             w += (int64_t)gridDim.x * 256) {
            const int plane = (int)(w / p.row_words), word = (int)(w - (int64_t)plane * p.row_words);
            const int h = plane % p.heads, pl = (plane / p.heads) % p.n_pools,
                      layer = plane / (p.heads * p.n_pools);
            // word offset of position 0 of this plane's head, in a block
            V* mem = static_cast<V*>(pl ? p.pool[1] : p.pool[0]) + layer * p.layer_words +
                     (int64_t)h * p.block_size * p.row_words + word;
            for (int i0 = 0; i0 < count; i0 += 8) {
                V x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i0 + i < count && s_from[i0 + i] != s_to[i0 + i]) x[i] = mem[s_from[i0 + i]];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i0 + i < count && s_from[i0 + i] != s_to[i0 + i]) mem[s_to[i0 + i]] = x[i];
            }
        }
        if (!s_more) return;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int check_latent_pool(const cx_latent_pool* p) {
    if (!p) return fail(CX_ERR_SHAPE, "latent pool is NULL");
    if (!p->kv) return fail(CX_ERR_SHAPE, "latent pool buffer is NULL");
    if (p->n_layers <= 0 || p->n_blocks <= 0 || p->block_size <= 0 || p->latent_dim <= 0 ||
        p->rope_dim <= 0)
        return fail(CX_ERR_SHAPE, "latent pool sizes must be positive");
    if (p->rope_dim % 2 != 0) return fail(CX_ERR_SHAPE, "latent pool: rope_dim must be even");
    if (p->latent_dim > kLatMaxLatent || p->latent_dim + p->rope_dim > kLatMaxDim)
        return fail(CX_ERR_UNSUPPORTED,
                    "latent pool: latent_dim above 512 or latent_dim + rope_dim above 576");
    if (p->n_blocks > INT32_MAX || p->block_size > (1 << 24) ||
        p->n_layers * p->n_blocks > INT32_MAX)
        return fail(CX_ERR_UNSUPPORTED, "latent pool: too many blocks");
    if (elem_bytes(p->dtype) == 0) return fail(CX_ERR_DTYPE, "unknown latent pool dtype");
    return CX_OK;
}

static int latent_append(const cx_latent_pool* pool, int64_t layer, const cx_latent_rows* rows,
                         const int64_t* slots, const int64_t* positions,
                         const cx_norm_rope* how, void* q_out, int32_t q_out_dtype,
                         cudaStream_t st) {
    const char* me = "cx_latent_append: ";
    auto bad = [&](int code, const char* what) { return fail(code, std::string(me) + what); };
    int rc = check_latent_pool(pool);
    if (rc) return rc;
    if (layer < 0 || layer >= pool->n_layers) return bad(CX_ERR_RANGE, "layer out of range");
    if (!rows || !how) return bad(CX_ERR_SHAPE, "NULL rows or how");
    if (rows->n_tokens < 0 || rows->n_q_heads < 0)
        return bad(CX_ERR_SHAPE, "negative token or head count");
    if (rows->n_tokens > INT32_MAX || rows->n_q_heads > (1 << 20))
        return bad(CX_ERR_UNSUPPORTED, "too many tokens or heads");
    const int src = elem_bytes(rows->dtype);
    if (src == 0) return bad(CX_ERR_DTYPE, "unknown row type");
    const bool has_q = rows->n_q_heads > 0;
    if (has_q && elem_bytes(q_out_dtype) == 0) return bad(CX_ERR_DTYPE, "unknown output type");
    const void* weight = how->k_weight;
    if (weight && how->k_weight_dtype != CX_F32 && how->k_weight_dtype != rows->dtype)
        return bad(CX_ERR_DTYPE, "weights must be float32 or the rows' type");
    if (weight && !(how->eps >= 0.f && isfinite(how->eps)))
        return bad(CX_ERR_SHAPE, "eps must be finite and >= 0");
    if (positions) {
        if (!how->cos_table || !how->sin_table || how->table_rows < 0)
            return bad(CX_ERR_SHAPE, "positions without cos / sin tables");
        if (how->rot_dim != pool->rope_dim)
            return bad(CX_ERR_SHAPE, "the tables' rot_dim must be the pool's rope_dim");
    } else if (has_q) {
        return bad(CX_ERR_SHAPE, "queries without positions");
    }
    if (rows->latent_token_stride < 0 || rows->rope_token_stride < 0 ||
        rows->q_token_stride < 0 || rows->q_head_stride < 0)
        return bad(CX_ERR_SHAPE, "negative stride");
    if (rows->n_tokens == 0) return CX_OK;
    if (!rows->latent || !rows->rope || !slots || (has_q && (!rows->q || !q_out)))
        return bad(CX_ERR_SHAPE, "NULL array");
    LatAppendParams p{};
    p.latent = rows->latent;
    p.rope = rows->rope;
    p.q = has_q ? rows->q : nullptr;
    p.latent_tok = rows->latent_token_stride;
    p.rope_tok = rows->rope_token_stride;
    p.q_tok = rows->q_token_stride;
    p.q_head = rows->q_head_stride;
    p.slots = slots;
    p.positions = positions;
    p.cos_table = how->cos_table;
    p.sin_table = how->sin_table;
    p.table_rows = how->table_rows;
    p.n_slots = pool->n_blocks * pool->block_size;
    p.layer_row0 = layer * p.n_slots;
    p.weight = weight;
    p.pool = pool->kv;
    p.q_out = q_out;
    p.n_tokens = (int)rows->n_tokens;
    p.heads = (int)rows->n_q_heads;
    p.dc = (int)pool->latent_dim;
    p.dr = (int)pool->rope_dim;
    p.dtype = rows->dtype;
    p.pool_dtype = pool->dtype;
    p.weight_dtype = how->k_weight_dtype;
    p.q_out_dtype = q_out_dtype;
    p.interleaved = how->interleaved != 0;
    p.eps = how->eps;
    // 16-byte rows on both sides, and heads of 8, 16 .. 256 pairs, so that a warp's lanes
    // keep their units
    const int units = p.dr / 16;
    auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    const uintptr_t bytes = al(p.latent) | al(p.rope) | al(p.pool) | al(weight) |
                            (positions ? al(p.cos_table) | al(p.sin_table) : 0) |
                            (uintptr_t)(p.latent_tok * src) | (uintptr_t)(p.rope_tok * src) |
                            (has_q ? al(p.q) | al(q_out) | (uintptr_t)(p.q_tok * src) |
                                         (uintptr_t)(p.q_head * src)
                                   : 0);
    const bool vec = (bytes & 15) == 0 && p.dc % 8 == 0 && p.dr % 16 == 0 && 32 % units == 0;
    if (vec) {
        const int per_warp = 32 / units;
        const int per_q = per_warp * kLaHeads;
        const int warps = !has_q ? 1 : std::min(kLaWarps, 1 + (p.heads + per_q - 1) / per_q);
        const unsigned n = (unsigned)p.n_tokens;
        if (p.dtype == CX_F32)
            latent_append_vec_kernel<float><<<n, warps * 32, 0, st>>>(p);
        else if (p.dtype == CX_BF16)
            latent_append_vec_kernel<__nv_bfloat16><<<n, warps * 32, 0, st>>>(p);
        else
            latent_append_vec_kernel<__half><<<n, warps * 32, 0, st>>>(p);
        return check_launch("latent_append_vec_kernel");
    }
    latent_append_kernel<<<(unsigned)p.n_tokens, 128, 0, st>>>(p);
    return check_launch("latent_append_kernel");
}

static int accept_paths(AcceptParams p, int64_t batch, int64_t row_bytes, int64_t layers,
                        uintptr_t align, cudaStream_t st) {
    align |= (uintptr_t)row_bytes;
    const int v = (align & 15) == 0 ? 16 : (align & 7) == 0 ? 8 : (align & 3) == 0 ? 4 : 2;
    p.row_words = (int)(row_bytes / v);
    p.layer_words = p.n_blocks * p.heads * p.block_size * p.row_words;
    const int64_t planes = layers * p.n_pools * p.heads;
    // (about eight CTAs an SM in all)
    const int64_t most = (planes * p.row_words + 255) / 256, fair = 8ll * num_sms() / batch;
    const int64_t blocks = std::max<int64_t>(1, std::min(most, fair));
    if (planes > INT32_MAX || blocks > INT32_MAX || batch > 65535)
        return fail(CX_ERR_UNSUPPORTED, "accepted paths: pool or batch too large");
    p.planes = (int)planes;
    const dim3 grid((unsigned)blocks, (unsigned)batch);
    switch (v) {
        case 16: accept_kernel<uint4><<<grid, 256, 0, st>>>(p); break;
        case 8: accept_kernel<uint2><<<grid, 256, 0, st>>>(p); break;
        case 4: accept_kernel<uint32_t><<<grid, 256, 0, st>>>(p); break;
        default: accept_kernel<uint16_t><<<grid, 256, 0, st>>>(p);
    }
    return check_launch("accept_kernel");
}

// The batch half of cx_kv_accept / cx_latent_accept; 1: nothing to do.
static int accept_setup(AcceptParams& p, const char* me, const cx_attn_batch* b,
                        const int32_t* paths, int64_t path_stride, int64_t path_len) {
    auto bad = [&](int code, const char* what) { return fail(code, std::string(me) + what); };
    if (!b) return bad(CX_ERR_SHAPE, "NULL batch");
    if (b->batch < 0 || path_len < 0 || path_stride < path_len)
        return bad(CX_ERR_SHAPE, "negative sizes or path_stride below path_len");
    if (b->batch == 0 || path_len == 0) return -1;
    if (!b->block_tables || !b->ctx_lens || b->table_stride <= 0 || !paths)
        return bad(CX_ERR_SHAPE, "NULL array or empty table");
    p.tables = b->block_tables;
    p.table_stride = b->table_stride;
    p.ctx_lens = b->ctx_lens;
    p.q_start = b->q_start;
    p.paths = paths;
    p.path_stride = path_stride;
    p.path_len = path_len;
    return CX_OK;
}

}  // namespace cx

extern "C" {

int cx_kv_accept(const cx_pool* pool, const cx_attn_batch* batch, const int32_t* paths,
                 int64_t path_stride, int64_t path_len, void* stream) {
    using namespace cx;
    int rc = check_pool(pool);
    if (rc) return rc;
    AcceptParams p{};
    rc = accept_setup(p, "cx_kv_accept: ", batch, paths, path_stride, path_len);
    if (rc) return rc < 0 ? CX_OK : rc;
    if (pool->block_size > (1 << 24) || pool->n_kv_heads > (1 << 20) || pool->head_dim > (1 << 20))
        return fail(CX_ERR_UNSUPPORTED, "cx_kv_accept: pool too large");
    p.pool[0] = pool->k;
    p.pool[1] = pool->v;
    p.n_pools = 2;
    p.n_blocks = pool->n_blocks;
    p.block_size = (int)pool->block_size;
    p.heads = (int)pool->n_kv_heads;
    return accept_paths(p, batch->batch, pool->head_dim * elem_bytes(pool->dtype), pool->n_layers,
                        reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v),
                        as_stream(stream));
}

int cx_latent_accept(const cx_latent_pool* pool, const cx_attn_batch* batch, const int32_t* paths,
                     int64_t path_stride, int64_t path_len, void* stream) {
    using namespace cx;
    int rc = check_latent_pool(pool);
    if (rc) return rc;
    AcceptParams p{};
    rc = accept_setup(p, "cx_latent_accept: ", batch, paths, path_stride, path_len);
    if (rc) return rc < 0 ? CX_OK : rc;
    p.pool[0] = pool->kv;
    p.n_pools = 1;
    p.n_blocks = pool->n_blocks;
    p.block_size = (int)pool->block_size;
    p.heads = 1;
    return accept_paths(p, batch->batch,
                        (pool->latent_dim + pool->rope_dim) * elem_bytes(pool->dtype),
                        pool->n_layers, reinterpret_cast<uintptr_t>(pool->kv), as_stream(stream));
}

int cx_latent_append(const cx_latent_pool* pool, int64_t layer, const cx_latent_rows* rows,
                     const int64_t* slot_mapping, const int64_t* positions,
                     const cx_norm_rope* how, void* q_out, int32_t q_out_dtype, void* stream) {
    return cx::latent_append(pool, layer, rows, slot_mapping, positions, how, q_out, q_out_dtype,
                             cx::as_stream(stream));
}

int cx_latent_gather(const cx_latent_pool* pool, int64_t layer, const int32_t* block_table,
                     int64_t n_tokens, void* latent_out, void* rope_out, void* stream) {
    using namespace cx;
    int rc = check_latent_pool(pool);
    if (rc) return rc;
    if (layer < 0 || layer >= pool->n_layers)
        return fail(CX_ERR_RANGE, "cx_latent_gather: layer out of range");
    if (n_tokens < 0) return fail(CX_ERR_SHAPE, "cx_latent_gather: negative token count");
    if (n_tokens == 0) return CX_OK;
    if (!block_table || !latent_out || !rope_out)
        return fail(CX_ERR_SHAPE, "cx_latent_gather: NULL array");
    if (n_tokens > INT32_MAX)
        return fail(CX_ERR_UNSUPPORTED, "cx_latent_gather: too many tokens");
    const int64_t row0 = layer * pool->n_blocks * pool->block_size;
    const int bs = (int)pool->block_size, dc = (int)pool->latent_dim, dr = (int)pool->rope_dim;
    cudaStream_t st = as_stream(stream);
    auto go = [&](auto e) {
        using E = decltype(e);
        latent_gather_kernel<E><<<(unsigned)n_tokens, 128, 0, st>>>(
            static_cast<const E*>(pool->kv), row0, pool->n_blocks, bs, block_table, n_tokens, dc,
            dr, static_cast<E*>(latent_out), static_cast<E*>(rope_out));
    };
    if (pool->dtype == CX_F32)
        go(uint32_t{});
    else
        go(uint16_t{});
    return check_launch("latent_gather_kernel");
}

int cx_latent_block_copy(const cx_latent_pool* pool, int64_t layer, const int32_t* src,
                         const int32_t* dst, const int32_t* n_valid, int64_t n, int64_t n_slots,
                         void* stream) {
    using namespace cx;
    int rc = check_latent_pool(pool);
    if (rc) return rc;
    if (layer >= pool->n_layers)
        return fail(CX_ERR_RANGE, "cx_latent_block_copy: layer out of range");
    if (n < 0 || n_slots < 0 || n_slots > pool->block_size)
        return fail(CX_ERR_SHAPE, "cx_latent_block_copy: negative count or too many slots");
    if (n == 0) return CX_OK;
    if (!src || !dst) return fail(CX_ERR_SHAPE, "cx_latent_block_copy: NULL array");
    const int64_t layers = layer < 0 ? pool->n_layers : 1;
    if (n > INT32_MAX || layers > 65535)
        return fail(CX_ERR_UNSUPPORTED, "cx_latent_block_copy: too many blocks or layers");
    const int64_t row = (pool->latent_dim + pool->rope_dim) * elem_bytes(pool->dtype);
    const uintptr_t al = reinterpret_cast<uintptr_t>(pool->kv) | (uintptr_t)row;
    const dim3 grid((unsigned)n, (unsigned)layers);
    cudaStream_t st = as_stream(stream);
    auto go = [&](auto e) {
        using V = decltype(e);
        const int64_t rw = row / (int64_t)sizeof(V), bw = rw * pool->block_size;
        latent_copy_kernel<V><<<grid, 256, 0, st>>>(
            static_cast<V*>(pool->kv), bw * pool->n_blocks, bw, rw, pool->n_blocks,
            layer < 0 ? 0 : layer, src, dst, n_valid, n_slots, pool->block_size);
    };
    if ((al & 15) == 0)
        go(uint4{});
    else if ((al & 3) == 0)
        go(uint32_t{});
    else
        go(uint16_t{});
    return check_launch("latent_copy_kernel");
}

}  // extern "C"
