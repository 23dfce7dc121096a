// Attention over a latent cache on CUDA cores, fp32 throughout: fp32 pools, block
// sizes that are no multiple of 8, rows that TMA cannot load.  Two kernels:
//
// latent_generic_kernel, up to 16 rows (query token x head) of a sequence: a warp takes 2
// or 4 neighbouring keys of its CTA's part of the context at a time and holds 4 packed
// rows' queries and outputs in registers, one element in 32 a lane: a key's row is
// read once, from global memory, and serves the score and the output.  Four dot products
// are summed over the lanes with 6 + 4 shuffles.  4 sequences of up to 1,024 fp32 keys
// of 128 + 32, 8 heads: one key at a time 29 us and 27 to join its parts, 16 and 10 with
// four and the parts' references side by side.
//
// latent_rows_kernel, more rows: 32 rows share tiles of 32 keys in shared memory, two
// in turn.  A warp has 4 rows: a lane's key against them for the scores (a query
// element is one broadcast read), a lane's columns of every key for the outputs.  It
// is bound by shared memory (in passes of 128 bytes a warp: 8 for 16 products a lane of the
// scores, 17 for 64 of the outputs of 512) and by one CTA an SM: 14 TFLOP/s for 62 tokens of 64 heads behind 1,200
// keys of 384 + 64, 558 us.
//
// Parts of a context that is split over CTAs are joined by their maxima.
#pragma once

#include "latent_attn_tc.cuh"

namespace cx {

constexpr int kLgRows = 4, kLgWarps = 4;
constexpr int kLrRows = 32, kLrKeys = 32, kLrWarps = 8;

struct LatGenParams {
    LatParams a;
    const void* pool;
    int64_t n_blocks64, layer64;
    int32_t n_split, row_tiles;
    int32_t unit_rows;        // rows of a unit: kLgRows or kLrRows
    float scale;
    float* part;              // [unit][split][unit_rows][dc + 2]
};

// Sums of a[0 .. 3] over the warp, in every lane.
__device__ __forceinline__ void warp_sum4(float (&a)[4], int lane) {
    const bool up = lane & 16, mid = lane & 8;
    float x = up ? a[2] : a[0], y = up ? a[3] : a[1];
    x += __shfl_xor_sync(0xffffffffu, up ? a[0] : a[2], 16);
    y += __shfl_xor_sync(0xffffffffu, up ? a[1] : a[3], 16);
    float z = mid ? y : x;
    z += __shfl_xor_sync(0xffffffffu, mid ? x : y, 8);
    z += __shfl_xor_sync(0xffffffffu, z, 4);
    z += __shfl_xor_sync(0xffffffffu, z, 2);
    z += __shfl_xor_sync(0xffffffffu, z, 1);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = __shfl_sync(0xffffffffu, z, r * 8);
}

template <typename KT, int KE>
__global__ void __launch_bounds__(kLgWarps * 32) latent_generic_kernel(const LatGenParams g) {
    const LatParams& p = g.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit = (int)blockIdx.x, b = unit / g.row_tiles, rt = unit - b * g.row_tiles;
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T_raw = p.q_start ? p.q_start[b + 1] - qs : 1;
    const int T = min(max(T_raw, 0), p.max_q);
    const int raw = p.ctx_lens[b];
    const int64_t cap = p.table_stride * p.block_size;
    const int ctx = (int)min((int64_t)max(raw, 0), cap), base = ctx - T;
    if (rt == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        if (raw > cap) raise_flag(CX_DEV_TABLE_OVERRUN);
        if (T != T_raw || (raw > 0 && T > ctx)) raise_flag(CX_DEV_BAD_QLEN);
    }
    const int rows = T * p.heads, r0 = rt * kLgRows, nr = min(kLgRows, rows - r0);
    if (nr <= 0) return;

    // ---- queries, each row's plain run [lo, up], its last node ----
    float q[kLgRows][KE];
    int lo[kLgRows], up[kLgRows], last[kLgRows];
    int lo_all = ctx, hi_all = -1;
#pragma unroll
    for (int r = 0; r < kLgRows; ++r) {
        lo[r] = 0;
        up[r] = last[r] = -1;
#pragma unroll
        for (int e = 0; e < KE; ++e) q[r][e] = 0.f;
        if (r >= nr) continue;
        const int t = (r0 + r) / p.heads, h = (r0 + r) - t * p.heads;
        const int64_t ql = (qs + t) * p.ql_tok + h * p.ql_head;
        const int64_t qr = (qs + t) * p.qr_tok + h * p.qr_head;
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            const int d = lane + 32 * e;
            if (d >= p.dim) continue;
            const void* s = d < p.dc ? p.q_lat : p.q_rope;
            const int64_t i = d < p.dc ? ql + d : qr + d - p.dc;
            q[r][e] = p.q_dtype == CX_F32    ? static_cast<const float*>(s)[i]
                      : p.q_dtype == CX_BF16 ? __bfloat162float(
                                                   static_cast<const __nv_bfloat16*>(s)[i])
                                             : __half2float(static_cast<const __half*>(s)[i]);
        }
        int pos = base + t;
        last[r] = up[r] = pos;
        if (p.tree.masks) {
            pos = base + p.tree.depths[qs + t];
            up[r] = base - 1;
        }
        if (p.window > 0) lo[r] = max(0, pos - p.window + 1);
        lo_all = min(lo_all, p.tree.masks ? min(lo[r], max(base, 0)) : lo[r]);
        hi_all = max(hi_all, last[r]);
    }
    hi_all = min(hi_all, ctx - 1);
    // this CTA's keys
    const int n_keys = max(0, hi_all - lo_all + 1);
    const int per = (n_keys + g.n_split - 1) / g.n_split;
    const int k_lo = lo_all + (int)blockIdx.y * per, k_hi = min(hi_all + 1, k_lo + per);

    float o[kLgRows][KE], m[kLgRows], l[kLgRows];
#pragma unroll
    for (int r = 0; r < kLgRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < KE; ++e) o[r][e] = 0.f;
    }
    const int32_t* tab = p.tables + (int64_t)b * p.table_stride;
    const KT* pool = static_cast<const KT*>(g.pool);
    // the row of key k (nullptr: a bad block)
    auto row_of = [&](int k) -> const KT* {
        const int blk = k / p.block_size, id = tab[blk];
        if (id < 0 || id >= p.n_blocks) {
            if (lane == 0) raise_flag(CX_DEV_BAD_BLOCK);
            return nullptr;
        }
        return pool + ((g.layer64 * g.n_blocks64 + id) * p.block_size + (k - blk * p.block_size)) *
                          p.dim;
    };
    constexpr int NK = KE <= 10 ? 4 : 2;
    for (int k0 = k_lo + warp * NK; k0 < k_hi; k0 += kLgWarps * NK) {
        unsigned sees[NK];                        // bit r: row r sees the key
        const KT* src[NK];
        float x[NK][KE];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int k = k0 + j;
            sees[j] = 0;
#pragma unroll
            for (int r = 0; r < kLgRows; ++r) {
                bool see = k >= lo[r] && k <= up[r];
                if (p.tree.masks && k >= base && k <= last[r]) {
                    const int t = (r0 + r) / p.heads;
                    see = tree_bits(p.tree, qs + t, t, k - base) & 1u;
                }
                if (k < k_hi && see) sees[j] |= 1u << r;
            }
            src[j] = sees[j] ? row_of(k) : nullptr;
            if (!src[j]) sees[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < KE; ++e) {
                const int d = lane + 32 * e;
                x[j][e] = sees[j] && d < p.dim ? Conv<KT>::to_f(src[j][d]) : 0.f;
            }
        float s[NK][kLgRows];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
#pragma unroll
            for (int r = 0; r < kLgRows; ++r) {
                float a0 = 0.f, a1 = 0.f;
#pragma unroll
                for (int e = 0; e < KE; e += 2) {
                    a0 = fmaf(q[r][e], x[j][e], a0);
                    if (e + 1 < KE) a1 = fmaf(q[r][e + 1], x[j][e + 1], a1);
                }
                s[j][r] = a0 + a1;
            }
            warp_sum4(s[j], lane);
        }
#pragma unroll
        for (int r = 0; r < kLgRows; ++r) {
            float top = m[r];
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                s[j][r] *= g.scale;
                if ((sees[j] >> r) & 1u) top = fmaxf(top, s[j][r]);
            }
            if (top > m[r]) {
                const float f = expf(m[r] - top);
                m[r] = top;
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < KE; ++e) o[r][e] *= f;
            }
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                if (!((sees[j] >> r) & 1u)) continue;     // adds nothing, whatever it holds
                const float w = expf(s[j][r] - ref_base(top));
                l[r] += w;
#pragma unroll
                for (int e = 0; e < KE; ++e) o[r][e] = fmaf(w, x[j][e], o[r][e]);
            }
        }
    }
    asm volatile("griddepcontrol.launch_dependents;");
    // ---- the four warps' states, then the output or this CTA's part ----
    extern __shared__ float gsm[];                // [warp][row][dc + 2]
    const int mrow = p.dc + 2;
#pragma unroll
    for (int r = 0; r < kLgRows; ++r) {
        float* dst = gsm + ((size_t)warp * kLgRows + r) * mrow;
#pragma unroll
        for (int e = 0; e < KE; ++e)
            if (lane + 32 * e < p.dc) dst[lane + 32 * e] = o[r][e];
        if (lane == 0) {
            dst[p.dc] = m[r];
            dst[p.dc + 1] = l[r];
        }
    }
    __syncthreads();
    const int64_t row0 = (int64_t)qs * p.heads + r0;
    for (int e = threadIdx.x; e < nr * p.dc; e += blockDim.x) {
        const int r = e / p.dc, d = e - r * p.dc;
        const float* src = gsm + (size_t)r * mrow;
        const size_t step = (size_t)kLgRows * mrow;
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int w = 0; w < kLgWarps; ++w) M = fmaxf(M, src[w * step + p.dc]);
        for (int w = 0; w < kLgWarps; ++w) {
            const float f = expf(src[w * step + p.dc] - ref_base(M));
            L = fmaf(src[w * step + p.dc + 1], f, L);
            O = fmaf(src[w * step + d], f, O);
        }
        if (g.n_split > 1) {
            float* dst = g.part +
                         (((int64_t)unit * g.n_split + blockIdx.y) * kLgRows + r) * mrow;
            dst[d] = O;
            if (d == 0) {
                dst[p.dc] = M;
                dst[p.dc + 1] = L;
            }
        } else {
            store_as(p.out, p.out_dtype, (row0 + r) * p.dc + d, L == 0.f ? 0.f : O / L);
        }
    }
}

// Floats between rows in shared memory: 4 modulo 32, so that eight lanes' 16-byte reads
// of their own rows meet no bank twice.
__host__ __device__ inline int latent_rows_stride(int dim) { return (dim + 31) / 32 * 32 + 4; }

template <typename KT, int NC>
__global__ void __launch_bounds__(kLrWarps * 32, 1) latent_rows_kernel(const LatGenParams g) {
    const LatParams& p = g.a;
    extern __shared__ float gsm[];                // queries, two key tiles, probabilities
    const int SD = latent_rows_stride(p.dim), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* s_q = gsm;
    float* s_k = s_q + kLrRows * SD;
    float4* s_p = reinterpret_cast<float4*>(s_k + 2 * kLrKeys * SD) + warp * kLrKeys;
    const int unit = (int)blockIdx.x, b = unit / g.row_tiles, rt = unit - b * g.row_tiles;
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T_raw = p.q_start ? p.q_start[b + 1] - qs : 1;
    const int T = min(max(T_raw, 0), p.max_q);
    const int raw = p.ctx_lens[b];
    const int64_t cap = p.table_stride * p.block_size;
    const int ctx = (int)min((int64_t)max(raw, 0), cap), base = ctx - T;
    if (rt == 0 && blockIdx.y == 0 && tid == 0) {
        if (raw > cap) raise_flag(CX_DEV_TABLE_OVERRUN);
        if (T != T_raw || (raw > 0 && T > ctx)) raise_flag(CX_DEV_BAD_QLEN);
    }
    const int rows = T * p.heads, r0 = rt * kLrRows, nr = min(kLrRows, rows - r0);
    if (nr <= 0) return;

    // ---- queries as fp32, zeros behind the width and the rows ----
    for (int r = warp; r < kLrRows; r += kLrWarps) {
        const int t = (r0 + r) / p.heads, h = (r0 + r) - t * p.heads;
        for (int d = lane; d < SD; d += 32) {
            float x = 0.f;
            if (r < nr && d < p.dim) {
                const bool in_lat = d < p.dc;
                x = load_as(in_lat ? p.q_lat : p.q_rope, p.q_dtype,
                            in_lat ? (qs + t) * p.ql_tok + h * p.ql_head + d
                                   : (qs + t) * p.qr_tok + h * p.qr_head + d - p.dc);
            }
            s_q[r * SD + d] = x;
        }
    }
    // this warp's rows: plain runs [lo, up], last nodes; the range of keys of the CTA
    const int R0 = 4 * warp;
    int lo[4], up[4], last[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        lo[r] = 0;
        up[r] = last[r] = -1;
        if (R0 + r >= nr) continue;
        const int t = (r0 + R0 + r) / p.heads;
        int pos = base + t;
        last[r] = up[r] = pos;
        if (p.tree.masks) {
            pos = base + p.tree.depths[qs + t];
            up[r] = base - 1;
        }
        if (p.window > 0) lo[r] = max(0, pos - p.window + 1);
    }
    const int t_first = r0 / p.heads, t_last = (r0 + nr - 1) / p.heads;
    const int hi_all = min(base + t_last, ctx - 1);
    const int lo_all =
        p.window > 0 ? max(0, base + (p.tree.masks ? 0 : t_first) - p.window + 1) : 0;
    const int n_keys = max(0, hi_all - lo_all + 1);
    const int per = ((n_keys + g.n_split - 1) / g.n_split + kLrKeys - 1) / kLrKeys * kLrKeys;
    const int k_lo = lo_all + (int)blockIdx.y * per, k_hi = min(hi_all + 1, k_lo + per);

    const int32_t* tab = p.tables + (int64_t)b * p.table_stride;
    const KT* pool = static_cast<const KT*>(g.pool);
    const bool async16 = sizeof(KT) == 4 && p.dim % 4 == 0 &&
                         (reinterpret_cast<uintptr_t>(g.pool) & 15) == 0;
    bool bad = false;                             // this warp's keys of the tile: a bad block
    // keys k0 .. k0 + 31 into buffer `buf`, four a warp; zeros for what is not there
    auto load = [&](int k0, int buf) {
        float* dst = s_k + (buf * kLrKeys + R0) * SD;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + R0 + i;
            const KT* src = nullptr;
            if (k < k_hi) {
                const int blk = k / p.block_size, id = tab[blk];
                if (id >= 0 && id < p.n_blocks)
                    src = pool + ((g.layer64 * g.n_blocks64 + id) * p.block_size +
                                  (k - blk * p.block_size)) * p.dim;
                else
                    bad = true;
            }
            float* row = dst + i * SD;
            if (async16) {
                for (int c = lane; c < p.dim / 4; c += 32)
                    cp_async16(row + c * 4, src ? src + c * 4 : pool, src != nullptr);
            } else {
                for (int d = lane; d < p.dim; d += 32)
                    row[d] = src ? Conv<KT>::to_f(src[d]) : 0.f;
            }
            for (int d = p.dim + lane; d < SD; d += 32) row[d] = 0.f;
        }
    };
    float o[4][4 * NC], m[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < 4 * NC; ++e) o[r][e] = 0.f;
    }
    if (k_lo < k_hi) load(k_lo, 0);
    int buf = 0;
    for (int k0 = k_lo; k0 < k_hi; k0 += kLrKeys, buf ^= 1) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();                          // the tile is there; the other buffer was read
        if (k0 + kLrKeys < k_hi) load(k0 + kLrKeys, buf ^ 1);
        // ---- scores of key k0 + lane ----
        const float4* kr = reinterpret_cast<const float4*>(s_k + (buf * kLrKeys + lane) * SD);
        const float4* qr = reinterpret_cast<const float4*>(s_q + R0 * SD);
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = 0; c < (p.dim + 3) / 4; ++c) {
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
        const int k = k0 + lane;
        bool there = k < k_hi;
        if (there) {
            const int id = tab[k / p.block_size];
            there = id >= 0 && id < p.n_blocks;
        }
        float pr[4];
        bool moved = false;
        float corr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bool see = there && k >= lo[r] && k <= up[r];
            if (p.tree.masks && there && k >= base && k <= last[r]) {
                const int t = (r0 + R0 + r) / p.heads;
                see = tree_bits(p.tree, qs + t, t, k - base) & 1u;
            }
            const float x = see ? a[r] * g.scale : -INFINITY;
            float top = x;
#pragma unroll
            for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            corr[r] = 1.f;
            if (top > m[r]) {
                corr[r] = expf(m[r] - top);
                m[r] = top;
                moved = true;
            }
            pr[r] = see ? expf(x - ref_base(m[r])) : 0.f;
            l[r] = fmaf(l[r], corr[r], pr[r]);
        }
        s_p[lane] = make_float4(pr[0], pr[1], pr[2], pr[3]);
        __syncwarp();
        if (moved) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < 4 * NC; ++e) o[r][e] *= corr[r];
        }
        // ---- columns 128 c + 4 lane of every key ----
        const float* vt = s_k + buf * kLrKeys * SD + 4 * lane;
#pragma unroll 2
        for (int j = 0; j < kLrKeys; ++j) {
            const float4 w = s_p[j];
            // (a key that none of the rows sees adds nothing, whatever it holds)
            if (w.x == 0.f && w.y == 0.f && w.z == 0.f && w.w == 0.f) continue;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float4 v = *reinterpret_cast<const float4*>(vt + j * SD + 128 * c);
                const float x[4] = {v.x, v.y, v.z, v.w}, y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[r][4 * c + e] = fmaf(y[r], x[e], o[r][4 * c + e]);
            }
        }
        __syncwarp();
    }
    asm volatile("griddepcontrol.launch_dependents;");
    if (bad && lane == 0) raise_flag(CX_DEV_BAD_BLOCK);
    const int64_t row0 = (int64_t)qs * p.heads + r0;
    const int mrow = p.dc + 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float L = l[r];
#pragma unroll
        for (int w = 16; w; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
        if (R0 + r >= nr) continue;
        float* dst = g.n_split > 1
                         ? g.part + (((int64_t)unit * g.n_split + blockIdx.y) * kLrRows + R0 + r) *
                                        mrow
                         : nullptr;
        const float inv = sum_inv(L);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 128 * c + 4 * lane + e;
                if (d >= p.dc) continue;
                if (dst)
                    dst[d] = o[r][4 * c + e];
                else
                    store_as(p.out, p.out_dtype, (row0 + R0 + r) * p.dc + d, o[r][4 * c + e] * inv);
            }
        if (dst && lane == 0) {
            dst[p.dc] = m[r];
            dst[p.dc + 1] = L;
        }
    }
}

// Joins the parts of a context that was split: one CTA per row.  Lanes fetch the parts'
// references side by side; there are at most 256.
__global__ void __launch_bounds__(128) latent_generic_join(const LatGenParams g) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const LatParams& p = g.a;
    const int unit = (int)blockIdx.x, b = unit / g.row_tiles, rt = unit - b * g.row_tiles;
    const int r = blockIdx.y, lane = threadIdx.x & 31;
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T = p.q_start ? min(max(p.q_start[b + 1] - qs, 0), p.max_q) : 1;
    const int r0 = rt * g.unit_rows;
    if (r0 + r >= T * p.heads) return;
    const int mrow = p.dc + 2;
    const float* src = g.part + ((int64_t)unit * g.n_split * g.unit_rows + r) * mrow;
    const int64_t step = (int64_t)g.unit_rows * mrow;
    __shared__ float s_f[256];
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < g.n_split; s += 32) M = fmaxf(M, src[s * step + p.dc]);
#pragma unroll
    for (int w = 16; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    for (int s = lane; s < g.n_split; s += 32) {
        const float f = expf(src[s * step + p.dc] - ref_base(M));
        L = fmaf(src[s * step + p.dc + 1], f, L);
        if (threadIdx.x < 32) s_f[s] = f;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
    __syncthreads();
    for (int d = threadIdx.x; d < p.dc; d += 128) {
        float O = 0.f;
        // (the branch around the loop: with a choice behind it 4 x 1k tokens took 20 us, not 16)
        if (L != 0.f) {
#pragma unroll 8
            for (int s = 0; s < g.n_split; ++s) O = fmaf(src[s * step + d], s_f[s], O);
            O /= L;
        }
        store_as(p.out, p.out_dtype, ((int64_t)qs * p.heads + r0 + r) * p.dc + d, O);
    }
}

static int launch_latent_generic_join(const LatGenParams& g, int64_t units, cudaStream_t st) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)units, g.unit_rows);
    cfg.blockDim = 128;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, latent_generic_join, g));
    return check_launch("latent_generic_join");
}

template <typename KT>
static int launch_latent_generic(const LatGenParams& g, cudaStream_t st) {
    const int64_t units = (int64_t)g.a.batch * g.row_tiles;
    if (units <= 0) return CX_OK;
    const size_t smem = (size_t)kLgWarps * kLgRows * (g.a.dc + 2) * 4;
    const dim3 grid((unsigned)units, (unsigned)g.n_split);
    if (g.unit_rows == kLrRows) {
        // (behind the last key's row the outputs' reads may go on into the probabilities)
        const int sd = latent_rows_stride(g.a.dim);
        const int bytes = (kLrRows + 2 * kLrKeys) * sd * 4 + kLrWarps * kLrKeys * 16;
        auto go = [&](auto kern) {
            CX_CUDA_CHECK(
                cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
            kern<<<grid, kLrWarps * 32, bytes, st>>>(g);
            return check_launch("latent_rows_kernel");
        };
        const int nc = (g.a.dc + 127) / 128;
        const int rc = nc == 1   ? go(latent_rows_kernel<KT, 1>)
                       : nc == 2 ? go(latent_rows_kernel<KT, 2>)
                       : nc == 3 ? go(latent_rows_kernel<KT, 3>)
                                 : go(latent_rows_kernel<KT, 4>);
        if (rc || g.n_split == 1) return rc;
        return launch_latent_generic_join(g, units, st);
    }
    if (g.a.dim <= 192)
        latent_generic_kernel<KT, 6><<<grid, kLgWarps * 32, smem, st>>>(g);
    else if (g.a.dim <= 320)
        latent_generic_kernel<KT, 10><<<grid, kLgWarps * 32, smem, st>>>(g);
    else
        latent_generic_kernel<KT, 18><<<grid, kLgWarps * 32, smem, st>>>(g);
    int rc = check_launch("latent_generic_kernel");
    if (rc || g.n_split == 1) return rc;
    return launch_latent_generic_join(g, units, st);
}

}  // namespace cx
