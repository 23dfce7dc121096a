// Attention over a latent cache on CUDA cores, fp32 throughout: fp32 pools, block
// sizes other than 16, 32 and 64, rows that TMA cannot load.
//
// A warp takes 2 or 4 neighbouring keys of its CTA's part of the context at a time and
// holds 4 packed rows' queries and outputs in registers, one element in 32 a lane: a
// key's row is read once, from global memory, and serves the score and the output.  Four
// dot products are summed over the lanes with 6 + 4 shuffles.  The four warps, and
// the parts of a context that is split over CTAs, are joined by their maxima.
// 4 sequences of up to 1,024 fp32 keys of 128 + 32, 8 heads: one key at a time 29 us and
// 27 to join its parts, 16 and 10 with four and the parts' references side by side.
#pragma once

#include "latent_attn_tc.cuh"

namespace cx {

constexpr int kLgRows = 4, kLgWarps = 4;

struct LatGenParams {
    LatParams a;
    const void* pool;
    int64_t n_blocks64, layer64;
    int32_t n_split, row_tiles;
    float scale;
    float* part;              // [unit][split][4][dc + 2]
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
                const float w = expf(s[j][r] - top);
                l[r] += w;
#pragma unroll
                for (int e = 0; e < KE; ++e) o[r][e] = fmaf(w, x[j][e], o[r][e]);
            }
        }
    }
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
        for (int w = 0; M != -INFINITY && w < kLgWarps; ++w) {
            const float f = expf(src[w * step + p.dc] - M);
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
            store_as(p.out, p.out_dtype, (row0 + r) * p.dc + d, L > 0.f ? O / L : 0.f);
        }
    }
}

// Joins the parts of a context that was split: one CTA per row.  Lanes fetch the parts'
// references side by side; there are at most 256.
__global__ void __launch_bounds__(128) latent_generic_join(const LatGenParams g) {
    const LatParams& p = g.a;
    const int unit = (int)blockIdx.x, b = unit / g.row_tiles, rt = unit - b * g.row_tiles;
    const int r = blockIdx.y, lane = threadIdx.x & 31;
    const int qs = p.q_start ? p.q_start[b] : b;
    const int T = p.q_start ? min(max(p.q_start[b + 1] - qs, 0), p.max_q) : 1;
    const int r0 = rt * kLgRows;
    if (r0 + r >= T * p.heads) return;
    const int mrow = p.dc + 2;
    const float* src = g.part + ((int64_t)unit * g.n_split * kLgRows + r) * mrow;
    const int64_t step = (int64_t)kLgRows * mrow;
    __shared__ float s_f[256];
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < g.n_split; s += 32) M = fmaxf(M, src[s * step + p.dc]);
#pragma unroll
    for (int w = 16; w; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    for (int s = lane; s < g.n_split; s += 32) {
        const float f = M == -INFINITY ? 0.f : expf(src[s * step + p.dc] - M);
        L = fmaf(src[s * step + p.dc + 1], f, L);
        if (threadIdx.x < 32) s_f[s] = f;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
    __syncthreads();
    for (int d = threadIdx.x; d < p.dc; d += 128) {
        float O = 0.f;
#pragma unroll 8
        for (int s = 0; s < g.n_split; ++s) O = fmaf(src[s * step + d], s_f[s], O);
        store_as(p.out, p.out_dtype, ((int64_t)qs * p.heads + r0 + r) * p.dc + d,
                 L > 0.f ? O / L : 0.f);
    }
}

template <typename KT>
static int launch_latent_generic(const LatGenParams& g, cudaStream_t st) {
    const int64_t units = (int64_t)g.a.batch * g.row_tiles;
    if (units <= 0) return CX_OK;
    const size_t smem = (size_t)kLgWarps * kLgRows * (g.a.dc + 2) * 4;
    const dim3 grid((unsigned)units, (unsigned)g.n_split);
    if (g.a.dim <= 192)
        latent_generic_kernel<KT, 6><<<grid, kLgWarps * 32, smem, st>>>(g);
    else if (g.a.dim <= 320)
        latent_generic_kernel<KT, 10><<<grid, kLgWarps * 32, smem, st>>>(g);
    else
        latent_generic_kernel<KT, 18><<<grid, kLgWarps * 32, smem, st>>>(g);
    int rc = check_launch("latent_generic_kernel");
    if (rc || g.n_split == 1) return rc;
    latent_generic_join<<<dim3((unsigned)units, kLgRows), 128, 0, st>>>(g);
    return check_launch("latent_generic_join");
}

}  // namespace cx
