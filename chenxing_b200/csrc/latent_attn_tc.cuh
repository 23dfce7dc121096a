// Attention over a latent cache on tcgen05, absorbed form: one row a token,
// [latent (dc) | rotated shared key part (dr)], is the key of every query head and
// its latent part is their value.
//
//     s[t, h, j] = scale * (q_latent[t, h] . c[j] + q_rope[t, h] . r[j])
//     o[t, h]    = sum_j softmax_j(s[t, h, :])[j] c[j]
//
// Packed rows (row = query token x head) are cut into tiles of N = 16, 32 or 64.
// Both products run transposed, so that the tile of keys is the M operand, any
// number of rows is the N operand, and one copy of the keys in shared memory
// serves both:
//
//     S^T (64 keys x N)  = C (64 x dim, K-major)   . Q^T   (N x dim, K-major)
//     O^T (dc   x N)    += C^T (dc x 64, MN-major) . P^T   (N x 64, MN-major)
//
// O^T takes 4 N TMEM columns (dc <= 512: four tiles of 128 lanes), S^T two buffers
// of N.  With the rows as M, 512 value columns would fill the TMEM and leave S no
// room, and 16 rows (16 heads, one token) would run MMAs of 128.
//
// A CTA has a contiguous run of the batch's 64-key tiles, which are dealt out evenly
// over the CTAs (every CTA works its share out from the lengths); a (sequence, row
// tile) that is cut is joined by latent_join_kernel.  Roles:
//
//   4 or 8 warps: softmax of a tile's 64 keys (16 keys and all or half of the rows a
//              warp), Q tiles in, output out.
//   2 warps  : issue the MMAs: one S^T of a tile piece by piece as it arrives, up to two
//              tiles ahead, the other O^T.  (One warp that polled for whichever could run
//              took 150 to 350 cycles to see either.)
//   2 warps  : producers, one for either chunk of a piece.  A tile is [64-column chunk]
//              [64 keys][128 bytes] (128-byte swizzle) and arrives in pieces of two
//              chunks, which O^T's MMAs free one after the other; a TMA box is a block's
//              rows of a chunk.  (Boxes of 16 rows of a chunk take the SM's TMA unit 25
//              cycles; 8 rows of two chunks in one box, 2 KB as well, 72, and of nine
//              113.)  Blocks past the sequence and ids outside the pool are read outside
//              the tensor map, which fills zeros.
//
// The reference of a row's exponentials follows its maximum as in the kernels beside
// this one (Half16), so that a tile nearly always needs one pass and one vote.
// Tiles that some row sees only in part are masked by one 64-bit word a row, which
// also holds the nodes that a row of a drafted tree sees; keys that no row of
// the CTA sees are zeroed in shared memory first (0 * NaN is NaN).
// Every wait is bounded.
#pragma once

#include "attn_prefill_tc.cuh"
#include "tma_map.cuh"

namespace cx {

constexpr int kLatKeys = 64;          // keys per tile
constexpr int kLatMaxDim = 576;       // latent + rotary part
constexpr int kLatMaxLatent = 512;
constexpr int kLatChunk = kLatKeys * 128;      // 64 columns of a tile
constexpr int kLatP = kLatKeys * 128;          // P^T: a line of up to 64 rows per key
constexpr int kLatProd = 2;                   // producer warps
constexpr int kLatMaxStages = 4;
constexpr int kLatMaxPieces = (kLatMaxDim + 127) / 128;
constexpr int kLatMinTiles = 4;       // cost (in tiles) of a CTA before another starts

// What a range costs its CTA beside its tiles (output, first tile), in tiles.  With
// shares of equal tiles the CTAs that two ranges meet in took 72 us where the others
// took 66 (64 x 8k tokens, 16 heads).  In time it is about the same for all widths, and a
// tile's time goes with its width: 5 tiles of 576 columns (3: 70.0, 5: 69.5, 7: 70.4 us), 9
// of 320 (trees over latents of 256 + 64, 3: 78, 5: 72, 9: 69).
static int lat_range_cost(int dim) {
    const int c = 2880 / dim;
    return c < 4 ? 4 : c > 12 ? 12 : c;
}

struct LatParams {
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* ctx_lens;
    const int32_t* q_start;     // NULL: one query token per sequence
    TreeMask tree;
    const void* q_lat;
    const void* q_rope;
    int64_t ql_tok, ql_head, qr_tok, qr_head;
    void* out;                  // [rows][heads][dc]
    float* part_o;              // [CTA][2][N][dc]
    float* part_ml;             // [CTA][2][N][2]
    int32_t* desc;              // [CTA][8] the range that a CTA's last partial opens
    int32_t batch, heads, max_q, rtiles, sub, n_units;
    int32_t n_blocks, block_size, layer, window, dc, dim;
    int32_t q_dtype, out_dtype, q_vec;
    int32_t stages;             // tiles in shared memory
    int32_t box_rows, range_cost;
    float scale_log2;
    uint32_t tries;             // of a wait
};

// One (sequence, row tile) and its key tiles.
struct LatUnit {
    int b, T, qs, ctx, base;    // base: committed tokens (ctx - T)
    int r0, n_rows;             // packed rows [r0, r0 + n_rows) of the sequence
    int tile0, n_tiles;         // of the `sub` row tiles that run side by side
    __device__ __forceinline__ int cost(const LatParams& p) const {
        return n_tiles > 0 ? n_tiles + p.range_cost : 0;
    }
};

__device__ __forceinline__ LatUnit lat_unit(const LatParams& p, int u, int sub_id, int N) {
    const int per_seq = (p.rtiles + p.sub - 1) / p.sub;
    LatUnit x;
    x.b = u / per_seq;
    const int s = u - x.b * per_seq;
    x.qs = p.q_start ? p.q_start[x.b] : x.b;
    x.T = p.q_start ? min(max(p.q_start[x.b + 1] - x.qs, 0), p.max_q) : 1;
    x.ctx = (int)min((int64_t)max(p.ctx_lens[x.b], 0), p.table_stride * p.block_size);
    x.base = x.ctx - x.T;
    const int rows = x.T * p.heads, first = s * p.sub * N, end = min(rows, first + p.sub * N);
    x.r0 = first + sub_id * N;
    x.n_rows = min(max(rows - x.r0, 0), N);
    x.tile0 = x.n_tiles = 0;
    if (end <= first || x.ctx == 0) return x;
    const int hi = min(x.ctx - 1, x.base + (end - 1) / p.heads);
    int lo = 0;
    if (p.window > 0) lo = max(0, x.base + (p.tree.masks ? 0 : first / p.heads) - p.window + 1);
    if (hi >= lo) x.tile0 = lo / kLatKeys;
    x.n_tiles = hi >= lo ? hi / kLatKeys - x.tile0 + 1 : 1;
    return x;
}

// A run of tiles of one unit.  Shares are counted in cost: a unit's first range_cost
// are no tiles.
struct LatSeg {
    LatUnit x;
    int from, to;
    __device__ __forceinline__ bool whole() const { return from == 0 && to == x.n_tiles; }
};

struct LatCursor {
    int u, off, left;
    __device__ __forceinline__ bool next(const LatParams& p, int sub_id, int N, LatSeg& s) {
        while (left > 0 && u < p.n_units) {
            s.x = lat_unit(p, u, sub_id, N);
            const int take = min(left, s.x.cost(p) - off);
            s.from = max(off - p.range_cost, 0);
            s.to = off + take - p.range_cost;
            left -= max(take, 0);
            ++u;
            off = 0;
            // (a side-by-side tile past the rows: none)
            if (s.to > s.from && s.x.n_rows > 0) return true;
        }
        return false;
    }
};

// Bytes of a tile in shared memory: its chunks, and as many as O^T's MMAs of 128
// columns read.
__host__ __device__ inline int lat_stage(int dc, int dim) {
    const int nch = (dim + 63) / 64, read = (dc + 127) / 128 * 2;
    return (nch > read ? nch : read) * kLatChunk;
}

template <int N>
struct LatCfg {
    // softmax warps: rows of 64 in two halves, so that a tile takes half as long (the way
    // from S^T to P^T is part of what a tile in shared memory waits for: 163 us for 32 x
    // 16k tokens of 128 heads with four warps)
    static constexpr int SW = N == 64 ? 8 : 4;
    static constexpr int ST = SW * 32;
    static constexpr int NW = N / (SW / 4);       // rows of a warp
    static constexpr int THREADS = (SW + 2 + kLatProd) * 32;
    static constexpr int Q_CHUNK = N * 128;
    static constexpr int MISC = 2048;
    static constexpr int TMEM_COLS = 512;
    static constexpr int S_COL = 4 * N;
    __host__ static void ring(int dc, int dim, int& stages, int& smem) {
        const int nch = (dim + 63) / 64, stage = lat_stage(dc, dim);
        const int fixed = 1024 + nch * Q_CHUNK + kLatP + MISC;
        stages = (232448 - fixed) / stage;
        if (stages > kLatMaxStages) stages = kLatMaxStages;
        smem = fixed + stages * stage;
        // above half of the SM's shared memory: one CTA an SM, which owns the TMEM
        if (smem < 117 * 1024) smem = 117 * 1024;
    }
};

// OR of `pred` over the `nthreads` threads that meet at named barrier `id`.
__device__ __forceinline__ bool bar_red_or(int id, int nthreads, bool pred) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "bar.red.or.pred p, %1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(nthreads), "r"((uint32_t)pred)
        : "memory");
    return r != 0;
}

// N columns of 16 TMEM lanes: v[4 j + e] is lane `lane / 4 + 8 (e / 2)`, column
// 8 j + 2 (lane % 4) + e % 2.
template <int N>
__device__ __forceinline__ void lat_ld_s(uint32_t taddr, float (&v)[N / 2]) {
    uint32_t r[N / 2];
    if constexpr (N == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
              "=r"(r[6]), "=r"(r[7])
            : "r"(taddr));
    } else if constexpr (N == 32) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
              "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
              "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
            "[%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
              "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
              "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
              "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
              "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
              "=r"(r[30]), "=r"(r[31])
            : "r"(taddr));
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = __uint_as_float(r[i]);
}

// 64-bit word with bits [a, b) set, 0 <= a, b <= 64 (none when b <= a).
__device__ __forceinline__ uint64_t bit_run(int a, int b) {
    if (b <= a) return 0;
    const uint64_t upto = b >= 64 ? ~0ull : (1ull << b) - 1;
    return a >= 64 ? 0 : upto & ~((1ull << a) - 1);
}

// Which of the keys [k0, k0 + 64) packed row r of the unit sees.
__device__ __forceinline__ uint64_t lat_visible(const LatParams& p, const LatUnit& x, int r,
                                                int k0) {
    const int t = r / p.heads, last = x.base + t;
    int pos = last, up = last;                 // `up`: the last key of the plain run
    if (p.tree.masks) {
        pos = x.base + p.tree.depths[x.qs + t];
        up = x.base - 1;
    }
    const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    uint64_t v = bit_run(min(max(lo - k0, 0), 64), min(max(up + 1 - k0, 0), 64));
    if (p.tree.masks && last >= k0 && x.base < k0 + kLatKeys) {
        const int u0 = k0 - x.base;
        v |= tree_bits(p.tree, x.qs + t, t, u0) |
             (uint64_t)tree_bits(p.tree, x.qs + t, t, u0 + 32) << 32;
    }
    return v;
}

// 8 consecutive elements of a query row (latent part, then rotary part) as 16-bit
// type E; zeros past the row.
template <typename E>
__device__ __forceinline__ uint4 lat_q8(const LatParams& p, int64_t lat, int64_t rope, int d) {
    if (p.q_vec) {            // both parts, rows and widths: multiples of 8 elements
        if (d >= p.dim) return make_uint4(0, 0, 0, 0);
        const bool in_lat = d < p.dc;
        const int64_t at = in_lat ? lat + d : rope + (d - p.dc);
        const void* base = in_lat ? p.q_lat : p.q_rope;
        if (p.q_dtype != CX_F32)
            return __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(base) + at));
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 a = __ldg(s), b = __ldg(s + 1);
        return make_uint4(Half16<E>::pack(a.x, a.y), Half16<E>::pack(a.z, a.w),
                          Half16<E>::pack(b.x, b.y), Half16<E>::pack(b.z, b.w));
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = d + e;
        x[e] = 0.f;
        if (i < p.dim) {
            const bool in_lat = i < p.dc;
            const int64_t at = in_lat ? lat + i : rope + (i - p.dc);
            const void* base = in_lat ? p.q_lat : p.q_rope;
            x[e] = p.q_dtype == CX_F32 ? static_cast<const float*>(base)[at]
                                       : Conv<E>::to_f(static_cast<const E*>(base)[at]);
        }
    }
    return make_uint4(Half16<E>::pack(x[0], x[1]), Half16<E>::pack(x[2], x[3]),
                      Half16<E>::pack(x[4], x[5]), Half16<E>::pack(x[6], x[7]));
}

template <typename E>
__host__ __device__ constexpr uint32_t lat_idesc(int m, int n, int a_mn, int b_mn) {
    return sc_idesc<E>(m, n, b_mn) | ((uint32_t)a_mn << 15);
}

// A call of f(std::integral_constant<int, n>), 1 <= n <= MAX.
template <int MAX, typename F>
__device__ __forceinline__ void with_constant(int n, const F& f) {
    if constexpr (MAX > 1) {
        if (n < MAX) {
            with_constant<MAX - 1>(n, f);
            return;
        }
    }
    f(std::integral_constant<int, MAX>{});
}

template <int N, typename E>
__global__ void __launch_bounds__(LatCfg<N>::THREADS, 1)
    latent_tc_kernel(const __grid_constant__ CUtensorMap tm, const LatParams p) {
    using C = LatCfg<N>;
    constexpr int SW = C::SW, SMT = C::ST, NW = C::NW, NJ = NW / 8;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = (int)warp_uniform(tid >> 5);
    const int sub_id = (int)blockIdx.x % p.sub, g = (int)blockIdx.x / p.sub;
    const int G = (int)gridDim.x / p.sub;
    const int NM = (p.dc + 127) / 128, NCH = (p.dim + 63) / 64;
    const int ST = p.stages, STAGE = lat_stage(p.dc, p.dim), NP = (NCH + 1) / 2;

    unsigned char* s_q = sm;
    unsigned char* s_p = s_q + NCH * C::Q_CHUNK;
    unsigned char* s_c = s_p + kLatP;
    unsigned char* misc = s_c + ST * STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(misc);
    // [stage][piece] two chunks of a tile
    uint64_t* empty = full + kLatMaxStages * kLatMaxPieces;
    uint64_t* s_full = empty + kLatMaxStages * kLatMaxPieces;     // [2] S^T of a tile is there
    uint64_t* p_full = s_full + 2;                // [2] P^T written, O^T rescaled
    uint64_t* o_done = p_full + 2;                // O^T of a tile is done
    // [2] Q of a range is there, by the range's parity: behind a range of one tile the
    // softmax warps come to the next range's before the PV warp need have seen this one's
    uint64_t* q_full = o_done + 1;
    uint64_t* drain = q_full + 2;                 // [2] last commits of the MMA warps
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drain + 2);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile int* s_issued = s_abort + 1;         // [kLatProd] tiles whose loads were begun
    int* s_start = const_cast<int*>(s_issued) + kLatProd;     // [4] unit, offset, share, all shares
    volatile int* s_n = s_start + 4;              // [2] tiles of a range (by its parity); 0: no more
    int* s_warp = s_start + 6;                    // [C::THREADS / 32]
    uint64_t* s_vis = reinterpret_cast<uint64_t*>(misc + 512);        // [64]
    float* s_alpha = reinterpret_cast<float*>(misc + 512);            // [64], after s_vis
    float* s_red = reinterpret_cast<float*>(misc + 1024);             // [4][64]

    // ---- what needs nothing of the kernels before: it may still run beside them ----
    if (tid == 0) {
        for (int s = 0; s < ST * kLatMaxPieces; ++s) {
            mbar_init(&full[s], kLatProd);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&s_full[0], 1);
        mbar_init(&s_full[1], 1);
        mbar_init(&p_full[0], SW);
        mbar_init(&p_full[1], SW);
        mbar_init(o_done, 1);
        mbar_init(&q_full[0], SW);
        mbar_init(&q_full[1], SW);
        mbar_init(&drain[0], 1);
        mbar_init(&drain[1], 1);
        *s_abort = 0;
        for (int k = 0; k < kLatProd; ++k) s_issued[k] = 0;
        fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) p.desc[(int64_t)blockIdx.x * 8] = 0;

    // rows of sequences without a key: zeros (threads t0, t0 + n_t, ..)
    auto zero_rows = [&](int t0, int n_t) {
        for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
            const int raw = p.ctx_lens[b];
            const int qs = p.q_start ? p.q_start[b] : b;
            const int n = p.q_start ? p.q_start[b + 1] - qs : 1;
            const int64_t cap = p.table_stride * p.block_size;
            if (t0 == 0) {
                if (raw > cap) raise_flag(CX_DEV_TABLE_OVERRUN);
                if (n < 0 || n > p.max_q || (raw > 0 && n > min((int64_t)raw, cap)))
                    raise_flag(CX_DEV_BAD_QLEN);
            }
            if (raw > 0) continue;
            const int64_t o0 = (int64_t)qs * p.heads * p.dc;
            const int64_t cnt = (int64_t)min(max(n, 0), p.max_q) * p.heads * p.dc;
            for (int64_t i = t0; i < cnt; i += n_t) store_as(p.out, p.out_dtype, o0 + i, 0.f);
        }
    };

    // ---- this CTA's share of the tiles ----
    {
        const int per = (p.n_units + C::THREADS - 1) / C::THREADS;
        const int u0 = min(p.n_units, tid * per), u1 = min(p.n_units, u0 + per);
        int sum = 0;
        for (int u = u0; u < u1; ++u) sum += lat_unit(p, u, 0, N).cost(p);
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        int before = incl - sum, W = 0;
#pragma unroll
        for (int w = 0; w < C::THREADS / 32; ++w) {
            if (w < warp) before += s_warp[w];
            W += s_warp[w];
        }
        W = (int)warp_uniform(W);     // (the branch below is then one for the whole warp)
        const int P = min(G, max(1, (W + kLatMinTiles - 1) / kLatMinTiles));
        const int w0 = g < P ? (int)((int64_t)g * W / P) : W;
        const int w1 = g < P ? (int)((int64_t)(g + 1) * W / P) : W;
        if (w1 <= w0) {
            zero_rows(tid, C::THREADS);
            return;
        }
        if (before <= w0 && w0 < before + sum) {
            int u = u0, at = before;
            for (; u < u1; ++u) {
                const int n = lat_unit(p, u, 0, N).cost(p);
                if (w0 < at + n) break;
                at += n;
            }
            s_start[0] = u;
            s_start[1] = w0 - at;
            s_start[2] = w1 - w0;
            s_start[3] = W;
        }
    }
    if (warp == SW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(s_tmem)),
                     "r"(C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    LatCursor cur{s_start[0], s_start[1], s_start[2]};
    LatSeg seg;
    int tile = 0;               // tiles of this CTA before the range
    const int bs = p.block_size;                  // (a multiple of 8)

    if (warp < SW) {
        // ---------------- Q in, softmax, output ----------------
        const int quad = warp & 3, wg = warp >> 2;    // keys [16 quad, ..), rows [NW wg, ..)
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const int tq = lane >> 2, c = lane & 3;
        const int tok0 = quad * 16 + tq, tok1 = tok0 + 8;
        const int col0 = wg * NW + 2 * c;             // this thread's first row
        constexpr float kGrow = Half16<E>::kGrowLog2, kLead = Half16<E>::kLeadLog2;
        bool ok = true;
        int slot = 0;
        // A range's queries, 16-bit, K-major, swizzled, zero padding rows.  Of the pool's
        // type and on 16-byte rows they are copied asynchronously.
        const bool q_async = p.q_vec && p.q_dtype != CX_F32;
        auto load_q = [&](const LatUnit& x) {
            if (q_async) {
                // a warp per row; lane k first finds the warp's k-th row
                const E *lat = static_cast<const E*>(p.q_lat), *rope = lat;
                const int r_k = warp + SW * lane;
                if (r_k < x.n_rows) {
                    const int R = x.r0 + r_k, t = R / p.heads, h = R - t * p.heads;
                    lat += (x.qs + t) * p.ql_tok + h * p.ql_head;
                    rope = static_cast<const E*>(p.q_rope) + (x.qs + t) * p.qr_tok +
                           h * p.qr_head - p.dc;
                }
#pragma unroll 2
                for (int k = 0; k < N / SW; ++k) {
                    const int r = warp + SW * k;
                    const E* l_k = reinterpret_cast<const E*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(lat), k));
                    const E* r_k = reinterpret_cast<const E*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(rope), k));
                    unsigned char* dst = s_q + r * 128;
                    for (int ch = lane; ch < NCH * 8; ch += 32) {
                        const int d = ch * 8;
                        const bool there = r < x.n_rows && d < p.dim;
                        const E* src = (d < p.dc ? l_k : r_k) + d;
                        cp_async16(dst + (ch >> 3) * C::Q_CHUNK + (((ch & 7) ^ (r & 7)) << 4),
                                   there ? src : static_cast<const E*>(p.q_lat), there);
                    }
                }
                return;
            }
            for (int i = tid; i < N * NCH * 8; i += SMT) {
                const int r = i / (NCH * 8), ch = i - r * (NCH * 8);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < x.n_rows) {
                    const int t = (x.r0 + r) / p.heads, h = (x.r0 + r) - t * p.heads;
                    v = lat_q8<E>(p, (x.qs + t) * p.ql_tok + h * p.ql_head,
                                  (x.qs + t) * p.qr_tok + h * p.qr_head, ch * 8);
                }
                *reinterpret_cast<uint4*>(s_q + (ch >> 3) * C::Q_CHUNK + r * 128 +
                                          (((ch & 7) ^ (r & 7)) << 4)) = v;
            }
        };
        int ranges = 0;
        auto q_ready = [&](int n) {                  // n tiles; 0: no further range
            uint64_t* there = &q_full[ranges & 1];
            if (tid == 0) s_n[ranges & 1] = n;
            ++ranges;
            if (q_async) asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(there);
        };
        bool more = cur.next(p, sub_id, N, seg);
        if (more) load_q(seg.x);
        q_ready(more ? seg.to - seg.from : 0);
        while (more) {
            const LatUnit x = seg.x;
            const int n = seg.to - seg.from, from = seg.from;
            const bool whole = seg.whole();
            const int32_t* tab = p.tables + (int64_t)x.b * p.table_stride;
            const int nblk = (x.ctx + bs - 1) / bs;
            const int first_k = (x.tile0 + from) * kLatKeys;
            bool bad = false;
            for (int k = first_k / bs + tid; k < nblk && k * bs < first_k + n * kLatKeys; k += SMT) {
                const int id = tab[k];
                bad |= id < 0 || id >= p.n_blocks;
            }
            const bool any_bad = bar_red_or(1, SMT, bad);
            // keys up to `all_hi` and from `all_lo` on are seen by every row
            const int t_first = x.r0 / p.heads, t_last = (x.r0 + x.n_rows - 1) / p.heads;
            const int all_hi = p.tree.masks ? x.base - 1 : x.base + t_first;
            const int all_lo = p.window > 0 ? x.base + t_last - p.window + 1 : 0;

            float m[NJ][2], l[NJ][2];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                m[j][0] = m[j][1] = -INFINITY;
                l[j][0] = l[j][1] = 0.f;
            }
            for (int i = 0; i < n; ++i, ++tile) {
                const int k0 = first_k + i * kLatKeys;
                ok = el_wait(&s_full[tile & 1], (tile >> 1) & 1, s_abort, p.tries);
                tc_fence_after();
                float v[NW / 2];
                lat_ld_s<NW>(tmem + C::S_COL + (tile & 1) * N + wg * NW + lane_base, v);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < NW / 2; ++e) v[e] *= p.scale_log2;
                const bool edge = any_bad || k0 + kLatKeys - 1 > all_hi || k0 < all_lo;
                uint64_t dead = 0;
                if (edge) {
                    uint64_t vis = 0;
                    if (tid < x.n_rows) {
                        vis = lat_visible(p, x, x.r0 + tid, k0);
                        for (int k = 0; any_bad && k < kLatKeys / 8; ++k) {
                            const int blk = (k0 + 8 * k) / bs, id = blk < nblk ? tab[blk] : 0;
                            if (id < 0 || id >= p.n_blocks) vis &= ~(0xffull << 8 * k);
                        }
                    }
                    if (tid < 64) s_vis[tid] = vis;
                    named_bar_sync(1, SMT);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint64_t w = s_vis[col0 + 8 * j + e];
                            if (!((w >> tok0) & 1)) v[4 * j + e] = -INFINITY;
                            if (!((w >> tok1) & 1)) v[4 * j + 2 + e] = -INFINITY;
                        }
                    }
                    // keys that no row sees
                    uint64_t any = s_vis[lane] | s_vis[lane + 32];
                    const uint32_t a0 = __reduce_or_sync(0xffffffffu, (uint32_t)any);
                    const uint32_t a1 = __reduce_or_sync(0xffffffffu, (uint32_t)(any >> 32));
                    dead = ~((uint64_t)a1 << 32 | a0);
                }
                // ---- the references; again with a maximum that outgrew one ----
                bool grow = false;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        grow |= fmaxf(v[4 * j + e], v[4 * j + 2 + e]) > m[j][e] + kGrow;
                if (bar_red_or(1, SMT, grow || !ok)) {
                    if (!(ok = bar_red_and(1, SMT, ok))) break;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float y = fmaxf(v[4 * j + e], v[4 * j + 2 + e]);
                            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                            if (lane < 4) s_red[quad * 64 + col0 + 8 * j + e] = y;
                        }
                    named_bar_sync(1, SMT);
                    bool moved = false;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float* q = s_red + col0 + 8 * j + e;
                            const float y = fmaxf(fmaxf(q[0], q[64]), fmaxf(q[128], q[192]));
                            float alpha = 1.f;
                            if (y > m[j][e] + kGrow) {      // (m -inf: any score that is not)
                                const float mn = y + kLead;
                                alpha = ex2_sfu(m[j][e] - mn);
                                m[j][e] = mn;
                                moved = true;
                            }
                            l[j][e] *= alpha;
                            if (quad == 0 && lane < 4) s_alpha[col0 + 8 * j + e] = alpha;
                        }
                    // (every thread of a column c has the same alphas)
                    moved = bar_red_or(1, SMT, moved);
                    if (moved && i > 0) {
                        // O^T holds the tiles before this one
                        ok = el_wait(o_done, (tile - 1) & 1, s_abort, p.tries);
                        if (!(ok = bar_red_and(1, SMT, ok))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int k = wg; k < NM * (N / 16); k += SW / 4) {
                            const int col = (k / (N / 16)) * N + (k % (N / 16)) * 16;
                            const uint32_t at = tmem + col + lane_base;
                            float o[16];
                            sc_ld16(at, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= s_alpha[(k % (N / 16)) * 16 + e];
                            sc_st16(at, reinterpret_cast<const uint32_t(&)[16]>(o));
                        }
                        tc_wait_st();
                    }
                    named_bar_sync(1, SMT);     // s_alpha and s_red are read
                }
                uint32_t pk[NW / 4];
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const float b0 = ref_base(m[j][0]), b1 = ref_base(m[j][1]);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        pk[2 * j + t] = Half16<E>::pack(ex2_sfu(v[4 * j + 2 * t] - b0),
                                                        ex2_sfu(v[4 * j + 2 * t + 1] - b1));
                }
                // ---- P^T over the last tile's, when O^T has read that ----
                if (tile > 0)
                    ok = el_wait(o_done, (tile - 1) & 1, s_abort, p.tries);
                if (!ok) {
                    *s_abort = 1;               // the next vote ends the loop for all
                    continue;
                }
                if (dead != 0) {
                    const int tok = tid & 63;
                    if ((dead >> tok) & 1) {
                        unsigned char* line = s_c + (tile % ST) * STAGE + tok * 128;
                        for (int ch = tid >> 6; ch < min(2 * NM, NCH); ch += SMT / 64) {
                            uint4* z = reinterpret_cast<uint4*>(line + ch * kLatChunk);
#pragma unroll
                            for (int k = 0; k < 8; ++k) z[k] = make_uint4(0, 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int ch = wg * NJ + j;
                    *reinterpret_cast<uint32_t*>(s_p + tok0 * 128 + ((ch ^ (tok0 & 7)) << 4) +
                                                 c * 4) = pk[2 * j];
                    *reinterpret_cast<uint32_t*>(s_p + tok1 * 128 + ((ch ^ (tok1 & 7)) << 4) +
                                                 c * 4) = pk[2 * j + 1];
                }
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[tile & 1]);
                // (the sums of what the second product gets: numerator and denominator round
                // alike)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float e0, e1, f0, f1;
                    f2_get(Half16<E>::unpack(pk[2 * j]), e0, e1);
                    f2_get(Half16<E>::unpack(pk[2 * j + 1]), f0, f1);
                    l[j][0] += e0 + f0;
                    l[j][1] += e1 + f1;
                }
                if (i == n - 1) {
                    // every MMA that reads this range's queries is done: the next range's
                    more = cur.next(p, sub_id, N, seg);
                    if (more) load_q(seg.x);
                }
            }
            // (a wait before the last P^T may have given up in some threads only)
            if (!(ok = bar_red_and(1, SMT, ok))) break;
            q_ready(more ? seg.to - seg.from : 0);      // S^T of the next range runs beside what follows
            // ---- denominators, then O^T to the output or to this CTA's part ----
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float y = l[j][e];
                    y += __shfl_xor_sync(0xffffffffu, y, 4);
                    y += __shfl_xor_sync(0xffffffffu, y, 8);
                    y += __shfl_xor_sync(0xffffffffu, y, 16);
                    if (lane < 4) s_red[quad * 64 + col0 + 8 * j + e] = y;
                }
            ok = el_wait(o_done, (tile - 1) & 1, s_abort, p.tries);
            if (!(ok = bar_red_and(1, SMT, ok))) break;
            tc_fence_after();
            const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * N;
            if (tid < N) {
                const float L = (s_red[tid] + s_red[64 + tid]) + (s_red[128 + tid] + s_red[192 + tid]);
                s_alpha[tid] = whole ? sum_inv(L) : 1.f;
                if (!whole) p.part_ml[(part + tid) * 2 + 1] = L;
            }
            if (!whole && quad == 0 && lane < 4) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        p.part_ml[(part + col0 + 8 * j + e) * 2] = m[j][e];
            }
            named_bar_sync(1, SMT);
            const int64_t row0 = (int64_t)x.qs * p.heads + x.r0;
#pragma unroll 1
            for (int k = wg; k < NM * (N / 16); k += SW / 4) {
                const int mm = k / (N / 16), n0 = (k % (N / 16)) * 16;
                const int d = mm * 128 + quad * 32 + lane, rows = x.n_rows - n0;
                if (rows <= 0) continue;                     // (the same for the warp)
                float o[16];
                sc_ld16(tmem + mm * N + n0 + lane_base, o);
                tc_wait_ld();
                if (!whole) {
                    float* dst = p.part_o + (part + n0) * p.dc + d;
                    if (d < p.dc) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (e < rows) dst[(int64_t)e * p.dc] = o[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= s_alpha[n0 + e];
                    if (p.out_dtype == CX_F32 || (p.dc & 1) ||
                        (reinterpret_cast<uintptr_t>(p.out) & 3)) {
                        if (d < p.dc) {
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (e < rows)
                                    store_as(p.out, p.out_dtype, (row0 + n0 + e) * p.dc + d, o[e]);
                        }
                    } else {
                        // pairs of columns: an even lane writes the even rows of both, its
                        // neighbour the odd ones
                        uint32_t* dst = static_cast<uint32_t*>(p.out) +
                                        ((row0 + n0 + (lane & 1)) * p.dc + (d & ~1)) / 2;
                        const bool bf = p.out_dtype == CX_BF16, in = (d & ~1) < p.dc;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float give = lane & 1 ? o[e] : o[e + 1];
                            const float keep = lane & 1 ? o[e + 1] : o[e];
                            const float got = __shfl_xor_sync(0xffffffffu, give, 1);
                            const float a = lane & 1 ? got : keep, b = lane & 1 ? keep : got;
                            const uint32_t u = bf ? Half16<__nv_bfloat16>::pack(a, b)
                                                  : Half16<__half>::pack(a, b);
                            if (in && e + (lane & 1) < rows) dst[(int64_t)e * p.dc / 2] = u;
                        }
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
            if (!whole && from == 0 && tid == 0) {
                // the unit starts here and goes on: who has the rest of it
                const int W = s_start[3];
                const int P = min(G, max(1, (W + kLatMinTiles - 1) / kLatMinTiles));
                const int end = (int)((int64_t)(g + 1) * W / P) + x.n_tiles - (from + n);
                int last = g + 1;
                while (last + 1 < P && (int)((int64_t)(last + 1) * W / P) < end) ++last;
                int32_t* d = p.desc + (int64_t)blockIdx.x * 8;
                d[1] = slot;
                d[2] = x.n_rows;
                d[3] = (int32_t)(row0 & 0xffffffff);
                d[4] = (int32_t)(row0 >> 32);
                d[0] = last - g + 1;
            }
            slot = 1;
            named_bar_sync(1, SMT);             // s_alpha and s_red are read
        }
        if (!ok) {
            *s_abort = 1;
            if (tid == 0) raise_flag(CX_DEV_WAIT_TIMEOUT);
        }
        zero_rows(tid, SMT);
    } else if (warp >= SW + 2) {
        // ---------------- producers: one for either chunk of a piece ----------------
        const int br = p.box_rows, nb = kLatKeys / br, w0 = warp - SW - 2;
        bool go = true;
        while (go && warp_uniform(cur.next(p, sub_id, N, seg))) {
            const LatUnit& x = seg.x;
            const int32_t* tab = p.tables + (int64_t)x.b * p.table_stride;
            const int n = (int)warp_uniform(seg.to - seg.from);
            const int key0 = (x.tile0 + seg.from) * kLatKeys;
            // lane l < nb: block (INT32_MIN: none) and row of box l of tile i
            auto place = [&](int i, int& id, int& row) {
                const int key = key0 + i * kLatKeys + br * lane, blk = key / bs;
                row = key - blk * bs;
                id = lane < nb && i < n && key < x.ctx ? tab[blk] : INT32_MIN;
            };
            int id, row, id_next, row_next;
            place(0, id, row);
            place(1, id_next, row_next);
            for (int i = 0; go && i < n; ++i, ++tile) {
                int z = -1;           // outside the map: the copy fills zeros
                if (id >= 0 && id < p.n_blocks)
                    z = p.layer * p.n_blocks + id;
                else if (id != INT32_MIN)
                    raise_flag(CX_DEV_BAD_BLOCK);
                const int s = tile % ST, use = tile / ST;
                const uint32_t dst0 = warp_uniform(smem_addr(s_c + s * STAGE));
                const uint32_t bar0 = warp_uniform(smem_addr(full + s * kLatMaxPieces));
                if (lane == 0) s_issued[w0] = tile + 1;
                // (what the boxes of every piece share; for other block sizes see below)
                int z4[4], row4[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    z4[k] = __shfl_sync(0xffffffffu, z, k);
                    row4[k] = __shfl_sync(0xffffffffu, row, k);
                }
                for (int j = 0; j < NP; ++j) {
                    // the pieces that O^T does not read are free first
                    const int q = j + NM < NP ? j + NM : j + NM - NP, ch = 2 * q + w0;
                    if (use > 0) {
                        go = el_wait(&empty[s * kLatMaxPieces + q], (use - 1) & 1, s_abort,
                                      p.tries);
                        if (!go) break;
                    }
                    const uint32_t bar = bar0 + q * 8, dst = dst0 + ch * kLatChunk;
                    el_expect(bar, ch < NCH ? kLatChunk : 0);
                    if (ch >= NCH) continue;
                    // (a condition at every box would triple what they take)
                    if (nb == 4) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            el_tma(dst + k * 2048, &tm, bar, ch * 64, row4[k], z4[k]);
                    } else {
                        for (int k = 0; k < nb; ++k)
                            el_tma(dst + k * br * 128, &tm, bar, ch * 64,
                                    __shfl_sync(0xffffffffu, row, k),
                                    __shfl_sync(0xffffffffu, z, k));
                    }
                }
                id = id_next;
                row = row_next;
                place(i + 2, id_next, row_next);
            }
        }
        if (!go && lane == 0) {
            *s_abort = 1;
            raise_flag(CX_DEV_WAIT_TIMEOUT);
        }
    } else {
        // ---------------- MMA issuers: whole warps, one thread's instructions ----------------
        const bool is_s = warp == SW;
        const uint32_t tm = warp_uniform(tmem);
        const uint32_t c_lo = warp_uniform(el_desc_lo(s_c, kLatChunk));
        const uint32_t b_lo = warp_uniform(el_desc_lo(is_s ? s_q : s_p, 16));
        bool ok = true;
        int st = 0;                               // stage of the next tile
        uint32_t use = 0;                         // parity of its fill
        for (int range = 0;; ++range) {
            ok = el_wait(&q_full[range & 1], (range >> 1) & 1, s_abort, p.tries);
            const int n = (int)warp_uniform(s_n[range & 1]);
            if (!ok || n == 0) break;
            for (int i = 0; ok && i < n; ++i, ++tile) {
                const uint32_t cd = warp_uniform(c_lo + (uint32_t)(st * STAGE >> 4));
                if (is_s) {
                    constexpr uint32_t idesc = lat_idesc<E>(kLatKeys, N, 0, 0);
                    const int b = tile & 1;
                    const uint32_t d = warp_uniform(tm + C::S_COL + b * N);
                    // S^T of two tiles before was read
                    if (tile >= 2)
                        ok = el_wait(&p_full[b], ((tile >> 1) - 1) & 1, s_abort, p.tries);
                    for (int j = 0; ok && j < NP; ++j) {
                        const int q = j + NM < NP ? j + NM : j + NM - NP;
                        ok = el_wait(&full[st * kLatMaxPieces + q], use, s_abort,
                                                   p.tries);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t ad = warp_uniform(cd + (uint32_t)(q * 2 * kLatChunk >> 4));
                        const uint32_t qd = warp_uniform(b_lo + (uint32_t)(q * 2 * C::Q_CHUNK >> 4));
                        const uint32_t acc = warp_uniform(j > 0);
                        // (a condition at every MMA triples what they take)
                        auto steps = [&](auto k_end) {
#pragma unroll
                            for (int k = 0; k < decltype(k_end)::value; ++k)
                                el_mma(d, ad + (((k >> 2) * kLatChunk + (k & 3) * 32) >> 4),
                                        qd + (((k >> 2) * C::Q_CHUNK + (k & 3) * 32) >> 4), idesc,
                                        k > 0 ? 1u : acc);
                        };
                        if (2 * q + 1 < NCH)
                            steps(std::integral_constant<int, 8>{});
                        else
                            steps(std::integral_constant<int, 4>{});
                        if (q >= NM) el_commit(&empty[st * kLatMaxPieces + q]);
                    }
                    if (ok) el_commit(&s_full[b]);
                } else {
                    constexpr uint32_t idesc = lat_idesc<E>(128, N, 1, 1);
                    ok = el_wait(&p_full[tile & 1], (tile >> 1) & 1, s_abort,
                                               p.tries);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t acc = warp_uniform(i > 0);
                    with_constant<kLatMaxLatent / 128>(NM, [&](auto nm) {
#pragma unroll
                        for (int mm = 0; mm < decltype(nm)::value; ++mm) {
#pragma unroll
                            for (int kk = 0; kk < kLatKeys / 16; ++kk)
                                el_mma(tm + mm * N, cd + ((mm * 2 * kLatChunk + kk * 2048) >> 4),
                                        b_lo + kk * (2048 >> 4), idesc, kk > 0 ? 1u : acc);
                            el_commit(&empty[st * kLatMaxPieces + mm]);
                        }
                    });
                    el_commit(o_done);
                }
                if (++st == ST) {
                    st = 0;
                    use ^= 1;
                }
            }
            if (!ok) break;
        }
        if (!ok && lane == 0) {
            *s_abort = 1;
            raise_flag(CX_DEV_WAIT_TIMEOUT);
        }
        el_commit(&drain[is_s ? 0 : 1]);         // completes once this warp's MMAs have
    }

    // ---- teardown: drain this CTA's own copies and MMAs, then free TMEM ----
    tc_fence_before();
    __syncthreads();
    if (*s_abort && tid == 0) {
        // (a tile that was given up in the middle never completes: what of it was issued
        // ends well within the wait)
        int issued = 0;
        for (int k = 0; k < kLatProd; ++k) issued = max(issued, s_issued[k]);
        for (int s = 0; s < ST; ++s) {
            const int uses = issued > s ? (issued - 1 - s) / ST + 1 : 0;
            for (int q = 0; uses > 0 && q < NP; ++q)
                mbar_wait_bounded(&full[s * kLatMaxPieces + q], (uses - 1) & 1, nullptr,
                                  20000000ull);
        }
    }
    if (tid == SW * 32 || tid == SW * 32 + 32)
        mbar_wait_bounded(&drain[tid == SW * 32 ? 0 : 1], 0, nullptr, kWaitLimitNs);
    __syncthreads();
    tc_fence_after();
    if (warp == SW)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(C::TMEM_COLS)
                     : "memory");
}

// Joins the parts of cut ranges: block (x, y) has rows 2 y and 2 y + 1 of the range that
// CTA x's last partial opens, 128 threads a row.  Lanes fetch the parts' references
// side by side, then every thread adds up four columns of all parts.
template <int N>
__global__ void __launch_bounds__(256) latent_join_kernel(const LatParams p) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 d = *reinterpret_cast<const int4*>(p.desc + (int64_t)blockIdx.x * 8);
    const int parts = d.x, slot = d.y, n_rows = d.z;
    const int r = blockIdx.y * 2 + (threadIdx.x >> 7), lane = threadIdx.x & 31;
    if (parts < 2 || r >= n_rows) return;
    const int64_t row = ((int64_t)(uint32_t)d.w |
                         (int64_t)p.desc[(int64_t)blockIdx.x * 8 + 4] << 32) + r;
    auto at = [&](int k) {
        return (((int64_t)blockIdx.x + (int64_t)k * p.sub) * 2 + (k == 0 ? slot : 0)) * N + r;
    };
    const int col = (threadIdx.x & 127) * 4;
    float M = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < parts; k0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (k0 + lane < parts) ml = *reinterpret_cast<const float2*>(p.part_ml + at(k0 + lane) * 2);
        float top = fmaxf(ml.x, M);
#pragma unroll
        for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        // (parts that saw no key: weight 0; of parts of NaN the sums are NaN)
        const float base = ref_base(top), old = exp2f(M - base), f = exp2f(ml.x - base);
        M = top;
        float sum = ml.y * f;
#pragma unroll
        for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        L = fmaf(L, old, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= old;
        const int n = min(32, parts - k0);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float* src = p.part_o + at(k0 + k) * p.dc + col;
            if (fk == 0.f) continue;              // (also what a part without a key left)
            if (p.dc % 4 == 0) {
                const float4 v = col < p.dc ? *reinterpret_cast<const float4*>(src)
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
                o[0] = fmaf(v.x, fk, o[0]);
                o[1] = fmaf(v.y, fk, o[1]);
                o[2] = fmaf(v.z, fk, o[2]);
                o[3] = fmaf(v.w, fk, o[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < p.dc) o[e] = fmaf(src[e], fk, o[e]);
            }
        }
    }
    const float inv = sum_inv(L);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < p.dc) store_as(p.out, p.out_dtype, row * p.dc + col + e, o[e] * inv);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Rows of a TMA box: of one block, and of a tile.
static int latent_box_rows(int64_t block_size) {
    return block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : block_size % 16 == 0 ? 16 : 8;
}

// View of a 16-bit latent pool: (row, slot, layer * block), box of 64 columns x some slots.
static int make_latent_tmap(CUtensorMap* m, const cx_latent_pool* p) {
    auto enc = tmap_encoder();
    if (!enc) return fail(CX_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dim = (cuuint64_t)(p->latent_dim + p->rope_dim);
    const cuuint64_t dims[3] = {dim, (cuuint64_t)p->block_size,
                                (cuuint64_t)(p->n_layers * p->n_blocks)};
    const cuuint64_t strides[2] = {dim * 2, dim * 2 * (cuuint64_t)p->block_size};
    const cuuint32_t box[3] = {64, (cuuint32_t)latent_box_rows(p->block_size), 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, p->dtype == CX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           3, p->kv, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(CX_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    return CX_OK;
}

template <int N, typename E>
static int launch_latent_tc(const CUtensorMap& tm, LatParams p, int grid, cudaStream_t st) {
    int smem = 0;
    LatCfg<N>::ring(p.dc, p.dim, p.stages, smem);
    auto kern = latent_tc_kernel<N, E>;
    CX_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    // (both kernels start beside the end of the one before them and wait for it)
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = LatCfg<N>::THREADS;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tm, p));
    int rc = check_launch("latent_tc_kernel");
    if (rc) return rc;
    cfg.gridDim = dim3(grid, N / 2);
    cfg.blockDim = 256;
    cfg.dynamicSmemBytes = 0;
    CX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, latent_join_kernel<N>, p));
    return check_launch("latent_join_kernel");
}

}  // namespace cx
