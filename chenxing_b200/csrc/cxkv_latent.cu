// Third translation unit of libcxkv.so: the latent cache and its attention, and the
// move of accepted nodes.  It keeps a device flag word of its own, like the others.
#include "cx_common.cuh"
#include "latent_attn_generic.cuh"
#include "latent_ops.cuh"

namespace cx {

unsigned int* dev_flags_latent() { return dev_flags(); }

// Whether the tcgen05 kernel takes the call: 16-bit pools whose rows TMA can load
// (queries of any alignment), with queries of the pool's type or fp32, which are rounded to
// it as by the kernels over K/V pools (fp32 beyond fp16's 65504 becomes infinite, and the row
// NaN).  Queries of the other 16-bit type are rare and lose range or precision: they go to
// the fp32 kernels, which convert nothing.
static bool latent_tc(const cx_latent_pool* pool, int32_t q_dtype) {
    const int64_t dim = pool->latent_dim + pool->rope_dim;
    return pool->dtype != CX_F32 && (q_dtype == CX_F32 || q_dtype == pool->dtype) &&
           dim % 8 == 0 && dim >= 64 && (reinterpret_cast<uintptr_t>(pool->kv) & 15) == 0 &&
           pool->block_size % 8 == 0;
}

// Rows of a tile, row tiles of the longest sequence, how many of them run side by
// side, and the CTAs.
struct LatPlan {
    int n, rtiles, sub, grid;
    int64_t units;
};

static LatPlan latent_plan(const cx_latent_pool* pool, const cx_attn_batch* b) {
    const int64_t rows = b->n_q_heads * b->max_q_len;
    LatPlan x{};
    x.n = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    x.rtiles = (int)((rows + x.n - 1) / x.n);
    // two row tiles of a sequence read the same keys at the same time: once from HBM
    x.sub = x.rtiles == 2 ? 2 : 1;
    x.units = b->batch * ((x.rtiles + x.sub - 1) / x.sub);
    const int sms = std::max(num_sms(), x.sub);
    int64_t keys = b->table_stride * pool->block_size;
    if (b->window > 0) keys = std::min(keys, b->window + b->max_q_len + 2 * kLatKeys);
    const int cost = lat_range_cost((int)(pool->latent_dim + pool->rope_dim));
    const int64_t tiles = x.units * ((keys + kLatKeys - 1) / kLatKeys + cost);
    const int64_t want = std::max<int64_t>(1, (tiles + kLatMinTiles - 1) / kLatMinTiles);
    x.grid = (int)std::min<int64_t>(sms / x.sub, want) * x.sub;
    return x;
}

// Rows of a unit of the fp32 kernels: latent_rows_kernel from 17 rows of a sequence on (62
// tokens of 64 heads behind 1,200 keys of 384 + 64: 1,188 us with units of 4 rows, 558 with
// 32; 16 rows behind 4,000 of 512 + 64: 150 and 174).
static int generic_unit_rows(const cx_attn_batch* b) {
    return b->n_q_heads * b->max_q_len > 16 ? kLrRows : kLgRows;
}

static int64_t generic_tiles(const cx_attn_batch* b) {
    const int64_t u = generic_unit_rows(b);
    return (b->n_q_heads * b->max_q_len + u - 1) / u;
}

// Parts that the fp32 kernels split a context into: CTAs for four an SM (of 32 rows: two),
// at least 32 keys a part, at most 256 parts (latent_generic_join).
static int latent_split(const cx_latent_pool* pool, const cx_attn_batch* b, int64_t units) {
    int64_t keys = b->table_stride * pool->block_size;
    if (b->window > 0) keys = std::min(keys, b->window + b->max_q_len);
    const int64_t want = (generic_unit_rows(b) == kLrRows ? 2ll : 4ll) * std::max(num_sms(), 1) /
                         std::max<int64_t>(units, 1);
    return (int)std::max<int64_t>(1, std::min(std::min(want, keys / 32), (int64_t)256));
}

static size_t latent_workspace(const cx_latent_pool* pool, const cx_attn_batch* b, bool tc) {
    if (tc) {
        const LatPlan x = latent_plan(pool, b);
        const size_t rows = (size_t)x.grid * 2 * x.n;
        return 256 + (size_t)x.grid * 32 + rows * (pool->latent_dim + 2) * 4;
    }
    const int64_t units = b->batch * generic_tiles(b);
    const int s = latent_split(pool, b, units);
    return s == 1 ? 256 : 256 + (size_t)units * s * generic_unit_rows(b) * (pool->latent_dim + 2) * 4;
}

static int latent_attend(const cx_latent_pool* pool, int64_t layer, const cx_attn_batch* bt,
                         const cx_tree* tree, const cx_latent_q* q, void* out, int32_t out_dtype,
                         void* ws, size_t ws_bytes, cudaStream_t st) {
    auto bad = [&](int code, const char* what) {
        return fail(code, std::string("cx_latent_attend: ") + what);
    };
    int rc = check_latent_pool(pool);
    if (rc) return rc;
    if (!bt || !q) return bad(CX_ERR_SHAPE, "NULL batch or queries");
    if (layer < 0 || layer >= pool->n_layers) return bad(CX_ERR_RANGE, "layer out of range");
    if (bt->batch < 0 || bt->n_q_heads <= 0)
        return bad(CX_ERR_SHAPE, "batch must be >= 0 and n_q_heads positive");
    if (bt->q_start && bt->max_q_len < 1) return bad(CX_ERR_SHAPE, "max_q_len must be at least 1");
    if (elem_bytes(q->dtype) == 0 || elem_bytes(out_dtype) == 0)
        return bad(CX_ERR_DTYPE, "unknown query or output type");
    if (q->latent_token_stride < 0 || q->latent_head_stride < 0 || q->rope_token_stride < 0 ||
        q->rope_head_stride < 0)
        return bad(CX_ERR_SHAPE, "negative stride");
    if (tree && (!bt->q_start || !tree->masks || !tree->depths || tree->words < 1 ||
                 tree->words * 32 < bt->max_q_len))
        return bad(CX_ERR_SHAPE, "a tree needs q_start, masks of max_q_len bits and depths");
    if (bt->batch == 0) return CX_OK;
    if (!bt->block_tables || !bt->ctx_lens || !q->latent || !q->rope || !out ||
        bt->table_stride <= 0)
        return bad(CX_ERR_SHAPE, "NULL array or empty table");
    cx_attn_batch b = *bt;
    if (!b.q_start) b.max_q_len = 1;
    const int64_t cap = b.table_stride * pool->block_size;
    if (b.table_stride > (1ll << 26) || cap > (1ll << 30) || b.batch > (1 << 24) ||
        b.max_q_len > (1 << 24) || b.n_q_heads > (1 << 16) ||
        b.max_q_len * b.n_q_heads > (1ll << 30) || (tree && tree->words > (1 << 20)))
        return bad(CX_ERR_UNSUPPORTED, "batch, table or rows too large");
    const bool tc = latent_tc(pool, q->dtype);
    const size_t need = latent_workspace(pool, &b, tc);
    if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255) != 0)
        return bad(CX_ERR_WORKSPACE, "workspace missing, too small or not 256-byte aligned");
    const float scale =
        isnan(b.scale) ? 1.0f / sqrtf((float)(pool->latent_dim + pool->rope_dim)) : b.scale;
    LatParams p{};
    p.tables = b.block_tables;
    p.table_stride = b.table_stride;
    p.ctx_lens = b.ctx_lens;
    p.q_start = b.q_start;
    if (tree) p.tree = {tree->masks, tree->depths, tree->words};
    p.q_lat = q->latent;
    p.q_rope = q->rope;
    p.ql_tok = q->latent_token_stride;
    p.ql_head = q->latent_head_stride;
    p.qr_tok = q->rope_token_stride;
    p.qr_head = q->rope_head_stride;
    p.out = out;
    p.batch = (int)b.batch;
    p.heads = (int)b.n_q_heads;
    p.max_q = (int)b.max_q_len;
    p.n_blocks = (int)pool->n_blocks;
    p.block_size = (int)pool->block_size;
    p.layer = (int)layer;
    p.window = b.window > 0 ? (int)std::min<int64_t>(b.window, 1 << 30) : 0;
    p.dc = (int)pool->latent_dim;
    p.dim = (int)(pool->latent_dim + pool->rope_dim);
    p.q_dtype = q->dtype;
    p.out_dtype = out_dtype;
    p.scale_log2 = scale * 1.4426950408889634f;
    // (a try suspends for half a microsecond at most)
    p.tries = (uint32_t)std::min<unsigned long long>(1ull << 30, wait_limit_ns() / 500 + 1);
    if (!tc) {
        LatGenParams g{};
        g.a = p;
        g.pool = pool->kv;
        g.n_blocks64 = pool->n_blocks;
        g.layer64 = layer;
        const int64_t tiles = generic_tiles(&b), units = b.batch * tiles;
        if (units > INT32_MAX) return bad(CX_ERR_UNSUPPORTED, "too many rows");
        g.row_tiles = (int)tiles;
        g.unit_rows = generic_unit_rows(&b);
        g.n_split = latent_split(pool, &b, units);
        g.scale = scale;
        g.part = reinterpret_cast<float*>(static_cast<char*>(ws) + 256);
        switch (pool->dtype) {
            case CX_F32: return launch_latent_generic<float>(g, st);
            case CX_BF16: return launch_latent_generic<__nv_bfloat16>(g, st);
            default: return launch_latent_generic<__half>(g, st);
        }
    }
    const LatPlan x = latent_plan(pool, &b);
    if (x.units * (cap / kLatKeys + 13) > INT32_MAX)
        return bad(CX_ERR_UNSUPPORTED, "batch x context too large");
    p.rtiles = x.rtiles;
    p.sub = x.sub;
    p.n_units = (int)x.units;
    const int e = elem_bytes(q->dtype);
    const uintptr_t al =
        reinterpret_cast<uintptr_t>(q->latent) | reinterpret_cast<uintptr_t>(q->rope) |
        (uintptr_t)((p.ql_tok | p.ql_head | p.qr_tok | p.qr_head) * e);
    p.q_vec = (al & 15) == 0 && p.dc % 8 == 0;
    char* w = static_cast<char*>(ws);
    p.desc = reinterpret_cast<int32_t*>(w);
    p.part_ml = reinterpret_cast<float*>(w + (size_t)x.grid * 32);
    p.part_o = p.part_ml + (size_t)x.grid * 2 * x.n * 2;   // (16-byte aligned)
    p.range_cost = lat_range_cost(p.dim);
    p.box_rows = latent_box_rows(pool->block_size);
    CUtensorMap tm;
    rc = make_latent_tmap(&tm, pool);
    if (rc) return rc;
    auto go = [&](auto e16) {
        using E = decltype(e16);
        return x.n == 16   ? launch_latent_tc<16, E>(tm, p, x.grid, st)
               : x.n == 32 ? launch_latent_tc<32, E>(tm, p, x.grid, st)
                           : launch_latent_tc<64, E>(tm, p, x.grid, st);
    };
    return pool->dtype == CX_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

}  // namespace cx

extern "C" {

int cx_latent_attend(const cx_latent_pool* pool, int64_t layer, const cx_attn_batch* batch,
                     const cx_tree* tree, const cx_latent_q* q, void* out, int32_t out_dtype,
                     void* workspace, size_t workspace_bytes, void* stream) {
    return cx::latent_attend(pool, layer, batch, tree, q, out, out_dtype, workspace,
                             workspace_bytes, cx::as_stream(stream));
}

// (for the larger of the two kernels' needs: which one runs depends on the queries)
size_t cx_latent_attend_workspace_bytes(const cx_latent_pool* pool, const cx_attn_batch* batch) {
    if (!pool || !batch || batch->n_q_heads <= 0 || batch->batch < 0) return 0;
    if (cx::check_latent_pool(pool) != CX_OK) return 0;
    cx_attn_batch b = *batch;
    if (!b.q_start || b.max_q_len < 1) b.max_q_len = 1;
    const size_t g = cx::latent_workspace(pool, &b, false);
    return cx::latent_tc(pool, CX_F32) ? std::max(g, cx::latent_workspace(pool, &b, true)) : g;
}

int cx_latent_attend_kind(const cx_latent_pool* pool, const cx_attn_batch* batch,
                          int32_t q_dtype) {
    if (!pool || !batch || cx::check_latent_pool(pool) != CX_OK) return CX_KERNEL_GENERIC;
    return cx::latent_tc(pool, q_dtype) ? CX_KERNEL_TCGEN05 : CX_KERNEL_GENERIC;
}

}  // extern "C"
