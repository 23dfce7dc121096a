"""Attention of drafted trees and the move of accepted paths."""
import numpy as np
import pytest
import torch

from scored_cases import alibi
from tree_cases import TreeCase, random_tree

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_flags():
    from chenxing_b200 import _lib
    _lib.device_flags(clear=True)
    yield
    flags = _lib.device_flags(clear=True)
    assert flags == 0, f"device error flags raised: {_lib.describe_flags(flags)}"


MODS = {
    "plain": dict(),
    "cap-window": dict(softcap=30.0, window=19, q_scale=4.0),
    "alibi": dict(slopes="alibi"),
    "alibi-cap-window": dict(slopes="alibi", softcap=20.0, window=3, q_scale=3.0),
    "prefix-window": dict(prefix=11, window=9),
}


def _case(mods, kind, hq, sizes, ctx, **kw):
    m = dict(MODS[mods])
    if m.get("slopes"):
        m["slopes"] = alibi(hq)
    if m.get("prefix"):
        m["prefix"] = [m["prefix"] + 40 * (b % 2) for b in range(len(ctx))]
    m.update(kw)
    rng = np.random.default_rng(hq + sum(sizes))
    return TreeCase(hq=hq, ctx=ctx, parents=[random_tree(rng, n, kind) for n in sizes], **m)


SHAPES = [
    # fp32, mma.sync and generic kernels
    (8, 2, 64, F32, [1, 8, 5, 0, 13], [1, 8, 300, 40, 77]),
    (4, 4, 128, F32, [16, 3], [16, 700]),
    (8, 2, 128, BF, [1, 8, 5, 0, 6], [1, 8, 290, 16, 95]),
    (8, 8, 64, F16, [32, 7, 20], [32, 500, 49]),
    (6, 2, 128, BF, [10, 9], [200, 64]),
    (4, 1, 64, BF, [4, 2], [1030, 2]),
    (4, 2, 80, BF, [9, 21], [50, 300]),
    (6, 3, 40, F32, [12, 1], [100, 17]),
    (8, 2, 64, F32, [40, 20], [100, 317]),
    (4, 1, 64, F32, [2, 1, 0], [700, 20, 9]),
    (3, 1, 128, F32, [3, 40], [5000, 41]),
    # tcgen05: one query tile in two places
    (8, 2, 128, BF, [26, 10, 1, 0, 17], [26, 600, 129, 16, 140]),
    (32, 8, 128, BF, [26, 12], [1000, 127]),
    (8, 8, 64, F16, [60, 7, 33], [60, 500, 49]),
    (4, 1, 64, BF, [15, 9], [1030, 9]),
    (12, 4, 128, F16, [11, 40, 3], [128, 385, 257]),
    # and two, or their keys over many CTAs
    (4, 4, 64, F16, [130, 64, 200], [130, 500, 333]),
    (14, 2, 64, BF, [40, 19], [300, 19]),
    (6, 2, 128, F16, [90, 43], [211, 43]),
    (5, 1, 128, F16, [30, 13], [4000, 40]),
    (2, 1, 128, BF, [30], [9000]),
]


@pytest.mark.parametrize("mods", list(MODS))
@pytest.mark.parametrize("kind", ["random", "star", "deep"])
@pytest.mark.parametrize("hq,hk,d,dtype,sizes,ctx", SHAPES)
def test_trees(mods, kind, hq, hk, d, dtype, sizes, ctx):
    c = _case(mods, kind, hq, sizes, ctx, hk=hk, d=d, dtype=dtype, seed=hq + d)
    c.check(c.run(out_dtype=dtype))


def test_kernels_of_the_shapes():
    kinds = []
    for hq, hk, d, dtype, sizes, ctx in SHAPES:
        kinds.append(_case("plain", "star", hq, sizes, ctx, hk=hk, d=d, dtype=dtype)
                     .batch().kernel_kind(dtype, dtype))
    assert kinds == ["fma", "fma", "mma", "mma", "mma", "mma", "generic", "generic", "fma", "fma",
                     "fma"] + ["tcgen05"] * 10


@pytest.mark.parametrize("hq,hk,d,dtype,n", [(8, 2, 128, BF, 7), (8, 2, 128, BF, 13),
                                             (8, 2, 128, BF, 40),
                                             (8, 2, 64, F32, 8), (4, 2, 96, F16, 8)])
def test_a_chain_is_what_verify_gives(hq, hk, d, dtype, n):
    """A tree without branches has the bits of the chain's verification."""
    c = _case("cap-window", "chain", hq, [n, n], [n + 200, n + 31], hk=hk, d=d, dtype=dtype)
    tree = c.run(out_dtype=dtype)
    from chenxing_b200 import PagedBatch
    chain = PagedBatch(c.cache, c.tables, c.ctx, n_q_heads=hq, q_lens=c.q_lens, window=c.window,
                       softcap=c.softcap, scale=c.scale)
    c.check(tree)
    c.check(c.run(chain, out_dtype=dtype))


@pytest.mark.parametrize("dtype,q_dtype,out_dtype", [(BF, F32, F32), (F16, F16, F32),
                                                     (F32, BF, F16), (BF, F16, BF)])
@pytest.mark.parametrize("n", [6, 40])
def test_type_mixes(dtype, q_dtype, out_dtype, n):
    c = _case("plain", "random", 8, [n, 3], [70, 300], hk=2, d=128, dtype=dtype, q_dtype=q_dtype,
              strided=True)
    c.check(c.run(out_dtype=out_dtype))


@pytest.mark.parametrize("bs", [1, 5, 64])
def test_blocks_of_other_sizes(bs):
    c = _case("alibi-cap-window", "random", 8, [21, 0, 4], [150, 7, 4], hk=2, d=64, dtype=F32, bs=bs)
    assert c.batch().kernel_kind(F32) == "fma"
    c.check(c.run())


@pytest.mark.parametrize("hq,dtype,n", [(8, F32, 2), (8, F32, 9), (8, BF, 6), (8, BF, 26)])
@pytest.mark.parametrize("prefix", [None, [21]])
def test_bad_block_ids_leave_their_keys_out(hq, dtype, n, prefix):
    from chenxing_b200 import _lib
    c = _case("plain", "random", hq, [n], [200 + n], hk=2, d=64, dtype=dtype, prefix=prefix)
    batch = c.batch()
    batch.block_tables[0, 3] = 10 ** 6
    batch.block_tables[0, 7] = -5
    out = c.run(batch, out_dtype=dtype)
    assert _lib.device_flags(clear=True) == 2
    c.check(out, list(range(48, 64)) + list(range(112, 128)))


def test_batches_on_two_streams_at_once():
    """A batch a stream, each with a workspace of its own; the same calls one by one."""
    shapes = [(8, 2, 64, F32, [9, 12]), (8, 2, 128, BF, [26, 12]), (8, 2, 128, BF, [3, 6])]
    for hq, hk, d, dtype, sizes in shapes:
        c = _case("alibi", "random", hq, sizes, [2500, 333], hk=hk, d=d, dtype=dtype)
        batches = [c.batch() for _ in range(2)]
        want = c.run(batches[0])
        c.check(want)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for _ in range(5):
            for b, st in zip(batches, streams):
                with torch.cuda.stream(st):
                    outs.append(c.run(b))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_two_graphs_share_a_workspace():
    c = _case("plain", "deep", 8, [9, 30], [1500, 333], hk=2, d=64, dtype=F32)
    batch = c.batch()
    want = c.run(batch)
    outs = [torch.empty_like(want) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o in zip(graphs, outs):
        with torch.cuda.graph(g):
            c.run(batch, out=o)
    for _ in range(2):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_float32_output_takes_the_tree_too():
    """The default output type of a batch without score modifiers is fp32."""
    c = _case("plain", "random", 8, [7, 12], [70, 300], hk=2, d=128, dtype=BF)
    c.check(c.run())


def test_set_takes_new_trees_and_graphs_replay():
    c = _case("plain", "random", 8, [9, 12], [90, 333], hk=2, d=128, dtype=BF, seed=1)
    batch = c.batch()
    c.check(c.run(batch, out_dtype=BF))
    rng = np.random.default_rng(5)
    c.parents = [random_tree(rng, 9, "deep"), random_tree(rng, 12, "star")]
    batch.set(c.tables, c.ctx, c.q_lens, tree_parents=c.parents)
    want = c.run(batch, out_dtype=BF)
    c.check(want)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(batch, out=out)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# accepted paths
# ---------------------------------------------------------------------------
def _caches(latent, layers, hk, d, dtype, bs, nb):
    from chenxing_b200 import LatentPagedKVCache, RadixPagedKVCache
    if latent:
        c = LatentPagedKVCache(nb, bs, layers, d - d // 8 // 2 * 2, d // 8 // 2 * 2, dtype=dtype, host_io=False)
        return c, [c.kv_pool[:, :, :, None]]
    c = RadixPagedKVCache(nb, bs, layers, hk, d, dtype=dtype, host_io=False)
    return c, [c.k_pool, c.v_pool]


def _batch(cache, latent, tables, ctx, q_lens):
    from chenxing_b200 import LatentBatch, PagedBatch
    if latent:
        return LatentBatch(cache, tables, ctx, n_q_heads=4, q_lens=q_lens, scale=1.0)
    return PagedBatch(cache, tables, ctx, n_q_heads=cache.n_kv_heads, q_lens=q_lens)


PATHS = [[0, 2, 3, 7], [], [0], [5], [0, 1, 2, 3, 4, 5], list(range(0, 80, 2)), list(range(33)),
         [3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 79]]
SIZES = [8, 4, 1, 6, 6, 80, 33, 80]


@pytest.mark.parametrize("latent,hk,d,dtype,bs", [
    (False, 2, 64, F32, 16), (False, 8, 128, BF, 16), (False, 3, 5, F16, 4), (False, 1, 6, BF, 1),
    (True, 1, 576, BF, 16), (True, 1, 33 * 2, F16, 16), (True, 1, 34, F32, 8)])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_accept_paths(latent, hk, d, dtype, bs, as_tensor):
    gen = torch.Generator().manual_seed(d)
    ctx = [n + 5 * i for i, n in enumerate(SIZES)]
    need = [-(-c // bs) for c in ctx]
    cache, pools = _caches(latent, 3, hk, d, dtype, bs, sum(need) + 2)
    perm = np.random.default_rng(d).permutation(sum(need) + 2)
    off = np.concatenate([[0], np.cumsum(need)])
    tables = [perm[off[b]:off[b + 1]].tolist() for b in range(len(ctx))]
    for p in pools:
        p.copy_(torch.randn(p.shape, generator=gen).to(dtype))
    want = [p.cpu().clone() for p in pools]
    for p in want:
        old = p.clone()
        for b, path in enumerate(PATHS):
            for k, n in enumerate(path):
                f, t = ctx[b] - SIZES[b] + n, ctx[b] - SIZES[b] + k
                p[:, tables[b][t // bs], t % bs] = old[:, tables[b][f // bs], f % bs]
    batch = _batch(cache, latent, tables, ctx, SIZES)
    paths = PATHS
    if as_tensor:
        width = max(map(len, PATHS)) + 2
        paths = torch.tensor([p + [-1] * (width - len(p)) for p in PATHS], device="cuda")
    cache.accept_paths(batch, paths)
    for p, w in zip(pools, want):
        assert torch.equal(p.cpu(), w)


def test_bad_paths_raise_a_flag_and_stop():
    from chenxing_b200 import _lib
    cache, pools = _caches(False, 1, 2, 8, F32, 16, 4)
    for p in pools:
        p.copy_(torch.arange(p.numel(), dtype=torch.float32).reshape(p.shape))
    old = pools[0].cpu().clone()
    batch = _batch(cache, False, [[0, 1], [2]], [20, 10], [8, 4])
    cache.accept_paths(batch, torch.tensor([[1, 3, 3, 5], [2, 9, -1, -1]], dtype=torch.int32))
    assert _lib.device_flags(clear=True) == 64
    new = pools[0].cpu()
    want = old.clone()
    want[0, 0, 12], want[0, 0, 13] = old[0, 0, 13], old[0, 0, 15]
    want[0, 2, 6] = old[0, 2, 8]
    assert torch.equal(new, want)


def test_accept_in_a_graph_reads_each_replays_paths():
    cache, pools = _caches(True, 2, 1, 64, BF, 16, 4)
    data = torch.randn(pools[0].shape, generator=torch.Generator().manual_seed(0)).to(BF).cuda()
    batch = _batch(cache, True, [[3, 1]], [20], [8])
    paths = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    cache.accept_paths(batch, paths)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.accept_paths(batch, paths)
    for path in ([2, 5], [0, 1, 6, 7], [4]):
        pools[0].copy_(data)
        paths.fill_(-1)
        paths[0, :len(path)] = torch.tensor(path)
        g.replay()
        torch.cuda.synchronize()
        at = [(3, p) if p < 16 else (1, p - 16) for p in range(20)]
        for k, n in enumerate(path):
            (tb, ts), (fb, fs) = at[12 + k], at[12 + n]
            assert torch.equal(pools[0][:, tb, ts], data[:, fb, fs])


# ---------------------------------------------------------------------------
# a speculative step of the engine, as it is used: append with rotation, attention of
# the trees, one path kept, and the next step over what was kept
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("latent", [False, True])
def test_engine_steps(latent):
    """The kept path must leave the cache as if its tokens had been decoded one by one."""
    from chenxing_b200 import (BatchedKVEngine, LatentPagedKVCache, RadixPagedKVCache, RopeTables)
    hq, L = 8, 2
    if latent:
        cache = LatentPagedKVCache(64, 16, L, 128, 64, dtype=F32, host_io=False)
        ref = LatentPagedKVCache(64, 16, L, 128, 64, dtype=F32, host_io=False)
        rope, kw = RopeTables(256, 64), dict(scale=0.07)
        widths, q_width = (128, 64), 64
    else:
        cache = RadixPagedKVCache(64, 16, L, 2, 64, dtype=F32, host_io=False)
        ref = RadixPagedKVCache(64, 16, L, 2, 64, dtype=F32, host_io=False)
        rope, kw = RopeTables(256, 64), {}
        widths, q_width = (64, 64), 64
    gen = torch.Generator().manual_seed(1)

    def rows(n, *shape):
        return torch.randn(n, *shape, generator=gen).cuda()

    def kv(n):
        return [(rows(n, widths[0]), rows(n, widths[1])) if latent else
                (rows(n, 2, 64), rows(n, 2, 64)) for _ in range(L)]

    def step(eng, ids, q_lens, new, qs, **plan_kw):
        plan = eng.plan(ids, q_lens, verify=True, **plan_kw)
        outs = []
        for layer, (k, v) in enumerate(new):
            q = eng.append_rope(plan, layer, k, v, rope, qs[layer][..., -q_width:],
                                q_out_dtype=F32, **({} if latent else dict(k_weight=one)))
            outs.append(eng.attend(plan, layer, (qs[layer][..., :128], q) if latent else q))
        return plan, outs

    one = torch.ones(64, device="cuda")
    eng = BatchedKVEngine(cache, n_q_heads=hq, **kw)
    want = BatchedKVEngine(ref, n_q_heads=hq, **kw)
    prompt = {7: 21, 9: 40}
    for e in (eng, want):
        for i, n in prompt.items():
            e.add(i, list(range(100 * i, 100 * i + n)))
    first, q0 = kv(61), [rows(61, hq, 192 if latent else 64) for _ in range(L)]
    for e in (eng, want):
        plan, _ = step(e, [7, 9], [21, 40], first, q0)
        e.commit(plan)
    trees = [[-1, 0, 0, 1, 2, 2, 4], [-1, -1, 1, 1, 3]]
    paths = [[0, 2, 4, 6], [1, 3, 4]]
    sizes = [7, 5]
    new, qs = kv(12), [rows(12, hq, 192 if latent else 64) for _ in range(L)]
    plan, outs = step(eng, [7, 9], sizes, new, qs, tree_parents=trees)
    eng.accept(plan, paths)
    keep = torch.tensor([n for b, p in enumerate(paths) for n in [x + 7 * b for x in p]]).cuda()
    got = [o[keep] for o in outs]
    plan, exp = step(want, [7, 9], [4, 3], [(k[keep], v[keep]) for k, v in new],
                     [q[keep] for q in qs])
    want.commit(plan)
    for a, b in zip(got, exp):       # the same keys in fp32, summed in another order
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
    for i, n in ((7, 25), (9, 43)):
        assert eng.seqs[i].n_tokens == want.seqs[i].n_tokens == n
        for layer in range(L):
            for x, y in zip(cache.read_layer(eng.seqs[i].block_table, n, layer),
                            ref.read_layer(want.seqs[i].block_table, n, layer)):
                assert torch.equal(x, y)
    more, q1 = kv(2), [rows(2, hq, 192 if latent else 64) for _ in range(L)]
    results = []
    for e in (eng, want):
        plan, o = step(e, [7, 9], [1, 1], more, q1)
        e.commit(plan)
        results.append(o)
    for a, b in zip(*results):
        assert torch.equal(a, b)
