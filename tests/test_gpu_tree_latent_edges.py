"""Edges of the drafted trees, the accepted paths and the latent cache (bounds:
tree_cases)."""
import math

import numpy as np
import pytest
import torch

from scored_cases import HALF, ScoredCase, alibi
from tree_cases import LatentCase, TreeCase, random_tree

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_flags():
    from chenxing_b200 import _lib
    _lib.device_flags(clear=True)
    yield
    flags = _lib.device_flags(clear=True)
    assert flags == 0, f"device error flags raised: {_lib.describe_flags(flags)}"


@pytest.mark.parametrize("hq,dc,dr,dtype,q_lens", [
    (16, 512, 64, BF, None), (16, 128, 64, F16, None), (64, 256, 64, BF, None), (20, 128, 64, BF, 2)])
def test_many_ranges_of_one_tile(hq, dc, dr, dtype, q_lens):
    """2,000 sequences of 1 to 64 tokens: every range of a CTA has one key tile."""
    ctx = [1 + (37 * i) % 64 for i in range(2000)]
    if q_lens:
        q_lens = [min(q_lens, c) for c in ctx]
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=ctx, q_lens=q_lens, dtype=dtype, seed=hq)
    batch = c.batch()
    assert batch.kernel_kind(dtype) == "tcgen05"
    a = c.run(batch, out_dtype=dtype)
    c.check(a)
    for _ in range(5):
        assert torch.equal(a, c.run(batch, out_dtype=dtype))


@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 128, BF), (4, 4, 64, F16)])
def test_two_places_that_end_apart(hq, hk, d, dtype):
    """Trees of one query tile, held in two places, behind 1 to 10 key tiles: the places
    have as many or differ by one, and each is read by the other's warps."""
    rng = np.random.default_rng(d)
    ctx = [60 + 128 * i for i in range(10)] + [128 * i + 1 for i in range(1, 10)]
    n = 15 if hq > hk else 40
    parents = [random_tree(rng, n, "random") for _ in ctx]
    c = TreeCase(hq=hq, hk=hk, d=d, dtype=dtype, ctx=ctx, parents=parents, seed=d)
    batch = c.batch()
    assert batch.kernel_kind(dtype, dtype) == "tcgen05"
    a = c.run(batch, out_dtype=dtype)
    c.check(a)
    for _ in range(30):
        assert torch.equal(a, c.run(batch, out_dtype=dtype))


def _check_nan_rows(c, out, rows):
    """`rows` (token, head) hold NaN throughout, every other row is as without them."""
    bad = torch.zeros(out.shape[:2], dtype=torch.bool)
    for r in rows:
        bad[r] = True
    got = out.double().cpu()
    assert bool(torch.isnan(got[bad]).all()), "a row of NaN queries came out finite"
    got[bad] = c.expected(out.dtype, "any")[0][bad] if isinstance(c, LatentCase) \
        else c.expected(out.dtype)[0][bad]
    c.check(got.to(out.dtype))


@pytest.mark.parametrize("ctx", [[40, 200], [3000, 70]])
@pytest.mark.parametrize("hq,hk,d,dtype,n", [
    (8, 2, 64, F32, 2), (8, 2, 64, F32, 8), (8, 2, 128, BF, 7), (32, 4, 64, F16, 6),
    (8, 2, 128, BF, 9), (4, 4, 64, F16, 9), (8, 2, 80, BF, 9)])
# (a capped infinity is the cap)
@pytest.mark.parametrize("value,mods", [
    (math.nan, dict()), (math.inf, dict()), (math.nan, dict(softcap=20.0, slopes="alibi"))])
def test_nan_queries_of_trees(value, ctx, hq, hk, d, dtype, n, mods):
    """A NaN or infinite query element gives NaN scores (an infinite one scores +inf and
    -inf, whose softmax is NaN): the row is NaN whatever kernel takes it and however its
    keys are cut, and the others are untouched."""
    mods = dict(mods)
    if mods.get("slopes"):
        mods["slopes"] = alibi(hq)
    rng = np.random.default_rng(d)
    c = TreeCase(hq=hq, hk=hk, d=d, dtype=dtype, ctx=ctx,
                 parents=[random_tree(rng, n, "random") for _ in ctx], seed=d, **mods)
    rows = [(0, 1), (n + 1, hq - 1)]
    for r in rows:
        c.q_dev[r][3] = value
    _check_nan_rows(c, c.run(out_dtype=dtype), rows)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("ctx", [[40, 200], [3000, 70]])
@pytest.mark.parametrize("hq,dc,dr,dtype,n", [
    (4, 128, 32, F32, 1), (6, 300, 6, F32, 2), (20, 256, 64, F32, 3), (16, 512, 64, BF, 1),
    (16, 256, 64, F16, 3), (40, 512, 64, BF, 9)])
def test_nan_queries_of_latents(value, ctx, hq, dc, dr, dtype, n):
    c = LatentCase(hq=hq, dc=dc, dr=dr, dtype=dtype, ctx=ctx, q_lens=[n, n], seed=dc)
    rows = [(0, 1), (2 * n - 1, hq - 1)]
    for r in rows:
        c.q_dev[0][r][3] = value
    _check_nan_rows(c, c.run(out_dtype=dtype), rows)


@pytest.mark.parametrize("ctx", [[40, 200], [3000, 70]])
@pytest.mark.parametrize("hq,hk,d,dtype,n", [(8, 2, 64, F32, 3), (8, 2, 128, BF, 5),
                                             (4, 4, 64, F16, 100), (8, 2, 80, BF, 9)])
def test_nan_queries_of_scored_chains(ctx, hq, hk, d, dtype, n):
    n = min(n, min(ctx))
    c = ScoredCase(hq=hq, hk=hk, d=d, dtype=dtype, ctx=ctx, q_lens=[n, n], softcap=20.0,
                   slopes=alibi(hq), seed=d)
    rows = [(0, 1), (2 * n - 1, hq - 1)]
    for r in rows:
        c.q_dev[r][3] = math.nan
    _check_nan_rows(c, c.run(out_dtype=dtype), rows)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_accept_of_rows_without_nodes(latent, as_tensor):
    """A padded row (no context) of a decode batch, and a sequence without nodes: empty
    paths raise nothing, and the others move; a path that asks such a row for a node
    raises the flag of its fault."""
    from chenxing_b200 import (LatentBatch, LatentPagedKVCache, PagedBatch, RadixPagedKVCache,
                               _lib)
    if latent:
        cache = LatentPagedKVCache(6, 16, 2, 64, 16, dtype=BF, host_io=False)
        pools, make = [cache.kv_pool], LatentBatch
        kw = dict(n_q_heads=4, scale=1.0)
    else:
        cache = RadixPagedKVCache(6, 16, 2, 2, 64, dtype=BF, host_io=False)
        pools, make = [cache.k_pool, cache.v_pool], PagedBatch
        kw = dict(n_q_heads=4)
    gen = torch.Generator().manual_seed(1)
    for p in pools:
        p.copy_(torch.randn(p.shape, generator=gen).to(BF))
    before = [p.clone() for p in pools]

    def accept(batch, paths):
        width = max(map(len, paths)) + 1
        cache.accept_paths(batch, torch.tensor([p + [-1] * (width - len(p)) for p in paths],
                                               device="cuda") if as_tensor else paths)
        return _lib.device_flags(clear=True)

    decode = make(cache, [[1], [], [3, 4]], [5, 0, 20], **kw)
    assert accept(decode, [[0], [], [0]]) == 0             # (in place already)
    drafted = make(cache, [[1], [], [3, 4], [5]], [5, 0, 20, 7], q_lens=[3, 0, 4, 0], **kw)
    assert all(torch.equal(p, b) for p, b in zip(pools, before))
    assert accept(drafted, [[1, 2], [], [0, 3], []]) == 0
    for p, b in zip(pools, before):
        assert torch.equal(p[:, 1, 2:4], b[:, 1, 3:5])
        assert torch.equal(p[:, 4, 1], b[:, 4, 3]) and torch.equal(p[:, 4, 0], b[:, 4, 0])
    if as_tensor:
        assert accept(drafted, [[], [], [], [0]]) == 64    # no such node
        assert accept(decode, [[], [0], []]) == 16         # no context


def test_fp32_queries_beyond_fp16():
    """Rounded to the pool's type they are infinite: the row is NaN, no other is touched.
    Over a bf16 pool, and where the fp32 kernels take the call, the same query is finite."""
    for dtype, bs in ((F16, 16), (BF, 16), (F16, 20)):
        c = LatentCase(hq=16, dc=128, dr=64, ctx=[200, 70], dtype=dtype, q_dtype=F32, bs=bs, seed=3)
        kind = c.batch().kernel_kind(F32)
        assert kind == ("generic" if bs == 20 else "tcgen05")
        c.q_dev[0][1, 2, 5] = 1e5
        if dtype == F16 and kind == "tcgen05":
            _check_nan_rows(c, c.run(out_dtype=F32), [(1, 2)])
        else:
            assert bool(torch.isfinite(c.run(out_dtype=F32)).all())


# ---------------------------------------------------------------------------
# placement of tcgen05 trees, chains as trees, long chunks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B", [32, 33, 64, 100, 128, 129])
@pytest.mark.parametrize("lengths", ["equal", "distinct", "some"])
def test_many_trees_on_tcgen05(B, lengths):
    """The longest contexts start first, ranked 32 at a time up to 128 sequences: every
    sequence's rows are written once, with ties, ranks across the groups of 32 and
    sequences without nodes; long tables cut the keys over several CTAs up to 64."""
    rng = np.random.default_rng(B)
    sizes = [9 if lengths == "equal" or i % 7 else 0 for i in range(B)]
    if lengths == "equal":
        ctx = [40] * B
    elif lengths == "distinct":
        ctx = (12 + rng.permutation(B)).tolist()
    else:
        ctx = [12 + int(x) for x in rng.integers(0, 4, B) * 16]
    ctx[B // 2] = 1100
    c = TreeCase(hq=4, hk=1, d=64, dtype=BF, ctx=ctx, seed=B,
                 parents=[random_tree(rng, n, "random") for n in sizes])
    batch = c.batch()
    assert batch.kernel_kind(BF, BF) == "tcgen05"
    a = c.run(batch, out_dtype=BF)
    c.check(a)
    assert torch.equal(a, c.run(batch, out_dtype=BF))


@pytest.mark.parametrize("hq,hk,d,dtype,n,same", [
    (8, 2, 128, BF, 7, True), (8, 8, 64, F16, 20, True), (4, 2, 96, F16, 8, True),
    (8, 2, 64, F32, 2, True), (8, 2, 128, BF, 13, False), (8, 2, 64, F32, 8, False),
    (8, 2, 128, BF, 40, False)])
def test_a_chain_as_a_tree(hq, hk, d, dtype, n, same):
    """`same`: chain and tree run one kernel, whose sums then have one order, bit for bit;
    elsewhere both are within their bounds, and so of each other."""
    from chenxing_b200 import PagedBatch
    c = TreeCase(hq=hq, hk=hk, d=d, dtype=dtype, ctx=[n + 200, n + 31], softcap=30.0, window=19,
                 q_scale=4.0, parents=[random_tree(None, n, "chain")] * 2, seed=d)
    tree_batch = c.batch()
    chain_batch = PagedBatch(c.cache, c.tables, c.ctx, n_q_heads=hq, q_lens=c.q_lens,
                             window=c.window, softcap=c.softcap, scale=c.scale)
    tree, chain = c.run(tree_batch, out_dtype=dtype), c.run(chain_batch, out_dtype=dtype)
    c.check(tree)
    c.check(chain)
    if same:
        assert tree_batch.kernel_kind(dtype, dtype) == chain_batch.kernel_kind(dtype, dtype)
        assert torch.equal(tree, chain)
    _, tol = c.expected(dtype)
    assert bool(((tree - chain).double().abs().cpu() <= 2 * tol).all())


@pytest.mark.parametrize("hq,dc,dr,dtype", [(16, 512, 64, BF), (4, 256, 64, F16), (3, 128, 32, F32)])
@pytest.mark.parametrize("window", [None, 100])
def test_long_chunks_over_latents(hq, dc, dr, dtype, window):
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=[700, 301, 64], q_lens=[300, 301, 5], dtype=dtype,
                   window=window, seed=dr)
    c.check(c.run(out_dtype=dtype))


# ---------------------------------------------------------------------------
# the engine: 16-bit pools, a tree behind a tail block that two sequences share
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("latent", [False, True])
def test_engine_tree_behind_a_shared_tail(latent, dtype):
    """Sequence 1 shares sequence 0's partly filled tail block, drafts a tree behind it and
    keeps a path: the block is copied first, sequence 0 keeps its rows, and the cache holds
    for sequence 1 what decoding the path alone would have left."""
    from chenxing_b200 import BatchedKVEngine, LatentPagedKVCache, RadixPagedKVCache, RopeTables
    hq, L = 8, 2

    def engine():
        if latent:
            return BatchedKVEngine(LatentPagedKVCache(32, 16, L, 128, 64, dtype=dtype,
                                                      host_io=False), n_q_heads=hq, scale=0.07)
        return BatchedKVEngine(RadixPagedKVCache(32, 16, L, 2, 64, dtype=dtype, host_io=False),
                               n_q_heads=hq)

    gen = torch.Generator().manual_seed(3)
    rope = RopeTables(256, 64)
    one = torch.ones(64, device="cuda")

    def rows(n):
        make = (lambda *s: torch.randn(n, *s, generator=gen).to(dtype).cuda())
        kv = [(make(128), make(64)) if latent else (make(2, 64), make(2, 64)) for _ in range(L)]
        return kv, [make(hq, 192 if latent else 64) for _ in range(L)]

    def step(eng, ids, q_lens, new, qs, **kw):
        plan = eng.plan(ids, q_lens, verify=True, **kw)
        outs = []
        for layer, (k, v) in enumerate(new):
            q = eng.append_rope(plan, layer, k, v, rope, qs[layer][..., -64:],
                                **({} if latent else dict(k_weight=one)))
            outs.append(eng.attend(plan, layer, (qs[layer][..., :128], q) if latent else q))
        return plan, outs

    def read(eng, i, layer, n):
        return eng.cache.read_layer(eng.seqs[i].block_table, n, layer)

    eng, ref = engine(), engine()
    tokens = list(range(21))
    first, q0 = rows(21)
    n0 = 15                                        # committed of sequence 1, in a shared block
    for e, i, n in ((eng, 0, 21), (ref, 0, 21), (ref, 1, n0)):
        e.add(i, tokens[:n])
        plan, _ = step(e, [i], [n], [(k[:n], v[:n]) for k, v in first], [q[:n] for q in q0])
        e.commit(plan)
    assert eng.add(1, tokens[:n0] + [90], share_tail_from=0).n_tokens == n0
    assert eng.seqs[1].block_table == eng.seqs[0].block_table[:1]
    kept = [[t.clone() for t in read(eng, 0, layer, 21)] for layer in range(L)]
    new, qs = rows(6)
    plan, outs = step(eng, [1], [6], new, qs, tree_parents=[[-1, -1, 0, 1, 1, 4]])
    assert eng.seqs[1].block_table[0] != eng.seqs[0].block_table[0]
    path = [1, 4, 5]
    eng.accept(plan, [path])
    keep = torch.tensor(path).cuda()
    plan, want = step(ref, [1], [3], [(k[keep], v[keep]) for k, v in new], [q[keep] for q in qs])
    ref.commit(plan)
    assert eng.seqs[1].n_tokens == ref.seqs[1].n_tokens == n0 + 3
    for layer in range(L):
        for x, y in zip(read(eng, 1, layer, n0 + 3), read(ref, 1, layer, n0 + 3)):
            assert torch.equal(x, y)
        for x, y in zip(read(eng, 0, layer, 21), kept[layer]):
            assert torch.equal(x, y)
        # the same scores to fp32; each side rounds its probabilities to the pool's type (of
        # sums of p |v| up to max |v|), fp16 those below its smallest step too
        v = read(ref, 1, layer, n0 + 3)[0 if latent else 1].float().abs().max()
        bound = 2 * (HALF[dtype] + 2.0 ** -16 + (n0 + 3) * 2.0 ** -25) * v
        assert bool(((outs[layer][keep] - want[layer]).abs() <= bound).all())


# ---------------------------------------------------------------------------
# device flags
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("unit", ["scored", "tree", "latent"])
def test_flags_of_every_unit_are_read_and_cleared(unit):
    from chenxing_b200 import _lib
    if unit == "latent":
        c = LatentCase(hq=4, dc=128, dr=64, ctx=[100], dtype=BF, poison=False)
    elif unit == "tree":
        c = TreeCase(hq=8, hk=2, d=64, ctx=[100], parents=[[-1, 0]], poison=False)
    else:
        c = ScoredCase(hq=8, hk=2, d=64, ctx=[100], softcap=30.0, poison=False)
    batch = c.batch()
    batch.block_tables[0, 2] = c.cache.n_blocks + 5
    c.run(batch, out_dtype=BF)
    assert [_lib.device_flags(clear=x) for x in (False, False, True, True, False)] == [2, 2, 2, 0, 0]


@pytest.mark.parametrize("clear", [False, True])
def test_reading_the_flags_copies_once(clear):
    """One launch collects the words of all units, one copy brings them to the host."""
    from torch.profiler import ProfilerActivity, profile

    from chenxing_b200 import _lib
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA],
                 acc_events=True) as prof:
        assert _lib.device_flags(clear=clear) == 0
    calls = {e.key: e.count for e in prof.key_averages()}
    if not calls.get("cudaStreamSynchronize"):
        pytest.skip("the profiler sees no runtime calls here")
    assert calls["cudaStreamSynchronize"] == calls.get("cudaMemcpyAsync") == 1
    assert calls.get("cudaLaunchKernel", 0) + calls.get("cudaLaunchKernelExC", 0) == 1


def test_flags_read_on_streams_by_many_threads():
    from concurrent.futures import ThreadPoolExecutor

    from chenxing_b200 import _lib

    def read(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            return [_lib.device_flags(clear=i % 2 == 0) for _ in range(50)]
    with ThreadPoolExecutor(8) as pool:
        assert not any(sum(pool.map(read, range(8)), []))
