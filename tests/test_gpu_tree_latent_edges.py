"""Edges of the drafted trees, the accepted paths and the latent cache (bounds:
tree_cases)."""
import math

import numpy as np
import pytest
import torch

from scored_cases import ScoredCase, alibi
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
