"""Edges of the drafted trees, the accepted paths and the latent cache (bounds:
tree_cases)."""
import numpy as np
import pytest
import torch

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
