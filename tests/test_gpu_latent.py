"""The latent cache and its attention against their definitions in float64 (bounds:
tree_cases)."""
import numpy as np
import pytest
import torch

from tree_cases import LatentCase, random_tree

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_flags():
    from chenxing_b200 import _lib
    _lib.device_flags(clear=True)
    yield
    flags = _lib.device_flags(clear=True)
    assert flags == 0, f"device error flags raised: {_lib.describe_flags(flags)}"


CTX = [1, 15, 63, 64, 65, 0, 300, 129, 1000]


@pytest.mark.parametrize("hq,dc,dr,dtype,bs", [
    (16, 512, 64, BF, 16), (1, 512, 64, BF, 16), (128, 512, 64, BF, 16), (32, 512, 64, F16, 16),
    (64, 256, 64, BF, 16), (20, 320, 64, F16, 16), (16, 128, 32, BF, 16), (5, 384, 64, BF, 32),
    (40, 448, 64, BF, 64), (8, 88, 8, BF, 16), (3, 200, 40, F16, 16), (7, 512, 16, BF, 16),
    (80, 64, 64, BF, 16), (8, 128, 32, F32, 16), (3, 512, 64, F32, 16), (16, 256, 32, BF, 8),
    (4, 50, 6, BF, 16), (9, 300, 2, F32, 1), (2, 31, 2, F16, 128)])
def test_decode(hq, dc, dr, dtype, bs):
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=CTX, dtype=dtype, bs=bs, seed=hq + dc)
    c.check(c.run(out_dtype=dtype))


@pytest.mark.parametrize("hq,dc,dr,dtype", [
    (16, 512, 64, BF), (5, 256, 64, F16), (128, 512, 64, BF), (1, 128, 32, BF), (3, 128, 32, F32),
    (16, 512, 64, F32), (12, 300, 6, F32), (5, 50, 6, BF), (2, 383, 10, F16), (9, 257, 2, F32)])
@pytest.mark.parametrize("window", [None, 1, 37, 100])
@pytest.mark.parametrize("ctx,q_lens", [
    ([1, 5, 17, 64, 200, 66, 333], [1, 5, 4, 0, 5, 2, 3]),
    ([70, 500, 129], [70, 1, 33])])
def test_chains(hq, dc, dr, dtype, window, ctx, q_lens):
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=ctx, q_lens=q_lens, dtype=dtype, window=window, seed=dc)
    c.check(c.run(out_dtype=dtype))


@pytest.mark.parametrize("hq,dc,dr,dtype,bs", [
    (16, 512, 64, BF, 16), (4, 256, 64, F16, 32), (2, 128, 32, F32, 16), (128, 512, 64, BF, 16),
    (1, 64, 8, F32, 16), (7, 320, 64, F32, 5), (3, 64, 16, BF, 24)])
@pytest.mark.parametrize("kind", ["random", "star", "chain", "deep"])
@pytest.mark.parametrize("window", [None, 3, 50])
def test_trees(hq, dc, dr, dtype, bs, kind, window):
    rng = np.random.default_rng(dc + len(kind))
    sizes, ctx = [1, 16, 7, 0, 33, 70], [1, 16, 260, 40, 97, 200]
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=ctx, dtype=dtype, bs=bs, window=window, seed=3,
                   parents=[random_tree(rng, n, kind) for n in sizes])
    c.check(c.run(out_dtype=dtype))


@pytest.mark.parametrize("dtype,q_dtype,out_dtype", [
    (BF, F32, F32), (BF, BF, F16), (F16, F32, BF), (F16, BF, F16), (F32, BF, F32), (F32, F16, BF),
    (BF, F16, BF)])
@pytest.mark.parametrize("strides", ["plain", "heads", "one", "odd"])
def test_types_and_strides(dtype, q_dtype, out_dtype, strides):
    c = LatentCase(hq=6, dc=256, dr=64, ctx=[70, 300], q_lens=[3, 20], dtype=dtype,
                   q_dtype=q_dtype, strides=strides, seed=11)
    c.check(c.run(out_dtype=out_dtype))


@pytest.mark.parametrize("ctx,q_lens,hq", [
    ([20000], None, 16), ([9000, 3, 5000], None, 128), ([12000, 40], [2, 40], 64),
    ([64 * 5] * 40, None, 16), ([700] * 300, None, 4)])
def test_cut_ranges(ctx, q_lens, hq):
    """Contexts cut over many CTAs, many sequences a CTA; bit-equal from call to call."""
    c = LatentCase(hq=hq, dc=512, dr=64, ctx=ctx, q_lens=q_lens, dtype=BF, seed=5)
    batch = c.batch()
    a = c.run(batch, out_dtype=BF)
    c.check(a)
    assert torch.equal(a, c.run(batch, out_dtype=BF))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("scale", [0.0, -0.05, 0.5])
def test_scales_and_growing_scores(dtype, scale):
    """Scores that grow along the context, so that the references move."""
    c = LatentCase(hq=20, dc=256, dr=64, ctx=[900, 333], q_lens=[2, 5], dtype=dtype, scale=scale,
                   seed=8)
    for b, rows in enumerate(c.rows):
        rows *= torch.linspace(0.05, 2.0, rows.shape[0])[:, None]
        rows.copy_(rows.to(dtype).double())
        t, pos = torch.tensor(c.tables[b]), torch.arange(rows.shape[0])
        c.cache.kv_pool[0][t.cuda()[pos.cuda() // 16], pos.cuda() % 16] = rows.to(dtype).cuda()
    c.check(c.run(out_dtype=F32))


@pytest.mark.parametrize("hq,dc,dr,dtype,bs", [(8, 128, 32, F32, 16), (64, 384, 64, F32, 16),
                                               (3, 50, 6, BF, 16), (40, 70, 2, F16, 1)])
def test_cut_contexts_of_the_fp32_kernels(hq, dc, dr, dtype, bs):
    c = LatentCase(hq=hq, dc=dc, dr=dr, ctx=[3000, 1, 0, 777], dtype=dtype, bs=bs, seed=12)
    batch = c.batch()
    assert batch.kernel_kind(dtype) == "generic"
    a = c.run(batch, out_dtype=F32)
    c.check(a)
    assert torch.equal(a, c.run(batch, out_dtype=F32))


def test_last_layer_and_larger_table():
    c = LatentCase(hq=16, dc=128, dr=64, ctx=[130, 64], dtype=BF, n_layers=3, layer=2, seed=4)
    c.check(c.run(c.batch(table_stride=500), out_dtype=BF))


def test_out_given_and_rows_behind_the_last_sequence():
    c = LatentCase(hq=16, dc=256, dr=64, ctx=[130, 64], q_lens=[3, 2], dtype=BF, seed=4)
    room = torch.full((9, 16, 256), 7.0, dtype=BF, device="cuda")
    out = c.run(out=room[:5])
    c.check(out)
    assert out.data_ptr() == room.data_ptr() and bool((room[5:] == 7.0).all())


def test_other_stream_and_graph():
    c = LatentCase(hq=16, dc=512, dr=64, ctx=[700, 64, 90], dtype=BF, seed=6)
    batch = c.batch()
    want = c.run(batch, out_dtype=BF)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = c.run(batch, out_dtype=BF)
    side.synchronize()
    assert torch.equal(want, got)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(batch, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, out)


def test_bad_block_ids_leave_their_keys_out():
    from chenxing_b200 import _lib
    c = LatentCase(hq=16, dc=128, dr=64, ctx=[200, 64], dtype=BF, seed=9)
    batch = c.batch()
    batch.block_tables[0, 3] = 10 ** 6
    batch.block_tables[0, 7] = -5
    out = c.run(batch, out_dtype=F32)
    assert _lib.device_flags(clear=True) == 2
    hidden = list(range(48, 64)) + list(range(112, 128))
    want, tol = c.expected(F32, "tcgen05", hidden)
    assert bool(((out[0].double().cpu() - want[0]).abs() <= tol[0]).all())


@pytest.mark.parametrize("hq,q_lens", [(4, None), (16, [3])])
def test_bad_block_ids_in_fp32(hq, q_lens):
    from chenxing_b200 import _lib
    c = LatentCase(hq=hq, dc=128, dr=32, ctx=[200], q_lens=q_lens, dtype=F32, seed=9)
    batch = c.batch()
    batch.block_tables[0, 3] = 10 ** 6
    batch.block_tables[0, 7] = -5
    out = c.run(batch)
    assert _lib.device_flags(clear=True) == 2
    c.check(out, hidden=list(range(48, 64)) + list(range(112, 128)))


@pytest.mark.parametrize("hq,dtype", [(16, BF), (64, F16), (8, F32), (40, F32)])
def test_batches_on_two_streams_at_once(hq, dtype):
    """A batch a stream, each with a workspace of its own; the same calls one by one."""
    c = LatentCase(hq=hq, dc=256, dr=64, ctx=[2500, 333], dtype=dtype, seed=4)
    batches = [c.batch() for _ in range(2)]
    want = c.run(batches[0], out_dtype=dtype)
    c.check(want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for b, st in zip(batches, streams):
            with torch.cuda.stream(st):
                outs.append(c.run(b, out_dtype=dtype))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_wait_limit():
    """Waits that run out end the call with an error, and the next call is right."""
    from chenxing_b200 import _lib
    c = LatentCase(hq=64, dc=512, dr=64, ctx=[30000, 20000], dtype=BF, seed=2)
    batch = c.batch()
    _lib.lib().cx_set_wait_limit_ns(1)
    try:
        c.run(batch, out_dtype=BF)
        torch.cuda.synchronize()
        flags = _lib.device_flags(clear=True)
    finally:
        _lib.lib().cx_set_wait_limit_ns(0)
    assert flags == 8
    c.check(c.run(batch, out_dtype=BF))


# ---------------------------------------------------------------------------
# append, read, copies
# ---------------------------------------------------------------------------
def _turned(x, cos, sin, inter):
    """x (T, .., dr) float64 turned by table rows (T, dr)."""
    half = x.shape[-1] // 2
    y = x.clone()
    shape = (x.shape[0],) + (1,) * (x.dim() - 2)
    for p in range(half):
        a, b = (2 * p, 2 * p + 1) if inter else (p, p + half)
        ta, tb = (p, p) if inter else (p, p + half)
        ca, sa, cb, sb = (t.reshape(shape) for t in (cos[:, ta], sin[:, ta], cos[:, tb],
                                                     sin[:, tb]))
        y[..., a] = x[..., a] * ca - x[..., b] * sa
        y[..., b] = x[..., b] * cb + x[..., a] * sb
    return y


@pytest.mark.parametrize("T,hq,dc,dr,src,pool_dtype", [
    (1, 16, 512, 64, BF, BF), (8, 16, 512, 64, F32, BF), (37, 5, 320, 32, BF, F16),
    (300, 32, 256, 64, F16, F16), (9, 128, 512, 64, BF, F32), (5, 3, 50, 6, F32, F32),
    (4, 0, 512, 64, BF, BF), (6, 2, 136, 48, BF, BF), (3, 1, 128, 128, F32, BF)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fused", [True, False])
def test_append(T, hq, dc, dr, src, pool_dtype, inter, norm, fused):
    """Bounds: the rotation's two products and one sum, 3 roundings of fp32 relative to
    |x| + |y|; the norm's sum of dc squares, its root and two products, (dc / 2 + 6)
    2^-24; one rounding to the destination: half a step, relative to the value, or in
    fp16 below 2^-14, where its step is 2^-24 whatever the value, 2^-25."""
    from chenxing_b200 import LatentPagedKVCache, RopeTables
    gen = torch.Generator().manual_seed(T + dc)
    h = {F32: 2.0 ** -24, BF: 2.0 ** -8, F16: 2.0 ** -11}
    if fused:
        kv = torch.randn(T, dc + dr, generator=gen).to(src).cuda()
        lat, kr = kv[:, :dc], kv[:, dc:]
        q = torch.randn(T, max(hq, 1), 16 + dr, generator=gen).to(src).cuda()[..., 16:]
    else:
        lat = torch.randn(T, dc, generator=gen).to(src).cuda()
        kr = torch.randn(T, dr, generator=gen).to(src).cuda()
        q = torch.randn(T, max(hq, 1), dr, generator=gen).to(src).cuda()
    w = (1 + 0.3 * torch.randn(dc, generator=gen)).to(src).cuda() if norm else None
    cache = LatentPagedKVCache(2 * T // 16 + 3, 16, 2, dc, dr, dtype=pool_dtype, host_io=False)
    cache.kv_pool.fill_(3.0)
    slots = torch.randperm(cache.n_blocks * 16, generator=gen)[:T]
    if T > 3:
        slots[2] = -1
    pos = torch.randint(0, 500, (T,), generator=gen)
    rope = RopeTables(500, dr, interleaved=inter)
    got = cache.append_norm_rope(1, lat, kr, slots, pos, rope, q if hq else None, weight=w,
                                 eps=1e-5)
    cos, sin = rope.cos.cpu().double()[pos], rope.sin.cpu().double()[pos]

    def near(a, b, bound, dt):
        tol = bound + h[dt] * (b.abs() + bound) + (2.0 ** -25 if dt == F16 else 0.0)
        over = float(((a.double().cpu() - b).abs() - tol).max()) if b.numel() else 0.0
        assert over <= 0.0, f"{over} above the bound"

    x = lat.double().cpu()
    want, bound = x, torch.zeros_like(x)
    if norm:
        want = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double().cpu()
        bound = want.abs() * (dc / 2 + 6) * 2.0 ** -24
    live = slots >= 0
    flat = cache.kv_pool[1].reshape(-1, dc + dr)
    rows = flat[slots[live].cuda()]
    near(rows[:, :dc], want[live], bound[live], pool_dtype)

    def turn_bound(x):
        y = x.abs()
        return (y + y.amax(-1, keepdim=True)) * 3 * 2.0 ** -24

    k = kr.double().cpu()
    near(rows[:, dc:], _turned(k, cos, sin, inter)[live], turn_bound(k)[live], pool_dtype)
    if hq:
        near(got, _turned(q.double().cpu(), cos, sin, inter), turn_bound(q.double().cpu()), src)
    else:
        assert got is None
    # nothing else was written
    other = torch.ones(flat.shape[0], dtype=torch.bool)
    other[slots[live]] = False
    assert bool((flat[other.cuda()] == 3.0).all()) and bool((cache.kv_pool[0] == 3.0).all())


def test_positions_and_slots_out_of_range():
    from chenxing_b200 import LatentPagedKVCache, RopeTables, _lib
    cache = LatentPagedKVCache(2, 16, 1, 128, 64, dtype=BF, host_io=False)
    rope = RopeTables(10, 64)
    lat, kr = torch.ones(3, 128, dtype=BF, device="cuda"), torch.ones(3, 64, dtype=BF, device="cuda")
    cache.append_norm_rope(0, lat, kr, torch.tensor([0, 1, 2]), torch.tensor([0, 10, -1]), rope)
    assert _lib.device_flags(clear=True) == 32
    assert float(cache.kv_pool[0, 0, 1:3].abs().sum()) == 0.0
    cache.append_norm_rope(0, lat, kr, torch.tensor([32, 5, 6]), torch.tensor([0, 1, 2]), rope)
    assert _lib.device_flags(clear=True) == 1


@pytest.mark.parametrize("dtype,dc,dr,bs", [(F32, 128, 32, 16), (BF, 512, 64, 16), (F16, 50, 6, 5),
                                            (BF, 31, 2, 7)])
def test_write_read_copy(dtype, dc, dr, bs):
    from chenxing_b200 import LatentPagedKVCache
    gen = torch.Generator().manual_seed(dc)
    cache = LatentPagedKVCache(12, bs, 2, dc, dr, dtype=dtype, host_io=False)
    n = 3 * bs - 2
    lat, kr = torch.randn(n, dc, generator=gen).to(dtype), torch.randn(n, dr, generator=gen).to(dtype)
    table = [7, 2, 9]
    for layer in (0, 1):
        cache.write_layer(table, 0, layer, lat * (layer + 1), kr)
        a, b = cache.read_layer(table, n, layer)
        assert torch.equal(a.cpu(), lat * (layer + 1)) and torch.equal(b.cpu(), kr)
    cache.copy_blocks([7, 2, 9], [0, 1, 3])
    for layer in (0, 1):
        a, b = cache.read_layer([0, 1, 3], n, layer)
        assert torch.equal(a.cpu(), lat * (layer + 1)) and torch.equal(b.cpu(), kr)
    cache.append_batch(1, lat[:1] * 0, kr[:1] * 0, [4 * bs + bs - 1],
                       cow=([7], [4], [bs - 1]))
    a, _ = cache.read_layer([4], bs, 1)
    assert torch.equal(a[:bs - 1].cpu(), lat[:bs - 1] * 2) and float(a[-1].abs().sum()) == 0.0
    assert cache.read_layer([], 5, 0)[0].shape == (0, dc)
