"""Paged attention with capped scores, distance bias, visible prefixes and
16-bit outputs against its definition in float64 (bounds: scored_cases)."""
import pytest
import torch

from scored_cases import ScoredCase, alibi

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
    "cap": dict(softcap=30.0, q_scale=4.0),
    "tight-cap": dict(softcap=3.0, q_scale=6.0),
    "alibi": dict(slopes="alibi"),
    "cap-alibi-window": dict(softcap=20.0, slopes="alibi", window=37, q_scale=3.0),
    "window-prefix": dict(window=40, prefix=21),
    "prefix": dict(prefix=50),
    "window-prefix-cap": dict(window=100, prefix=33, softcap=50.0, q_scale=3.0),
    "plain": dict(),
}


def _case(mods, hq, ctx, **kw):
    m = dict(MODS[mods])
    if m.get("slopes"):
        m["slopes"] = alibi(hq)
    if m.get("prefix"):
        m["prefix"] = [min(m["prefix"] + 3 * b, 2 * c + 1) for b, c in enumerate(ctx)]
    m.update(kw)
    return ScoredCase(hq=hq, ctx=ctx, **m)


def _out(mods, dtype):
    """The pool's type; bf16 where an unmodified fp32 output would be
    cx_paged_decode's or cx_paged_verify's, which promise less of dead slots."""
    return BF if mods == "plain" and dtype == F32 else dtype


DECODE_CTX = [1, 15, 16, 17, 300, 33, 0, 129, 640]


@pytest.mark.parametrize("mods", list(MODS))
@pytest.mark.parametrize("hq,hk,d,dtype", [
    (8, 2, 64, F32), (8, 8, 128, F32), (32, 8, 128, BF), (16, 16, 64, BF), (7, 1, 128, F16),
    (24, 8, 64, F16), (12, 4, 96, BF), (4, 2, 256, F16), (6, 3, 40, F32), (20, 1, 128, BF),
    (64, 1, 64, BF)])
def test_decode(mods, hq, hk, d, dtype):
    c = _case(mods, hq, DECODE_CTX, hk=hk, d=d, dtype=dtype, seed=hq + d)
    c.check(c.run(out_dtype=_out(mods, dtype)))


@pytest.mark.parametrize("mods", list(MODS))
@pytest.mark.parametrize("hq,hk,d,dtype", [
    (8, 2, 64, F32), (4, 4, 128, F32), (32, 8, 128, BF), (8, 8, 64, F16), (6, 2, 128, BF),
    (5, 1, 64, F16), (4, 2, 80, BF)])
def test_verify_chains(mods, hq, hk, d, dtype):
    ctx = [1, 5, 17, 31, 200, 64, 333]
    q_lens = [1, 5, 4, 0, 5, 2, 3]
    c = _case(mods, hq, ctx, q_lens=q_lens, hk=hk, d=d, dtype=dtype, seed=d)
    c.check(c.run(out_dtype=_out(mods, dtype)))


@pytest.mark.parametrize("mods", list(MODS))
@pytest.mark.parametrize("hq,hk,d,dtype,q_lens,ctx", [
    (8, 2, 128, BF, [70, 16, 1, 33], [70, 500, 129, 127]),       # one query tile
    (8, 2, 128, BF, [200, 64, 131, 1], [200, 777, 131, 90]),     # several tiles, ragged
    (4, 4, 64, F16, [300, 129], [300, 1000]),
    (6, 2, 128, F16, [90, 43], [211, 43]),                       # 3 heads a group: 126 of 128 rows
    (14, 2, 64, BF, [40, 19], [300, 19]),                        # 7 heads a group
    (2, 1, 96, BF, [50], [130]),
])
def test_prompt_chunks(mods, hq, hk, d, dtype, q_lens, ctx):
    c = _case(mods, hq, ctx, q_lens=q_lens, hk=hk, d=d, dtype=dtype, seed=sum(ctx))
    c.check(c.run(out_dtype=_out(mods, dtype)))


@pytest.mark.parametrize("dtype,out_dtype,q_dtype", [
    (BF, F32, BF), (BF, F16, F32), (F16, BF, F16), (F16, F32, F32), (F32, BF, F32),
    (F32, F16, BF), (BF, BF, F16)])
@pytest.mark.parametrize("q_lens", [None, [3, 40]])
def test_type_mixes(dtype, out_dtype, q_dtype, q_lens):
    c = _case("cap", 8, [70, 300], hk=2, d=128, dtype=dtype, q_dtype=q_dtype, q_lens=q_lens)
    c.check(c.run(out_dtype=out_dtype))


@pytest.mark.parametrize("mods", ["cap", "alibi", "window-prefix-cap", "prefix"])
@pytest.mark.parametrize("hq,hk,d,dtype,q_lens,ctx", [
    (4, 1, 128, BF, [33], [5000]),                    # one tile, its keys over many CTAs
    (2, 2, 64, F16, [300, 70], [4100, 70]),           # two sequences, one too short to split
    (96, 1, 64, BF, None, [3000, 1, 0]),              # one token of 96 heads on one KV head
    (5, 1, 128, F16, [1, 60, 0], [2500, 900, 40]),
])
def test_key_tiles_split_over_ctas(mods, hq, hk, d, dtype, q_lens, ctx):
    c = _case(mods, hq, ctx, q_lens=q_lens, hk=hk, d=d, dtype=dtype, seed=7)
    batch = c.batch()
    assert batch.kernel_kind(dtype) == "tcgen05"
    a = c.run(batch, out_dtype=dtype)
    c.check(a)
    assert torch.equal(a, c.run(batch, out_dtype=dtype))


@pytest.mark.parametrize("softcap", [3e-6, 1e-3, 0.3, 3e3, 1e5])
@pytest.mark.parametrize("q_lens", [None, [40, 60]])
def test_extreme_caps(softcap, q_lens):
    """Coefficients beyond fp32's range on either side, rows of zero scores."""
    c = _case("plain", 8, [70, 300], hk=2, d=128, dtype=BF, q_lens=q_lens, softcap=softcap)
    c.check(c.run(out_dtype=BF))
    c.q_dev.zero_()
    c.q.zero_()
    c.check(c.run(out_dtype=BF))


@pytest.mark.parametrize("hq,hk,ctx", [(8, 2, [120000, 300, 80000]), (32, 8, [50000, 300, 20000])])
def test_wait_timeout_returns_and_flags(hq, hk, ctx):
    """Pipeline waits that run out (more K and V than L2 holds, a limit of a few
    ns; four producer warps and one): the call returns with the flag raised, and
    the next one has the bits of the one before."""
    from chenxing_b200 import _lib
    c = _case("cap", hq, ctx, hk=hk, d=128, dtype=BF)
    batch = c.batch()
    ref = c.run(batch, out_dtype=BF)
    lib = _lib.lib()
    try:
        lib.cx_set_wait_limit_ns(5)
        c.run(batch, out_dtype=BF)
        flags = _lib.device_flags(clear=True)
    finally:
        lib.cx_set_wait_limit_ns(0)
    assert flags & 8, f"expected a wait timeout, flags = {_lib.describe_flags(flags)}"
    batch.needs_plan = True
    assert torch.equal(c.run(batch, out_dtype=BF), ref)
    assert _lib.device_flags(clear=True) == 0


def test_no_query_row():
    c = _case("cap", 8, [70, 300], hk=2, d=64, dtype=BF, q_lens=[0, 0])
    assert c.run(out_dtype=BF).shape == (0, 8, 64)


@pytest.mark.parametrize("q_scale", [1.0, 12.0])
def test_scores_on_both_sides_of_the_polynomial(q_scale):
    """|z| = |score| / cap below 0.8 for every key, and beyond it for most."""
    c = _case("plain", 8, [700, 640], hk=4, d=128, dtype=F16, q_lens=[300, 90], softcap=12.0,
              q_scale=q_scale)
    c.check(c.run(out_dtype=F16))


@pytest.mark.parametrize("q_lens", [None, [3, 5], [3, 80]])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_query_heads_of_a_fused_projection(dtype, q_lens):
    c = _case("alibi", 8, [90, 222], hk=2, d=128, dtype=dtype, q_lens=q_lens, strided=True)
    assert not c.q_dev.is_contiguous()
    c.check(c.run(out_dtype=dtype))


@pytest.mark.parametrize("bs", [1, 8, 32])
def test_other_block_sizes(bs):
    c = _case("window-prefix-cap", 8, [70, 300, 1], hk=2, d=64, dtype=BF, bs=bs, seed=bs)
    c.check(c.run(out_dtype=BF))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
@pytest.mark.parametrize("q_lens", [None, [4, 5], [40, 60]])
def test_scales(scale, q_lens):
    c = _case("cap", 8, [70, 300], hk=2, d=128, q_lens=q_lens, scale=scale)
    c.check(c.run(out_dtype=BF))


def test_long_context_is_split_and_joined():
    """One sequence over all SMs, its ranges merged by ticket; twice the same bits."""
    c = _case("alibi", 8, [20000], hk=8, d=64, dtype=F16, seed=3)
    batch = c.batch()
    a = c.run(batch, out_dtype=F16)
    b = c.run(batch, out_dtype=F16)
    c.check(a)
    assert torch.equal(a, b)


@pytest.mark.parametrize("hq,hk,d,dtype,q", [
    (8, 2, 64, BF, 7), (8, 2, 64, F16, 5), (4, 4, 64, BF, 20), (4, 1, 128, BF, 1), (8, 2, 128, F16, 6),
    (8, 1, 64, BF, 1), (4, 2, 128, F32, 1), (4, 1, 128, F32, 2), (8, 8, 64, F32, 1),
    (4, 2, 64, F32, 3), (12, 4, 128, F32, 4)])
def test_rings_that_wrap_many_times(hq, hk, d, dtype, q):
    """Contexts of several hundred blocks a CTA: every ring length goes round often
    under all its producer warps (their number divides it), twice the same bits."""
    ctx = [30000, 33, 9001, 25000]
    c = _case("plain", hq, ctx, hk=hk, d=d, dtype=dtype, q_lens=None if q == 1 else [q] * 4,
              softcap=30.0)
    batch = c.batch()
    a = c.run(batch, out_dtype=dtype)
    c.check(a)
    for _ in range(3):
        assert torch.equal(a, c.run(batch, out_dtype=dtype))


@pytest.mark.parametrize("mods", ["cap-alibi-window", "window-prefix-cap", "prefix", "alibi"])
@pytest.mark.parametrize("hq,hk,d,dtype,ctx,q_lens", [
    (16, 4, 128, BF, [6000], [6]),                          # one range over every CTA
    (8, 8, 64, F16, [40, 4000, 0, 900], None),              # two head groups, an empty sequence
    (4, 2, 128, F32, [33, 5000, 20], [2, 3, 0]),
    (3, 1, 64, F32, [2500], None),
    (8, 4, 64, F16, [40] * 40 + [9000] + [25] * 39, [3] * 80),   # more ranges than half the CTAs
    (8, 1, 128, BF, [9000, 7000] + [70] * 98, [5, 1] + [2] * 98),
])
def test_ranges_cut_into_many_partials(mods, hq, hk, d, dtype, ctx, q_lens):
    c = _case(mods, hq, ctx, q_lens=q_lens, hk=hk, d=d, dtype=dtype, seed=11)
    batch = c.batch()
    a = c.run(batch, out_dtype=dtype)
    c.check(a)
    b = a.clone().fill_(float("nan"))
    for _ in range(2):
        c.run(batch, out=b)
        assert torch.equal(a, b)


@pytest.mark.parametrize("hq,hk,d,q_lens", [(8, 2, 128, None), (32, 8, 64, [5, 3]),
                                            (8, 2, 128, [64, 100])])
def test_no_modifier_matches_the_plain_entry_point(hq, hk, d, q_lens):
    c = _case("plain", hq, [100, 513], hk=hk, d=d, dtype=BF, q_lens=q_lens, poison=False)
    a = c.run(out_dtype=BF)
    b = c.run()                        # cx_paged_decode / cx_paged_verify, fp32 output
    assert b.dtype == F32
    c.check(a)
    c.check(b)


def test_one_batch_through_both_entry_points():
    """Each entry point makes its own plan; neither reads the other's."""
    c = _case("plain", 8, [100, 513, 40], hk=2, d=64, dtype=F16, poison=False)
    batch = c.batch()
    for dt in (F16, F32, F16, BF, F32):
        c.check(c.run(batch, out_dtype=dt))


def test_plan_of_a_generic_call_serves_the_next_layer():
    """The first layer's queries are off 16 bytes (generic kernel), the second's
    are not: its split-K kernel finds the step's plan."""
    c = _case("cap", 8, [100, 513, 40], hk=2, d=64, dtype=BF)
    odd = torch.zeros(3 * 8 * 64 + 1, dtype=BF, device="cuda")[1:].view(3, 8, 64)
    odd.copy_(c.q_dev)
    batch = c.batch()
    c.check(c.cache.decode_batch(0, odd, batch, out_dtype=BF))
    assert not batch.needs_plan
    c.check(c.run(batch, out_dtype=BF))


KIND = {"decode": None, "chain": [3, 5], "chunk": [40, 70]}


@pytest.mark.parametrize("shape,dtype,d,kind", [
    ("decode", BF, 64, "mma"), ("decode", F16, 128, "mma"), ("chain", F16, 64, "mma"),
    ("decode", F32, 64, "fma"), ("chain", F32, 128, "fma"), ("decode", BF, 96, "generic"),
    ("chunk", F32, 64, "generic"), ("chunk", BF, 128, "tcgen05"), ("chunk", F16, 64, "tcgen05")])
def test_kernel_choice(shape, dtype, d, kind):
    c = _case("cap", 8, [70, 300], hk=2, d=d, dtype=dtype, q_lens=KIND[shape])
    assert c.batch().kernel_kind(dtype) == kind


def test_out_argument_and_untouched_rows():
    c = _case("cap", 8, [70, 300], hk=2, d=64, dtype=BF, q_lens=[3, 2])
    buf = torch.full((9, 8, 64), 7.0, dtype=BF, device="cuda")
    out = c.run(out=buf[2:7])
    assert out.data_ptr() == buf[2:7].data_ptr()
    c.check(out)
    assert (buf[:2] == 7).all() and (buf[7:] == 7).all()


def test_batch_reload_keeps_or_replaces_the_prefix():
    c = _case("window-prefix", 8, [70, 300], hk=2, d=64, dtype=BF)
    batch = c.batch()
    c.check(c.run(batch, out_dtype=BF))
    batch.set(c.tables, c.ctx)
    c.check(c.run(batch, out_dtype=BF))
    c.prefix = [0, 9]                  # inside the old one: what it showed holds no NaN
    batch.set(c.tables, c.ctx, prefix_lens=c.prefix)
    c.check(c.run(batch, out_dtype=BF))
    with pytest.raises(ValueError):
        batch.set(c.tables[:1], c.ctx[:1])


def test_second_layer_and_other_stream():
    c = _case("cap", 8, [70, 300], hk=2, d=64, dtype=BF, n_layers=3, layer=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = c.run(out_dtype=BF)
    torch.cuda.current_stream().wait_stream(s)
    c.check(out)


@pytest.mark.parametrize("q_lens,dtype", [(None, BF), (None, F32), ([3, 5], BF), ([40, 70], F16)])
def test_captured_and_replayed(q_lens, dtype):
    c = _case("cap-alibi-window", 8, [70, 300], hk=2, d=64, dtype=dtype, q_lens=q_lens)
    batch = c.batch()
    out = c.run(batch, out_dtype=dtype)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(batch, out=out, replan=True)
        c.run(batch, out=out, replan=False)
    for _ in range(3):
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        c.check(out)


def test_bad_block_id_is_left_out_and_flagged():
    """Ids outside the pool can only be written past the host check."""
    from chenxing_b200 import _lib
    for q_lens, dtype in ((None, BF), ([3], BF), ([40], BF), (None, F32)):
        c = _case("cap", 8, [100], hk=2, d=64, dtype=dtype, q_lens=q_lens)
        batch = c.batch()
        batch.block_tables[0, 2] = c.cache.n_blocks + 5
        out = c.run(batch, out_dtype=dtype)
        assert _lib.device_flags(clear=True) == 2
        c.check(out, hidden=range(32, 48))


def test_refusals():
    from chenxing_b200 import PagedBatch
    c = _case("cap", 8, [70], hk=2, d=64, dtype=BF)
    b = c.batch()
    with pytest.raises(ValueError):
        c.run(b, out=torch.empty(1, 8, 64, dtype=BF, device="cuda"), out_dtype=F16)
    with pytest.raises(ValueError):
        c.run(b, out=torch.empty(1, 8, 128, dtype=BF, device="cuda")[:, :, ::2])
    with pytest.raises(TypeError):
        c.run(b, out_dtype=torch.float64)
    with pytest.raises(IndexError):
        c.cache.decode_batch(1, c.q_dev, b, out_dtype=BF)
    with pytest.raises(ValueError):
        c.cache.decode_batch(0, c.q_dev[:, :4], b, out_dtype=BF)
    for kw in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=float("inf")),
               dict(softcap=float("nan")), dict(alibi_slopes=[0.1] * 7),
               dict(alibi_slopes=[-0.1] * 8), dict(alibi_slopes=[float("nan")] * 8),
               dict(prefix_lens=[1, 2]), dict(prefix_lens=[-1])):
        with pytest.raises(ValueError):
            PagedBatch(c.cache, c.tables, c.ctx, n_q_heads=8, **kw)
