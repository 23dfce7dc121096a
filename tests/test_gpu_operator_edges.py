"""Calls at the edges of the normalised append's and the scored attention's
documented ranges (definitions and bounds: test_gpu_norm_rope, scored_cases)."""
import pytest
import torch

from scored_cases import ScoredCase, alibi
from test_gpu_norm_rope import Rows

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_flags():
    from chenxing_b200 import _lib
    _lib.device_flags(clear=True)
    yield
    flags = _lib.device_flags(clear=True)
    assert flags == 0, f"device error flags raised: {_lib.describe_flags(flags)}"


@pytest.mark.parametrize("off_k,off_v", [(0, 8), (8, 8), (8, 0)])
@pytest.mark.parametrize("dtype,pool", [(BF, BF), (F32, F16)])
def test_append_of_much_data_into_pools_off_16_bytes(off_k, off_v, dtype, pool):
    """A pool of the caller's own (C interface) may start at any element."""
    r = Rows(2100, 24, 8, 96, 96, dtype=dtype, pool=pool, seed=off_k + off_v)
    pool_c, cache = r.cache._pool, r.cache
    at = pool_c.k, pool_c.v
    moved = []
    try:
        for name, off in (("k", off_k), ("v", off_v)):
            was = getattr(cache, "_" + name)
            buf = torch.zeros(was.numel() + 8, dtype=pool, device="cuda")
            assert buf.data_ptr() % 16 == 0
            part = buf[off // 2:][:was.numel()].view_as(was)
            part.copy_(was)
            setattr(pool_c, name, part.data_ptr())
            moved.append((was, part, buf))
        out = r.call(q_out_dtype=pool)
        for was, part, _ in moved:
            was.copy_(part)
    finally:
        pool_c.k, pool_c.v = at
    r.check(out)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("softcap,q_scale", [(10.0, 12.0), (30.0, 25.0)])
def test_biased_scores_far_beyond_the_cap(softcap, q_scale, dtype):
    """Raw scores of several caps on either side, with a distance bias, on tiles
    that every row sees: the reference maximum follows capped scores only."""
    c = ScoredCase(hq=8, hk=2, d=128, ctx=[900, 700, 333], q_lens=[64, 90, 40], dtype=dtype,
                   softcap=softcap, slopes=alibi(8), q_scale=q_scale, seed=4)
    assert c.batch().kernel_kind(dtype) == "tcgen05"
    c.check(c.run(out_dtype=dtype))


@pytest.mark.parametrize("dtype,rows,kinds", [
    (BF, BF, ("mma", "tcgen05")), (F16, F16, ("mma", "tcgen05")), (F32, F32, ("fma", "generic")),
    (BF, F32, ("mma", "tcgen05")), (F16, BF, ("mma", "tcgen05"))])
def test_engine_step_keeps_the_pools_type(dtype, rows, kinds):
    """Norms, append and attention over bf16, fp16 and fp32 pools: Q comes in the
    pool's type, and the pool's kernel attends."""
    from chenxing_b200 import BatchedKVEngine, RadixPagedKVCache, RopeTables
    hq, hk, d, cap = 8, 2, 64, 15.0
    cache = RadixPagedKVCache(64, 16, 1, hk, d, dtype=dtype, host_io=False)
    eng = BatchedKVEngine(cache, n_q_heads=hq, softcap=cap)
    rope = RopeTables(512, d)
    gen = torch.Generator().manual_seed(6)
    lens = [70, 33]
    for i, n in enumerate(lens):
        eng.add(i, list(range(1000 * i, 1000 * i + n)))
    w = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(rows).cuda()
    for q_lens, kind in ((lens, kinds[1]), ([1, 1], kinds[0])):
        plan = eng.plan([0, 1], q_lens)
        x = torch.randn(sum(q_lens), hq + 2 * hk, d, generator=gen).to(rows).cuda()
        q = eng.append_rope(plan, 0, x[:, hq:hq + hk], x[:, hq + hk:], rope, x[:, :hq],
                            q_weight=w[0], k_weight=w[1])
        assert q.dtype == dtype
        assert plan.batch.kernel_kind(q.dtype) == kind
        out = eng.attend(plan, 0, q, out_dtype=dtype)
        c = object.__new__(ScoredCase)
        c.hq, c.hk, c.d, c.dtype, c.q_dtype = hq, hk, d, dtype, dtype
        c.softcap, c.window, c.slopes, c.prefix = cap, None, None, None
        c.scale, c.q, c.q_lens = d ** -0.5, q.double().cpu(), q_lens
        c.ctx = [int(s.n_tokens + n) for s, n in zip(plan.seqs, q_lens)]
        kv = [cache.read_layer(s.block_table, n, 0) for s, n in zip(plan.seqs, c.ctx)]
        c.k = [a.double().cpu() for a, _ in kv]
        c.v = [b.double().cpu() for _, b in kv]
        c.check(out)
        eng.commit(plan)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_plan_of_another_call_is_refused_on_the_device(dtype):
    """A plan of cx_paged_decode, of another window or without the prefix, given
    to cx_paged_attend with replan = 0 (the C interface does not see whose it is)."""
    from chenxing_b200 import _lib
    c = ScoredCase(hq=8, hk=2, d=64, ctx=[700, 333], dtype=dtype, window=100, prefix=[40, 60],
                   poison=False)
    batch = c.batch()

    def left(plan, out_dtype):
        """Makes `batch` plan as ``plan`` says, then calls it without a plan."""
        good, kept = batch._c, batch.prefix_lens
        plan()
        batch._c, batch.prefix_lens, batch._planned_by = good, kept, None
        out = torch.full((2, 8, 64), 7.0, dtype=out_dtype, device="cuda")
        c.run(batch, out=out, out_dtype=out_dtype, replan=False)
        flags = _lib.device_flags(clear=True)
        return flags, bool((out == 7).all())

    def plain():
        batch.prefix_lens = None
        c.run(batch, out_dtype=F32, replan=True)

    def no_prefix():
        batch.prefix_lens = None
        c.run(batch, out_dtype=BF, replan=True)

    def other_window():
        batch._c = _lib.CxAttnBatch.from_buffer_copy(batch._c)
        batch._c.window = 50
        c.run(batch, out_dtype=BF, replan=True)

    for plan in (plain, no_prefix, other_window):
        assert left(plan, BF) == (16, True), plan.__name__
    batch.needs_plan = True
    c.check(c.run(batch, out_dtype=dtype))


@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** -60])
@pytest.mark.parametrize("q_lens,ctx", [(None, 60000), ([5], 60000), ([60], 1300), ([2, 70], 2500)])
def test_large_and_small_values_under_scores_that_jump(q_lens, ctx, size):
    """Row maxima that grow by 50 powers of two between tiles, in either order of
    the keys, times V far from 1: what is finite stays finite."""
    hq, hk, d = 8, 2, 128
    n = len(q_lens or [1])
    c = ScoredCase(hq=hq, hk=hk, d=d, ctx=[ctx - 300 * b for b in range(n)], q_lens=q_lens,
                   softcap=200.0, poison=False, q_scale=0.0)
    c.q = (1.0 + 0.1 * torch.randn(c.q.shape, generator=torch.Generator().manual_seed(1))).to(BF)
    c.q_dev = c.q.cuda()
    c.q = c.q.double()
    top = 50 * 0.6931 / (d * c.scale)          # adds 50 to a score in base 2
    for b in range(n):
        j = torch.arange(c.ctx[b])
        k = c.k[b] * 0.05 + (top * ((j // 128) % 2))[:, None, None]
        c.k[b] = k.to(BF).double()
        c.v[b] = (c.v[b] * size).to(BF).double()
        t = torch.tensor(c.tables[b])
        c.cache.k_pool[0][t[j // 16].cuda(), (j % 16).cuda()] = c.k[b].to(BF).cuda()
        c.cache.v_pool[0][t[j // 16].cuda(), (j % 16).cuda()] = c.v[b].to(BF).cuda()
    c.check(c.run(out_dtype=BF))


@pytest.mark.parametrize("softcap", [1e-30, 1e30])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64), (F32, 64), (BF, 96)])
@pytest.mark.parametrize("q_lens", [None, [40, 60]])
def test_smallest_and_largest_cap(softcap, dtype, d, q_lens):
    """The mean of the visible V under the one, no cap at all under the other."""
    c = ScoredCase(hq=8, hk=2, d=d, ctx=[70, 300], q_lens=q_lens, dtype=dtype, softcap=softcap)
    batch = c.batch()
    out = c.run(batch, out_dtype=dtype)
    if softcap > 1:
        c.softcap = None
    c.check(out)


@pytest.mark.parametrize("hq,hk,d,dtype,q_lens,ctx", [
    (4, 1, 128, BF, [33], 5000), (8, 2, 64, F16, [200], 3000), (96, 1, 64, BF, None, 3000),
    (8, 2, 128, BF, None, 6000), (4, 2, 64, F32, [3], 5000), (4, 2, 96, BF, [5], 700)])
def test_steepest_slopes(hq, hk, d, dtype, q_lens, ctx):
    """A bias that leaves each row its own key alone: the output is that V row."""
    steep = 2.0 ** 23 / (ctx + 1)
    c = ScoredCase(hq=hq, hk=hk, d=d, ctx=[ctx], q_lens=q_lens, dtype=dtype,
                   slopes=[steep / (1 + h % 3) for h in range(hq)])
    out = c.run(out_dtype=dtype).cpu()
    own = c.v[0][-len(out):].to(dtype).repeat_interleave(hq // hk, 1)
    assert torch.equal(out, own)


def timed_out(call):
    """Flags of ``call`` under a wait limit of a few ns."""
    from chenxing_b200 import _lib
    try:
        _lib.lib().cx_set_wait_limit_ns(5)
        call()
        return _lib.device_flags(clear=True)
    finally:
        _lib.lib().cx_set_wait_limit_ns(0)


@pytest.mark.parametrize("hq,hk,q_lens,ctx", [
    (32, 8, [300, 200, 300, 129], [9000, 3000, 300, 6000]),       # a CTA a pair of query tiles
    (4, 1, [33], [20000])])                                       # keys split over many CTAs
@pytest.mark.parametrize("mods", [dict(softcap=30.0), dict(slopes=True)])
def test_tcgen05_waits_that_run_out_return_and_flag(hq, hk, q_lens, ctx, mods):
    """The call returns with the flag raised; the next one has the bits of the
    one before."""
    if mods.get("slopes"):
        mods = dict(slopes=alibi(hq))
    c = ScoredCase(hq=hq, hk=hk, d=128, ctx=ctx, q_lens=q_lens, **mods)
    batch = c.batch()
    assert batch.kernel_kind() == "tcgen05"
    ref = c.run(batch, out_dtype=BF)
    assert timed_out(lambda: c.run(batch, out_dtype=BF)) == 8
    assert torch.equal(c.run(batch, out_dtype=BF), ref)


def test_staged_append_waits_that_run_out_return_and_flag():
    """Q stored to pinned host memory, which takes a token's rows much longer to
    leave the stage than a copy takes to fill it."""
    from chenxing_b200 import _lib
    r = Rows(3000, 32, 8, 128, 128)
    slots, pos, rope = r.slots.cuda(), r.pos.cuda(), r.rope
    w = [x.cuda() for x in (r.qw, r.kw)]
    st = [n for x in r.dev for n in (x.stride(0), x.stride(1))]
    rows = _lib.CxQkv(*(x.data_ptr() for x in r.dev), *st, r.T, r.hq, _lib.CX_BF16, 0)
    how = _lib.CxNormRope(w[0].data_ptr(), w[1].data_ptr(), _lib.CX_BF16, _lib.CX_BF16, r.eps, 0,
                          rope.cos.data_ptr(), rope.sin.data_ptr(), rope.rows, rope.head_dim)
    host = torch.zeros(r.T, r.hq, r.d, dtype=BF).pin_memory()

    def call():
        _lib.check(_lib.lib().cx_kv_append_norm_rope(
            r.cache.cx_pool(), 0, rows, slots.data_ptr(), pos.data_ptr(), how, host.data_ptr(),
            _lib.CX_BF16, _lib.stream_ptr()), "cx_kv_append_norm_rope")
        torch.cuda.synchronize()
    assert timed_out(call) == 8
    for pool, fill in ((r.cache.k_pool, 3.0), (r.cache.v_pool, 5.0)):
        pool.fill_(fill)
    call()
    r.check(host.cuda())


@pytest.mark.parametrize("clear,most", [(False, 1), (True, 2)])
def test_reading_the_flags_waits_once(clear, most):
    """Two flag words, one wait for both (and one for clearing them)."""
    from torch.profiler import ProfilerActivity, profile

    from chenxing_b200 import _lib
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA],
                 acc_events=True) as prof:
        assert _lib.device_flags(clear=clear) == 0
    waits = sum(e.count for e in prof.key_averages() if e.key == "cudaStreamSynchronize")
    if not waits:
        pytest.skip("the profiler sees no runtime calls here")
    assert waits <= most


@pytest.mark.parametrize("scored", [False, True])
def test_flags_of_both_units_are_read_and_cleared(scored):
    from chenxing_b200 import _lib
    c = ScoredCase(hq=8, hk=2, d=64, ctx=[100], softcap=30.0 if scored else None, poison=False)
    batch = c.batch()
    batch.block_tables[0, 2] = c.cache.n_blocks + 5
    c.run(batch)
    assert _lib.device_flags(clear=False) == 2
    assert _lib.device_flags(clear=True) == 2
    assert _lib.device_flags(clear=True) == 0


@pytest.mark.parametrize("hq,hk,d,dtype,q_lens,ctx", [
    (8, 2, 128, BF, None, [900, 20000, 33]), (8, 2, 64, F16, [6, 3], [9000, 70]),
    (4, 2, 128, F32, [3], [7000]), (8, 2, 128, BF, [300, 64], [700, 129]),
    (4, 1, 64, F16, [40], [9000]), (6, 3, 96, BF, [5, 50], [300, 77])])
def test_output_in_place_of_the_queries(hq, hk, d, dtype, q_lens, ctx):
    c = ScoredCase(hq=hq, hk=hk, d=d, ctx=ctx, q_lens=q_lens, dtype=dtype, softcap=20.0)
    batch = c.batch()
    apart = c.run(batch, out_dtype=dtype)
    c.check(apart)
    own = c.q_dev.clone()
    for _ in range(2):
        c.q_dev = own.clone()
        assert c.run(batch, out=c.q_dev).data_ptr() == c.q_dev.data_ptr()
        assert torch.equal(c.q_dev, apart)


def test_output_over_part_of_the_queries_is_refused():
    c = ScoredCase(hq=8, hk=2, d=64, ctx=[70, 300], q_lens=[3, 2], softcap=20.0)
    buf = torch.zeros(6, 8, 64, dtype=BF, device="cuda")
    buf[:5] = c.q_dev
    c.q_dev = buf[:5]
    with pytest.raises(ValueError):
        c.run(out=buf[1:])
    with pytest.raises(ValueError):        # the same memory as another type
        c.run(out=buf[:5].view(F16))
    wide = torch.zeros(5, 12, 64, dtype=BF, device="cuda")
    wide[:, :8] = c.q_dev
    c.q_dev = wide[:, :8]
    with pytest.raises(ValueError):
        c.run(out=wide.flatten()[:5 * 8 * 64].view(5, 8, 64))
    c.check(c.run(out=torch.empty(5, 8, 64, dtype=BF, device="cuda")))
