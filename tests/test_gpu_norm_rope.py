"""append_norm_rope against its definition in float64.

Bound per rotated element, ``u`` = 2^-24: the mean of squares (a sum of D
products in fp32: relative ``(D + 2) u``, halved by the root), rsqrt (2 ulp)
and three products give each normed element a relative error below
``e = (D / 2 + 10) u``; a pair's rotation adds two products and a sum, so
``|error| <= (e + 4 u) (|a cos| + |b sin|)``, plus half a step of the type it
is stored in.  Rows that are copied keep their bits.
"""
import numpy as np
import pytest
import torch

from conftest import record_margin
from scored_cases import HALF

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_flags():
    from chenxing_b200 import _lib
    _lib.device_flags(clear=True)
    yield
    flags = _lib.device_flags(clear=True)
    assert flags == 0, f"device error flags raised: {_lib.describe_flags(flags)}"


def tables(rows, rot, **kw):
    from chenxing_b200 import build_rope_cache
    return build_rope_cache(rows, rot, **kw)


class Rows:
    """A step's rows and where they go."""

    def __init__(self, T, hq, hk, d, rot, *, dtype=BF, pool=None, inter=False, norm="qk",
                 w_dtype=None, layout="fused", bs=16, seed=0, eps=1e-6, max_pos=600, skip=(),
                 n_layers=1, layer=0, x_scale=1.0):
        from chenxing_b200 import RadixPagedKVCache, RopeTables
        gen = torch.Generator().manual_seed(seed)
        self.T, self.hq, self.hk, self.d, self.rot, self.inter = T, hq, hk, d, rot, inter
        self.eps, self.layer, self.bs = eps, layer, bs
        pool = pool or dtype
        nb = -(-max(T, 1) // bs) + 4
        self.cache = RadixPagedKVCache(nb, bs, n_layers, hk, d, dtype=pool, host_io=False)
        self.cache.k_pool.fill_(3.0)
        self.cache.v_pool.fill_(5.0)
        x = (torch.randn(T, hq + 2 * hk, d, generator=gen) * x_scale).to(dtype)
        self.q, self.k, self.v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        if layout == "fused":
            y = x.cuda()
            self.dev = (y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:])
        elif layout == "heads-first":       # (H, T, D) seen as (T, H, D)
            self.dev = tuple(a.permute(1, 0, 2).contiguous().cuda().permute(1, 0, 2)
                             for a in (self.q, self.k, self.v))
        elif layout == "odd":               # rows that start off 16 bytes
            y = torch.zeros(T, (hq + 2 * hk) * d + 3, dtype=dtype)
            y[:, 1:-2] = x.reshape(T, -1)
            y = y.cuda()[:, 1:-2].view(T, hq + 2 * hk, d) if T else x.cuda()
            self.dev = (y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:])
        else:
            self.dev = tuple(a.contiguous().cuda() for a in (self.q, self.k, self.v))
        w = (1 + 0.3 * torch.randn(2, d, generator=gen)).to(w_dtype or dtype)
        self.qw = w[0] if "q" in norm else None
        self.kw = w[1] if "k" in norm else None
        self.slots = torch.randperm(nb * bs, generator=gen)[:T]
        for t in skip:
            self.slots[t] = -1
        self.pos = torch.randint(0, max_pos, (T,), generator=gen)
        if T:
            self.pos[0], self.pos[-1] = max_pos - 1, 0
        self.cos, self.sin = tables(max_pos, rot)
        self.rope = RopeTables(max_pos, rot, interleaved=inter, tables=(self.cos, self.sin))

    def call(self, **kw):
        q, k, v = self.dev
        cu = lambda w: None if w is None else w.cuda()  # noqa: E731
        return self.cache.append_norm_rope(self.layer, k, v, self.slots.cuda(), self.pos.cuda(),
                                           self.rope, q, q_weight=cu(self.qw),
                                           k_weight=cu(self.kw), eps=self.eps, **kw)

    def turned(self, x, w, out_dtype):
        """(values, bounds) in float64."""
        u = 2.0 ** -24
        e = 0.0
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.eps) * w.double()
            e = (self.d / 2 + 10) * u
        y, tol = x.clone(), x.abs() * e
        c = torch.from_numpy(self.cos).double()[self.pos][:, None]
        s = torch.from_numpy(self.sin).double()[self.pos][:, None]
        half = self.rot // 2
        if self.inter:
            ia, ib = torch.arange(half) * 2, torch.arange(half) * 2 + 1
            ta = tb = torch.arange(half)
        else:
            ia, ib = torch.arange(half), torch.arange(half) + half
            ta, tb = ia, ib
        a, b = x[..., ia], x[..., ib]
        y[..., ia] = a * c[..., ta] - b * s[..., ta]
        y[..., ib] = b * c[..., tb] + a * s[..., tb]
        tol[..., ia] = (e + 4 * u) * ((a * c[..., ta]).abs() + (b * s[..., ta]).abs())
        tol[..., ib] = (e + 4 * u) * ((b * c[..., tb]).abs() + (a * s[..., tb]).abs())
        least = 2.0 ** -25 if out_dtype == F16 else 2.0 ** -134
        return y, tol + HALF[out_dtype] * (y.abs() + tol) + least

    def check(self, q_out):
        def near(got, want, tol):
            worst = float(((got.double().cpu() - want).abs() / tol).max()) if want.numel() else 0.
            assert torch.isfinite(got).all()
            record_margin(worst)
            assert worst <= 1.0, f"error {worst:.3f} times its bound"

        want, tol = self.turned(self.q, self.qw, q_out.dtype)
        near(q_out, want, tol)
        pool_dt = self.cache.torch_dtype
        kp, vp = self.cache.k_pool.cpu(), self.cache.v_pool.cpu()
        kept = self.slots >= 0
        at = self.slots[kept]
        want, tol = self.turned(self.k, self.kw, pool_dt)
        near(kp[self.layer, at // self.bs, at % self.bs], want[kept], tol[kept])
        assert torch.equal(vp[self.layer, at // self.bs, at % self.bs],
                           self.v[kept].float().to(pool_dt))
        kp[self.layer, at // self.bs, at % self.bs] = 3.0     # all else is as it was
        vp[self.layer, at // self.bs, at % self.bs] = 5.0
        assert (kp == 3).all() and (vp == 5).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 32), (64, 64), (64, 16), (80, 80), (80, 20),
                                   (96, 48), (256, 256), (256, 64), (40, 2), (6, 4), (33, 12),
                                   (72, 72), (160, 96)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_heads_and_rotations(d, rot, inter, dtype):
    r = Rows(19, 6, 2, d, rot, dtype=dtype, inter=inter, seed=d + rot)
    r.check(r.call())


@pytest.mark.parametrize("T", [1, 2, 7, 64, 333, 2049])
@pytest.mark.parametrize("hq,hk", [(8, 2), (1, 1), (7, 7), (32, 8)])
def test_token_and_head_counts(T, hq, hk):
    r = Rows(T, hq, hk, 64, 64, dtype=F16, seed=T, skip=range(T // 3, T // 2))
    r.check(r.call())


@pytest.mark.parametrize("T,d,rot,dtype,pool,hq,hk", [
    (1400, 128, 128, BF, BF, 32, 8), (3000, 64, 16, F32, F32, 17, 3),
    (2600, 96, 24, F16, F16, 24, 4), (2000, 256, 128, F32, BF, 4, 2), (3000, 80, 40, BF, BF, 24, 4)])
@pytest.mark.parametrize("inter", [False, True])
def test_staged_form_for_much_data(T, d, rot, dtype, pool, hq, hk, inter):
    """From 14 MB of rows a CTA copies several tokens ahead into shared memory."""
    r = Rows(T, hq, hk, d, rot, dtype=dtype, pool=pool, inter=inter, seed=d, skip=range(0, T, 7))
    r.check(r.call(q_out_dtype=pool))


@pytest.mark.parametrize("layout", ["fused", "heads-first", "odd", "contiguous"])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("norm", ["qk", "q", "k", ""])
def test_layouts_and_norms(layout, dtype, norm):
    r = Rows(21, 4, 2, 128, 64, dtype=dtype, layout=layout, norm=norm)
    r.check(r.call())


@pytest.mark.parametrize("dtype,pool,q_out,w", [
    (F32, BF, BF, F32), (BF, F32, F32, F32), (BF, F16, F16, BF), (F16, F16, F32, F32),
    (F16, BF, BF, F16), (F32, F16, F32, F32)])
@pytest.mark.parametrize("d", [64, 36])
def test_type_mixes(dtype, pool, q_out, w, d):
    r = Rows(9, 4, 2, d, d, dtype=dtype, pool=pool, w_dtype=w)
    out = r.call(q_out_dtype=q_out)
    assert out.dtype == q_out
    r.check(out)


@pytest.mark.parametrize("bs", [1, 7, 32])
def test_block_sizes_and_layers(bs):
    r = Rows(50, 4, 2, 64, 32, bs=bs, n_layers=3, layer=1)
    r.check(r.call())


def test_zero_rows_and_large_values():
    r = Rows(8, 2, 2, 64, 64, dtype=F32, x_scale=1e15)       # squares up to 1e31
    r.check(r.call())
    r = Rows(8, 2, 2, 64, 64, dtype=F32, x_scale=0.0)        # 0 * rsqrt(eps) = 0
    r.check(r.call())


def test_no_query_and_no_token():
    r = Rows(5, 2, 2, 64, 64)
    _, k, v = r.dev
    assert r.cache.append_norm_rope(0, k, v, r.slots.cuda(), r.pos.cuda(), r.rope,
                                    k_weight=r.kw.cuda()) is None
    want, tol = r.turned(r.k, r.kw, BF)
    got = r.cache.k_pool.cpu()[0, r.slots // 16, r.slots % 16].double()
    assert bool(((got - want).abs() <= tol).all())
    e = Rows(0, 2, 2, 64, 64)
    assert e.call().shape == (0, 2, 64)


def test_plain_rotation_has_the_bits_of_append_rope():
    """Whole heads, no norm, fp32: the same products and sums as append_rope up
    to contraction (one rounding of a product), the same pool rows for V."""
    r = Rows(40, 4, 2, 64, 64, dtype=F32, norm="")
    r.check(r.call())
    q, k, v = r.dev
    other = Rows(40, 4, 2, 64, 64, dtype=F32, norm="")
    qo = other.cache.append_rope(0, k, v, r.slots.cuda(), r.pos.cuda(), r.rope, q,
                                 q_out_dtype=F32)
    other.check(qo)
    assert torch.equal(other.cache.v_pool, r.cache.v_pool)


def test_scaled_tables_for_long_contexts():
    from chenxing_b200 import RopeTables
    r = Rows(30, 4, 2, 128, 64, dtype=F32, max_pos=20000)
    r.cos, r.sin = tables(20000, 64, scaling_factor=8.0, original_max_pos=2048)
    for dev in ("numpy", "cpu", "cuda"):
        tabs = [x if dev == "numpy" else torch.from_numpy(x).to(dev) for x in (r.cos, r.sin)]
        r.rope = RopeTables(20000, 64, tables=tabs)
        r.check(r.call())
    with pytest.raises(ValueError):
        RopeTables(20000, 32, tables=tabs)


def test_bad_position_and_slot_are_skipped_and_flagged():
    from chenxing_b200 import _lib
    r = Rows(6, 2, 2, 64, 64)
    r.slots[2] = r.cache.n_blocks * r.bs
    out = r.call()
    assert _lib.device_flags(clear=True) == 1
    r.slots[2] = -1
    r.check(out)
    for T, hq, bad in ((6, 2, 3), (3000, 40, 2500)):
        r = Rows(T, hq, 2, 64, 64)
        r.pos[bad] = 600
        out = r.call()
        assert _lib.device_flags(clear=True) == 32
        at = int(r.slots[bad])
        assert (r.cache.k_pool[0, at // 16, at % 16] == 3).all()
        assert (r.cache.v_pool[0, at // 16, at % 16] == 5).all()
        r.pos[bad], r.slots[bad] = 0, -1        # all other rows are right
        want, _ = r.turned(r.q, r.qw, BF)
        out[bad] = want[bad].to(BF).cuda()
        r.check(out)


def test_numpy_rows():
    r = Rows(5, 2, 2, 64, 64, dtype=F32)
    out = r.cache.append_norm_rope(0, r.k.numpy(), r.v.numpy(), r.slots.numpy(), r.pos.numpy(),
                                   r.rope, r.q.numpy(), q_weight=r.qw.numpy(),
                                   k_weight=r.kw.numpy())
    r.check(out)


def test_captured_and_replayed():
    r = Rows(33, 4, 2, 128, 128)
    q, k, v = r.dev
    args = (0, k, v, r.slots.cuda(), r.pos.cuda(), r.rope, q)
    kw = dict(q_weight=r.qw.cuda(), k_weight=r.kw.cuda())
    r.cache.append_norm_rope(*args, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = r.cache.append_norm_rope(*args, **kw)
    r.cache.k_pool.fill_(3.0)
    r.cache.v_pool.fill_(5.0)
    g.replay()
    torch.cuda.synchronize()
    r.check(out)


def test_refusals():
    r = Rows(6, 2, 2, 64, 64)
    q, k, v = r.dev
    s, p = r.slots.cuda(), r.pos.cuda()
    call = r.cache.append_norm_rope
    with pytest.raises(TypeError):
        call(0, k.float(), v, s, p, r.rope, q)
    with pytest.raises(TypeError):
        call(0, k, v, s, p, r.rope, q.half())
    with pytest.raises(ValueError):
        call(0, k[:, :1], v, s, p, r.rope, q)
    with pytest.raises(ValueError):
        call(0, k, v, s, p, r.rope, q[:3])
    with pytest.raises(ValueError):
        call(0, k, v, s[:3], p, r.rope, q)
    with pytest.raises(ValueError):
        call(0, k, v, s, p, r.rope, q, q_weight=torch.ones(63, device="cuda"))
    with pytest.raises(IndexError):
        call(1, k, v, s, p, r.rope, q)
    with pytest.raises(ValueError):
        call(0, k, v, s, p, r.rope, q, eps=-1.0)
    with pytest.raises(ValueError):
        call(0, k, v, s, p, r.rope, q, eps=float("nan"))
    with pytest.raises(TypeError):
        call(0, k, v, s, p, r.rope, q, q_out_dtype=torch.float64)
    wide = Rows(6, 2, 2, 128, 128)
    with pytest.raises(ValueError):
        call(0, k, v, s, p, wide.rope, q)


def test_engine_step_norm_rope_append_attend_with_modifiers():
    """A prompt chunk, a decode step and a speculative chain through the engine:
    append_rope with norms and part-of-head tables, then attend with a cap,
    against the definition on the K/V the pool holds."""
    from chenxing_b200 import BatchedKVEngine, RadixPagedKVCache, RopeTables
    from scored_cases import ScoredCase
    hq, hk, d, rot, cap = 8, 2, 64, 32, 15.0
    cache = RadixPagedKVCache(64, 16, 2, hk, d, dtype=BF, host_io=False)
    eng = BatchedKVEngine(cache, n_q_heads=hq, window=50, softcap=cap)
    rope = RopeTables(512, rot, tables=tables(512, rot))
    gen = torch.Generator().manual_seed(5)
    lens = [70, 33]
    for i, n in enumerate(lens):
        eng.add(i, list(range(1000 * i, 1000 * i + n)))
    w = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(BF).cuda()
    for q_lens in (lens, [1, 1], [4, 3]):
        plan = eng.plan([0, 1], q_lens, prefix_lens=[20, 5])
        T = sum(q_lens)
        for layer in range(2):
            x = torch.randn(T, hq + 2 * hk, d, generator=gen).to(BF).cuda()
            q = eng.append_rope(plan, layer, x[:, hq:hq + hk], x[:, hq + hk:], rope, x[:, :hq],
                                q_weight=w[0], k_weight=w[1])
            out = eng.attend(plan, layer, q, out_dtype=BF)
            c = object.__new__(ScoredCase)
            c.hq, c.hk, c.d, c.dtype, c.q_dtype = hq, hk, d, BF, BF
            c.softcap, c.window, c.slopes, c.prefix = cap, 50, None, [20, 5]
            c.scale, c.q, c.q_lens = d ** -0.5, q.double().cpu(), q_lens
            c.ctx = [int(s.n_tokens + n) for s, n in zip(plan.seqs, q_lens)]
            kv = [cache.read_layer(s.block_table, n, layer) for s, n in zip(plan.seqs, c.ctx)]
            c.k = [a.double().cpu() for a, _ in kv]
            c.v = [b.double().cpu() for _, b in kv]
            c.check(out)
        eng.commit(plan)


def test_ids_are_distinct():
    assert len(np.unique(Rows(300, 1, 1, 8, 8).slots.numpy())) == 300
