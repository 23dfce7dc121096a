"""Argument checks of the norm + rotation append and of the scored attention:
every refusal comes from the host, before any launch (no GPU needed)."""
import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from chenxing_b200 import PagedBatch, _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def _pool(**kw):
    a = dict(k=0x1000, v=0x9000, n_layers=2, n_blocks=8, block_size=16, n_kv_heads=2, head_dim=64,
             dtype=_lib.CX_BF16, reserved=0)
    a.update(kw)
    return _lib.CxPool(*a.values())


def _append(lib, pool=None, layer=0, slots=0x100, positions=0x200, q_out=0x300,
            q_out_dtype=_lib.CX_BF16, rows=None, how=None):
    r = dict(q=0x400, k=0x500, v=0x600, qt=128, qh=64, kt=128, kh=64, vt=128, vh=64, n_tokens=3,
             n_q_heads=2, dtype=_lib.CX_BF16, reserved=0)
    r.update(rows or {})
    h = dict(q_weight=0x700, k_weight=None, q_weight_dtype=_lib.CX_F32,
             k_weight_dtype=_lib.CX_F32, eps=1e-6, interleaved=0, cos=0x800, sin=0x900,
             table_rows=10, rot_dim=64)
    h.update(how or {})
    return lib.cx_kv_append_norm_rope(pool or _pool(), layer, _lib.CxQkv(*r.values()), slots,
                                      positions, _lib.CxNormRope(*h.values()), q_out, q_out_dtype,
                                      None)


@pytest.mark.parametrize("want,kw", [
    ("CX_ERR_RANGE", dict(layer=2)), ("CX_ERR_RANGE", dict(layer=-1)),
    ("CX_ERR_SHAPE", dict(slots=None)), ("CX_ERR_SHAPE", dict(positions=None)),
    ("CX_ERR_SHAPE", dict(q_out=None)), ("CX_ERR_DTYPE", dict(q_out_dtype=9)),
    ("CX_ERR_SHAPE", dict(rows=dict(q=None))), ("CX_ERR_SHAPE", dict(rows=dict(k=None))),
    ("CX_ERR_SHAPE", dict(rows=dict(n_tokens=-1))), ("CX_ERR_SHAPE", dict(rows=dict(qt=-1))),
    ("CX_ERR_DTYPE", dict(rows=dict(dtype=7), how=dict(q_weight=None))),
    ("CX_ERR_UNSUPPORTED", dict(rows=dict(n_q_heads=1 << 21))),
    ("CX_ERR_SHAPE", dict(how=dict(rot_dim=0))), ("CX_ERR_SHAPE", dict(how=dict(rot_dim=3))),
    ("CX_ERR_SHAPE", dict(how=dict(rot_dim=66))), ("CX_ERR_SHAPE", dict(how=dict(eps=-1.0))),
    ("CX_ERR_SHAPE", dict(how=dict(eps=math.nan))), ("CX_ERR_SHAPE", dict(how=dict(eps=math.inf))),
    ("CX_ERR_SHAPE", dict(how=dict(cos=None))), ("CX_ERR_SHAPE", dict(how=dict(table_rows=-1))),
    ("CX_ERR_DTYPE", dict(how=dict(q_weight_dtype=_lib.CX_F16))),
    ("CX_ERR_SHAPE", dict(pool=_pool(n_blocks=0))), ("CX_ERR_DTYPE", dict(pool=_pool(dtype=5))),
    ("CX_OK", dict(rows=dict(n_tokens=0))),
])
def test_append_norm_rope(lib, want, kw):
    assert _append(lib, **kw) == getattr(_lib, want)


def _attend(lib, pool=None, layer=0, q=0x100, q_dtype=_lib.CX_BF16, out=0x200, batch=None,
            mods=None):
    b = dict(tables=0x1000, stride=4, ctx=0x2000, q_start=None, batch=2, max_q=1, hq=4,
             scale=math.nan, reserved=0, window=0)
    b.update(batch or {})
    m = dict(softcap=30.0, out_dtype=_lib.CX_BF16, slopes=None, prefix=None, q_stride=0)
    m.update(mods or {})
    return lib.cx_paged_attend(pool or _pool(), layer, _lib.CxAttnBatch(*b.values()),
                               _lib.CxAttnMods(*m.values()), q, q_dtype, out, None, 0, 1, None)


@pytest.mark.parametrize("want,kw", [
    ("CX_ERR_RANGE", dict(layer=2)), ("CX_ERR_SHAPE", dict(q=None)),
    ("CX_ERR_SHAPE", dict(out=None)), ("CX_ERR_DTYPE", dict(q_dtype=4)),
    ("CX_ERR_SHAPE", dict(batch=dict(hq=3))), ("CX_ERR_SHAPE", dict(batch=dict(hq=0))),
    ("CX_ERR_SHAPE", dict(batch=dict(batch=-1))), ("CX_ERR_SHAPE", dict(batch=dict(tables=None))),
    ("CX_ERR_SHAPE", dict(batch=dict(stride=0))),
    ("CX_ERR_SHAPE", dict(batch=dict(q_start=0x40, max_q=0))),
    ("CX_ERR_SHAPE", dict(mods=dict(softcap=-1.0))),
    ("CX_ERR_SHAPE", dict(mods=dict(softcap=math.nan))),
    ("CX_ERR_SHAPE", dict(mods=dict(softcap=math.inf))),
    ("CX_ERR_DTYPE", dict(mods=dict(out_dtype=3))),
    ("CX_ERR_SHAPE", dict(mods=dict(q_stride=255))), ("CX_ERR_SHAPE", dict(mods=dict(q_stride=-4))),
    ("CX_ERR_UNSUPPORTED", dict(pool=_pool(head_dim=264))),
    ("CX_ERR_SHAPE", dict(pool=_pool(k=None))), ("CX_OK", dict(batch=dict(batch=0))),
])
def test_paged_attend(lib, want, kw):
    assert _attend(lib, **kw) == getattr(_lib, want)


def test_null_structs(lib):
    assert lib.cx_paged_attend(_pool(), 0, None, None, 1, 1, 1, None, 0, 0, None) \
        == _lib.CX_ERR_SHAPE
    assert lib.cx_kv_append_norm_rope(_pool(), 0, None, 1, 1, None, 1, 1, None) \
        == _lib.CX_ERR_SHAPE


def test_struct_sizes():
    assert ctypes.sizeof(_lib.CxQkv) == 3 * 8 + 6 * 8 + 2 * 8 + 2 * 4
    assert ctypes.sizeof(_lib.CxNormRope) == 2 * 8 + 4 * 4 + 2 * 8 + 2 * 8
    assert ctypes.sizeof(_lib.CxAttnMods) == 2 * 4 + 3 * 8


def _cache():
    return SimpleNamespace(device=torch.device("cpu"), n_kv_heads=2, head_dim=64, block_size=16,
                           n_blocks=8, cx_pool=_pool)


@pytest.mark.parametrize("kw", [
    dict(softcap=0.0), dict(softcap=-2.0), dict(softcap=math.inf), dict(softcap=math.nan),
    dict(alibi_slopes=[0.5] * 3), dict(alibi_slopes=[0.5, 0.5, 0.5, -0.5]),
    dict(alibi_slopes=[math.inf] * 4), dict(prefix_lens=[1]), dict(prefix_lens=[1, -1])])
def test_paged_batch_modifiers(lib, kw):
    with pytest.raises(ValueError):
        PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4, **kw)


def test_paged_batch_counts_and_reload(lib):
    b = PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4, window=4, prefix_lens=[3, 9])
    assert b.scored and b.kv_tokens == (4 + 3) + (4 + 1)
    b.advance()
    assert b.prefix_lens.tolist() == [3, 9] and b.ctx_host.tolist() == [21, 6]
    with pytest.raises(ValueError):
        b.set([[0]], [4])
    b.set([[0]], [4], prefix_lens=[2])
    assert b.prefix_lens.tolist() == [2]
    assert not PagedBatch(_cache(), [[0]], [4], n_q_heads=4).scored
