"""What the engine and the batch pass on to the normalised append and the scored
attention, and what they refuse: host logic only (no GPU needed)."""
import math
from types import SimpleNamespace

import pytest
import torch

from chenxing_b200 import BatchedKVEngine, PagedBatch, _lib
from test_scored_refusals_cpu import _attend, _cache, _pool


class CallsOnly:
    """Stands in for a cache: notes which append an engine makes, and how."""

    head_dim, torch_dtype = 64, torch.float16

    def append_rope(self, layer, k, v, slots, positions, rope, q, q_out_dtype):
        if rope.head_dim != self.head_dim:
            raise ValueError("RoPE tables were built for another head_dim")
        self.last = "append_rope", q_out_dtype

    def append_norm_rope(self, layer, k, v, slots, positions, rope, q, *, q_weight, k_weight, eps,
                         q_out_dtype):
        self.last = "append_norm_rope", q_out_dtype


def append(rot=64, **kw):
    eng = object.__new__(BatchedKVEngine)
    eng.cache = CallsOnly()
    plan = SimpleNamespace(cow_host=[], cow_done=False, positions=torch.zeros(1), slots=None,
                           appended=set())
    eng.append_rope(plan, 0, None, None, SimpleNamespace(head_dim=rot), None, **kw)
    return eng.cache.last


@pytest.mark.parametrize("kw,want", [
    (dict(), ("append_rope", torch.bfloat16)),
    (dict(q_out_dtype=torch.float32), ("append_rope", torch.float32)),
    (dict(q_weight=1), ("append_norm_rope", torch.float16)),    # the pool's type
    (dict(k_weight=1), ("append_norm_rope", torch.float16)),
    (dict(q_weight=1, rot=32), ("append_norm_rope", torch.float16)),
    (dict(k_weight=1, q_out_dtype=torch.float32), ("append_norm_rope", torch.float32))])
def test_engine_query_type(kw, want):
    assert append(**kw) == want


def test_engine_refuses_narrow_tables_unless_they_are_meant():
    with pytest.raises(ValueError):
        append(rot=32)
    with pytest.raises(ValueError):
        append(rot=32, rot_dim=16)
    with pytest.raises(ValueError):
        append(rot=32, rot_dim=16, q_weight=1)
    assert append(rot=32, rot_dim=32)[0] == "append_norm_rope"
    assert append(rot=64, rot_dim=64)[0] == "append_norm_rope"


def test_replan_false_needs_a_plan_of_the_same_entry_point():
    from chenxing_b200.batch import _plans
    b = SimpleNamespace(needs_plan=False, _planned_by="plain")
    assert not _plans(b, None, "plain") and _plans(b, None, "scored")
    assert not _plans(b, False, "plain") and _plans(b, True, "scored")
    with pytest.raises(ValueError):
        _plans(b, False, "scored")
    b._planned_by = "scored"
    with pytest.raises(ValueError):
        _plans(b, False, "plain")
    b._planned_by = None                     # never planned here: the device checks
    assert not _plans(b, False, "plain")


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


@pytest.mark.parametrize("softcap", [1e-50, 1e-40, 9e-31, 2e30, 3e38])
def test_caps_outside_fp32_arithmetic_are_refused(lib, softcap):
    """1e-50 is 0 in fp32, which would mean no cap."""
    with pytest.raises(ValueError):
        PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4, softcap=softcap)
    if softcap > 1e-45:
        assert _attend(lib, mods=dict(softcap=softcap)) == _lib.CX_ERR_SHAPE


@pytest.mark.parametrize("scale", [1e9, -1e9, math.inf])
def test_scale_over_cap_must_be_finite(lib, scale):
    assert _attend(lib, batch=dict(scale=scale), mods=dict(softcap=1e-30)) == _lib.CX_ERR_SHAPE


def test_steep_slopes_are_refused_for_long_contexts(lib):
    """fp32 loses half a unit of a score beside a bias of 2^23."""
    def batch(slope):
        return PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4,
                          alibi_slopes=[0.5, slope, 0.0, 1.0])
    for slope in (2.0 ** 23 / 20, 1e30):
        with pytest.raises(ValueError):
            batch(slope)
    b = batch(2.0 ** 23 / 21)
    with pytest.raises(ValueError):
        b.advance()
    assert b.ctx_host.tolist() == [20, 5]          # as it was


def test_slopes_of_a_bf16_tensor(lib):
    b = PagedBatch(_cache(), [[0]], [4], n_q_heads=2,
                   alibi_slopes=torch.tensor([0.5, 0.25], dtype=torch.bfloat16))
    assert b.alibi_slopes.tolist() == [0.5, 0.25]


def test_kernel_kind_knows_the_output_type(lib):
    """A batch without modifiers changes the entry point with its output type."""
    f16 = _cache()
    f16.cx_pool = lambda: _pool(dtype=_lib.CX_F16)
    b = PagedBatch(f16, [[0, 1], [2]], [20, 5], n_q_heads=4)
    assert b.kernel_kind(torch.float16) == "generic"
    assert b.kernel_kind(torch.float16, torch.float16) == "mma"
    assert b.kernel_kind(torch.float16, out_dtype=torch.bfloat16) == "mma"
    b = PagedBatch(f16, [[0, 1], [2]], [20, 5], n_q_heads=4, softcap=5.0)
    assert b.kernel_kind(torch.float16) == b.kernel_kind(torch.float16, torch.float16) == "mma"
    b = PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4)
    assert b.kernel_kind() == b.kernel_kind(out_dtype=torch.float16) == "mma"


@pytest.mark.parametrize("dtype", [_lib.CX_BF16, _lib.CX_F16, _lib.CX_F32])
def test_prompt_chunks_size_no_split_workspace(lib, dtype):
    """Above 64 packed rows no kernel of either entry point reads a split-K plan."""
    pool = _pool(dtype=dtype, n_kv_heads=8, head_dim=128)

    def need(fn, max_q):
        return fn(pool, _lib.CxAttnBatch(0x100, 512, 0x200, 0x300, 4, max_q, 32, 0.1, 0, 0))
    assert need(lib.cx_paged_workspace_bytes, 1024) <= 1 << 20
    assert need(lib.cx_paged_attend_workspace_bytes, 1024) <= 1 << 20
    assert need(lib.cx_paged_workspace_bytes, 17) <= 1 << 20
    rows = 4 * 8 * 15 * 4                    # partial rows of the batch's ranges at least
    assert need(lib.cx_paged_workspace_bytes, 15) > rows * 130 * 4
    assert need(lib.cx_paged_attend_workspace_bytes, 15) > rows * 130 * 4


def test_kept_prefixes_are_for_the_same_sequences(lib):
    def batch():
        return PagedBatch(_cache(), [[0, 1], [2], []], [20, 5, 0], n_q_heads=4,
                          prefix_lens=[3, 9, 0])
    for tables, ctx in (([[0, 1, 4], [2, 5], []], [40, 17, 0]),     # grown
                        ([[0], [2], []], [16, 4, 0]), ([[0, 1], [2], []], [21, 6, 0])):
        b = batch()
        b.set(tables, ctx)
        assert b.prefix_lens.tolist() == [3, 9, 0]
    for tables, ctx in (([[2], [0, 1], []], [5, 20, 0]), ([[0, 3], [2], []], [20, 5, 0]),
                        ([[0, 1], [6], []], [20, 5, 0]), ([[0, 1], [2], [3]], [20, 5, 1]),
                        ([[0, 1], [], []], [20, 0, 0])):
        b = batch()
        with pytest.raises(ValueError):
            b.set(tables, ctx)
        assert b.ctx_host.tolist() == [20, 5, 0]
        b.set(tables, ctx, prefix_lens=[1, 1, 1])
        assert b.prefix_lens.tolist() == [1, 1, 1]


@pytest.mark.parametrize("kw", [
    dict(q_lens=[9, 1]), dict(q_lens=[1]), dict(q_lens=[-1, 2]), dict(q_lens=None),
    dict(q_lens=[1, 1], prefix_lens=[1]), dict(q_lens=[1, 1], ctx=[99, 1])])
def test_a_refused_reload_leaves_the_batch_as_it_was(lib, kw):
    """Its struct's pointers are those of the tensors it holds."""
    b = PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4, q_lens=[3, 2],
                   prefix_lens=[2, 0])

    def state():
        c = b.c_struct()
        return (b.batch, b.max_q, b.total_q, b.ctx_host.tolist(), b.q_lens_host.tolist(),
                b.block_tables.tolist(), b.ctx_lens.tolist(), b.q_start.tolist(),
                b.prefix_lens.tolist(), c.batch, c.max_q_len, c.block_tables, c.ctx_lens,
                c.q_start, b.block_tables.data_ptr(), b.ctx_lens.data_ptr(), b.q_start.data_ptr())
    was = state()
    with pytest.raises((ValueError, TypeError)):
        b.set([[0, 3], [2]], kw.pop("ctx", [8, 8]), **{"prefix_lens": [1, 1], **kw})
    assert state() == was


def test_a_device_without_an_index_is_the_current_one(monkeypatch):
    """A cache made on "cuda" stays on that device when another becomes current."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for dev in (None, "cuda", torch.device("cuda")):
        assert _lib.require_cuda(dev) == torch.device("cuda", 3)
    assert _lib.require_cuda("cuda:1") == torch.device("cuda", 1)
    with pytest.raises(_lib.CxError):
        _lib.require_cuda("cpu")


def test_overlap():
    from chenxing_b200._arrays import overlap
    x = torch.zeros(4, 6, 8)
    assert overlap(x, x) and overlap(x[1:], x[:2]) and overlap(x[:, :2], x[:, 3:])
    assert not overlap(x[:2], x[2:]) and not overlap(x[0, :3], x[0, 3:])
    assert not overlap(x[:0], x) and not overlap(x, torch.zeros(4))
    assert overlap(x[:1].expand(4, 6, 8), x[0]) and not overlap(x[:1].expand(4, 6, 8), x[1])
