"""Argument checks of the drafted trees, of the accepted paths and of the latent
cache: every refusal comes from the host, before any launch (no GPU needed).  The
masks of a tree are checked against the definition."""
import contextlib
import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from chenxing_b200 import BatchedKVEngine, LatentBatch, PagedBatch, _lib
from chenxing_b200.batch import decode_batch, tree_arrays, verify_batch
from chenxing_b200.engine import KVSequence, StepPlan
from chenxing_b200.latent import LatentPagedKVCache
from chenxing_b200.radix_kv import RadixIndex, _BlockPool


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def _pool(**kw):
    a = dict(k=0x1000, v=0x9000, n_layers=2, n_blocks=8, block_size=16, n_kv_heads=2, head_dim=64,
             dtype=_lib.CX_BF16, reserved=0)
    a.update(kw)
    return _lib.CxPool(*a.values())


def _latent_pool(**kw):
    a = dict(kv=0x1000, n_layers=2, n_blocks=8, block_size=16, latent_dim=128, rope_dim=64,
             dtype=_lib.CX_BF16, reserved=0)
    a.update(kw)
    return _lib.CxLatentPool(*a.values())


def _batch(**kw):
    b = dict(tables=0x1000, stride=4, ctx=0x2000, q_start=0x40, batch=2, max_q=3, hq=4,
             scale=0.1, reserved=0, window=0)
    b.update(kw)
    return _lib.CxAttnBatch(*b.values())


def _tree(**kw):
    t = dict(masks=0x100, words=1, depths=0x200)
    t.update(kw)
    return _lib.CxTree(*t.values())


BAD_POOLS = [("CX_ERR_SHAPE", dict(kv=None)), ("CX_ERR_SHAPE", dict(n_blocks=0)),
             ("CX_ERR_SHAPE", dict(latent_dim=0)), ("CX_ERR_SHAPE", dict(rope_dim=0)),
             ("CX_ERR_SHAPE", dict(rope_dim=63)), ("CX_ERR_UNSUPPORTED", dict(latent_dim=520)),
             ("CX_ERR_UNSUPPORTED", dict(latent_dim=512, rope_dim=66)),
             ("CX_ERR_UNSUPPORTED", dict(n_layers=1 << 16, n_blocks=1 << 16)),
             ("CX_ERR_DTYPE", dict(dtype=5))]


@pytest.mark.parametrize("want,batch,tree,mods", [
    ("CX_ERR_SHAPE", dict(q_start=None), {}, {}), ("CX_ERR_SHAPE", {}, dict(masks=None), {}),
    ("CX_ERR_SHAPE", {}, dict(depths=None), {}), ("CX_ERR_SHAPE", {}, dict(words=0), {}),
    ("CX_ERR_SHAPE", dict(max_q=33), {}, {}), ("CX_ERR_SHAPE", dict(max_q=0), {}, {}),
    ("CX_ERR_SHAPE", {}, dict(words=(1 << 20) + 1), {}), ("CX_ERR_SHAPE", dict(hq=3), {}, {}),
    ("CX_ERR_SHAPE", {}, {}, dict(softcap=math.nan)), ("CX_ERR_DTYPE", {}, {}, dict(out=9)),
    ("CX_ERR_WORKSPACE", {}, {}, {}), ("CX_OK", dict(batch=0), {}, {})])
def test_attend_tree(lib, want, batch, tree, mods):
    m = dict(softcap=0.0, out=_lib.CX_BF16, slopes=None, prefix=None, q_stride=0)
    m.update(mods)
    got = lib.cx_paged_attend_tree(_pool(), 0, _batch(**batch), _lib.CxAttnMods(*m.values()),
                                   _tree(**tree), 0x300, _lib.CX_BF16, 0x400, None, 0, 1, None)
    assert got == getattr(_lib, want)


def test_null_structs(lib):
    assert lib.cx_paged_attend_tree(_pool(), 0, _batch(), None, None, 1, 1, 1, None, 0, 1, None) \
        == _lib.CX_ERR_SHAPE
    assert lib.cx_paged_attend_tree_workspace_bytes(_pool(), None) == 0
    assert lib.cx_latent_attend_workspace_bytes(_latent_pool(), None) == 0
    assert lib.cx_latent_attend_workspace_bytes(_latent_pool(rope_dim=3), _batch()) == 0
    assert lib.cx_latent_attend(_latent_pool(), 0, None, None, None, 1, 0, None, 0, None) \
        == _lib.CX_ERR_SHAPE
    assert lib.cx_latent_append(_latent_pool(), 0, None, 1, None, None, None, 0, None) \
        == _lib.CX_ERR_SHAPE
    assert lib.cx_kv_accept(_pool(), None, 1, 1, 1, None) == _lib.CX_ERR_SHAPE


def test_struct_sizes():
    assert ctypes.sizeof(_lib.CxTree) == 3 * 8
    assert ctypes.sizeof(_lib.CxLatentPool) == 6 * 8 + 2 * 4
    assert ctypes.sizeof(_lib.CxLatentRows) == 3 * 8 + 4 * 8 + 2 * 8 + 2 * 4
    assert ctypes.sizeof(_lib.CxLatentQ) == 2 * 8 + 4 * 8 + 2 * 4


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("want,batch,paths", [
    ("CX_ERR_SHAPE", dict(batch=-1), {}), ("CX_ERR_SHAPE", {}, dict(length=-1)),
    ("CX_ERR_SHAPE", {}, dict(stride=1)), ("CX_ERR_SHAPE", {}, dict(paths=None)),
    ("CX_ERR_SHAPE", dict(tables=None), {}), ("CX_ERR_SHAPE", dict(ctx=None), {}),
    ("CX_ERR_SHAPE", dict(stride=0), {}), ("CX_ERR_UNSUPPORTED", dict(batch=1 << 16), {}),
    ("CX_OK", dict(batch=0), {}), ("CX_OK", {}, dict(length=0))])
def test_accept(lib, latent, want, batch, paths):
    p = dict(paths=0x500, stride=2, length=2)
    p.update(paths)
    fn, pool = (lib.cx_latent_accept, _latent_pool()) if latent else (lib.cx_kv_accept, _pool())
    assert fn(pool, _batch(**batch), *p.values(), None) == getattr(_lib, want)


@pytest.mark.parametrize("want,pool", BAD_POOLS)
def test_latent_pools(lib, want, pool):
    p = _latent_pool(**pool)
    want = getattr(_lib, want)
    q = _lib.CxLatentQ(0x100, 0x200, 512, 128, 256, 64, _lib.CX_BF16, 0)
    rows = _lib.CxLatentRows(0x100, 0x200, None, 128, 64, 0, 0, 3, 0, _lib.CX_BF16, 0)
    how = _lib.CxNormRope(None, None, 0, 0, 0.0, 0, None, None, 0, 0)
    assert lib.cx_latent_attend(p, 0, _batch(), None, q, 0x300, 0, 0x1000, 1 << 30, None) == want
    assert lib.cx_latent_append(p, 0, rows, 0x400, None, how, None, 0, None) == want
    assert lib.cx_latent_gather(p, 0, 0x400, 3, 0x500, 0x600, None) == want
    assert lib.cx_latent_block_copy(p, -1, 0x400, 0x500, None, 1, 1, None) == want
    assert lib.cx_latent_accept(p, _batch(), 0x400, 2, 2, None) == want


@pytest.mark.parametrize("want,kw", [
    ("CX_ERR_RANGE", dict(layer=2)), ("CX_ERR_RANGE", dict(layer=-1)),
    ("CX_ERR_SHAPE", dict(n_tokens=-1)), ("CX_ERR_SHAPE", dict(heads=-1)),
    ("CX_ERR_UNSUPPORTED", dict(n_tokens=1 << 31)), ("CX_ERR_UNSUPPORTED", dict(heads=1 << 21)),
    ("CX_ERR_DTYPE", dict(dtype=4)), ("CX_ERR_DTYPE", dict(q_out_dtype=7)),
    ("CX_ERR_DTYPE", dict(w_dtype=_lib.CX_F16)), ("CX_ERR_SHAPE", dict(eps=-1.0)),
    ("CX_ERR_SHAPE", dict(eps=math.inf)), ("CX_ERR_SHAPE", dict(cos=None)),
    ("CX_ERR_SHAPE", dict(table_rows=-1)), ("CX_ERR_SHAPE", dict(rot_dim=32)),
    ("CX_ERR_SHAPE", dict(positions=None)), ("CX_ERR_SHAPE", dict(lt=-8)),
    ("CX_ERR_SHAPE", dict(slots=None)), ("CX_ERR_SHAPE", dict(latent=None)),
    ("CX_ERR_SHAPE", dict(q=None)), ("CX_ERR_SHAPE", dict(q_out=None)),
    ("CX_OK", dict(n_tokens=0))])
def test_latent_append(lib, want, kw):
    a = dict(layer=0, latent=0x100, rope=0x200, q=0x300, lt=128, n_tokens=3, heads=2,
             dtype=_lib.CX_BF16, slots=0x400, positions=0x500, q_out=0x600,
             q_out_dtype=_lib.CX_BF16, weight=0x700, w_dtype=_lib.CX_F32, eps=1e-6, cos=0x800,
             table_rows=10, rot_dim=64)
    a.update(kw)
    rows = _lib.CxLatentRows(a["latent"], a["rope"], a["q"], a["lt"], 64, 128, 64, a["n_tokens"],
                             a["heads"], a["dtype"], 0)
    how = _lib.CxNormRope(None, a["weight"], 0, a["w_dtype"], a["eps"], 0, a["cos"], 0x900,
                          a["table_rows"], a["rot_dim"])
    assert lib.cx_latent_append(_latent_pool(), a["layer"], rows, a["slots"], a["positions"], how,
                                a["q_out"], a["q_out_dtype"], None) == getattr(_lib, want)


@pytest.mark.parametrize("want,batch,kw", [
    ("CX_ERR_RANGE", {}, dict(layer=2)), ("CX_ERR_SHAPE", dict(batch=-1), {}),
    ("CX_ERR_SHAPE", dict(hq=0), {}), ("CX_ERR_SHAPE", dict(max_q=0), {}),
    ("CX_ERR_DTYPE", {}, dict(dtype=3)), ("CX_ERR_DTYPE", {}, dict(out_dtype=3)),
    ("CX_ERR_SHAPE", {}, dict(stride=-1)), ("CX_ERR_SHAPE", {}, dict(latent=None)),
    ("CX_ERR_SHAPE", {}, dict(out=None)), ("CX_ERR_SHAPE", dict(tables=None), {}),
    ("CX_ERR_SHAPE", dict(stride=0), {}), ("CX_ERR_SHAPE", {}, dict(tree=dict(words=0))),
    ("CX_ERR_SHAPE", dict(max_q=40), dict(tree={})),
    ("CX_ERR_SHAPE", dict(q_start=None), dict(tree={})),
    ("CX_ERR_UNSUPPORTED", dict(stride=1 << 27), {}), ("CX_ERR_UNSUPPORTED", dict(hq=1 << 17), {}),
    ("CX_ERR_UNSUPPORTED", dict(max_q=1 << 20, hq=1 << 12), {}),
    ("CX_ERR_WORKSPACE", {}, dict(ws=None)), ("CX_ERR_WORKSPACE", {}, dict(ws_bytes=64)),
    ("CX_ERR_WORKSPACE", {}, dict(ws=0x1010)), ("CX_OK", dict(batch=0), {})])
def test_latent_attend(lib, want, batch, kw):
    a = dict(layer=0, latent=0x100, stride=128, dtype=_lib.CX_BF16, out=0x300,
             out_dtype=_lib.CX_F32, ws=0x1000, ws_bytes=1 << 40, tree=None)
    a.update(kw)
    q = _lib.CxLatentQ(a["latent"], 0x200, 512, a["stride"], 256, 64, a["dtype"], 0)
    tree = None if a["tree"] is None else _tree(**a["tree"])
    assert lib.cx_latent_attend(_latent_pool(), a["layer"], _batch(**batch), tree, q, a["out"],
                                a["out_dtype"], a["ws"], a["ws_bytes"], None) \
        == getattr(_lib, want)


@pytest.mark.parametrize("want,args", [
    ("CX_ERR_RANGE", (2, 0x400, 3, 0x500, 0x600)), ("CX_ERR_RANGE", (-1, 0x400, 3, 0x500, 0x600)),
    ("CX_ERR_SHAPE", (0, 0x400, -1, 0x500, 0x600)), ("CX_ERR_SHAPE", (0, None, 3, 0x500, 0x600)),
    ("CX_ERR_SHAPE", (0, 0x400, 3, None, 0x600)), ("CX_OK", (0, None, 0, None, None))])
def test_latent_gather(lib, want, args):
    assert lib.cx_latent_gather(_latent_pool(), *args, None) == getattr(_lib, want)


@pytest.mark.parametrize("want,args", [
    ("CX_ERR_RANGE", (2, 0x400, 0x500, None, 1, 1)), ("CX_ERR_SHAPE", (0, 0x400, 0x500, None, -1, 1)),
    ("CX_ERR_SHAPE", (0, 0x400, 0x500, None, 1, 17)), ("CX_ERR_SHAPE", (0, None, 0x500, None, 1, 1)),
    ("CX_OK", (0, None, None, None, 0, 0))])
def test_latent_block_copy(lib, want, args):
    assert lib.cx_latent_block_copy(_latent_pool(), *args, None) == getattr(_lib, want)


def test_latent_kinds(lib):
    kind = lib.cx_latent_attend_kind
    tc, gen = (k for k in sorted(_lib.KERNEL_KINDS, reverse=True) if _lib.KERNEL_KINDS[k] in
               ("tcgen05", "generic"))
    assert kind(_latent_pool(), _batch(), _lib.CX_BF16) == tc
    assert kind(_latent_pool(), _batch(), _lib.CX_F32) == tc
    for q, kw in ((_lib.CX_F16, {}), (_lib.CX_F32, dict(dtype=_lib.CX_F32)),
                  (_lib.CX_BF16, dict(block_size=20)), (_lib.CX_BF16, dict(kv=0x1008)),
                  (_lib.CX_BF16, dict(latent_dim=50, rope_dim=6)),
                  (_lib.CX_BF16, dict(latent_dim=130, rope_dim=64))):
        assert kind(_latent_pool(**kw), _batch(), q) == gen
    assert kind(_latent_pool(block_size=8), _batch(), _lib.CX_BF16) == tc


# ---------------------------------------------------------------------------
# trees
# ---------------------------------------------------------------------------
def _ancestors(parents, i):
    out = [i]
    while parents[i] >= 0:
        i = parents[i]
        out.append(i)
    return out


@pytest.mark.parametrize("window", [0, 1, 2, 5])
@pytest.mark.parametrize("kind", ["random", "chain", "star", "mixed"])
def test_tree_arrays(kind, window):
    rng = np.random.default_rng(1)
    sizes = [0, 1, 7, 32, 33, 70]
    make = {"random": lambda n: [int(rng.integers(-1, i)) if i else -1 for i in range(n)],
            "chain": lambda n: list(range(-1, n - 1)), "star": lambda n: [-1] * n,
            "mixed": lambda n: [(i - 1) // 2 if i else -1 for i in range(n)]}[kind]
    parents = [make(n) for n in sizes]
    masks, depths = tree_arrays(parents, sizes, window)
    assert masks.shape == (sum(sizes), 3) and masks.dtype == np.uint32
    row = 0
    for p in parents:
        for i in range(len(p)):
            up = _ancestors(p, i)
            want = set(up[:window] if window else up)
            assert {u for u in range(96) if masks[row, u // 32] >> (u % 32) & 1} == want
            assert depths[row] == len(up) - 1
            row += 1


@pytest.mark.parametrize("parents,q_lens", [
    ([[0]], [1]), ([[-1, 1]], [2]), ([[-2]], [1]), ([[-1, 2, 0]], [3]), ([[-1]], [2]),
    ([[-1]], [1, 1]), ([[]], [-1])])
def test_tree_arrays_refuses(parents, q_lens):
    with pytest.raises(ValueError):
        tree_arrays(parents, q_lens)


def test_no_tree_at_all():
    masks, depths = tree_arrays([], [])
    assert masks.shape == (0, 1) and depths.shape == (0,)


def _cache():
    return SimpleNamespace(device=torch.device("cpu"), n_kv_heads=2, head_dim=64, block_size=16,
                           n_blocks=8, cx_pool=_pool)


def test_paged_batch_of_trees(lib):
    with pytest.raises(ValueError):
        PagedBatch(_cache(), [[0, 1]], [20], n_q_heads=4, tree_parents=[[-1]])
    b = PagedBatch(_cache(), [[0, 1], [2]], [20, 5], n_q_heads=4, q_lens=[3, 0],
                   tree_parents=[[-1, 0, 0], []])
    assert b.scored and b.depths_host.tolist() == [0, 1, 1]
    assert b.row_positions().tolist() == [17, 18, 18]
    before = b.ctx_host.tolist()
    for kw in (dict(), dict(tree_parents=[[-1, 0], []]), dict(tree_parents=[[-1, 0, 5], []])):
        with pytest.raises(ValueError):
            b.set([[0, 1], [2]], [21, 6], [3, 0], **kw)
        assert b.ctx_host.tolist() == before             # refused whole
    b.set([[0, 1], [2]], [21, 6], [2, 1], tree_parents=[[-1, -1], [-1]])
    assert b.row_positions().tolist() == [19, 19, 5]
    plain = PagedBatch(_cache(), [[0, 1]], [20], n_q_heads=4, q_lens=[2])
    assert plain.row_positions().tolist() == [18, 19]
    with pytest.raises(ValueError):
        plain.set([[0, 1]], [20], [2], tree_parents=[[-1, 0]])


# ---------------------------------------------------------------------------
# the latent cache without its pool in HBM
# ---------------------------------------------------------------------------
def _latent_cache(**kw):
    c = object.__new__(LatentPagedKVCache)
    RadixIndex.__init__(c, 8, 16)
    c.device = torch.device("cpu")
    c.n_layers, c.latent_dim, c.rope_dim, c.n_kv_heads, c.head_dim = 2, 128, 64, 1, 192
    c.torch_dtype, c.host_io = torch.bfloat16, False
    c._pool = _latent_pool(n_blocks=8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw", [dict(latent_dim=0), dict(rope_dim=0), dict(rope_dim=7),
                                dict(latent_dim=513), dict(latent_dim=512, rope_dim=66),
                                dict(n_blocks=0), dict(block_size=0), dict(n_layers=0)])
def test_latent_cache_sizes(kw):
    a = dict(n_blocks=4, block_size=16, n_layers=1, latent_dim=64, rope_dim=16)
    a.update(kw)
    with pytest.raises(ValueError):
        LatentPagedKVCache(**a)


def test_latent_batch(lib):
    c = _latent_cache()
    with pytest.raises(TypeError):
        LatentBatch(_cache(), [[0]], [4], n_q_heads=4, scale=0.1)
    with pytest.raises(TypeError):
        PagedBatch(c, [[0]], [4], n_q_heads=4)
    with pytest.raises(ValueError):
        LatentBatch(c, [[0]], [4], n_q_heads=0, scale=0.1)
    with pytest.raises(ValueError):
        LatentBatch(c, [[0]], [4], n_q_heads=4, scale=0.1, window=0)
    b = LatentBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, scale=0.1, q_lens=[3, 2],
                    tree_parents=[[-1, 0, 0], [-1, 0]])
    assert b.kernel_kind() == "tcgen05" and b.kernel_kind(torch.float16) == "generic"
    assert b.workspace.numel() >= lib.cx_latent_attend_workspace_bytes(c.cx_pool(), b.c_struct())
    with pytest.raises(ValueError):
        b.set([[0, 1], [2]], [20, 5], [3, 2], prefix_lens=[1, 1],
              tree_parents=[[-1, 0, 0], [-1, 0]])
    for fn in (decode_batch, verify_batch):
        with pytest.raises((TypeError, ValueError)):
            fn(c, 0, torch.zeros(5, 4, 192, dtype=torch.bfloat16), b)


def test_latent_calls(lib, monkeypatch):
    monkeypatch.setattr(_lib, "same_device", lambda a, b: a == b)
    c = _latent_cache()
    b = LatentBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, scale=0.1)
    v = LatentBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, scale=0.1, q_lens=[1, 1])
    ql, qr = torch.zeros(2, 4, 128), torch.zeros(2, 4, 64)
    with pytest.raises(ValueError):
        c.decode_batch(0, (ql, qr), v)
    with pytest.raises(ValueError):
        c.verify_batch(0, (ql, qr), b)
    with pytest.raises(ValueError):
        _latent_cache().decode_batch(0, (ql, qr), b)      # another cache's batch
    for bad in ((ql[:1], qr), (ql[:, :3], qr), (ql, qr[..., :32]), torch.zeros(2, 4, 200)):
        with pytest.raises(ValueError):
            c.decode_batch(0, bad, b)
    with pytest.raises(TypeError):
        c.decode_batch(0, (ql, qr.half()), b)
    for out in (torch.zeros(2, 4, 64), torch.zeros(2, 4, 256)[..., :128]):
        with pytest.raises(ValueError):
            c.decode_batch(0, (ql, qr), b, out=out)
    both = torch.zeros(2 * 4 * 192)
    with pytest.raises(ValueError):
        c.decode_batch(0, both.view(2, 4, 192), b, out=both[:2 * 4 * 128].view(2, 4, 128))


def test_latent_rows():
    c = _latent_cache()
    lt, kr, slots = torch.zeros(3, 128), torch.zeros(3, 64), torch.arange(3)
    for bad in ((lt[:, :64], kr, slots), (lt, kr[:2], slots), (lt, kr, slots[:2]),
                (lt[0], kr, slots)):
        with pytest.raises(ValueError):
            c.append_batch(0, *bad)
    with pytest.raises(TypeError):
        c.append_batch(0, lt, kr.half(), slots)
    rope = SimpleNamespace(head_dim=32, device=torch.device("cpu"))
    with pytest.raises(ValueError):
        c.append_norm_rope(0, lt, kr, slots, slots, rope)
    rope = SimpleNamespace(head_dim=64, device=torch.device("cpu"))
    with pytest.raises(ValueError):
        c.append_norm_rope(0, lt, kr, slots, slots, rope, torch.zeros(3, 4, 32))
    with pytest.raises(ValueError):
        c.append_norm_rope(0, lt, kr, slots, slots, rope, weight=torch.ones(64))
    with pytest.raises(ValueError):
        c.write_layer([0], 15, 0, lt, kr)
    with pytest.raises(IndexError):
        c.write_layer([0], 0, 2, lt, kr)
    with pytest.raises(IndexError):
        c.write_layer([9], 0, 0, lt, kr)
    with pytest.raises(IndexError):
        c.read_layer([0], 3, 2)


# ---------------------------------------------------------------------------
# accepted paths and the engine
# ---------------------------------------------------------------------------
class _Recorder(_BlockPool):
    """A pool whose moves are written down."""

    def __init__(self):
        super().__init__(8, 16)
        self.device, self.moves = torch.device("cpu"), []
        self.n_kv_heads, self.head_dim, self.cx_pool = 2, 64, _pool

    def _accept_launch(self, batch, paths, stride, length):
        self.moves.append((paths.tolist(), stride, length))


def test_accept_paths_arguments(lib, monkeypatch):
    monkeypatch.setattr(_lib, "on_device", lambda d: contextlib.nullcontext())
    c = _Recorder()
    b = PagedBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, q_lens=[3, 2])
    for bad in ([[0]], [[0], [2]], [[1, 0], []], [[0, 0], []], [[-1], []]):
        with pytest.raises(ValueError):
            c.accept_paths(b, bad)
    for bad in (torch.zeros(3, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            c.accept_paths(b, bad)
    for bad in (torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.bool)):
        with pytest.raises(TypeError):
            c.accept_paths(b, bad)
    with pytest.raises(ValueError):
        _Recorder().accept_paths(b, [[0], [0]])
    assert c.moves == []
    c.accept_paths(b, [[], []])
    assert c.moves == []                                   # nothing to move: no launch
    c.accept_paths(b, [[0, 2], [1]])
    # (numbers outside 32 bits stay outside the tree)
    c.accept_paths(b, torch.tensor([[0, 1 << 32], [-(1 << 40), 1]]))
    assert c.moves == [([[0, 2], [1, -1]], 2, 2), ([[0, 2 ** 31 - 1], [-1, 1]], 2, 2)]
    # rows that overlap or lie apart in memory
    c.accept_paths(b, torch.tensor([[0, 1]], dtype=torch.int32).expand(2, 2))
    c.accept_paths(b, torch.arange(6, dtype=torch.int32).view(2, 3)[:, :2])
    assert c.moves[2:] == [([[0, 1], [0, 1]], 2, 2), ([[0, 1], [3, 4]], 3, 2)]


def test_engine_refusals(lib):
    with pytest.raises(ValueError):
        BatchedKVEngine(_latent_cache(), n_q_heads=4)
    with pytest.raises(ValueError):
        BatchedKVEngine(_latent_cache(), n_q_heads=4, scale=0.1, softcap=30.0)
    e = BatchedKVEngine(_latent_cache(), n_q_heads=4, scale=0.1)
    e.add(0, list(range(20)))
    free = e.cache.free_blocks
    for kw in (dict(tree_parents=[[-1]], attend=False), dict(prefix_lens=[1]),
               dict(tree_parents=[[0]]), dict(tree_parents=[[-1, 0]]),
               dict(q_lens=[2], tree_parents=[[-1]])):
        with pytest.raises(ValueError):
            e.plan([0], **kw)
        assert e.cache.free_blocks == free and e.seqs[0].block_table == []    # no table grew
    plan = StepPlan([], np.zeros(0, np.int64), np.zeros(0, np.int64), None, None, None, [])
    with pytest.raises(ValueError):                        # only the latent has a norm
        e.append_rope(plan, 0, None, None, SimpleNamespace(head_dim=64), q_weight=torch.ones(64))


def test_engine_accept_refusals():
    e = BatchedKVEngine(SimpleNamespace(accept_paths=lambda *a: None), n_q_heads=4)
    s = KVSequence(0, [1, 2, 3])
    plan = StepPlan([s], np.array([s.n_tokens]), np.array([2]), None, None, None, [])
    with pytest.raises(RuntimeError):
        e.accept(plan, [[0]])                              # no attention batch
    plan.batch, plan.tree = object(), True
    with pytest.raises(RuntimeError):
        e.commit(plan)                                     # a tree ends with accept
    e.accept(plan, [[0, 1]])
    assert s.n_tokens == plan.n_past[0] + 2
    with pytest.raises(RuntimeError):
        e.accept(plan, [[0]])                              # twice
    twice = StepPlan([s, s], np.array([s.n_tokens] * 2), np.array([1, 1]), None, object(), None, [])
    twice.batch = object()
    with pytest.raises(ValueError):
        e.accept(twice, [[0], [0]])
