"""Refusals of calls over drafted trees and the latent cache that would keep wrong rows
(no GPU needed: every one comes from the host, before any launch)."""
import contextlib
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from chenxing_b200 import BatchedKVEngine, PagedBatch, RadixPagedKVCache, _lib
from chenxing_b200.engine import KVSequence, StepPlan
from test_latent_refusals_cpu import _latent_cache, _Recorder


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


# ---------------------------------------------------------------------------
# accepted paths
# ---------------------------------------------------------------------------
TREES = [[-1, 0, 0, 1, 2, -1], [-1, 0]]


@pytest.mark.parametrize("path", [[1], [0, 3], [0, 1, 4], [0, 2, 5], [0, 5], [0, 1, 2], [2, 4],
                                  [0, 4]])
def test_paths_follow_the_parents(lib, monkeypatch, path):
    """[1] starts below the committed context's child, [0, 3] skips a level, [0, 1, 4] goes
    to another node's child, [0, 5] to another root."""
    monkeypatch.setattr(_lib, "on_device", lambda d: contextlib.nullcontext())
    c = _Recorder()
    b = PagedBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, q_lens=[6, 2], tree_parents=TREES)
    with pytest.raises(ValueError):
        c.accept_paths(b, [path, [0, 1]])
    with pytest.raises(ValueError):
        c.accept_paths(b, [[0, 2, 4], [1]])
    assert c.moves == []


def test_paths_of_the_tree_are_taken(lib, monkeypatch):
    monkeypatch.setattr(_lib, "on_device", lambda d: contextlib.nullcontext())
    c = _Recorder()
    b = PagedBatch(c, [[0, 1], [2]], [20, 5], n_q_heads=4, q_lens=[6, 2], tree_parents=TREES)
    c.accept_paths(b, [[0, 2, 4], []])
    c.accept_paths(b, [[5], [0, 1]])
    c.accept_paths(b, [[], []])
    assert c.moves == [([[0, 2, 4], [-1, -1, -1]], 3, 3), ([[5, -1], [0, 1]], 2, 2)]


def test_engine_keeps_the_first_rows_of_a_chain():
    moved = []
    e = BatchedKVEngine(SimpleNamespace(accept_paths=lambda b, p: moved.append(p)), n_q_heads=4)
    s = KVSequence(0, [1, 2, 3])
    plan = StepPlan([s], np.array([s.n_tokens]), np.array([3]), object(), None, None, [])
    for path in ([1], [0, 2], [1, 2]):
        with pytest.raises(ValueError):
            e.accept(plan, [path])
    assert moved == [] and s.n_tokens == plan.n_past[0]
    e.accept(plan, [[0, 1]])
    assert moved == [[[0, 1]]] and s.n_tokens == plan.n_past[0] + 2


# ---------------------------------------------------------------------------
# rows of the latent cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layer", [-1, 2])
def test_append_with_copies_checks_the_layer_first(monkeypatch, layer):
    """The block copy takes -1 for every layer: an append must not come that far."""
    called = []
    monkeypatch.setattr(_lib, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "raw_stream", lambda d: None)
    monkeypatch.setattr(_lib, "lib", lambda: SimpleNamespace(
        cx_latent_block_copy=lambda *a: called.append("copy") or 0,
        cx_latent_append=lambda *a: called.append("append") or 0))
    c = _latent_cache()
    rows = torch.zeros(1, 128), torch.zeros(1, 64), [40]
    with pytest.raises(IndexError):
        c.append_batch(layer, *rows, cow=([1], [2], [8]))
    with pytest.raises(IndexError):
        c.append_batch(layer, *rows)
    with pytest.raises(ValueError):                        # rows that are refused: no copy either
        c.append_batch(1, rows[0][:, :64], *rows[1:], cow=([1], [2], [8]))
    assert called == []
    c.append_batch(1, *rows, cow=([1], [2], [8]))
    assert called == ["copy", "append"]


@pytest.mark.parametrize("cow", [([1, 3], [2], [8]), ([1], [2, 4], [8]), ([1, 3], [2, 4], [8]),
                                 (torch.tensor([1, 3]), torch.tensor([2, 4]), torch.tensor([8]))])
@pytest.mark.parametrize("latent", [False, True])
def test_copies_of_one_length(cow, latent):
    """The copies read as many destinations and counts as there are sources."""
    if latent:
        c, rows = _latent_cache(), (torch.zeros(1, 128), torch.zeros(1, 64))
    else:
        c = object.__new__(RadixPagedKVCache)
        c.block_size, c.device = 16, torch.device("cpu")
        rows = torch.zeros(1, 2, 64), torch.zeros(1, 2, 64)
    c._append = c.append_slots = lambda *a: pytest.fail("came as far as the launch")
    with pytest.raises(ValueError):
        c.append_batch(0, *rows, [100], cow=cow)


def test_rotation_needs_positions(monkeypatch):
    """Without them the shared key part would be stored unrotated."""
    monkeypatch.setattr(_lib, "lib", lambda: pytest.fail("came as far as the launch"))
    c = _latent_cache()
    rope = SimpleNamespace(head_dim=64, device=torch.device("cpu"), interleaved=0, rows=8,
                           cos=torch.zeros(8, 64), sin=torch.zeros(8, 64))
    with pytest.raises(ValueError):
        c.append_norm_rope(0, torch.zeros(3, 128), torch.zeros(3, 64), torch.arange(3), None, rope)


def test_positions_of_padded_rows(lib):
    """A position of -1 is outside every rotation table and would raise a device flag."""
    b = PagedBatch(_Recorder(), [[0, 1], [], [2]], [20, 0, 5], n_q_heads=4)
    assert b.row_positions().tolist() == [19, 0, 4]
