"""Refusals of calls over drafted trees and the latent cache that would keep wrong rows
(no GPU needed: every one comes from the host, before any launch)."""
import contextlib
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from chenxing_b200 import BatchedKVEngine, PagedBatch, _lib
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
