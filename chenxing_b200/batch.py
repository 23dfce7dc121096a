"""Batched paged attention over a RadixPagedKVCache.

The reference decodes one sequence at a time (chenxing/engine/scheduler.py:59-74,
chenxing/engine/engine.py:110-129): per layer ``write_layer`` then
``read_layer`` + ``flash_attention``.  ``PagedBatch`` carries the same
per-sequence metadata (block tables, context lengths, query lengths) for a
whole batch as device arrays, so one ``cx_kv_append`` and one
``cx_paged_decode`` / ``cx_paged_verify`` launch serve every sequence of a
layer.  Tables and lengths are exactly the reference's ``Sequence.block_table``
and ``n_tokens`` values; nothing here changes them.

A batch may also change the scores (``softcap``, ``alibi_slopes``,
``prefix_lens``) or ask for a 16-bit output; ``cx_paged_attend`` serves those.
"""
from __future__ import annotations

import itertools
import math

import numpy as np
import torch

from . import _lib
from ._arrays import overlap, rows_on_device, to_device, upload

__all__ = ["PagedBatch", "slot_mapping", "decode_batch", "verify_batch"]


def slot_mapping(block_tables, starts, counts, block_size: int) -> np.ndarray:
    """Physical slots for positions [starts[b], starts[b] + counts[b]) of each
    sequence, concatenated: ``table[p // bs] * bs + p % bs`` (the placement
    rule of write_layer, chenxing/engine/radix_kv.py:123-128)."""
    starts = np.asarray(starts, dtype=np.int64).reshape(-1)
    counts = np.asarray(counts, dtype=np.int64).reshape(-1)
    bs = int(block_size)
    # only the table entries each write range touches, gathered in one pass
    parts, lens = [], []
    for bt, s, c in zip(block_tables, starts.tolist(), counts.tolist()):
        if c == 0:
            lens.append(0)
            continue
        if len(bt) * bs < s + c:
            raise ValueError("block_table too short for requested write range")
        seg = bt[s // bs:(s + c - 1) // bs + 1]
        parts.append(seg)
        lens.append(len(seg))
    total = int(counts.sum())
    if total == 0:
        return np.zeros(0, dtype=np.int64)
    ids = np.fromiter(itertools.chain.from_iterable(parts), dtype=np.int64, count=sum(lens))
    seg_off = np.zeros(len(lens), dtype=np.int64)
    np.cumsum(lens[:-1], out=seg_off[1:])
    row_off = np.zeros(len(counts), dtype=np.int64)
    np.cumsum(counts[:-1], out=row_off[1:])
    pos = np.arange(total, dtype=np.int64) + np.repeat(starts - row_off, counts)
    base = np.repeat(seg_off - starts // bs, counts)        # table index -> ids index
    return ids[base + pos // bs] * bs + pos % bs


def _same_start(a, b) -> bool:
    """Whether two block tables may be one sequence's: equal as far as both go."""
    n = min(len(a), len(b))
    return list(a[:n]) == list(b[:n]) and (n > 0 or len(a) == len(b))


class PagedBatch:
    """Device metadata + workspace for batched decode / verify on one cache.

    block_tables: list of per-sequence block-id lists; ctx_lens: cached tokens
    per sequence INCLUDING the query tokens being attended (they are appended
    first, as in transformer.py:87-88); q_lens: query tokens per sequence
    (None = decode, one each); window: sliding window or None.

    Score modifiers, none by default (the scaled score of a query at position
    ``pos`` and a key at ``j`` is ``s``):

    * ``softcap`` (1e-30 .. 1e30): ``s`` becomes ``softcap * tanh(s / softcap)``;
    * ``alibi_slopes`` (n_q_heads values >= 0, times the longest context below
      2^23): ``s -= slope[h] * |pos - j|``, after the cap;
    * ``prefix_lens`` (one per sequence): keys ``j < prefix_lens[b]`` are seen by
      every query row of the sequence, past the causal limit (a prompt whose
      first tokens see one another) and the window (tokens that a long stream
      keeps); what lies past the context is cut off.

    A batch holds one workspace: its calls run in order on one stream, the one
    it was made on.  A captured graph reads the device arrays of its capture:
    after ``set`` or ``advance`` it is captured again.
    """

    def __init__(self, cache, block_tables, ctx_lens, *, n_q_heads: int, q_lens=None,
                 window: int | None = None, scale: float | None = None,
                 table_stride: int | None = None, softcap: float | None = None,
                 alibi_slopes=None, prefix_lens=None) -> None:
        self.cache = cache
        self.device = cache.device
        self.n_q_heads = int(n_q_heads)
        if self.n_q_heads % cache.n_kv_heads:
            raise ValueError(f"GQA requires hq % hk == 0, got hq={n_q_heads}, hk={cache.n_kv_heads}")
        self.window = int(window) if window is not None else 0
        if window is not None and self.window <= 0:
            raise ValueError("window must be positive (or None)")
        self.scale = (1.0 / math.sqrt(cache.head_dim)) if scale is None else float(scale)
        self.verify = q_lens is not None
        self.table_stride = table_stride
        self.softcap = None if softcap is None else float(softcap)
        if softcap is not None and not (1e-30 <= self.softcap <= 1e30):
            raise ValueError("softcap must be None or 1e-30 .. 1e30")
        self.alibi_slopes = None
        self._steepest = 0.0
        if alibi_slopes is not None:
            sl = alibi_slopes.detach().float().cpu().numpy() \
                if isinstance(alibi_slopes, torch.Tensor) else alibi_slopes
            sl = np.asarray(sl, dtype=np.float32).reshape(-1)
            if sl.shape[0] != self.n_q_heads or not np.all(np.isfinite(sl)) or np.any(sl < 0):
                raise ValueError(f"alibi_slopes must be {self.n_q_heads} finite values >= 0")
            self._steepest = float(sl.max(initial=0.0))
            self.alibi_slopes = upload(sl, self.device)
        self.prefix_lens = None
        self.prefix_host = None
        self._planned_by = None          # entry point that made the workspace's plan
        self._ws = None
        self._ws_bytes = 0
        self.set(block_tables, ctx_lens, q_lens, prefix_lens)

    # ------------------------------------------------------------------ #
    def set(self, block_tables, ctx_lens, q_lens=None, prefix_lens=None) -> None:
        """(Re)load tables and lengths; the next attention call re-plans.  Without
        ``prefix_lens`` a batch that has some keeps them, for the same sequences:
        as many, and each table the one before, grown or cut."""
        bs = self.cache.block_size
        B = len(block_tables)
        ctx = np.asarray(ctx_lens, dtype=np.int64).reshape(-1)
        if ctx.shape[0] != B:
            raise ValueError("ctx_lens and block_tables differ in length")
        lens = np.fromiter(map(len, block_tables), dtype=np.int64, count=B)
        longest = int(lens.max(initial=0))
        stride = max(self.table_stride or 0, longest, 1)
        if self.table_stride is not None and longest > self.table_stride:
            raise ValueError("a block table is longer than table_stride")
        if np.any(ctx < 0) or np.any(ctx > lens * bs):
            raise ValueError("context length outside [0, len(block_table) * block_size]")
        # beside a bias of 2^23 fp32 loses half a unit of a score: more, and the
        # probabilities of far keys overflow fp16
        if self._steepest * int(ctx.max(initial=0)) >= 2 ** 23:
            raise ValueError("the steepest of alibi_slopes times the longest context must be "
                             "below 2**23")
        if prefix_lens is None:
            pre = self.prefix_host
            if pre is not None and pre.shape[0] != B:
                raise ValueError("prefix_lens must be given again for another batch size")
            if pre is not None and any(not _same_start(a, t) for a, t in
                                       zip(self.tables_host, block_tables)):
                raise ValueError("prefix_lens must be given again for other sequences")
        else:
            pre = np.asarray(prefix_lens, dtype=np.int64).reshape(-1)
            if pre.shape[0] != B or np.any(pre < 0):
                raise ValueError("prefix_lens must be one value >= 0 per sequence")
        ids = np.fromiter(itertools.chain.from_iterable(block_tables), dtype=np.int64,
                          count=int(lens.sum()))
        if ids.size and (ids.min() < 0 or ids.max() >= self.cache.n_blocks):
            raise IndexError(f"block id outside [0, {self.cache.n_blocks})")
        if self.verify:
            ql = np.asarray(q_lens, dtype=np.int64).reshape(-1)
            if ql.shape[0] != B or np.any(ql < 0) or np.any(ql > ctx):
                raise ValueError("q_lens must be per sequence and <= ctx_lens")
            qs = np.zeros(B + 1, dtype=np.int64)
            np.cumsum(ql, out=qs[1:])
        # nothing is refused from here on: a batch is reloaded whole or stays as it was
        self.needs_plan = True
        tab = np.zeros((B, stride), dtype=np.int32)
        tab[np.arange(stride) < lens[:, None]] = ids   # row-major mask order = concatenation
        self.batch = B
        self.stride = stride
        self.tables_host = [list(t) for t in block_tables]
        self.ctx_host = ctx
        self.block_tables = upload(tab, self.device)
        self.ctx_lens = upload(ctx.astype(np.int32), self.device)
        if self.verify:
            self.q_lens_host = ql
            self.q_start = upload(qs.astype(np.int32), self.device)
            self.max_q = int(ql.max(initial=1))
            self.total_q = int(qs[-1])
        else:
            self.q_lens_host = np.ones(B, dtype=np.int64)
            self.q_start = None
            self.max_q = 1
            self.total_q = B
        self._c = _lib.CxAttnBatch(self.block_tables.data_ptr(), self.stride,
                                   self.ctx_lens.data_ptr(),
                                   _lib.ptr(self.q_start), B, self.max_q, self.n_q_heads,
                                   self.scale, 0, self.window)
        if pre is not None:
            self.prefix_host = np.minimum(pre, np.iinfo(np.int32).max)
            self.prefix_lens = upload(self.prefix_host.astype(np.int32), self.device)
        need = max(int(_lib.lib().cx_paged_workspace_bytes(self.cache.cx_pool(), self._c)),
                   int(_lib.lib().cx_paged_attend_workspace_bytes(self.cache.cx_pool(), self._c)))
        if need > self._ws_bytes:
            self._ws = torch.zeros(need, dtype=torch.uint8, device=self.device)
            self._ws_bytes = need

    def advance(self, n: int = 1) -> None:
        """Every context grows by ``n`` tokens (one decode step); re-plans."""
        self.set(self.tables_host, self.ctx_host + n,
                 self.q_lens_host if self.verify else None)

    @property
    def kv_tokens(self) -> int:
        """Keys attended per layer (KV token-layers of one step and layer)."""
        if self.window:
            lo = np.maximum(0, self.ctx_host - self.q_lens_host - self.window + 1)
            pre = 0 if self.prefix_host is None else np.minimum(self.prefix_host, lo)
            return int(np.sum(self.ctx_host - lo + pre))
        return int(self.ctx_host.sum())

    def kernel_kind(self, q_dtype=torch.bfloat16, out_dtype=torch.float32) -> str:
        """Which libcxkv kernel attends this batch for queries and outputs of these
        types: "generic", "mma", "tcgen05" or "fma"."""
        if self.takes_attend(out_dtype):
            k = _lib.lib().cx_paged_attend_kind(self.cache.cx_pool(), self._c,
                                                _lib.cx_dtype(q_dtype))
        else:
            k = _lib.lib().cx_paged_kernel_kind(self.cache.cx_pool(), self._c,
                                                _lib.cx_dtype(q_dtype), int(self.verify))
        return _lib.KERNEL_KINDS[k]

    @property
    def scored(self) -> bool:
        """Whether the batch changes the scores or the visible keys."""
        return self.softcap is not None or self.alibi_slopes is not None \
            or self.prefix_lens is not None

    def takes_attend(self, out_dtype) -> bool:
        """Whether calls with this output type are ``cx_paged_attend``'s."""
        return self.scored or out_dtype != torch.float32

    def c_struct(self) -> _lib.CxAttnBatch:
        return self._c

    @property
    def workspace(self) -> torch.Tensor:
        return self._ws


def _attend(cache, layer: int, q, batch: PagedBatch, out, replan, out_dtype, fn_name: str):
    if batch.cache is not cache:
        raise ValueError("PagedBatch belongs to a different cache")
    if out_dtype is None:
        out_dtype = torch.float32 if out is None else out.dtype
    if batch.takes_attend(out_dtype):
        return _attend_scored(cache, layer, q, batch, out, replan, out_dtype)
    qt = to_device(q, cache.device)
    expect = (batch.total_q, batch.n_q_heads, cache.head_dim)
    if tuple(qt.shape) != expect:
        raise ValueError(f"q must have shape {expect}, got {tuple(qt.shape)}")
    if out is None:
        out = torch.empty(expect, dtype=torch.float32, device=cache.device)
    elif tuple(out.shape) != expect or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32 tensor of shape {expect}")
    do_plan = _plans(batch, replan, "plain")
    fn = getattr(_lib.lib(), fn_name)
    _lib.check(fn(cache.cx_pool(), int(layer), batch.c_struct(), qt.data_ptr(),
                  _lib.cx_dtype(qt.dtype), out.data_ptr(), batch.workspace.data_ptr(),
                  batch.workspace.numel(), int(do_plan), _lib.stream_ptr(cache.device)), fn_name)
    if do_plan:
        batch.needs_plan = False
        batch._planned_by = "plain"
    return out


def _plans(batch: PagedBatch, replan, by: str) -> bool:
    """Whether this call makes the plan: as asked, or when the batch was
    (re)loaded or its plan is the other entry point's (which serves no call
    of this one)."""
    if replan is None:
        return batch.needs_plan or batch._planned_by != by
    if not replan and batch._planned_by not in (None, by):
        raise ValueError("replan=False, but the batch's plan is that of calls "
                         f"{'with' if by == 'plain' else 'without'} score modifiers or a "
                         "16-bit output")
    return bool(replan)


def _attend_scored(cache, layer: int, q, batch: PagedBatch, out, replan, out_dtype):
    """``cx_paged_attend``: score modifiers, 16-bit outputs, strided query rows."""
    dev = cache.device
    qt = rows_on_device(q, dev)
    hq, d = batch.n_q_heads, cache.head_dim
    expect = (batch.total_q, hq, d)
    if tuple(qt.shape) != expect:
        raise ValueError(f"q must have shape {expect}, got {tuple(qt.shape)}")
    if not qt.is_contiguous() and (qt.stride(1) != d or qt.stride(0) < hq * d):
        qt = qt.contiguous()
    if out is None:
        out = qt.new_empty(expect, dtype=out_dtype)
    elif tuple(out.shape) != expect or out.dtype != out_dtype or not out.is_contiguous() \
            or not _lib.same_device(out.device, dev):
        raise ValueError(f"out must be a contiguous {out_dtype} tensor of shape {expect} "
                         f"on {dev}")
    elif overlap(out, qt) and not (out.data_ptr() == qt.data_ptr() and out.dtype == qt.dtype
                                   and qt.is_contiguous()):
        # (every kernel has read a row's queries when it stores that row)
        raise ValueError("out may be q itself, but not share part of its memory")
    if batch.total_q == 0:               # no query row at all
        return out
    mods = _lib.CxAttnMods(batch.softcap or 0.0, _lib.cx_dtype(out_dtype),
                           _lib.ptr(batch.alibi_slopes), _lib.ptr(batch.prefix_lens),
                           0 if qt.is_contiguous() else qt.stride(0))
    do_plan = _plans(batch, replan, "scored")
    with _lib.on_device(dev):
        _lib.check(_lib.lib().cx_paged_attend(
            cache.cx_pool(), int(layer), batch.c_struct(), mods, qt.data_ptr(),
            _lib.cx_dtype(qt.dtype), out.data_ptr(), batch.workspace.data_ptr(),
            batch.workspace.numel(), int(do_plan), _lib.raw_stream(dev)), "cx_paged_attend")
    if do_plan:
        batch.needs_plan = False
        batch._planned_by = "scored"
    return out


def decode_batch(cache, layer: int, q, batch: PagedBatch, out=None, replan=None,
                 out_dtype=None):
    """One query token per sequence: q (B, hq, D) -> (B, hq, D), float32 unless
    ``out`` or ``out_dtype`` says bfloat16 or float16.  With modifiers or a
    16-bit output, ``out`` may be ``q`` itself."""
    if batch.verify:
        raise ValueError("decode_batch needs a PagedBatch built without q_lens")
    return _attend(cache, layer, q, batch, out, replan, out_dtype, "cx_paged_decode")


def verify_batch(cache, layer: int, q, batch: PagedBatch, out=None, replan=None,
                 out_dtype=None):
    """q_lens[b] query tokens per sequence (speculative verify / prefill chunk):
    q (sum q_lens, hq, D) -> (sum q_lens, hq, D), float32 unless ``out`` or
    ``out_dtype`` says bfloat16 or float16."""
    if not batch.verify:
        raise ValueError("verify_batch needs a PagedBatch built with q_lens")
    return _attend(cache, layer, q, batch, out, replan, out_dtype, "cx_paged_verify")
