"""A paged cache of latent rows, and the attention that reads it.

Models whose keys and values are projected from one latent vector a token cache
that vector and a rotated key part that all heads share, instead of K and V of
every head.  In the absorbed form the key projection is multiplied into the
queries and the value projection into what follows the attention, so that the
row itself is every head's key, and its latent part every head's value:

    score[t, h, j] = scale * (q_latent[t, h] . latent[j] + q_rope[t, h] . k_rope[j])
    out[t, h]      = softmax(score[t, h]) @ latent                   (T, Hq, latent_dim)

``LatentPagedKVCache`` has the radix tree, the block rules and the errors of
``RadixPagedKVCache`` over a pool ``[n_layers][n_blocks][block_size][latent_dim +
rope_dim]`` (the reference has no such cache); ``LatentBatch`` is its
``PagedBatch``.  The projections stay with the model.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from ._arrays import (index_on_device, overlap, rows_on_device, to_device, to_numpy, torch_dtype,
                      upload)
from .batch import PagedBatch
from .radix_kv import _BlockPool, _check_cow_slots

__all__ = ["LatentPagedKVCache", "LatentBatch"]


def _rows2(x, device: torch.device) -> torch.Tensor:
    """``x`` (tokens, dim) on ``device`` with its innermost dimension contiguous."""
    if not (isinstance(x, torch.Tensor) and x.dtype != torch.float64 and x.device == device):
        x = to_device(x, device)
    if x.dim() != 2:
        raise ValueError(f"latent and k_rope must have two dimensions, got {tuple(x.shape)}")
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


class LatentBatch(PagedBatch):
    """``PagedBatch`` of a latent cache: tables, lengths, ``window`` and
    ``tree_parents`` as there, no score modifiers.  ``scale`` is that of the model's
    heads before they were absorbed (1 / sqrt of their query width).

    A batch holds one workspace: its calls run in order on one stream, the one it
    was made on.  A captured graph reads the device arrays of its capture: after
    ``set`` or ``advance`` it is captured again."""

    def __init__(self, cache, block_tables, ctx_lens, *, n_q_heads: int, scale: float,
                 q_lens=None, window: int | None = None, table_stride: int | None = None,
                 tree_parents=None) -> None:
        if int(n_q_heads) < 1:
            raise ValueError("n_q_heads must be positive")
        super().__init__(cache, block_tables, ctx_lens, n_q_heads=n_q_heads, q_lens=q_lens,
                         window=window, scale=float(scale), table_stride=table_stride,
                         tree_parents=tree_parents)

    def set(self, block_tables, ctx_lens, q_lens=None, prefix_lens=None,
            tree_parents=None) -> None:
        """``PagedBatch.set``, without ``prefix_lens``."""
        if prefix_lens is not None:
            raise ValueError("a latent cache takes no prefix_lens")
        super().set(block_tables, ctx_lens, q_lens, tree_parents=tree_parents)

    def _check_cache(self, cache) -> None:
        if not isinstance(cache, LatentPagedKVCache):
            raise TypeError("LatentBatch needs a LatentPagedKVCache")

    def _workspace_need(self) -> int:
        return int(_lib.lib().cx_latent_attend_workspace_bytes(self.cache.cx_pool(), self._c))

    def kernel_kind(self, q_dtype=torch.bfloat16, out_dtype=torch.float32) -> str:
        """Which kernel attends this batch: "tcgen05" or "generic"."""
        return _lib.KERNEL_KINDS[_lib.lib().cx_latent_attend_kind(
            self.cache.cx_pool(), self._c, _lib.cx_dtype(q_dtype))]


class LatentPagedKVCache(_BlockPool):
    """Pool of latent rows (all layers, in HBM) + logical radix prefix tree."""

    def __init__(self, n_blocks: int, block_size: int, n_layers: int, latent_dim: int,
                 rope_dim: int, dtype=np.float32, *, device=None, host_io: bool = True,
                 clock=None) -> None:
        if block_size <= 0 or n_blocks <= 0 or n_layers <= 0:
            raise ValueError("n_blocks, block_size, n_layers must be positive")
        if latent_dim <= 0 or rope_dim <= 0 or rope_dim % 2:
            raise ValueError("latent_dim must be positive, rope_dim positive and even")
        if latent_dim > 512 or latent_dim + rope_dim > 576:
            raise ValueError("latent_dim is at most 512, latent_dim + rope_dim at most 576")
        self.device = _lib.require_cuda(device)
        _lib.lib()
        super().__init__(n_blocks, block_size, clock)
        self.n_layers = int(n_layers)
        self.latent_dim = int(latent_dim)
        self.rope_dim = int(rope_dim)
        self.n_kv_heads, self.head_dim = 1, self.latent_dim + self.rope_dim
        self.dtype = dtype
        self.torch_dtype = torch_dtype(dtype)
        self.host_io = host_io
        self._kv = torch.zeros((self.n_layers, self.n_blocks, self.block_size, self.head_dim),
                               dtype=self.torch_dtype, device=self.device)
        self._pool = _lib.CxLatentPool(self._kv.data_ptr(), self.n_layers, self.n_blocks,
                                       self.block_size, self.latent_dim, self.rope_dim,
                                       _lib.cx_dtype(self.torch_dtype), 0)

    @property
    def kv_pool(self) -> torch.Tensor:
        """The pool (L, NB, bs, latent_dim + rope_dim)."""
        return self._kv

    @property
    def pool_bytes(self) -> int:
        return self._kv.numel() * self._kv.element_size()

    def cx_pool(self) -> _lib.CxLatentPool:
        return self._pool

    # ------------------------------------------------------------------ #
    # one sequence
    # ------------------------------------------------------------------ #
    def write_layer(self, block_table: list, slot_start: int, layer: int, latent, k_rope) -> None:
        """Store rows for positions [slot_start, slot_start + T) of one layer: latent
        (T, latent_dim) and k_rope (T, rope_dim), as they are, rounded to the pool's
        type.  Placement and errors are ``RadixPagedKVCache.write_layer``'s."""
        T = int(latent.shape[0])
        if len(block_table) * self.block_size < slot_start + T:
            raise ValueError("block_table too short for requested write range")
        if not 0 <= layer < self.n_layers:
            raise IndexError(f"layer {layer} outside [0, {self.n_layers})")
        if T == 0:
            return
        pos = np.arange(slot_start, slot_start + T, dtype=np.int64)
        used = np.asarray(block_table, dtype=np.int64)[pos // self.block_size]
        self._check_ids(np.unique(used))
        slots = used * self.block_size + pos % self.block_size
        self.append_batch(layer, latent, k_rope, upload(slots, self.device))

    def read_layer(self, block_table: list, n_tokens: int, layer: int):
        """Latent (n, latent_dim) and key part (n, rope_dim) of the first ``n_tokens``
        positions."""
        n = min(int(n_tokens), len(block_table) * self.block_size)
        out = [torch.empty((max(n, 0), d), dtype=self.torch_dtype, device=self.device)
               for d in (self.latent_dim, self.rope_dim)]
        if n > 0:
            if not 0 <= layer < self.n_layers:
                raise IndexError(f"layer {layer} outside [0, {self.n_layers})")
            used = list(block_table[:-(-n // self.block_size)])
            self._check_ids(used)
            table = upload(np.asarray(used, dtype=np.int32), self.device)
            with _lib.on_device(self.device):
                _lib.check(_lib.lib().cx_latent_gather(
                    self._pool, int(layer), table.data_ptr(), n, out[0].data_ptr(),
                    out[1].data_ptr(), _lib.raw_stream(self.device)), "cx_latent_gather")
        return tuple(map(to_numpy, out)) if self.host_io else tuple(out)

    # ------------------------------------------------------------------ #
    # many sequences
    # ------------------------------------------------------------------ #
    def append_batch(self, layer: int, latent, k_rope, slot_mapping, cow=None) -> None:
        """latent (T, latent_dim) and k_rope (T, rope_dim) go to ``slot_mapping`` (T,)
        as they are; a negative slot stores nothing.  ``cow``: (src, dst, n_valid), the
        first n_valid slots of block src are copied into block dst of this layer
        first."""
        if not 0 <= layer < self.n_layers:       # (to the block copy -1 is every layer)
            raise IndexError(f"layer {layer} outside [0, {self.n_layers})")
        if cow is not None:
            _check_cow_slots(slot_mapping, cow, self.block_size)
            cow = tuple(to_device(c, self.device, float_only=False).to(torch.int32) for c in cow)
        self._append(layer, latent, k_rope, slot_mapping, None, None, None, None, 0.0, None, cow)

    def append_norm_rope(self, layer: int, latent, k_rope, slot_mapping, positions, rope,
                         q_rope=None, *, weight=None, eps: float = 1e-6, q_out_dtype=None):
        """RMS norm of the latent, rotation of the shared key part and of the queries'
        rotary parts, and the append, in one launch; returns the rotated queries
        (T, Hq, rope_dim) of ``q_out_dtype`` (the rows' type by default), None without
        ``q_rope``.

        latent (T, latent_dim), k_rope (T, rope_dim), q_rope (T, Hq, rope_dim): one
        float type, any token and head strides (slices of a projection are read in
        place).  The latent x becomes ``x * rsqrt(mean(x^2) + eps) * weight`` (None: as
        it is; (latent_dim,), float32 or the rows' type); ``rope.head_dim`` is
        rope_dim.  fp32, rounded once.  A negative slot stores nothing (the queries
        are still returned); the slots of one call must differ."""
        if rope.head_dim != self.rope_dim:
            raise ValueError(f"RoPE tables of {rope.head_dim} dims for a rotary part of "
                             f"{self.rope_dim}")
        if rope.device != self.device and not _lib.same_device(rope.device, self.device):
            raise ValueError(f"RoPE tables on {rope.device}, the cache on {self.device}")
        if positions is None:
            raise ValueError("append_norm_rope needs positions (append_batch stores rows as they "
                             "are)")
        return self._append(layer, latent, k_rope, slot_mapping, positions, rope, q_rope, weight,
                            eps, q_out_dtype)

    def _append(self, layer, latent, k_rope, slots, positions, rope, q_rope, weight, eps,
                q_out_dtype, cow=None):
        dev, dc, dr = self.device, self.latent_dim, self.rope_dim
        lt, kt = _rows2(latent, dev), _rows2(k_rope, dev)
        dt, T = lt.dtype, lt.shape[0]
        if lt.shape[1] != dc or kt.shape != (T, dr):
            raise ValueError(f"latent and k_rope must be (T, {dc}) and (T, {dr}), got "
                             f"{tuple(lt.shape)} / {tuple(kt.shape)}")
        code = _lib.cx_dtype(dt)
        qt = qo = None
        hq, qs, q_code = 0, (0, 0), _lib.CX_F32
        if q_rope is not None:
            qt = rows_on_device(q_rope, dev)
            if qt.dim() != 3 or qt.shape[0] != T or qt.shape[2] != dr:
                raise ValueError(f"q_rope must be ({T}, Hq, {dr}), got {tuple(qt.shape)}")
            hq, qs = qt.shape[1], qt.stride()
        if kt.dtype != dt or (qt is not None and qt.dtype != dt):
            raise TypeError("latent, k_rope and q_rope must have one element type")
        st = index_on_device(slots, dev)
        ps = None if positions is None else index_on_device(positions, dev)
        if st.numel() != T or (ps is not None and ps.numel() != T):
            raise ValueError("slot_mapping and positions need one entry per token")
        w, w_code = weight, _lib.CX_F32
        if w is not None:
            if not (isinstance(w, torch.Tensor) and w.is_cuda and w.device == dev
                    and w.is_contiguous()):
                w = to_device(w, dev)
            if w.numel() != dc:
                raise ValueError(f"weight must have {dc} elements, got {w.numel()}")
            if w.dtype == dt:
                w_code = code
            elif w.dtype != torch.float32:
                w = w.float()
        if qt is not None:
            qo = qt.new_empty((T, hq, dr), dtype=q_out_dtype or dt)
            q_code = _lib.cx_dtype(qo.dtype)
        rows = _lib.CxLatentRows(lt.data_ptr(), kt.data_ptr(), _lib.ptr(qt), lt.stride(0),
                                 kt.stride(0), qs[0], qs[1], T, hq, code, 0)
        if rope is None:
            how = _lib.CxNormRope(None, _lib.ptr(w), 0, w_code, eps, 0, None, None, 0, 0)
        else:
            how = _lib.CxNormRope(None, _lib.ptr(w), 0, w_code, eps, rope.interleaved,
                                  rope.cos.data_ptr(), rope.sin.data_ptr(), rope.rows,
                                  rope.head_dim)
        with _lib.on_device(dev):
            if cow is not None:                  # (nothing is copied for rows that are refused)
                src, dst, n = cow
                _lib.check(_lib.lib().cx_latent_block_copy(
                    self._pool, int(layer), src.data_ptr(), dst.data_ptr(), n.data_ptr(),
                    src.numel(), self.block_size, _lib.raw_stream(dev)), "cx_latent_block_copy")
            _lib.check(_lib.lib().cx_latent_append(
                self._pool, int(layer), rows, st.data_ptr(), _lib.ptr(ps), how, _lib.ptr(qo),
                q_code, _lib.raw_stream(dev)), "cx_latent_append")
        return qo

    def decode_batch(self, layer: int, q, batch: LatentBatch, out=None, out_dtype=None):
        """One query token per sequence: q = (q_latent (B, Hq, latent_dim), q_rope (B,
        Hq, rope_dim)), of one type and any token and head strides, or one tensor
        (B, Hq, latent_dim + rope_dim) -> (B, Hq, latent_dim), float32 unless ``out`` or
        ``out_dtype`` says bfloat16 or float16.  Over a 16-bit pool the tcgen05 kernel
        rounds float32 queries to the pool's type first (over float16 those beyond 65504
        become infinite, and their rows NaN) and the probabilities before the second
        product; ``LatentBatch.kernel_kind`` names the kernel, "generic" is fp32
        throughout."""
        if batch.verify:
            raise ValueError("decode_batch needs a LatentBatch built without q_lens")
        return self._attend(layer, q, batch, out, out_dtype)

    def verify_batch(self, layer: int, q, batch: LatentBatch, out=None, out_dtype=None):
        """``decode_batch`` for q_lens[b] query tokens per sequence, rows concatenated
        (chains, prompt chunks, drafted trees)."""
        if not batch.verify:
            raise ValueError("verify_batch needs a LatentBatch built with q_lens")
        return self._attend(layer, q, batch, out, out_dtype)

    def _attend(self, layer, q, batch, out, out_dtype):
        if batch.cache is not self:
            raise ValueError("LatentBatch belongs to a different cache")
        dev, dc, dr = self.device, self.latent_dim, self.rope_dim
        rows, hq = batch.total_q, batch.n_q_heads
        if isinstance(q, (tuple, list)):
            ql, qr = q
            ql, qr = rows_on_device(ql, dev), rows_on_device(qr, dev)
        else:
            q = rows_on_device(q, dev)
            ql, qr = q[..., :dc], q[..., dc:]
        if ql.shape != (rows, hq, dc) or qr.shape != (rows, hq, dr):
            raise ValueError(f"q must be ({rows}, {hq}, {dc}) and ({rows}, {hq}, {dr}), got "
                             f"{tuple(ql.shape)} / {tuple(qr.shape)}")
        if ql.dtype != qr.dtype:
            raise TypeError("q_latent and q_rope must have one element type")
        if out_dtype is None:
            out_dtype = torch.float32 if out is None else out.dtype
        if out is None:
            out = ql.new_empty((rows, hq, dc), dtype=out_dtype)
        elif tuple(out.shape) != (rows, hq, dc) or out.dtype != out_dtype \
                or not out.is_contiguous() or not _lib.same_device(out.device, dev):
            raise ValueError(f"out must be a contiguous {out_dtype} tensor of shape "
                             f"{(rows, hq, dc)} on {dev}")
        elif overlap(out, ql) or overlap(out, qr):
            raise ValueError("out must not share memory with q")
        code, out_code = _lib.cx_dtype(ql.dtype), _lib.cx_dtype(out.dtype)
        if rows == 0:
            return out
        ls, rs = ql.stride(), qr.stride()
        qs = _lib.CxLatentQ(ql.data_ptr(), qr.data_ptr(), ls[0], ls[1], rs[0], rs[1], code, 0)
        with _lib.on_device(dev):
            _lib.check(_lib.lib().cx_latent_attend(
                self._pool, int(layer), batch.c_struct(), batch._tree, qs, out.data_ptr(),
                out_code, batch.workspace.data_ptr(), batch.workspace.numel(),
                _lib.raw_stream(dev)), "cx_latent_attend")
        return out

    # ------------------------------------------------------------------ #
    def _copy_launch(self, src: torch.Tensor, dst: torch.Tensor, n: int, n_slots: int) -> None:
        with _lib.on_device(self.device):
            _lib.check(_lib.lib().cx_latent_block_copy(
                self._pool, -1, src.data_ptr(), dst.data_ptr(), None, n, n_slots,
                _lib.raw_stream(self.device)), "cx_latent_block_copy")

    def _accept_launch(self, batch, paths: torch.Tensor, stride: int, length: int) -> None:
        _lib.check(_lib.lib().cx_latent_accept(self._pool, batch, paths.data_ptr(), stride, length,
                                               _lib.raw_stream(self.device)), "cx_latent_accept")
