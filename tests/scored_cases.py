"""Seeded cases for the paged attention with score modifiers, against its
definition in float64, with the error bound derived from the arithmetic.

Bound, per output element.  ``h`` is half a step of a type (bf16 2^-8, fp16
2^-11, fp32 2^-24), A = sum_j p_j |v_j| / sum_j p_j:

* the output's rounding: ``h_out |o|``;
* 16-bit pools round each probability before the PV product: ``h_pool A``
  (fp16 also loses what lies below its smallest step, 2^-25 a key relative to
  a row sum of at least 1: ``n 2^-25 max|v|``);
* a score error ``d`` moves the numerator and the denominator by at most
  ``e^d - 1`` each: ``2 d A``, where ``d`` = fp32 accumulation of head_dim
  products (``(head_dim + 4) 2^-24 sum_d |q_d k_d| scale``), the cap's tanh
  (absolute error up to ``2^-20``, times the cap), three roundings of the
  biased score (``2^-22 max|s|``) — all at their largest over the row;
* exponentials, row sums, split merges and the division: ``2^-18 A``;
* fp32 queries over a 16-bit pool are rounded to it first: ``d`` grows by
  ``h_pool sum_d |q_d k_d| scale``.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from conftest import record_margin

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def alibi(hq):
    return [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]


class ScoredCase:
    """Pools filled with K/V over scattered tables; what no query row may see
    (free blocks, slots past the context, keys left of every row's window)
    holds NaN and infinity."""

    def __init__(self, *, hq, hk, d, ctx, q_lens=None, dtype=torch.bfloat16, q_dtype=None,
                 softcap=None, slopes=None, prefix=None, window=None, bs=16, seed=0, q_scale=1.0,
                 n_layers=1, layer=0, scale=None, poison=True, strided=False):
        from chenxing_b200 import RadixPagedKVCache
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.hq, self.hk, self.d, self.bs, self.layer = hq, hk, d, bs, layer
        self.ctx = [int(c) for c in ctx]
        self.q_lens = None if q_lens is None else [int(n) for n in q_lens]
        self.softcap, self.window, self.dtype = softcap, window, dtype
        self.slopes, self.prefix = slopes, prefix
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        ql = self.q_lens or [1] * len(self.ctx)
        need = [max(1, -(-c // bs)) for c in self.ctx]
        nb = sum(need) + 5
        self.cache = RadixPagedKVCache(nb, bs, n_layers, hk, d, dtype=dtype, host_io=False)
        perm = rng.permutation(nb)
        off = np.concatenate([[0], np.cumsum(need)])
        self.tables = [perm[off[b]:off[b + 1]].tolist() for b in range(len(need))]
        k_all = torch.full((nb, bs, hk, d), math.nan if poison else 0.0)
        v_all = torch.full((nb, bs, hk, d), math.inf if poison else 0.0)
        self.k, self.v = [], []
        for b, c in enumerate(self.ctx):
            k = torch.randn(c, hk, d, generator=gen).to(dtype)
            v = torch.randn(c, hk, d, generator=gen).to(dtype)
            kk, vv = k.float(), v.float()
            if poison and window and ql[b]:
                dead = torch.arange(c) <= c - ql[b] - window
                dead &= torch.arange(c) >= (prefix[b] if prefix else 0)
                kk, vv = kk.clone(), vv.clone()
                kk[dead], vv[dead] = math.nan, math.nan
            if c:
                t = torch.tensor(self.tables[b])
                pos = torch.arange(c)
                k_all[t[pos // bs], pos % bs] = kk
                v_all[t[pos // bs], pos % bs] = vv
            self.k.append(k.double())
            self.v.append(v.double())
        self.cache.k_pool[layer].copy_(k_all)
        self.cache.v_pool[layer].copy_(v_all)
        self.q_dtype = q_dtype or dtype
        q = (torch.randn(sum(ql), hq, d, generator=gen) * q_scale).to(self.q_dtype)
        self.q = q.double()
        if strided:      # the query heads of a fused projection's rows
            wide = torch.full((sum(ql), hq + 2 * hk, d), math.nan, dtype=self.q_dtype)
            wide[:, :hq] = q
            self.q_dev = wide.cuda()[:, :hq]
        else:
            self.q_dev = q.cuda()

    def batch(self, **kw):
        from chenxing_b200 import PagedBatch
        return PagedBatch(self.cache, self.tables, self.ctx, n_q_heads=self.hq,
                          q_lens=self.q_lens, window=self.window, softcap=self.softcap,
                          scale=self.scale, alibi_slopes=self.slopes, prefix_lens=self.prefix,
                          **kw)

    def run(self, batch=None, out_dtype=None, **kw):
        batch = batch or self.batch()
        fn = self.cache.verify_batch if batch.verify else self.cache.decode_batch
        return fn(self.layer, self.q_dev, batch, out_dtype=out_dtype, **kw)

    def expected(self, out_dtype, hidden=()):
        """(values, bounds) in float64, rows concatenated; ``hidden``: positions
        that no row sees."""
        outs, tols, row = [], [], 0
        h_pool = HALF[self.dtype] if self.dtype != torch.float32 else 0.0
        for b, c in enumerate(self.ctx):
            n = 1 if self.q_lens is None else self.q_lens[b]
            q = self.q[row:row + n]
            row += n
            if c == 0 or n == 0:
                outs.append(torch.zeros(n, self.hq, self.d, dtype=torch.float64))
                tols.append(torch.zeros_like(outs[-1]))
                continue
            rep = self.hq // self.hk
            k = self.k[b].repeat_interleave(rep, 1)          # (c, hq, d)
            v = self.v[b].repeat_interleave(rep, 1)
            s = torch.einsum("nhd,chd->hnc", q, k) * self.scale
            mag = torch.einsum("nhd,chd->hnc", q.abs(), k.abs()) * abs(self.scale)
            pos = torch.arange(c - n, c)[:, None]
            j = torch.arange(c)[None, :]
            seen = j <= pos
            if self.window:
                seen &= j > pos - self.window
            if self.prefix:
                seen |= j < self.prefix[b]
            hid = [x for x in hidden if x < c]
            seen = seen.clone()
            seen[:, hid] = False
            if self.softcap:
                s = self.softcap * torch.tanh(s / self.softcap)
            if self.slopes is not None:
                sl = torch.as_tensor(self.slopes).double().float().double()
                s = s - sl[:, None, None] * (pos - j).abs()
            s = s.masked_fill(~seen, -math.inf)
            big = torch.where(seen, s.abs(), 0.0).amax(-1, keepdim=True)
            err = torch.where(seen, mag, 0.0).amax(-1, keepdim=True) * (self.d + 4) * 2.0 ** -24
            if self.q_dtype != self.dtype and self.dtype != torch.float32:
                err = err + h_pool * torch.where(seen, mag, 0.0).amax(-1, keepdim=True)
            err = err + big * 2.0 ** -22 + (self.softcap or 0.0) * 2.0 ** -20
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
            p = torch.where(seen, p, 0.0)
            den = p.sum(-1, keepdim=True)
            w = torch.where(den > 0, p / den, 0.0)
            o = torch.einsum("hnc,chd->nhd", w, v)
            a = torch.einsum("hnc,chd->nhd", w, v.abs())
            e = (2 * torch.expm1(err) + h_pool + 2.0 ** -18).permute(1, 0, 2) * a
            if self.dtype == torch.float16:
                e = e + c * 2.0 ** -25 * v.abs().max()
            outs.append(o)
            tols.append(e + HALF[out_dtype] * (o.abs() + e) + 1e-30)
        return torch.cat(outs), torch.cat(tols)

    def check(self, out, hidden=()):
        want, tol = self.expected(out.dtype, hidden)
        got = out.double().cpu()
        assert got.shape == want.shape
        assert torch.isfinite(got).all(), "non-finite output"
        worst = float(((got - want).abs() / tol.clamp_min(1e-30)).max()) if got.numel() else 0.0
        record_margin(worst)
        assert worst <= 1.0, f"error {worst:.3f} times its bound"
