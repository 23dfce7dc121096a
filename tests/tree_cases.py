"""Seeded cases for drafted trees over the K/V cache and for the latent cache,
against their definitions in float64.  Bounds are those of scored_cases, derived
there term by term; a latent row's score sums latent_dim + rope_dim products."""
from __future__ import annotations

import math

import numpy as np
import torch

from conftest import record_margin
from scored_cases import HALF, ScoredCase


def random_tree(rng, n, kind):
    """Parents of a tree of n nodes: a chain, a star of first tokens, or random."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] * n
    if kind == "deep":
        return [i - 1 if i == 0 or rng.random() < 0.7 else int(rng.integers(-1, i))
                for i in range(n)]
    return [int(rng.integers(max(-1, i // 3 - 2), i)) if i else -1 for i in range(n)]


def visible(n, c, parents=None, window=None, prefix=0):
    """(seen (n, c) bool, distance (n, c)) of n query rows behind c - n committed
    tokens, by the definition."""
    base = c - n
    rows, keys = list(range(base, c)), list(range(c))
    seen = np.zeros((n, c), dtype=bool)
    kin = [[] for _ in range(n)]
    if parents is not None:
        for i in range(n):
            u = i
            while u >= 0:
                kin[i].append(u)
                u = parents[u]
            rows[i] = base + len(kin[i]) - 1
        keys[base:] = rows
    dist = np.asarray(rows)[:, None] - np.asarray(keys)[None, :]
    for i in range(n):
        if parents is None:
            seen[i, :base + i + 1] = True
        else:
            seen[i, :base] = True
            seen[i, [base + u for u in kin[i]]] = True
    if window:
        seen &= dist < window
    seen[:, :min(prefix, base if parents is not None else c)] = True
    return torch.from_numpy(seen), torch.from_numpy(dist)


class TreeCase(ScoredCase):
    """A ScoredCase whose query rows are the nodes of a tree per sequence."""

    def __init__(self, *, parents, **kw):
        super().__init__(q_lens=[len(p) for p in parents], **kw)
        self.parents = parents

    def batch(self, **kw):
        from chenxing_b200 import PagedBatch
        return PagedBatch(self.cache, self.tables, self.ctx, n_q_heads=self.hq,
                          q_lens=self.q_lens, window=self.window, softcap=self.softcap,
                          scale=self.scale, alibi_slopes=self.slopes, prefix_lens=self.prefix,
                          tree_parents=self.parents, **kw)

    def expected(self, out_dtype, hidden=()):
        outs, tols, row = [], [], 0
        h_pool = HALF[self.dtype] if self.dtype != torch.float32 else 0.0
        for b, c in enumerate(self.ctx):
            n = self.q_lens[b]
            q = self.q[row:row + n]
            row += n
            if c == 0 or n == 0:
                outs.append(torch.zeros(n, self.hq, self.d, dtype=torch.float64))
                tols.append(torch.zeros_like(outs[-1]))
                continue
            rep = self.hq // self.hk
            k = self.k[b].repeat_interleave(rep, 1)
            v = self.v[b].repeat_interleave(rep, 1)
            s = torch.einsum("nhd,chd->hnc", q, k) * self.scale
            mag = torch.einsum("nhd,chd->hnc", q.abs(), k.abs()) * abs(self.scale)
            seen, dist = visible(n, c, self.parents[b], self.window,
                                 self.prefix[b] if self.prefix else 0)
            seen[:, [x for x in hidden if x < c]] = False
            if self.softcap:
                s = self.softcap * torch.tanh(s / self.softcap)
            if self.slopes is not None:
                sl = torch.as_tensor(self.slopes).double().float().double()
                s = s - sl[:, None, None] * dist.abs()
            o, e = attended(s, mag, seen, v, self.d, h_pool,
                            h_pool if self.q_dtype != self.dtype else 0.0, self.softcap or 0.0)
            if self.dtype == torch.float16:
                e = e + c * 2.0 ** -25 * v.abs().max()
            outs.append(o)
            tols.append(e + HALF[out_dtype] * (o.abs() + e) + 1e-30)
        return torch.cat(outs), torch.cat(tols)


def attended(s, mag, seen, v, width, h_pool, h_query, cap):
    """(output, bound) of scores s (h, n, c) over values v (c, h, d)."""
    s = s.masked_fill(~seen, -math.inf)
    big = torch.where(seen, s.abs(), 0.0).amax(-1, keepdim=True)
    top = torch.where(seen, mag, 0.0).amax(-1, keepdim=True)
    err = top * ((width + 4) * 2.0 ** -24 + h_query) + big * 2.0 ** -22 + cap * 2.0 ** -20
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
    p = torch.where(seen, p, 0.0)
    den = p.sum(-1, keepdim=True)
    w = torch.where(den > 0, p / den, 0.0)
    o = torch.einsum("hnc,chd->nhd", w, v)
    a = torch.einsum("hnc,chd->nhd", w, v.abs())
    return o, (2 * torch.expm1(err) + h_pool + 2.0 ** -18).permute(1, 0, 2) * a


class LatentCase:
    """A latent pool over scattered tables; what no query row may see (free blocks,
    slots past the context, keys left of every row's window) holds NaN."""

    def __init__(self, *, hq, dc, dr, ctx, q_lens=None, parents=None, dtype=torch.bfloat16,
                 q_dtype=None, window=None, bs=16, seed=0, q_scale=1.0, n_layers=1, layer=0,
                 scale=None, strides="plain", poison=True):
        from chenxing_b200 import LatentPagedKVCache
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.hq, self.dc, self.dr, self.layer, self.window = hq, dc, dr, layer, window
        self.ctx = [int(c) for c in ctx]
        self.parents = parents
        if parents is not None:
            q_lens = [len(p) for p in parents]
        self.q_lens = None if q_lens is None else [int(n) for n in q_lens]
        self.dtype, self.q_dtype = dtype, q_dtype or dtype
        self.scale = 1.0 / math.sqrt(dc + dr) if scale is None else scale
        ql = self.q_lens or [1] * len(self.ctx)
        need = [max(1, -(-c // bs)) for c in self.ctx]
        nb = sum(need) + 5
        self.cache = LatentPagedKVCache(nb, bs, n_layers, dc, dr, dtype=dtype, host_io=False)
        perm = rng.permutation(nb)
        off = np.concatenate([[0], np.cumsum(need)])
        self.tables = [perm[off[b]:off[b + 1]].tolist() for b in range(len(need))]
        pool = torch.full((nb, bs, dc + dr), math.nan if poison else 0.0)
        self.rows = []
        for b, c in enumerate(self.ctx):
            x = torch.randn(c, dc + dr, generator=gen).to(dtype)
            y = x.float().clone()
            if poison and window and ql[b]:
                y[torch.arange(c) <= c - ql[b] - window] = math.nan
            if c:
                t, pos = torch.tensor(self.tables[b]), torch.arange(c)
                pool[t[pos // bs], pos % bs] = y
            self.rows.append(x.double())
        self.cache.kv_pool[layer].copy_(pool)
        n = sum(ql)
        q = (torch.randn(n, hq, dc + dr, generator=gen) * q_scale).to(self.q_dtype)
        self.q = q.double()
        dev = q.cuda()
        if strides == "plain":
            self.q_dev = (dev[..., :dc].contiguous(), dev[..., dc:].contiguous())
        elif strides == "heads":      # head-major latents, rotary parts of wider heads
            wide = torch.full((n, hq, 24 + dr), math.nan, dtype=self.q_dtype, device="cuda")
            wide[..., 24:] = dev[..., dc:]
            self.q_dev = (dev[..., :dc].transpose(0, 1).contiguous().transpose(0, 1),
                          wide[..., 24:])
        elif strides == "one":        # one tensor
            self.q_dev = dev
        else:                         # rows that are not 16-byte aligned
            odd = torch.full((n, hq, dc + dr + 1), math.nan, dtype=self.q_dtype, device="cuda")
            odd[..., 1:] = dev
            self.q_dev = (odd[..., 1:1 + dc], odd[..., 1 + dc:])

    def batch(self, **kw):
        from chenxing_b200 import LatentBatch
        return LatentBatch(self.cache, self.tables, self.ctx, n_q_heads=self.hq, scale=self.scale,
                           q_lens=self.q_lens, window=self.window, tree_parents=self.parents, **kw)

    def run(self, batch=None, out_dtype=None, **kw):
        batch = batch or self.batch()
        fn = self.cache.verify_batch if batch.verify else self.cache.decode_batch
        return fn(self.layer, self.q_dev, batch, out_dtype=out_dtype, **kw)

    def expected(self, out_dtype, kernel, hidden=()):
        outs, tols, row = [], [], 0
        tc = kernel == "tcgen05"
        h_pool = HALF[self.dtype] if tc else 0.0
        h_query = h_pool if self.q_dtype != self.dtype else 0.0
        for b, c in enumerate(self.ctx):
            n = 1 if self.q_lens is None else self.q_lens[b]
            q = self.q[row:row + n]
            row += n
            if c == 0 or n == 0:
                outs.append(torch.zeros(n, self.hq, self.dc, dtype=torch.float64))
                tols.append(torch.zeros_like(outs[-1]))
                continue
            k = self.rows[b]
            v = k[:, None, :self.dc].expand(c, self.hq, self.dc)
            s = torch.einsum("nhd,cd->hnc", q, k) * self.scale
            mag = torch.einsum("nhd,cd->hnc", q.abs(), k.abs()) * abs(self.scale)
            seen, _ = visible(n, c, self.parents[b] if self.parents else None, self.window)
            seen[:, [x for x in hidden if x < c]] = False
            o, e = attended(s, mag, seen, v, self.dc + self.dr, h_pool, h_query, 0.0)
            if tc and self.dtype == torch.float16:
                e = e + c * 2.0 ** -25 * v.abs().max()
            outs.append(o)
            tols.append(e + HALF[out_dtype] * (o.abs() + e) + 1e-30)
        return torch.cat(outs), torch.cat(tols)

    def check(self, out, kernel=None, hidden=()):
        kernel = kernel or self.batch().kernel_kind(self.q_dtype)
        want, tol = self.expected(out.dtype, kernel, hidden)
        got = out.double().cpu()
        assert got.shape == want.shape
        assert torch.isfinite(got).all(), "non-finite output"
        worst = float(((got - want).abs() / tol.clamp_min(1e-30)).max()) if got.numel() else 0.0
        record_margin(worst)
        assert worst <= 1.0, f"error {worst:.3f} times its bound"
