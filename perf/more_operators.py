"""Cases, plain forms and exact values of operators for drafted trees and latent caches.

* ``tree`` — attention of a tree of drafted tokens per sequence over the paged
  K/V cache: each node sees the committed context and its own ancestors
  (``PagedBatch(..., tree_parents=)`` and ``verify_batch``).
* ``accept`` — the K/V of an accepted path moved to the positions behind the
  committed context, in every layer: ``accept_paths``.
* ``lappend`` — the append to a latent cache: RMS norm of the latent, rotation of
  the shared key part and of the queries' rotary part, in one call:
  ``LatentPagedKVCache.append_norm_rope``.
* ``lattend`` — attention over the latent cache in its absorbed form (one latent
  row a token is key and value of every head): a ``LatentBatch`` with
  ``decode_batch`` / ``verify_batch``; single tokens, chains, prompt chunks, trees.

``run`` computes the plain form (elementary torch operations, fp32, rounded
once at the end), or with ``own`` the framework's call.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
BLOCK = 16          # tokens per pool block
EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
SCORES = 1 << 29    # fp32 scores that the plain form holds at once


def _tree(name, B, lo, hi, n_lo, n_hi, roots, hq, hk, d, dtype, cap, alibi, window, prefix, seed):
    return {"name": name, "op": "tree", "B": B, "lo": lo, "hi": hi, "q_lo": n_lo, "q_hi": n_hi,
            "roots": roots, "hq": hq, "hk": hk, "d": d, "dtype": dtype, "cap": cap,
            "alibi": alibi, "window": window, "prefix": prefix, "lens_seed": seed}


def _accept(name, B, nodes, most, layers, hk, d, dtype, latent, seed):
    return {"name": name, "op": "accept", "B": B, "nodes": nodes, "most": most, "layers": layers,
            "hk": hk, "d": d, "dtype": dtype, "latent": latent, "lens_seed": seed}


def _lappend(name, T, hq, dc, dr, inter, dtype, fused, pad, max_pos):
    return {"name": name, "op": "lappend", "T": T, "hq": hq, "dc": dc, "dr": dr, "inter": inter,
            "dtype": dtype, "fused": fused, "pad": pad, "max_pos": max_pos}


def _lattend(name, kind, B, lo, hi, q_lo, q_hi, hq, dc, dr, dtype, window, empty, seed):
    return {"name": name, "op": "lattend", "kind": kind, "B": B, "lo": lo, "hi": hi, "q_lo": q_lo,
            "q_hi": q_hi, "roots": 1, "hq": hq, "dc": dc, "dr": dr, "dtype": dtype,
            "window": window, "empty": empty, "lens_seed": seed}


def listed():
    return [
        # 8 sequences with a tree of 8 nodes each, 8 / 2 heads of 64 in fp32: the smallest
        # verification, latency counts
        _tree("tree 8x8 f32", 8, 64, 512, 8, 8, 1, 8, 2, 64, "f32", 0.0, False, 0, 0, 1),
        # a serving batch: ragged trees of up to 26 nodes behind contexts of 1k to 8k
        _tree("tree 64x26 bf16", 64, 1024, 8192, 10, 26, 1, 32, 8, 128, "bf16", 0.0, False, 0, 0,
              2),
        # wide trees of up to 60 nodes from two first tokens, capped scores, a window
        _tree("tree 16x60 f16 cap", 16, 2048, 16384, 31, 60, 2, 32, 32, 64, "f16", 50.0, False,
              4096, 0, 3),
        # one user, 4 layers, a path of up to 5 of 16 nodes: the smallest move
        _accept("accept 1 f32", 1, 16, 5, 4, 2, 64, "f32", False, 4),
        # a batch of 64 after verification, 24 layers of 8 heads of 128
        _accept("accept 64 bf16", 64, 26, 6, 24, 8, 128, "bf16", False, 5),
        # one decode step of 8 sequences, 16 query heads
        _lappend("latent append 8 bf16", 8, 16, 512, 64, True, "bf16", True, 0, 32768),
        # prompt chunks: 8192 tokens in one call, 32 query heads
        _lappend("latent append 8192 bf16", 8192, 32, 512, 64, False, "bf16", True, 0, 32768),
        # the smallest decode: 4 fp32 sequences, narrow latents, one row of a padded batch empty
        _lattend("latent decode 4x1k f32", "decode", 4, 200, 1024, 1, 1, 8, 128, 32, "f32", 0, 1,
                 6),
        # a serving batch of 64 on one of several GPUs that share the heads: 16 heads
        _lattend("latent decode 64x8k bf16 h16", "decode", 64, 1024, 8192, 1, 1, 16, 512, 64,
                 "bf16", 0, 0, 7),
        # all 128 heads on one GPU, 32 sequences of up to 16k tokens
        _lattend("latent decode 32x16k bf16 h128", "decode", 32, 4096, 16384, 1, 1, 128, 512, 64,
                 "bf16", 0, 0, 8),
        # drafted trees of up to 16 nodes over latents of 256 in fp16
        _lattend("latent tree 32x16 f16", "tree", 32, 1024, 8192, 5, 16, 16, 256, 64, "f16", 0, 0,
                 9),
        # prompt chunks of 512 rows behind contexts of up to 6k
        _lattend("latent chunk 2x512 bf16", "chain", 2, 3000, 6144, 512, 512, 16, 512, 64, "bf16",
                 0, 0, 10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "accept", "lappend", "lattend", "lattend"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "tree":
        hk = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        d = rng.choice([64, 128])
        n = rng.randint(2, max(2, 64 // group)) if dtype == "f32" else _log(rng, 2, 128)
        hi = max(_log(rng, 64, 16384), n + 1)
        # no more keys, and no more (query, key) pairs, than the largest listed cases have
        keys = 2 ** 29 // (hk * d * BYTES[dtype])
        pairs = 2 ** 28 * 64 // (n * hk * group * d)
        hi = max(n + 1, min(hi, pairs, keys))
        B = _log(rng, 1, max(1, min(64, keys // hi, pairs // hi)))
        case = _tree("", B, rng.randint(max(n, hi // 8), hi), hi, rng.randint(1, n), n,
                     rng.choice([1, 1, 2, 4]), hk * group, hk, d, dtype,
                     rng.choice([0.0, 0.0, 30.0, 50.0]), rng.random() < 0.25,
                     rng.choice([0, 0, 100, 1000, 4096]), rng.choice([0, 0, 0, 40]),
                     rng.randint(0, 9999))
    elif op == "accept":
        most = rng.randint(1, 8)
        hk, d = (1, rng.choice([160, 320, 576])) if rng.random() < 0.4 else \
            (rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128]))
        case = _accept("", _log(rng, 1, 64), rng.randint(2 * most, 64), most, _log(rng, 1, 24),
                       hk, d, dtype, d in (160, 320, 576), rng.randint(0, 9999))
    elif op == "lappend":
        T = _log(rng, 1, 8192 if dtype != "f32" else 4096)
        case = _lappend("", T, rng.choice([1, 5, 16, 32]), rng.choice([128, 256, 320, 512]),
                        rng.choice([32, 64]), rng.random() < 0.5, dtype, rng.random() < 0.7,
                        rng.choice([0, 0, T // 7]), rng.choice([4096, 32768]))
    else:
        kind = rng.choice(["decode", "decode", "chain", "tree"])
        hq = rng.choice([1, 5, 8, 16, 32, 64, 128])
        dc, dr = rng.choice([(128, 32), (256, 32), (256, 64), (384, 64), (512, 64), (512, 64)])
        q = 1 if kind == "decode" else _log(rng, 2, 512) if kind == "chain" else _log(rng, 2, 64)
        f32 = dtype == "f32"
        hi = max(_log(rng, 64, 4096 if f32 else 16384), q + 1)
        keys = 2 ** (26 if f32 else 28) // (dc + dr)
        pairs = 2 ** (29 if f32 else 33) * 4 // (q * hq * (dc + dr))
        hi = max(q + 1, min(hi, pairs, keys))
        B = _log(rng, 1, max(1, min(64, keys // hi, pairs // hi)))
        case = _lattend("", kind, B, rng.randint(max(q, hi // 8), hi), hi, rng.randint(1, q), q,
                        hq, dc, dr, dtype, rng.choice([0, 0, 500, 4096]),
                        rng.choice([0, 0, 1]) if kind == "decode" else 0, rng.randint(0, 9999))
    del case["name"]
    return case


def _lens(case):
    """Context lengths (query tokens included) and query lengths, from the case alone."""
    r = random.Random(case["lens_seed"])
    ctx = [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    ctx[-1] = case["hi"]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["B"])]
    q[0] = case["q_hi"]
    for i in range(min(case.get("empty", 0), case["B"] - 1)):     # rows of a padded batch
        ctx[i] = 0
    return ctx, q


def _parents(case, q_lens):
    """A drafted tree a sequence: each node's parent (-1: behind the committed
    context), level by level, two to four children a node."""
    r = random.Random(case["lens_seed"] + 1)
    return [[-1 if i < case["roots"] else r.randint((i - 1) // 4, (i - 1) // 2)
             for i in range(n)] for n in q_lens]


def _ancestry(parents, Q):
    """(node sees node (Q, Q) bool, depth (Q,)) of one tree."""
    seen = np.zeros((Q, Q), dtype=bool)
    depth = np.zeros(Q, dtype=np.int64)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
            depth[i] = depth[p] + 1
        seen[i, i] = True
    return seen, depth


def _slopes(hq):
    """Slopes 2^(-8 (h + 1) / hq) of the distance bias."""
    return [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]


def _is_tree(case):
    return case["op"] == "tree" or case.get("kind") == "tree"


def prepare(case, seed):
    return {"tree": _prepare_attend, "lattend": _prepare_attend, "accept": _prepare_accept,
            "lappend": _prepare_lappend}[case["op"]](case, seed)


def _tables(nblk, nb, seed):
    """Block tables over scattered blocks of a pool of nb."""
    perm = np.random.default_rng(seed).permutation(nb)
    offs = np.concatenate([[0], np.cumsum(nblk)])
    return [perm[offs[b]:offs[b + 1]].tolist() for b in range(len(nblk))]


def _prepare_attend(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    ctx, q_lens = _lens(case)
    B, hq = case["B"], case["hq"]
    dt = DTYPES[case["dtype"]]
    nblk = [max(1, -(-c // BLOCK)) for c in ctx]
    width, nb = max(nblk), sum(nblk) + 5
    tables = _tables(nblk, nb, seed)
    padded = np.zeros((B, width), dtype=np.int64)
    for b in range(B):
        padded[b, :nblk[b]] = tables[b]
    rows, Q = sum(q_lens), max(q_lens)
    s = {"case": case, "max_q": Q, "width": width, "tables": torch.from_numpy(padded).to(DEV),
         "ctx": torch.tensor(ctx, device=DEV), "q_lens": torch.tensor(q_lens, device=DEV),
         "seq": torch.repeat_interleave(torch.arange(B), torch.tensor(q_lens)).to(DEV),
         "loc": torch.cat([torch.arange(n) for n in q_lens]).to(DEV)}
    parents = None
    if _is_tree(case):
        parents = _parents(case, q_lens)
        kin = [_ancestry(p, Q) for p in parents]
        s["sees"] = torch.from_numpy(np.stack([k[0] for k in kin])).to(DEV)     # (B, Q, Q)
        s["depth"] = torch.from_numpy(np.stack([k[1] for k in kin])).to(DEV)    # (B, Q)
    if case["op"] == "tree":
        hk, d = case["hk"], case["d"]
        # pools [block][slot][head][dim], scattered over by the block tables
        s["kp"] = torch.randn(nb, BLOCK, hk, d, generator=g, device=DEV).to(dt)
        s["vp"] = torch.randn(nb, BLOCK, hk, d, generator=g, device=DEV).to(dt)
        s["q"] = (3.0 * torch.randn(rows, hq, d, generator=g, device=DEV)).to(dt)
        prefix = [min(case["prefix"], c - n) for c, n in zip(ctx, q_lens)]
        s["prefix"] = torch.tensor(prefix, device=DEV)
        s["slopes"] = torch.tensor(_slopes(hq), dtype=torch.float32, device=DEV)
        if own:             # the program's cache and the batch it keeps for a step's layers
            from chenxing_b200 import PagedBatch, RadixPagedKVCache
            cache = RadixPagedKVCache(nb, BLOCK, 1, hk, d, dtype=dt, host_io=False)
            cache.k_pool.copy_(s["kp"][None])
            cache.v_pool.copy_(s["vp"][None])
            s["batch"] = PagedBatch(cache, tables, ctx, n_q_heads=hq, q_lens=q_lens,
                                    tree_parents=parents, window=case["window"] or None,
                                    softcap=case["cap"] or None,
                                    alibi_slopes=_slopes(hq) if case["alibi"] else None,
                                    prefix_lens=prefix if case["prefix"] else None)
            s["cache"] = cache
        return s
    dc, dr = case["dc"], case["dr"]
    s["pool"] = torch.randn(nb, BLOCK, dc + dr, generator=g, device=DEV).to(dt)
    # the absorbed queries come head by head from a product with each head's weight
    s["q_latent"] = (1.5 * torch.randn(hq, rows, dc, generator=g, device=DEV)).to(dt) \
        .transpose(0, 1)
    s["q_rope"] = (1.5 * torch.randn(rows, hq, dr, generator=g, device=DEV)).to(dt)
    s["scale"] = 1.0 / math.sqrt(128 + dr)
    if own:
        from chenxing_b200 import LatentBatch, LatentPagedKVCache
        cache = LatentPagedKVCache(nb, BLOCK, 1, dc, dr, dtype=dt, host_io=False)
        cache.kv_pool.copy_(s["pool"][None])
        s["batch"] = LatentBatch(cache, tables, ctx, n_q_heads=hq, scale=s["scale"],
                                 q_lens=None if case["kind"] == "decode" else q_lens,
                                 tree_parents=parents, window=case["window"] or None)
        s["cache"] = cache
    return s


def _accept_paths(case):
    """Context lengths (the nodes included), and the accepted nodes of each sequence:
    node 0, then later levels' nodes; -1 behind the last."""
    r = random.Random(case["lens_seed"])
    ctx, paths = [], []
    for b in range(case["B"]):
        ctx.append(case["nodes"] + r.randint(1, 100))
        n = case["most"] if b == 0 else r.randint(0, case["most"])
        nodes = [0] + sorted(r.sample(range(case["most"], case["nodes"]), max(0, n - 1)))
        paths.append(nodes[:n] + [-1] * (case["most"] - n))
    return ctx, paths


def _prepare_accept(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    ctx, paths = _accept_paths(case)
    nblk = [-(-c // BLOCK) for c in ctx]
    nb = sum(nblk) + 3
    tables = _tables(nblk, nb, seed)
    shape = (case["layers"], nb, BLOCK, case["hk"], case["d"])
    dt = DTYPES[case["dtype"]]
    s = {"case": case, "paths": torch.tensor(paths, dtype=torch.int32, device=DEV),
         "ctx": torch.tensor(ctx, device=DEV),
         "pools": [torch.randn(shape, generator=g, device=DEV).to(dt)
                   for _ in range(1 if case["latent"] else 2)]}
    padded = np.zeros((case["B"], max(nblk)), dtype=np.int64)
    for b in range(case["B"]):
        padded[b, :nblk[b]] = tables[b]
    s["tables"] = torch.from_numpy(padded).to(DEV)
    if own:
        from chenxing_b200 import LatentBatch, LatentPagedKVCache, PagedBatch, RadixPagedKVCache
        q_lens = [case["nodes"]] * case["B"]
        if case["latent"]:
            cache = LatentPagedKVCache(nb, BLOCK, case["layers"], case["d"] - 64, 64, dtype=dt,
                                       host_io=False)
            cache.kv_pool.copy_(s["pools"][0][..., 0, :])
            s["batch"] = LatentBatch(cache, tables, ctx, n_q_heads=1, q_lens=q_lens, scale=1.0)
            s["pools"] = [cache.kv_pool[:, :, :, None]]
        else:
            cache = RadixPagedKVCache(nb, BLOCK, case["layers"], case["hk"], case["d"], dtype=dt,
                                      host_io=False)
            cache.k_pool.copy_(s["pools"][0])
            cache.v_pool.copy_(s["pools"][1])
            s["batch"] = PagedBatch(cache, tables, ctx, n_q_heads=case["hk"], q_lens=q_lens)
            s["pools"] = [cache.k_pool, cache.v_pool]
        s["cache"] = cache
    return s


def _prepare_lappend(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    T, hq, dc, dr = case["T"], case["hq"], case["dc"], case["dr"]
    dt = DTYPES[case["dtype"]]
    if case["fused"]:       # slices of the projections' rows: [latent | k_rope], [q | q_rope]
        kv = torch.randn(T, dc + dr, generator=g, device=DEV).to(dt)
        latent, k_rope = kv[:, :dc], kv[:, dc:]
        q_rope = torch.randn(T, hq, 128 + dr, generator=g, device=DEV).to(dt)[..., 128:]
    else:
        latent = torch.randn(T, dc, generator=g, device=DEV).to(dt)
        k_rope = torch.randn(T, dr, generator=g, device=DEV).to(dt)
        q_rope = torch.randn(T, hq, dr, generator=g, device=DEV).to(dt)
    nb = 2 * (-(-T // BLOCK)) + 3
    slots = torch.randperm(nb * BLOCK, generator=g, device=DEV)[:T]
    if case["pad"]:         # padding rows of the batch: stored nowhere
        slots[T - case["pad"]:] = -1
    positions = torch.randint(0, case["max_pos"], (T,), generator=g, device=DEV)
    freq = 10000.0 ** (-torch.arange(0, dr, 2, dtype=torch.float64, device=DEV) / dr)
    ang = torch.arange(case["max_pos"], dtype=torch.float64, device=DEV)[:, None] * freq
    ang = torch.cat([ang, ang], -1)
    s = {"case": case, "latent": latent, "k_rope": k_rope, "q_rope": q_rope, "slots": slots,
         "positions": positions, "cos": ang.cos().float(), "sin": ang.sin().float(),
         "weight": (1 + 0.2 * torch.randn(dc, generator=g, device=DEV)).to(dt),
         # the pool, with one more row that takes what is stored nowhere
         "pool": torch.zeros(nb * BLOCK + 1, dc + dr, dtype=dt, device=DEV)}
    if own:                 # the program's cache and rotation tables
        from chenxing_b200 import LatentPagedKVCache, RopeTables
        s["cache"] = LatentPagedKVCache(nb, BLOCK, 1, dc, dr, dtype=dt, host_io=False)
        s["pool"] = s["cache"].kv_pool[0].view(nb * BLOCK, dc + dr)
        s["rope"] = RopeTables(case["max_pos"], dr, interleaved=case["inter"],
                               tables=(s["cos"].cpu().numpy(), s["sin"].cpu().numpy()))
    return s


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "accept":
        return _plain_accept(state)
    return _plain_lappend(state) if case["op"] == "lappend" else _plain_attend(state)


def _own(s, case):
    cache = s["cache"]
    if case["op"] == "accept":
        cache.accept_paths(s["batch"], s["paths"])
        return tuple(s["pools"])
    if case["op"] == "lappend":
        q_rope = cache.append_norm_rope(0, s["latent"], s["k_rope"], s["slots"], s["positions"],
                                        s["rope"], s["q_rope"], weight=s["weight"], eps=EPS)
        return q_rope, s["pool"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "tree":
        return cache.verify_batch(0, s["q"], s["batch"], out_dtype=dt)
    call = cache.decode_batch if case["kind"] == "decode" else cache.verify_batch
    return call(0, (s["q_latent"], s["q_rope"]), s["batch"], out_dtype=dt)


def _rotate(x, cos, sin, dr, inter):
    if inter:
        c, n = cos[:, None, :dr // 2], sin[:, None, :dr // 2]
        even, odd = x[..., 0::2], x[..., 1::2]
        return torch.stack([even * c - odd * n, even * n + odd * c], -1).flatten(-2)
    half = torch.cat([-x[..., dr // 2:], x[..., :dr // 2]], -1)
    return x * cos[:, None] + half * sin[:, None]


def _plain_lappend(s):
    case = s["case"]
    dt, dr = DTYPES[case["dtype"]], case["dr"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    c = s["latent"].float()
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    k = _rotate(s["k_rope"].float()[:, None], cos, sin, dr, case["inter"])[:, 0]
    q = _rotate(s["q_rope"].float(), cos, sin, dr, case["inter"]).to(dt)
    at = torch.where(s["slots"] < 0, s["pool"].shape[0] - 1, s["slots"])
    s["pool"][at] = torch.cat([c, k], -1).to(dt)
    return q, s["pool"][:-1]


def _plain_accept(s):
    case = s["case"]
    base = (s["ctx"] - case["nodes"])[:, None]
    node = s["paths"].long()
    to = base + torch.arange(case["most"], device=DEV)
    keep = node >= 0
    frm = torch.where(keep, base + node, to)     # what is not accepted stays where it is
    rows = torch.arange(case["B"], device=DEV)[:, None]
    src, dst = s["tables"][rows, frm // BLOCK], s["tables"][rows, to // BLOCK]
    for pool in s["pools"]:
        pool[:, dst, to % BLOCK] = pool[:, src, frm % BLOCK]
    return tuple(s["pools"])


def _plain_attend(s):
    case = s["case"]
    B, S, Q, hq = case["B"], s["width"] * BLOCK, s["max_q"], case["hq"]
    step = max(1, SCORES // (S * Q * hq))
    per = [_plain_some(s, slice(b, min(B, b + step))) for b in range(0, B, step)]
    return torch.cat(per)[s["seq"], s["loc"]].to(DTYPES[case["dtype"]])


def _plain_some(s, some):
    """The rows (b, Q, hq, dim of a value) of some sequences."""
    case = s["case"]
    tables = s["tables"][some]
    b, S, Q, hq = tables.shape[0], s["width"] * BLOCK, s["max_q"], case["hq"]
    at = (s["seq"] >= some.start) & (s["seq"] < some.stop)
    seq, loc = s["seq"][at] - some.start, s["loc"][at]
    if case["op"] == "tree":
        hk, d = case["hk"], case["d"]
        k = s["kp"][tables].view(b, S, hk, d).permute(0, 2, 3, 1).float()
        v = s["vp"][tables].view(b, S, hk, d).permute(0, 2, 1, 3).float()
        rows, scale = s["q"][at], 1.0 / math.sqrt(d)
    else:
        hk, d = 1, case["dc"] + case["dr"]
        kv = s["pool"][tables].view(b, 1, S, d).float()
        k, v = kv.transpose(2, 3), kv[..., :case["dc"]]
        rows, scale = torch.cat([s["q_latent"][at], s["q_rope"][at]], -1), s["scale"]
    q = torch.zeros(b, Q, hq, d, device=DEV)
    q[seq, loc] = rows.float()
    q = q.view(b, Q, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, hq // hk * Q, d)
    x = torch.matmul(q, k).mul_(scale).view(b, hk, hq // hk, Q, S)
    if case.get("cap"):
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    ctx, base = s["ctx"][some], (s["ctx"] - s["q_lens"])[some]
    key = torch.arange(S, device=DEV)
    node = key - base[:, None]                               # (b, S): < 0 in the committed context
    if _is_tree(case):
        depth = s["depth"][some]
        drafted = node.clamp(0, Q - 1)
        pos = base[:, None] + depth                          # (b, Q)
        key_pos = torch.where(node < 0, key, base[:, None] + depth.gather(1, drafted))
        kin = s["sees"][some].gather(2, drafted[:, None].expand(b, Q, S))
        seen = (node < 0)[:, None] | kin
    else:
        pos = base[:, None] + torch.arange(Q, device=DEV)
        key_pos = key.expand(b, S)
        seen = key_pos[:, None] <= pos[..., None]
    dist = pos[..., None] - key_pos[:, None]                 # (b, Q, S)
    if case.get("alibi"):
        x.sub_(s["slopes"].view(hk, hq // hk, 1, 1) * dist[:, None, None].abs())
    if case["window"]:
        seen = seen & (dist < case["window"])
    if case.get("prefix"):
        seen = seen | (key < s["prefix"][some][:, None])[:, None]
    seen = seen & (key < ctx[:, None])[:, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    den = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hk, hq // hk * Q, S), v).view(b, hk, hq // hk, Q, -1)
    return torch.where(den > 0, o / den, 0.0).permute(0, 3, 1, 2, 4).reshape(b, Q, hq, -1)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "lappend":
        T, hq, dc, dr = case["T"], case["hq"], case["dc"], case["dr"]
        kept = T - case["pad"]
        tables = min(T, case["max_pos"]) * dr * (1 if case["inter"] else 2) * 4
        return {"bytes": 2 * T * hq * dr * e + 2 * kept * (dc + dr) * e + tables + 16 * T + dc * e,
                "flops": kept * 4 * dc + (T * hq + kept) * 3 * dr}
    if case["op"] == "accept":
        moved = sum(n > k for p in _accept_paths(case)[1] for k, n in enumerate(p))
        row = case["layers"] * case["hk"] * case["d"] * e * (1 if case["latent"] else 2)
        return {"bytes": 2 * moved * row + 4 * case["B"] * case["most"], "flops": 0}
    ctx, q_lens = _lens(case)
    trees = _parents(case, q_lens) if _is_tree(case) else None
    keys = pairs = 0
    for b, (c, n) in enumerate(zip(ctx, q_lens)):
        if c == 0:
            continue
        base, w = c - n, case["window"]
        pre = min(case.get("prefix", 0), base)
        steps = _ancestry(trees[b], n)[1] if trees else np.arange(n)
        lo = np.maximum(0, base + steps - w + 1) if w else np.zeros(n, dtype=np.int64)
        far = np.maximum(0, base - np.maximum(lo, pre))          # committed keys past the prefix
        kin = np.minimum(steps + 1, w) if w else steps + 1       # nodes seen
        pairs += int(far.sum() + kin.sum()) + pre * n
        keys += pre + n + max(0, base - max(int(lo.min()), pre))
    rows, hq = sum(q_lens), case["hq"]
    if case["op"] == "tree":
        d = case["d"]
        return {"bytes": 2 * keys * case["hk"] * d * e + 2 * rows * hq * d * e
                + 4 * (keys // BLOCK) + 8 * case["B"], "flops": 4 * d * hq * pairs}
    dc, dr = case["dc"], case["dr"]
    return {"bytes": keys * (dc + dr) * e + rows * hq * (2 * dc + dr) * e + 4 * (keys // BLOCK)
            + 8 * case["B"], "flops": 2 * (2 * dc + dr) * hq * pairs}


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence and node by node."""
    if case["op"] == "lappend":
        return _exact_lappend(case, seed)
    s = prepare(case, seed)
    if case["op"] == "accept":
        ctx, paths = _accept_paths(case)
        out = [p.double() for p in s["pools"]]
        if own:
            out = [p.clone() for p in out]
        for b, path in enumerate(paths):
            table, base = s["tables"][b].tolist(), ctx[b] - case["nodes"]
            for k, n in enumerate(path):
                if n < 0:
                    break
                f, t = base + n, base + k
                for p in out:
                    p[:, table[t // BLOCK], t % BLOCK] = p[:, table[f // BLOCK], f % BLOCK]
        return tuple(out)
    ctx, q_lens = _lens(case)
    trees = _parents(case, q_lens) if _is_tree(case) else None
    hq, first, outs = case["hq"], 0, []
    for b, (c, n) in enumerate(zip(ctx, q_lens)):
        rows = slice(first, first + n)
        first += n
        if case["op"] == "tree":
            width, hk, scale = case["d"], case["hk"], case["d"] ** -0.5
            q = s["q"][rows].double()
        else:
            width, hk, scale = case["dc"], 1, s["scale"]
            q = torch.cat([s["q_latent"][rows].double(), s["q_rope"][rows].double()], -1)
        out = torch.zeros(n, hq, width, dtype=torch.float64, device=DEV)
        outs.append(out)
        if c == 0:
            continue
        blocks = s["tables"][b, :-(-c // BLOCK)]
        if case["op"] == "tree":
            k = s["kp"][blocks].flatten(0, 1)[:c].double()
            v = s["vp"][blocks].flatten(0, 1)[:c].double()
        else:
            k = s["pool"][blocks].flatten(0, 1)[:c, None].double()
            v = k[..., :width]
        # hidden[i, j], and how far key j lies behind row i
        base = c - n
        hidden = np.zeros((n, c), dtype=bool)
        at = np.arange(c, dtype=np.int64)                   # positions of the keys
        mine = np.arange(base, c, dtype=np.int64)           # and of the rows
        if trees:
            hidden[:, base:] = True
            for i in range(n):
                up, steps = i, 0
                while up >= 0:
                    hidden[i, base + up] = False
                    up, steps = trees[b][up], steps + 1
                mine[i] = base + steps - 1
            at[base:] = mine
        else:
            hidden |= at[None, :] > mine[:, None]
        dist = mine[:, None] - at[None, :]
        if case["window"]:
            hidden |= dist >= case["window"]
        pre = min(case.get("prefix", 0), base)
        hidden[:, :pre] = False
        hidden = torch.from_numpy(hidden).to(DEV)
        dist = torch.from_numpy(np.abs(dist)).to(DEV).double()
        for h in range(hq):
            g = h // (hq // hk)
            z = q[:, h] @ k[:, g].T * scale
            if case.get("cap"):
                z = case["cap"] * torch.tanh(z / case["cap"])
            if case.get("alibi"):
                z = z - 2.0 ** (-8.0 * (h + 1) / hq) * dist
            z[hidden] = -math.inf
            out[:, h] = torch.nan_to_num(torch.softmax(z, -1)) @ v[:, g]
    return torch.cat(outs)


def _exact_lappend(case, seed):
    s = prepare(case, seed)
    dc, dr, half = case["dc"], case["dr"], case["dr"] // 2
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]

    def turned(x):
        x = x.double()
        y = x.clone()
        shape = (-1,) + (1,) * (x.dim() - 2)
        for p in range(half):       # pair p of every row
            a, b = (2 * p, 2 * p + 1) if case["inter"] else (p, p + half)
            ta, tb = (p, p) if case["inter"] else (p, p + half)
            ca, sa = cos[:, ta].view(shape), sin[:, ta].view(shape)
            cb, sb = cos[:, tb].view(shape), sin[:, tb].view(shape)
            y[..., a] = x[..., a] * ca - x[..., b] * sa
            y[..., b] = x[..., b] * cb + x[..., a] * sb
        return y

    c = s["latent"].double()
    c = c / torch.sqrt(c.pow(2).sum(-1, keepdim=True) / dc + EPS) * s["weight"].double()
    kept = torch.nonzero(s["slots"] >= 0).flatten()
    n = s["pool"].shape[0] - (0 if own else 1)
    pool = torch.zeros(n, dc + dr, dtype=torch.float64, device=DEV)
    pool[s["slots"][kept]] = torch.cat([c, turned(s["k_rope"])], -1)[kept]
    return turned(s["q_rope"]), pool
