"""Cases, plain forms and exact values of three operators of the paged K/V cache.

* ``append`` — RMS norm of every query and key head, rotation of the leading
  ``rot`` dims (half-split or interleaved pairs) and the slot-mapped append of
  K and V, in one call: ``RadixPagedKVCache.append_norm_rope``.
* ``decode`` — attention of one new token per sequence over the paged cache,
  with scores capped by a tanh, a bias that falls with the distance, and a
  prefix that stays visible beside a sliding window: a ``PagedBatch`` with
  ``softcap`` / ``alibi_slopes`` / ``prefix_lens`` and ``decode_batch``.
* ``verify`` — the same scores for several query tokens per sequence
  (speculative chains and prompt chunks): ``verify_batch``.

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


def _append(name, T, hq, hk, d, rot, inter, dtype, norm, fused, pad, max_pos):
    return {"name": name, "op": "append", "T": T, "hq": hq, "hk": hk, "d": d, "rot": rot,
            "inter": inter, "dtype": dtype, "norm": norm, "fused": fused, "pad": pad,
            "max_pos": max_pos}


def _attend(name, op, B, lo, hi, q_lo, q_hi, hq, hk, d, dtype, cap, alibi, window, prefix, empty,
            lens_seed):
    return {"name": name, "op": op, "B": B, "lo": lo, "hi": hi, "q_lo": q_lo, "q_hi": q_hi,
            "hq": hq, "hk": hk, "d": d, "dtype": dtype, "cap": cap, "alibi": alibi,
            "window": window, "prefix": prefix, "empty": empty, "lens_seed": lens_seed}


def listed():
    return [
        # 8 sequences decoding with 8 / 2 heads of 64: the smallest step, latency counts
        _append("append step 8 f32", 8, 8, 2, 64, 64, False, "f32", True, False, 0, 1024),
        # one decode step of a batch of 64 padded to 72 rows, 32 / 8 heads of 128, Q / K / V
        # slices of one fused projection
        _append("append step 64 bf16", 72, 32, 8, 128, 128, False, "bf16", True, True, 8, 32768),
        # an odd prompt chunk, a quarter of each head rotated in interleaved pairs, no norm
        _append("append 1037 part f16", 1037, 16, 4, 128, 32, True, "f16", False, True, 0, 16384),
        # a batch of prompt chunks: 8192 tokens in one call
        _append("append 8192 bf16", 8192, 32, 8, 128, 128, False, "bf16", True, True, 0, 32768),
        # the smallest decode: 8 fp32 sequences of up to 512 tokens, capped scores
        _attend("decode 8x512 f32 cap", "decode", 8, 64, 512, 1, 1, 8, 2, 64, "f32", 30.0, False,
                0, 0, 0, 1),
        # a serving batch of 64 with contexts of 1k to 8k, capped scores
        _attend("decode 64x8k bf16 cap", "decode", 64, 1024, 8192, 1, 1, 32, 8, 128, "bf16", 50.0,
                False, 0, 0, 0, 2),
        # two users with long contexts and distance-biased scores, one KV head per query head
        _attend("decode 2x32k f16 alibi", "decode", 2, 30000, 32768, 1, 1, 32, 32, 64, "f16", 0.0,
                True, 0, 0, 0, 3),
        # long streams: a window of 4096 beside a prefix that stays visible, two empty rows
        _attend("decode 128 window+prefix", "decode", 128, 2048, 16384, 1, 1, 32, 8, 128, "bf16",
                0.0, False, 4096, 100, 2, 4),
        # speculative chains of up to 5 rows, capped, window 4096
        _attend("verify 128x5 bf16 cap", "verify", 128, 2048, 16384, 1, 5, 32, 8, 128, "bf16",
                50.0, False, 4096, 0, 0, 5),
        # a short fp32 chain
        _attend("verify 8x4 f32 alibi", "verify", 8, 64, 512, 4, 4, 8, 2, 64, "f32", 0.0, True,
                0, 0, 0, 6),
        # prompt chunks of 1024 rows behind contexts of up to 8k, capped scores
        _attend("prefill 4x1024 bf16 cap", "verify", 4, 4096, 8192, 1024, 1024, 32, 8, 128, "bf16",
                50.0, False, 0, 0, 0, 7),
        # prompts of ragged length whose first 300 tokens see one another, distance bias, heads of 64
        _attend("prefill 6x700 f16 prefix", "verify", 6, 701, 1500, 401, 700, 16, 16, 64, "f16",
                0.0, True, 0, 300, 0, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "verify"])
    hk = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "append":
        hq = hk * rng.choice([1, 2, 4, 7, 8])
        d = rng.choice([64, 80, 96, 128, 128, 256])
        most = 8192 * 48 * 128 // ((hq + 2 * hk) * d * BYTES[dtype] // 2)
        T = _log(rng, 1, min(8192, most))
        case = _append("", T, hq, hk, d, d // rng.choice([1, 1, 2, 4]) // 4 * 4,
                       rng.random() < 0.4, dtype, rng.random() < 0.8, rng.random() < 0.6,
                       rng.choice([0, 0, T // 7]), rng.choice([4096, 32768]))
    else:
        group = rng.choice([1, 2, 3, 4, 8])
        d = rng.choice([64, 128])
        f32 = dtype == "f32"
        # speculative chains or prompt chunks (fp32: chains)
        kind = "decode" if op == "decode" else rng.choice(["chain"] if f32 else ["chain", "chunk"])
        q_hi = {"decode": 1, "chain": rng.randint(2, 9), "chunk": _log(rng, 33, 1024)}[kind]
        if f32:
            q_hi = min(q_hi, max(1, 64 // group))
        hi = max(_log(rng, 64, 32768), q_hi + 1)
        # no more keys, and no more (query, key) pairs, than the largest listed cases have
        keys = 2 ** 30 // (hk * d * BYTES[dtype])
        pairs = 2 ** 30 * 64 // (q_hi * hk * group * d)
        hi = max(q_hi + 1, min(hi, pairs))
        B = _log(rng, 1, max(1, min(128, keys // hi, pairs // hi)))
        case = _attend("", op, B, rng.randint(max(q_hi, hi // 8), hi), hi,
                       1 if kind == "decode" else rng.randint(1, q_hi), q_hi,
                       hk * group, hk, d, dtype, rng.choice([0.0, 20.0, 30.0, 50.0]),
                       rng.random() < 0.4, rng.choice([0, 0, 128, 1000, 4096]),
                       rng.choice([0, 0, 4, 100, 300]),
                       rng.choice([0, 0, 1]) if kind == "decode" else 0, rng.randint(0, 9999))
    del case["name"]
    return case


def _lens(case):
    """Context and query lengths of the batch, from the case alone."""
    r = random.Random(case["lens_seed"])
    ctx = [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    ctx[-1] = case["hi"]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["B"])]
    q[0] = case["q_hi"]
    for i in range(min(case["empty"], case["B"] - 1)):     # rows of a padded batch
        ctx[i] = 0
    return ctx, q


def _slopes(hq):
    """Slopes 2^(-8 (h + 1) / hq) of the distance bias."""
    return [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]


def prepare(case, seed):
    return _prepare_append(case, seed) if case["op"] == "append" else _prepare_attend(case, seed)


def _prepare_append(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    T, hq, hk, d, rot = case["T"], case["hq"], case["hk"], case["d"], case["rot"]
    dt = DTYPES[case["dtype"]]
    if case["fused"]:       # one projection's rows [Q heads | K heads | V heads]
        qkv = torch.randn(T, hq + 2 * hk, d, generator=g, device=DEV).to(dt)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        q = torch.randn(T, hq, d, generator=g, device=DEV).to(dt)
        k = torch.randn(T, hk, d, generator=g, device=DEV).to(dt)
        v = torch.randn(T, hk, d, generator=g, device=DEV).to(dt)
    nb = 2 * (-(-T // BLOCK)) + 3
    slots = torch.randperm(nb * BLOCK, generator=g, device=DEV)[:T]
    if case["pad"]:         # padding rows of the batch: stored nowhere
        slots[T - case["pad"]:] = -1
    positions = torch.randint(0, case["max_pos"], (T,), generator=g, device=DEV)
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    ang = torch.arange(case["max_pos"], dtype=torch.float64, device=DEV)[:, None] * freq
    ang = torch.cat([ang, ang], -1)
    s = {"case": case, "q": q, "k": k, "v": v, "slots": slots, "positions": positions,
         "cos": ang.cos().float(), "sin": ang.sin().float(), "qw": None, "kw": None}
    if case["norm"]:
        s["qw"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
        s["kw"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dt)
    # the pools, with one more row that takes what is stored nowhere
    s["kp"] = torch.zeros(nb * BLOCK + 1, hk, d, dtype=dt, device=DEV)
    s["vp"] = torch.zeros(nb * BLOCK + 1, hk, d, dtype=dt, device=DEV)
    if own:                 # the program's cache and rotation tables
        from chenxing_b200 import RadixPagedKVCache, RopeTables
        # one block of all the slots, so that the pools seen token by token are views (the
        # slots are scattered rows either way)
        s["cache"] = RadixPagedKVCache(1, nb * BLOCK, 1, hk, d, dtype=dt, host_io=False)
        s["pools"] = s["cache"].k_pool[0, 0], s["cache"].v_pool[0, 0]
        s["rope"] = RopeTables(case["max_pos"], rot, interleaved=case["inter"],
                               tables=(s["cos"].cpu().numpy(), s["sin"].cpu().numpy()))
    return s


def _prepare_attend(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    ctx, q_lens = _lens(case)
    B, hk, hq, d = case["B"], case["hk"], case["hq"], case["d"]
    dt = DTYPES[case["dtype"]]
    nblk = [max(1, -(-c // BLOCK)) for c in ctx]
    width, nb = max(nblk), sum(nblk) + 5
    perm = np.random.default_rng(seed).permutation(nb)
    offs = np.concatenate([[0], np.cumsum(nblk)])
    tables = [perm[offs[b]:offs[b + 1]].tolist() for b in range(B)]
    padded = np.zeros((B, width), dtype=np.int64)
    for b in range(B):
        padded[b, :nblk[b]] = tables[b]
    # pools [block][slot][head][dim], scattered over by the block tables
    kp = torch.randn(nb, BLOCK, hk, d, generator=g, device=DEV).to(dt)
    vp = torch.randn(nb, BLOCK, hk, d, generator=g, device=DEV).to(dt)
    rows = sum(q_lens)
    q = (3.0 * torch.randn(rows, hq, d, generator=g, device=DEV)).to(dt)
    prefix = [min(case["prefix"], c) for c in ctx]
    cap = case["cap"] or None
    s = {"case": case, "kp": kp, "vp": vp, "q": q, "max_q": max(q_lens),
         "tables": torch.from_numpy(padded).to(DEV),
         "ctx": torch.tensor(ctx, device=DEV), "q_lens": torch.tensor(q_lens, device=DEV),
         "prefix": torch.tensor(prefix, device=DEV),
         "seq": torch.repeat_interleave(torch.arange(B), torch.tensor(q_lens)).to(DEV),
         "loc": torch.cat([torch.arange(n) for n in q_lens]).to(DEV),
         "slopes": torch.tensor(_slopes(hq), dtype=torch.float32, device=DEV),
         "width": width}
    if own:                 # the program's cache and the batch it keeps for a step's layers
        from chenxing_b200 import PagedBatch, RadixPagedKVCache
        cache = RadixPagedKVCache(nb, BLOCK, 1, hk, d, dtype=dt, host_io=False)
        cache.k_pool.copy_(kp[None])
        cache.v_pool.copy_(vp[None])
        s["cache"] = cache
        s["batch"] = PagedBatch(cache, tables, ctx, n_q_heads=hq,
                                q_lens=q_lens if case["op"] == "verify" else None,
                                window=case["window"] or None, softcap=cap,
                                alibi_slopes=_slopes(hq) if case["alibi"] else None,
                                prefix_lens=prefix if case["prefix"] else None)
    return s


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attend(state)


def _own(s):
    case = s["case"]
    cache = s["cache"]
    if case["op"] == "append":
        q_out = cache.append_norm_rope(0, s["k"], s["v"], s["slots"], s["positions"], s["rope"],
                                       s["q"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
        return (q_out, *s["pools"])
    call = cache.decode_batch if case["op"] == "decode" else cache.verify_batch
    return call(0, s["q"], s["batch"], out_dtype=DTYPES[case["dtype"]])


def _rotate(x, cos, sin, rot, inter):
    a = x[..., :rot]
    if inter:
        c, n = cos[:, None, :rot // 2], sin[:, None, :rot // 2]
        even, odd = a[..., 0::2], a[..., 1::2]
        y = torch.stack([even * c - odd * n, even * n + odd * c], -1).flatten(-2)
    else:
        half = torch.cat([-a[..., rot // 2:], a[..., :rot // 2]], -1)
        y = a * cos[:, None] + half * sin[:, None]
    return torch.cat([y, x[..., rot:]], -1)


def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _plain_append(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _rotate(_normed(s["q"].float(), s["qw"]), cos, sin, case["rot"], case["inter"]).to(dt)
    k = _rotate(_normed(s["k"].float(), s["kw"]), cos, sin, case["rot"], case["inter"]).to(dt)
    last = s["kp"].shape[0] - 1
    at = torch.where(s["slots"] < 0, last, s["slots"])
    s["kp"][at] = k
    s["vp"][at] = s["v"]
    return q, s["kp"][:-1], s["vp"][:-1]


def _plain_attend(s):
    case = s["case"]
    B, hk, hq, d = case["B"], case["hk"], case["hq"], case["d"]
    group, S, Q = hq // hk, s["width"] * BLOCK, s["max_q"]
    k = s["kp"][s["tables"]].view(B, S, hk, d).permute(0, 2, 3, 1).float()
    q = torch.zeros(B, Q, hq, d, device=DEV)
    q[s["seq"], s["loc"]] = s["q"].float()
    q = q.view(B, Q, hk, group, d).permute(0, 2, 3, 1, 4).reshape(B, hk, group * Q, d)
    x = (torch.matmul(q, k) * (1.0 / math.sqrt(d))).view(B, hk, group, Q, S)
    del k
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    key = torch.arange(S, device=DEV)
    pos = (s["ctx"] - s["q_lens"])[:, None] + torch.arange(Q, device=DEV)       # (B, Q)
    pos = pos[:, None, None, :, None]
    if case["alibi"]:
        x.sub_(s["slopes"].view(hk, group, 1, 1) * (pos - key).abs())
    seen = key <= pos
    if case["window"]:
        seen = seen & (key > pos - case["window"])
    seen = (seen | (key < s["prefix"][:, None, None, None, None])) \
        & (key < s["ctx"][:, None, None, None, None])
    x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    den = x.sum(-1, keepdim=True)
    v = s["vp"][s["tables"]].view(B, S, hk, d).permute(0, 2, 1, 3).float()
    o = torch.matmul(x.view(B, hk, group * Q, S), v).view(B, hk, group, Q, d)
    o = torch.where(den > 0, o / den, 0.0).permute(0, 3, 1, 2, 4).reshape(B, Q, hq, d)
    return o[s["seq"], s["loc"]].to(DTYPES[case["dtype"]])


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "append":
        T, hq, hk, d = case["T"], case["hq"], case["hk"], case["d"]
        kept = T - case["pad"]
        rows = 2 * T * hq * d * e + 4 * kept * hk * d * e    # Q in and out, K and V in and out
        tables = min(T, case["max_pos"]) * case["rot"] * (1 if case["inter"] else 2) * 4
        flops = (T * hq + kept * hk) * (4 * d if case["norm"] else 0) \
            + (T * hq + kept * hk) * 3 * case["rot"]
        return {"bytes": rows + tables + 16 * T + (2 * d * e if case["norm"] else 0),
                "flops": flops}
    ctx, q_lens = _lens(case)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    keys = pairs = 0
    for c, n in zip(ctx, q_lens):
        if c == 0:
            continue
        pre, w = min(case["prefix"], c), case["window"]
        pos = np.arange(c - n, c, dtype=np.int64)
        lo = np.maximum(0, pos - w + 1) if w else np.zeros_like(pos)
        run = np.maximum(0, pos + 1 - np.maximum(lo, pre))      # seen keys past the prefix
        pairs += int(run.sum()) + pre * n
        keys += pre + max(0, c - max(int(lo[0]), pre))
    rows = sum(q_lens)
    return {"bytes": 2 * keys * hk * d * e + 2 * rows * hq * d * e
            + 4 * (keys // BLOCK) + 8 * case["B"],
            "flops": 4 * d * hq * pairs}


def exact(case, seed):
    """The definition in 64 bits, token by token or sequence by sequence."""
    if case["op"] == "append":
        return _exact_append(case, seed)
    ctx, q_lens = _lens(case)
    # one head's scores of a sequence at a time; about a second per 1e10 products
    s = prepare(case, seed)
    d, hk, hq = case["d"], case["hk"], case["hq"]
    rows, outs = 0, []
    for b, (c, n) in enumerate(zip(ctx, q_lens)):
        q = s["q"][rows:rows + n].double()
        rows += n
        out = torch.zeros(n, hq, d, dtype=torch.float64, device=DEV)
        if c:
            blocks = s["tables"][b, :-(-c // BLOCK)]
            k = s["kp"][blocks].flatten(0, 1)[:c].double()
            v = s["vp"][blocks].flatten(0, 1)[:c].double()
            i = torch.arange(c - n, c, device=DEV)[:, None]
            j = torch.arange(c, device=DEV)[None, :]
            dist = (i - j).double()
            hidden = dist < 0
            if case["window"]:
                hidden |= dist >= case["window"]
            hidden &= j >= int(s["prefix"][b])
            for g0 in range(hk):
                kk, vv = k[:, g0], v[:, g0]
                for h in range(g0 * (hq // hk), (g0 + 1) * (hq // hk)):
                    z = q[:, h] @ kk.T / math.sqrt(d)
                    if case["cap"]:
                        z = case["cap"] * torch.tanh(z / case["cap"])
                    if case["alibi"]:
                        z = z - 2.0 ** (-8.0 * (h + 1) / hq) * dist.abs()
                    z[hidden] = -math.inf
                    out[:, h] = torch.nan_to_num(torch.softmax(z, -1)) @ vv
        outs.append(out)
    return torch.cat(outs)


def _exact_append(case, seed):
    s = prepare(case, seed)
    rot, half = case["rot"], case["rot"] // 2

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        y = x.clone()
        cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
        for p in range(half):       # pair p of every head
            a, b = (2 * p, 2 * p + 1) if case["inter"] else (p, p + half)
            ta, tb = (p, p) if case["inter"] else (p, p + half)
            y[..., a] = x[..., a] * cos[:, None, ta] - x[..., b] * sin[:, None, ta]
            y[..., b] = x[..., b] * cos[:, None, tb] + x[..., a] * sin[:, None, tb]
        return y

    kept = torch.nonzero(s["slots"] >= 0).flatten()
    kp, vp = s["kp"][:-1].double(), s["vp"][:-1].double()
    kp[s["slots"][kept]] = turned(s["k"], s["kw"])[kept]
    vp[s["slots"][kept]] = s["v"].double()[kept]
    return turned(s["q"], s["qw"]), kp, vp
