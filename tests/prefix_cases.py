"""Batches of rows that share prefixes, and the formula in 64 bits, row by row."""
import math
import random

import torch

from dew_b200.ops.prefix import Shared, group_rows


def batch(groups, heads, kv, dim, page, dtype=torch.bfloat16, pool=None, seed=0, device="cpu", garbage=True, alone=(), spare_columns=0, resting=()):
    """``groups``: (shared tokens, [own tokens of each row]).  Rows stand in a random order; ``resting`` rows (counted group by group) hold nothing; what no row's token stands in
    is NaN.  -> dict of ``shared_decode``'s arguments."""
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    tables, lengths = [], []
    fresh = iter(rng.sample(range(20000), 20000))
    for common, own in groups:
        whole = common // page
        first = [next(fresh) for _ in range(whole)]
        for n in own:
            tables.append(first + [next(fresh) for _ in range(-(-(common + n) // page) - whole)])
            lengths.append(common + n)
    place = rng.sample(range(len(tables)), len(tables))
    names = {p: i for i, p in enumerate(rng.sample(sorted({p for t in tables for p in t}), len({p for t in tables for p in t})))}
    pages = len(names) + 3                                               # pages that nobody has
    rows = [None] * len(tables)
    length = torch.zeros(len(tables), dtype=torch.int32)
    for i, (t, n) in enumerate(zip(tables, lengths)):
        rows[place[i]] = [names[p] for p in t]
        length[place[i]] = 0 if i in resting else n
    shape = (pages, page, kv, dim)
    stored = torch.zeros(pages, page, dtype=torch.bool)
    for t, n in zip(rows, [lengths[place.index(r)] for r in range(len(rows))]):
        for x in range(n):
            stored[t[x // page], x % page] = True
    make = lambda *s: torch.randn(*s, generator=g)
    out = dict(q=make(len(rows), heads, dim).to(dtype), scale=dim ** -0.5)
    if pool is None:
        k, v = (make(*shape).to(dtype) for _ in range(2))
        if garbage:
            k[~stored], v[~stored] = math.nan, math.nan
        out.update(k=k, v=v)
    else:
        limit = 127 if pool == torch.int8 else 448
        out.update({n: (make(*shape).clamp(-3, 3) / 3 * limit).to(pool) for n in ("k", "v")})
        for n in ("k_scale", "v_scale"):
            out[n] = (torch.rand(shape[:3], generator=g) + 0.5) / limit * 3
            if garbage:
                out[n][~stored] = math.nan
    columns = max([1] + [len(t) for t in rows]) + spare_columns
    table = torch.full((len(rows), columns), 12345678, dtype=torch.int32)      # (places past a row's tokens name nothing)
    for r, t in enumerate(rows):
        table[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
    order, first, tokens = group_rows([t if n not in alone else t for n, t in enumerate(rows)], page)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    out = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in out.items()}
    out.update(table=table.to(device), lengths=length.to(device), shared=Shared(ints(order), ints(first), ints(tokens)))
    return out


def truth(a, window=None, softcap=0.0, sinks=None):
    """``(o, sum p |v|, largest sum |q k| scale, longest)`` in 64 bits on the CPU."""
    c = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in a.items()}
    q, page = c["q"].double(), c["k"].shape[1]
    H, G = q.shape[1], c["k"].shape[2]
    out, size, most, longest = torch.zeros_like(q), torch.zeros_like(q), 0.0, 1
    for r, n in enumerate(c["lengths"].tolist()):
        if n == 0:
            continue
        lo = max(0, n - window) if window else 0
        held = c["table"][r, :-(-n // page)].long()
        k, v = (c[x][held].flatten(0, 1)[lo:n].double() for x in ("k", "v"))
        if "k_scale" in c:
            k, v = (t * c[x][held].flatten(0, 1)[lo:n].double()[..., None] for t, x in ((k, "k_scale"), (v, "v_scale")))
        k, v = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
        s = (k * q[r]).sum(-1) * c["scale"]
        most = max(most, float((k.abs() * q[r].abs()).sum(-1).max() * c["scale"]))
        longest = max(longest, n)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if sinks is not None:
            s = torch.cat([s, sinks.double().cpu()[None]])
        p = torch.softmax(s, 0)[:n - lo]
        out[r], size[r] = (p[..., None] * v).sum(0), (p[..., None] * v.abs()).sum(0)
    return out, size, most, longest


def allowed(a, found):
    """How far a kernel's output may be: its own rounding (half a step), weights rounded to bf16 in front of the second product (the same, of sum p |v|), scores summed in fp32
    over the head (a score's error times its weight, twice: in the weight and in the sum of weights), exponentials of 2^-21, values and weights summed over the keys."""
    o, size, most, longest = found
    dim, half = a["q"].shape[-1], torch.finfo(a["q"].dtype).eps / 2
    weights = half if a["q"].dtype == torch.bfloat16 else 0.0
    return half * o.abs() + size * (weights * 1.01 + 2 * ((dim + 4) * 2.0 ** -24 * most + 2.0 ** -21) + (longest + 64) * 2.0 ** -24) + 1e-30


def numbers_that_are_none(a, row, other):
    """``a`` with queries that no score of is a number (one head of ``row``; all of a resting row's), one whose every key scores minus infinity (a head of ``other``), and one
    that meets infinity: ``(arguments, rows x heads that are to be NaN, to be zero, as they were)``."""
    q, k = a["q"].clone(), a["k"].clone()
    R, H, _ = q.shape
    page, G = k.shape[1:3]
    q[row, 0] = math.nan
    q[a["lengths"] == 0] = math.nan
    nan, zero = torch.zeros(R, H, dtype=torch.bool), torch.zeros(R, H, dtype=torch.bool)
    nan[row, 0] = True
    # the last key head's first column: what one query multiplies with minus infinity, another with zero
    stored = torch.zeros(k.shape[:2], dtype=torch.bool)
    held = a["table"][other].tolist()
    n = int(a["lengths"][other])
    for x in range(n):
        stored[held[x // page], x % page] = True
    k[..., -1, 0] = 0
    k[..., -1, 0][stored.to(k.device)] = -math.inf
    q[:, (G - 1) * H // G:, 0] = 0                            # (0 times infinity: no number)
    q[other, H - 1, 0] = 1.0
    meets = torch.zeros(R, dtype=torch.bool)
    for r, length in enumerate(a["lengths"].tolist()):
        t = a["table"][r].tolist()
        meets[r] = any(bool(stored[t[x // page], x % page]) for x in range(length))
    nan[meets, (G - 1) * H // G:] = True
    nan[other, H - 1] = False
    zero[other, H - 1] = True
    zero[(a["lengths"] == 0).cpu()] = True
    nan &= ~zero
    same = ~nan & ~zero
    same[:, (G - 1) * H // G:] = False                        # (their queries and keys are others now)
    return {**a, "q": q, "k": k}, nan, zero, same
