"""What serving many requests of one model is measured on: pages of a cache that are copied as rows fork and the pool is compacted, a decode step of rows that share a
prefix, and low-rank adapters of many requests beside a shared projection.

``run`` computes each in plain torch, or, with ``own``, by the framework's calls on the same data.  ``exact`` restates them in 64 bits.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # eight rows of a small decoder fork in the middle of a page: launches
        dict(name="pages_fork_small", kind="pages", layers=4, pages=64, page=16, heads=4, dim=64, copies=8, times=4, rows=16, columns=8, changed=8, dtype="bf16"),
        # a batch of rollouts forks: every sample gets a last page of its own in sixteen layers of the dense 8 B configuration
        dict(name="pages_fork_rollouts", kind="pages", layers=16, pages=256, page=64, heads=8, dim=128, copies=112, times=7, rows=128, columns=64, changed=112, dtype="bf16"),
        # the server's default pages of 16 tokens moved to the front of their pool, and the tables that named them
        dict(name="pages_compact", kind="pages", layers=24, pages=4096, page=16, heads=2, dim=64, copies=1500, times=1, rows=256, columns=64, changed=100, dtype="bf16"),
        # four samples of one prompt, a decoder of width 1024: latency
        dict(name="prefix_small", kind="prefix", rows=4, groups=1, shared=448, shared_to=448, apart=1, apart_to=60, heads=8, kv=4, dim=128, page=64, window=0, softcap=0.0, sinks=False,
             resting=0, dtype="bf16"),
        # a batch of rollouts: sixteen prompts, each sampled several times, a layer of the dense 8 B configuration
        dict(name="prefix_rollouts", kind="prefix", rows=128, groups=16, shared=1000, shared_to=2048, apart=1, apart_to=1000, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0,
             sinks=False, resting=3, dtype="bf16"),
        # every request behind one long system prompt
        dict(name="prefix_system", kind="prefix", rows=128, groups=1, shared=8192, shared_to=8192, apart=16, apart_to=256, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0, sinks=False,
             resting=0, dtype="bf16"),
        # heads of 64 with sinks and a soft cap, the server's default pages, prefixes that end inside a page
        dict(name="prefix_sinks", kind="prefix", rows=61, groups=5, shared=0, shared_to=3001, apart=1, apart_to=333, heads=40, kv=8, dim=64, page=16, window=0, softcap=30.0, sinks=True,
             resting=4, dtype="bf16"),
        # a model in fp32, heads of a width of their own, a window that ends in the prefix
        dict(name="prefix_fp32", kind="prefix", rows=24, groups=3, shared=200, shared_to=700, apart=1, apart_to=99, heads=6, kv=2, dim=80, page=16, window=500, softcap=0.0, sinks=False,
             resting=1, dtype="fp32"),
        # one request with an adapter, a decoder of width 1024: latency
        dict(name="adapters_one", kind="adapters", tokens=1, adapters=4, used=1, rank=16, width=1024, out=2048, without=0, runs=False, dtype="bf16"),
        # a step of 128 requests, the packed projection of the dense 8 B configuration, 48 adapters among them
        dict(name="adapters_step", kind="adapters", tokens=128, adapters=64, used=48, rank=32, width=4096, out=6144, without=20, runs=False, dtype="bf16"),
        # the prompts of a dozen requests entering the cache, the output projection of that configuration
        dict(name="adapters_prompts", kind="adapters", tokens=8192, adapters=16, used=12, rank=64, width=4096, out=4096, without=700, runs=True, dtype="bf16"),
        # an fp32 model of odd widths with adapters of odd rank
        dict(name="adapters_fp32", kind="adapters", tokens=77, adapters=9, used=9, rank=5, width=520, out=1004, without=7, runs=False, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("pages", "prefix", "prefix", "adapters"))
    if kind == "pages":
        page, heads, dim = rng.choice((16, 32, 48, 64)), rng.choice((1, 2, 4, 8)), rng.choice((40, 64, 80, 128))
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        layers = _log(rng, 2, 32)
        most = (1 << 30) // (layers * page * heads * dim * (4 if dtype == "fp32" else 2))
        pages = _log(rng, 24, max(25, min(6000, most // 2)))
        copies = _log(rng, 1, pages // 3)
        rows, columns = _log(rng, 1, 256), _log(rng, 1, 128)
        return dict(kind=kind, layers=layers, pages=pages, page=page, heads=heads, dim=dim, copies=copies, times=rng.choice((1, 1, 3, 8)), rows=rows, columns=columns,
                    changed=rng.randint(0, min(rows, 8000 // columns)), dtype=dtype)
    if kind == "prefix":
        plain = rng.random() < 0.75
        rows = _log(rng, 1, 128 if plain else 32)
        kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)) if plain else rng.choice((48, 80, 128, 256))
        most = 8192 if plain else 1500
        shared = sorted(rng.randint(0, _log(rng, 64, most)) for _ in range(2))
        apart = sorted(_log(rng, 1, 1000 if plain else 200) for _ in range(2))
        return dict(kind=kind, rows=rows, groups=rng.randint(1, max(1, rows // 2)), shared=shared[0], shared_to=shared[1], apart=apart[0], apart_to=apart[1], heads=kv * rng.randint(1, 8), kv=kv, dim=dim,
                    page=rng.choice((16, 48, 64, 128)), window=rng.choice((0, 0, 0, rng.randint(1, 2000))), softcap=rng.choice((0.0, 0.0, 30.0)),
                    sinks=rng.random() < 0.3, resting=rng.randint(0, rows // 4), dtype="bf16" if plain else "fp32")
    runs = rng.random() < 0.4
    tokens = _log(rng, 257, 8192) if runs else _log(rng, 1, 512)
    adapters = _log(rng, 1, 128)
    without = rng.randint(0, tokens // 2)
    used = rng.randint(1, max(1, min(adapters, tokens - without, 16 if runs else 128)))
    dtype = "fp32" if tokens <= 512 and rng.random() < 0.25 else "bf16"
    width, out = (8 * _log(rng, 8, 512) for _ in range(2))
    return dict(kind=kind, tokens=tokens, adapters=adapters, used=used, rank=rng.choice((4, 8, 13, 16, 24, 32, 64, 128)), width=width, out=out, without=without,
                runs=runs, dtype=dtype)


def _spread(lo, hi, n):
    """``n`` whole numbers from ``lo`` to ``hi``."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """The groups' row counts and shared tokens, and the rows' own tokens (group by group); rows that rest hold nothing."""
    R, G = case["rows"], case["groups"]
    ends = [R * i * (i + G) // (2 * G * G) for i in range(G + 1)]
    return [b - a for a, b in zip(ends, ends[1:])], _spread(case["shared"], case["shared_to"], G), _spread(case["apart"], case["apart_to"], R)


def prepare(case, seed):
    return {"pages": _prepare_pages, "prefix": _prepare_prefix, "adapters": _prepare_adapters}[case["kind"]](case, seed)


def _prepare_pages(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    shape = (case["layers"], case["pages"], case["page"], case["heads"], case["dim"])
    k, v = (torch.randn(shape, generator=g, device=DEV, dtype=TYPES[case["dtype"]]) for _ in range(2))
    order, n = torch.randperm(case["pages"], generator=h), case["copies"]
    # a page is copied `times` times; what is written is written once, and not read
    src = order[n:][torch.arange(n) // case["times"]]
    table = torch.randint(case["pages"], (case["rows"], case["columns"]), generator=g, device=DEV, dtype=torch.int32)
    # pieces of rows' tables: (row, first column, pages)
    each = (case["columns"] + 1) // 2
    named = torch.randint(case["pages"], (case["changed"], each), generator=h).tolist()
    first = torch.randint(case["columns"] - each + 1, (case["changed"],), generator=h).tolist()
    tables = list(zip(torch.randperm(case["rows"], generator=h).tolist(), first, named))
    return dict(kind="pages", k=k, v=v, table=table, src=src.tolist(), dst=order[:n].tolist(), tables=tables)


def _prepare_prefix(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    R, page, dt = case["rows"], case["page"], TYPES[case["dtype"]]
    sizes, shared, apart = _lengths(case)
    # what is shared: whole pages; a row's own tokens begin in the page behind them
    whole = [s // page for s in shared]
    tables, lengths = [], []
    named = sum(whole) + sum(-(-(shared[j] + a) // page) - whole[j] for j, a in zip((j for j, n in enumerate(sizes) for _ in range(n)), apart))
    names = iter(torch.randperm(named, generator=h).tolist())
    for j, n in enumerate(sizes):
        first = [next(names) for _ in range(whole[j])]
        for _ in range(n):
            length = shared[j] + apart[len(tables)]
            tables.append(first + [next(names) for _ in range(-(-length // page) - whole[j])])
            lengths.append(length)
    place = torch.randperm(R, generator=h).tolist()                                     # where in the batch each of them stands
    for r in torch.randperm(R, generator=h)[:case["resting"]].tolist():
        lengths[r] = 0
    columns = max(len(t) for t in tables)
    table = torch.zeros(R, columns, dtype=torch.int32)
    length = torch.zeros(R, dtype=torch.int32)
    for i, (t, n) in enumerate(zip(tables, lengths)):
        table[place[i], :len(t)] = torch.tensor(t, dtype=torch.int32)
        length[place[i]] = n
    pages = int(table.max()) + 1
    shape = (pages, page, case["kv"], case["dim"])
    k, v = (torch.randn(shape, generator=g, device=DEV, dtype=dt) for _ in range(2))
    q = torch.randn(R, case["heads"], case["dim"], generator=g, device=DEV, dtype=dt)
    sinks = torch.randn(case["heads"], generator=g, device=DEV) if case["sinks"] else None
    ends = torch.tensor([0] + sizes).cumsum(0)
    ints = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEV)
    return dict(kind="prefix", q=q, k=k, v=v, table=table.to(DEV), lengths=length.to(DEV), sinks=sinks, window=case["window"], softcap=case["softcap"],
                scale=case["dim"] ** -0.5, longest=max(lengths),
                order=ints(place), first=ints(ends), tokens=ints([w * page for w in whole]))


def _prepare_adapters(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    T, n, r, K, N, dt = case["tokens"], case["adapters"], case["rank"], case["width"], case["out"], TYPES[case["dtype"]]
    make = lambda *shape, by=1.0: (torch.randn(shape, generator=g, device=DEV) * by).to(dt)
    names = torch.randperm(n, generator=h)[:case["used"]]
    with_one = max(0, T - case["without"])
    at = torch.arange(with_one)
    ids = torch.cat([names[at * len(names) // max(1, with_one)], torch.full((T - with_one,), -1)])
    if not case["runs"]:
        ids = ids[torch.randperm(T, generator=h)]
    return dict(kind="adapters", x=make(T, K), w=make(N, K, by=K ** -0.5), a=make(n, r, K, by=K ** -0.5), b=make(n, N, r, by=0.5 * r ** -0.5),
                scale=torch.rand(n, generator=g, device=DEV) + 0.5, ids=ids.to(DEV, torch.int32))


def run(state):
    return {"pages": _run_pages, "prefix": _run_prefix, "adapters": _run_adapters}[state["kind"]](state)


def _run_pages(s):
    k, v, table = s["k"], s["v"], s["table"]
    if own:
        from dew_b200.ops import pages
        pages.move_pages([k, v], s["src"], s["dst"], table, s["tables"])
    else:
        src, dst = torch.tensor([s["src"], s["dst"]], device=DEV)
        k[:, dst] = k[:, src]
        v[:, dst] = v[:, src]
        if s["tables"]:
            row, first, pages = (torch.tensor(x, device=DEV) for x in zip(*s["tables"]))
            table[row[:, None], first[:, None] + torch.arange(pages.shape[1], device=DEV)] = pages.int()
    return {"k": k, "v": v, "table": table}


def _run_prefix(s):
    q, table, lengths = s["q"], s["table"], s["lengths"]
    if own:
        from dew_b200.ops import prefix
        shared = prefix.Shared(s["order"], s["first"], s["tokens"])
        return prefix.shared_decode(q, s["k"], s["v"], table, lengths, shared, s["scale"], window=s["window"] or None, softcap=s["softcap"], sinks=s["sinks"])
    R, H, D = q.shape
    page, G = s["k"].shape[1:3]
    key = torch.arange(s["longest"], device=DEV)
    slots = table.long()[:, key // page] * page + key % page                            # [R, n]
    k, v = (t.view(-1, G, D)[slots].float() for t in (s["k"], s["v"]))
    score = torch.einsum("rghd,rngd->rghn", q.float().view(R, G, H // G, D), k) * s["scale"]
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    seen = key < lengths[:, None]
    if s["window"]:
        seen = seen & (key >= lengths[:, None] - s["window"])
    score = torch.where(seen[:, None, None], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    sink = None if s["sinks"] is None else s["sinks"].view(1, G, H // G, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True) + (0.0 if sink is None else torch.exp(sink - top))
    weight = torch.where(total > 0, weight / total, torch.zeros_like(weight))
    return torch.einsum("rghn,rngd->rghd", weight, v).reshape(R, H, D).to(q.dtype)


def _run_adapters(s):
    x, w, a, b, scale, ids = (s[n] for n in ("x", "w", "a", "b", "scale", "ids"))
    if own:
        from dew_b200.ops import adapters
        return adapters.adapted_linear(x, w, adapters.Bank(a, b, scale), ids)
    n, r, K = a.shape
    chosen = (ids[:, None] == torch.arange(n, device=DEV)).float() * scale               # [T, n]: a token's adapter, and its factor
    low = (x.float() @ a.float().reshape(n * r, K).T).view(-1, n, r) * chosen[..., None]
    return (x.float() @ w.float().T + low.reshape(-1, n * r) @ b.float().transpose(1, 2).reshape(n * r, -1)).to(x.dtype)


def work(case):
    if case["kind"] == "pages":
        size = case["layers"] * case["page"] * case["heads"] * case["dim"] * (4 if case["dtype"] == "fp32" else 2)
        return {"bytes": 2 * size * (-(-case["copies"] // case["times"]) + case["copies"]) + 4 * case["changed"] * ((case["columns"] + 1) // 2), "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "prefix":
        sizes, shared, apart = _lengths(case)
        whole = [s // case["page"] * case["page"] for s in shared]
        rows_of = [j for j, n in enumerate(sizes) for _ in range(n)]
        live = 1 - case["resting"] / case["rows"]
        seen = [min(shared[j] + a, case["window"] or math.inf) for j, a in zip(rows_of, apart)]
        own_keys = sum(min(n, shared[j] - whole[j] + a) for j, a, n in zip(rows_of, apart, seen)) * live
        shared_keys = sum(max([0] + [n - min(n, shared[j] - whole[j] + a) for i, a, n in zip(rows_of, apart, seen) if i == j]) for j in range(len(sizes)))
        return {"bytes": 2 * size * case["dim"] * (case["kv"] * (own_keys + shared_keys) + case["rows"] * case["heads"]),
                "flops": 4 * case["heads"] * case["dim"] * sum(seen) * live}
    T, r, K, N = case["tokens"], case["rank"], case["width"], case["out"]
    used = case["used"] if T > case["without"] else 0
    return {"bytes": size * (T * (K + N) + K * N + used * r * (K + N)), "flops": 2 * T * K * N + 2 * max(0, T - case["without"]) * r * (K + N)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        comes_from = torch.arange(case["pages"])
        for src, dst in zip(s["src"], s["dst"]):
            comes_from[dst] = src
        table = s["table"].clone().cpu()
        for row, first, pages in s["tables"]:
            for i, page in enumerate(pages):
                table[row, first + i] = page
        return {"k": s["k"].double().index_select(1, comes_from.to(DEV)), "v": s["v"].double().index_select(1, comes_from.to(DEV)), "table": table}
    if case["kind"] == "prefix":
        return _exact_prefix(s)
    out = []
    for t in range(0, case["tokens"], 512):
        x, ids = s["x"][t:t + 512].double(), s["ids"][t:t + 512].tolist()
        y = x @ s["w"].double().T
        for j in sorted(set(ids) - {-1}):
            at = torch.tensor([i for i, name in enumerate(ids) if name == j], device=DEV)
            y[at] += (x[at] @ s["a"][j].double().T) @ s["b"][j].double().T * s["scale"][j].double()
        out.append(y)
    return torch.cat(out)


def _exact_prefix(s):
    q, page = s["q"].double(), s["k"].shape[1]
    out = torch.zeros_like(q)
    each = q.shape[1] // s["k"].shape[2]
    for r, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        lo = max(0, n - s["window"]) if s["window"] else 0
        k, v = (t[s["table"][r, :-(-n // page)].long()].flatten(0, 1)[lo:n].double().repeat_interleave(each, 1) for t in (s["k"], s["v"]))
        z = (k * q[r]).sum(-1) * s["scale"]                                             # [n, H]
        if s["softcap"]:
            z = s["softcap"] * torch.tanh(z / s["softcap"])
        if s["sinks"] is not None:
            z = torch.cat([z, s["sinks"].double()[None]])
        p = torch.softmax(z, 0)[:n - lo]
        out[r] = (p[..., None] * v).sum(0)
    return out
