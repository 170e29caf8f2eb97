"""What models over a selective state are measured on: the selective scan of whole rows with its gradients, a call's rows against states that a store keeps (prompts of uneven lengths and
single tokens), the same for a state per head, and the norm behind the gate.

``run`` computes each in plain torch, or, with ``own``, by the framework's calls on the same data.  ``exact`` restates them in 64 bits.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
MOST = 4 * 2048 * 4096 * 16            # tokens x channels x states of the largest scan


def listed():
    return [
        # a training step of a small model on short rows: latency
        dict(name="scan_train_small", kind="scan", batch=2, tokens=256, channels=512, states=16, gate=True, skip=True, initial=False, backward=True, dtype="bf16"),
        # a training step at the batch and length of the dense configuration's microbatches, a model of width 2048
        dict(name="scan_train", kind="scan", batch=4, tokens=2048, channels=4096, states=16, gate=True, skip=True, initial=False, backward=True, dtype="bf16"),
        # an fp32 model of odd sizes, with a state that comes from earlier tokens and a gradient for it
        dict(name="scan_train_fp32", kind="scan", batch=3, tokens=333, channels=200, states=24, gate=False, skip=True, initial=True, backward=True, dtype="fp32"),
        # one long document is scored: few rows, so the tokens have to be shared out
        dict(name="scan_long", kind="scan", batch=1, tokens=16384, channels=2048, states=16, gate=True, skip=True, initial=False, backward=False, dtype="bf16"),
        # one request's next token, a model of width 1024: latency
        dict(name="tokens_one", kind="tokens", rows=1, width=1, shortest=1, channels=2048, states=16, fresh=0, resting=0, dtype="bf16"),
        # a decode step of 128 requests, a model of width 4096
        dict(name="tokens_step", kind="tokens", rows=128, width=1, shortest=1, channels=8192, states=16, fresh=2, resting=3, dtype="bf16"),
        # the server's chunks of prompts: eight rows of uneven lengths, half of them go on from an earlier chunk
        dict(name="tokens_prompts", kind="tokens", rows=8, width=512, shortest=37, channels=5120, states=16, fresh=4, resting=1, dtype="bf16"),
        # one request's next token, 32 heads of 64 over 128 states: latency
        dict(name="heads_one", kind="heads", rows=1, width=1, shortest=1, heads=32, groups=1, dim=64, states=128, fresh=0, resting=0, dtype="bf16"),
        # a decode step of 128 requests, 64 heads: the states are what it moves
        dict(name="heads_step", kind="heads", rows=128, width=1, shortest=1, heads=64, groups=1, dim=64, states=128, fresh=2, resting=3, dtype="bf16"),
        # prompts in an fp32 model of other widths, two groups
        dict(name="heads_prompts_fp32", kind="heads", rows=5, width=300, shortest=1, heads=24, groups=2, dim=48, states=80, fresh=3, resting=1, dtype="fp32"),
        # a decode step's norm: latency
        dict(name="norm_step", kind="norm", rows=16, width=4096, backward=False, dtype="bf16"),
        # a training step's norm, a model of width 4096
        dict(name="norm_train", kind="norm", rows=8192, width=8192, backward=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("scan", "scan", "tokens", "tokens", "heads", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    states = rng.choice((16, 16, 16, 4, 8, 24, 32, 64, 100, 128))
    if kind == "scan":
        batch, channels = _log(rng, 1, 8), _log(rng, 8, 8192)
        tokens = _log(rng, 1, min(4096, max(2, MOST // (batch * channels * states))))
        return dict(kind=kind, batch=batch, tokens=tokens, channels=channels, states=states, gate=rng.random() < 0.75, skip=rng.random() < 0.75, initial=rng.random() < 0.5,
                    backward=rng.random() < 0.6, dtype=dtype)
    width = 1 if rng.random() < 0.5 else _log(rng, 2, 1024)
    if kind == "norm":
        rows, width = _log(rng, 1, 8192), _log(rng, 40, 8192)
        return dict(kind=kind, rows=rows, width=width if rng.random() < 0.3 else (width + 7) // 8 * 8, backward=rng.random() < 0.6, dtype=dtype)
    rows = _log(rng, 1, 256 if width == 1 else 16)
    shared = dict(kind=kind, rows=rows, width=width, shortest=rng.randint(1, width), fresh=rng.randint(0, rows), resting=rng.randint(0, rows // 4), dtype=dtype)
    if kind == "tokens":
        return dict(**shared, channels=_log(rng, 8, min(8192, MOST // (rows * width * states))), states=states)
    groups, dim = rng.choice((1, 1, 2, 4)), rng.choice((16, 32, 48, 64, 64, 100, 128))
    states = rng.choice((16, 64, 128, 128, 80, 256))
    most = MOST // (rows * width * dim * states * groups)
    return dict(**shared, heads=groups * _log(rng, 1, max(1, min(96 // groups, most))), groups=groups, dim=dim, states=states)


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    make = lambda *shape, by=1.0, to=dt: (torch.randn(shape, generator=g, device=DEV) * by).to(to)
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEV)
    # logits of steps from a thousandth to a tenth
    steps = lambda *shape: (lambda d: d + torch.log(-torch.expm1(-d)))(torch.exp(uniform(*shape) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3)))
    if case["kind"] == "scan":
        return _prepare_scan(case, make, steps)
    if case["kind"] == "norm":
        # the gate is half of the layer's wider projection
        leaves = dict(x=make(case["rows"], case["width"]), z=make(case["rows"], 2 * case["width"])[:, case["width"]:], w=make(case["width"], by=0.1) + 1)
        return dict(kind="norm", backward=case["backward"], dy=make(case["rows"], case["width"]), **{n: t.detach().requires_grad_(case["backward"]) for n, t in leaves.items()})
    R, S, N = case["rows"], case["width"], case["states"]
    h = torch.Generator().manual_seed(seed)
    lengths = [case["shortest"] + (S - case["shortest"]) * i // max(1, R - 1) for i in range(R)]
    lengths[R // 2] = S
    order = torch.randperm(R, generator=h).tolist()
    first = [17 + 5 * i for i in range(R)]
    for r in order[:case["fresh"]]:
        first[r] = 0
    for r in order[len(order) - case["resting"]:]:
        first[r], lengths[r] = -1, 0
    at = torch.arange(S)
    positions = torch.stack([torch.where(at < n, at + max(p, 0), -torch.ones_like(at)) for p, n in zip(first, lengths)]).to(DEV, torch.int32)
    ends = torch.tensor([p + n if n else 0 for p, n in zip(first, lengths)], dtype=torch.int32, device=DEV)
    stored = R + 3
    ids = torch.randperm(stored, generator=h)[:R].to(DEV, torch.int32)
    rows = dict(positions=positions, lengths=ends, row_ids=ids)
    if case["kind"] == "tokens":
        C = case["channels"]
        rank = max(1, C // 32)
        low = make(R, S, rank + 2 * N)                                       # what the layer's narrow projection gives: the step's bottleneck, B and C
        a_log = torch.log(torch.arange(1, N + 1, device=DEV, dtype=torch.float32)).repeat(C, 1) + make(C, N, by=0.1, to=torch.float32)
        return dict(kind="tokens", x=make(R, S, C, by=0.5), dt=(steps(C) + make(R, S, C, by=0.5, to=torch.float32)).to(dt), a_log=a_log, b=low[..., rank:rank + N], c=low[..., rank + N:],
                    d=make(C, by=0.3, to=torch.float32) + 1, z=make(R, S, 2 * C)[..., C:], state=make(stored, C, N, by=0.3, to=torch.float32), **rows)
    H, G, P = case["heads"], case["groups"], case["dim"]
    wide = make(R, S, H * P + 2 * G * N, by=0.5)                             # what the layer's convolution gives: x, B and C
    return dict(kind="heads", H=H, G=G, x=wide[..., :H * P], b=wide[..., H * P:H * P + G * N], c=wide[..., H * P + G * N:], dt=make(R, S, H, by=0.5), dt_bias=steps(H),
                a_log=torch.log(uniform(H) * 15 + 1), d=make(H, by=0.3, to=torch.float32) + 1, state=make(stored, H, P, N, by=0.3, to=torch.float32), **rows)


def _prepare_scan(case, make, steps):
    B, T, C, N = (case[n] for n in ("batch", "tokens", "channels", "states"))
    rank = max(1, C // 32)
    low = make(B, T, rank + 2 * N)
    dt = TYPES[case["dtype"]]
    leaves = dict(x=make(B, T, C, by=0.5), dt=(steps(C) + make(B, T, C, by=0.5, to=torch.float32)).to(dt),
                  a=-torch.arange(1, N + 1, device=DEV, dtype=torch.float32).repeat(C, 1) * torch.exp(make(C, N, by=0.1, to=torch.float32)),
                  b=low[..., rank:rank + N], c=low[..., rank + N:], d=make(C, by=0.3, to=torch.float32) + 1 if case["skip"] else None,
                  z=make(B, T, 2 * C)[..., C:] if case["gate"] else None, initial=make(B, C, N, by=0.3, to=torch.float32) if case["initial"] else None)
    leaves = {n: None if t is None else t.detach().requires_grad_(case["backward"]) for n, t in leaves.items()}
    return dict(kind="scan", backward=case["backward"], dy=make(B, T, C), dlast=make(B, C, N, by=0.1, to=torch.float32), **leaves)


def run(state):
    return {"scan": _run_scan, "tokens": _run_tokens, "heads": _run_heads, "norm": _run_norm}[state["kind"]](state)


SCAN = ("x", "dt", "a", "b", "c", "d", "z", "initial")


def _run_scan(s):
    with torch.set_grad_enabled(s["backward"]):
        if own:
            from dew_b200.ops import scan
            y, last = scan.selective_scan(*(s[n] for n in SCAN), softplus=True)
        else:
            y, last = _plain_scan(*(s[n] for n in SCAN))
    if not s["backward"]:
        return {"y": y, "last": last}
    names = [n for n in SCAN if s[n] is not None]
    grads = torch.autograd.grad((y, last), [s[n] for n in names], (s["dy"], s["dlast"]))
    return {"y": y.detach(), "last": last.detach(), **{f"d{n}": g for n, g in zip(names, grads)}}


def _plain_scan(x, dt, a, b, c, d, z, initial):
    xf, bf, cf = x.float(), b.float(), c.float()
    step = torch.log(1 + torch.exp(-dt.float().abs())) + dt.float().clamp_min(0)
    h = torch.zeros(x.shape[0], *a.shape, device=x.device) if initial is None else initial
    ys = []
    for t in range(x.shape[1]):
        h = torch.exp(step[:, t, :, None] * a) * h + (step[:, t] * xf[:, t])[..., None] * bf[:, t, None]
        ys.append((h * cf[:, t, None]).sum(-1))
    y = torch.stack(ys, 1)
    if d is not None:
        y = y + d * xf
    if z is not None:
        y = y * (z.float() * torch.sigmoid(z.float()))
    return y.to(x.dtype), h


def _run_tokens(s):
    if own:
        from dew_b200.ops import selective, token_mix
        rows = token_mix.Rows(s["positions"], s["lengths"], s["row_ids"])
        return {"y": selective.selective_tokens(s["x"], s["dt"], s["a_log"], s["b"], s["c"], s["d"], s["z"], rows, s["state"]), "state": s["state"]}
    xf, z, bf, cf = (s[n].float() for n in ("x", "z", "b", "c"))
    dt = s["dt"].float()
    step = torch.log(1 + torch.exp(-dt.abs())) + dt.clamp_min(0)
    a = -torch.exp(s["a_log"])
    ids, h = _begin(s)
    ys = []
    for t in range(xf.shape[1]):
        new = torch.exp(step[:, t, :, None] * a) * h + (step[:, t] * xf[:, t])[..., None] * bf[:, t, None]
        h = torch.where((s["positions"][:, t] >= 0)[:, None, None], new, h)
        ys.append((h * cf[:, t, None]).sum(-1))
    return _end(s, ids, h, (torch.stack(ys, 1) + s["d"] * xf) * (z * torch.sigmoid(z)))


def _begin(s):
    """The store rows of a call's rows, and the states that they begin with."""
    ids = s["row_ids"].long()
    h = s["state"][ids]
    starts = s["positions"][:, 0] == 0
    return ids, torch.where(starts.view(-1, *([1] * (h.dim() - 1))), torch.zeros_like(h), h)


def _end(s, ids, h, y):
    s["state"][ids] = torch.where((s["positions"][:, 0] >= 0).view(-1, *([1] * (h.dim() - 1))), h, s["state"][ids])
    return {"y": torch.where((s["positions"] >= 0)[..., None], y, torch.zeros_like(y)).to(s["x"].dtype), "state": s["state"]}


def _run_heads(s):
    H, G = s["H"], s["G"]
    if own:
        from dew_b200.ops import selective, token_mix
        rows = token_mix.Rows(s["positions"], s["lengths"], s["row_ids"])
        return {"y": selective.ssd_tokens(s["x"], s["dt"], s["dt_bias"], s["a_log"], s["b"], s["c"], s["d"], H, G, rows, s["state"]), "state": s["state"]}
    R, S = s["x"].shape[:2]
    xf = s["x"].float().view(R, S, H, -1)
    bf, cf = (s[n].float().reshape(R, S, G, 1, -1).expand(-1, -1, -1, H // G, -1).reshape(R, S, H, 1, -1) for n in ("b", "c"))
    dt = s["dt"].float() + s["dt_bias"]
    step = torch.log(1 + torch.exp(-dt.abs())) + dt.clamp_min(0)
    decay = torch.exp(-step * torch.exp(s["a_log"]))
    ids, h = _begin(s)
    ys = []
    for t in range(S):
        new = decay[:, t, :, None, None] * h + (step[:, t, :, None] * xf[:, t])[..., None] * bf[:, t]
        h = torch.where((s["positions"][:, t] >= 0)[:, None, None, None], new, h)
        ys.append((h * cf[:, t]).sum(-1))
    return _end(s, ids, h, (torch.stack(ys, 1) + s["d"][:, None] * xf).flatten(2))


EPS = 1e-5


def _run_norm(s):
    x, z, w = s["x"], s["z"], s["w"]
    with torch.set_grad_enabled(s["backward"]):
        if own:
            from dew_b200 import ops
            y = ops.gated_rms_norm(x, z, w, EPS, gate_first=True)
        else:
            u = x.float() * (z.float() * torch.sigmoid(z.float()))
            y = (u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w.float()).to(x.dtype)
    if not s["backward"]:
        return y
    return {"y": y.detach(), **dict(zip(("dx", "dz", "dw"), torch.autograd.grad(y, (x, z, w), s["dy"])))}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": size * (n * (6 if case["backward"] else 3) + case["width"] * (2 if case["backward"] else 1)), "flops": n * (25 if case["backward"] else 9)}
    if case["kind"] == "scan":
        B, T, C, N = (case[n] for n in ("batch", "tokens", "channels", "states"))
        wide, extra = 3 + case["gate"], B * C * N * (1 + case["initial"]) + C * (N + case["skip"])
        if case["backward"]:                       # the gradients of y and of what it came from; of the last state, the first one and the weights
            return {"bytes": size * B * T * (2 * wide * C + 4 * N) + 4 * 2 * extra, "flops": 27 * B * T * C * N}
        return {"bytes": size * B * T * (wide * C + 2 * N) + 4 * extra, "flops": 7 * B * T * C * N}
    R, S, N = case["rows"], case["width"], case["states"]
    live = sum(case["shortest"] + (S - case["shortest"]) * i // max(1, R - 1) for i in range(R)) * (1 - case["resting"] / R)
    stays = (R - case["resting"]) + max(0, R - case["resting"] - case["fresh"])                 # states written, and read
    if case["kind"] == "tokens":
        C = case["channels"]
        return {"bytes": size * live * (4 * C + 2 * N) + 4 * C * (stays * N + N + 1), "flops": 7 * live * C * N}
    H, P = case["heads"], case["dim"]
    return {"bytes": size * live * (2 * H * P + H + 2 * case["groups"] * N) + 4 * H * P * N * stays, "flops": 5 * live * H * P * N}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    if case["kind"] == "scan":
        return _exact_scan(s)
    x, b, c, d = (s[n].double() for n in ("x", "b", "c", "d"))
    state = s["state"].double()
    if case["kind"] == "tokens":
        step = torch.nn.functional.softplus(s["dt"].double(), threshold=200)
        rate = -s["a_log"].double().exp()
        z = s["z"].double()
        gate = z * torch.sigmoid(z)
    else:
        H, G = s["H"], s["G"]
        step = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=200)
        rate = -s["a_log"].double().exp()[:, None, None]
        x = x.unflatten(-1, (H, -1))
        b, c = (t.unflatten(-1, (G, -1)).repeat_interleave(H // G, -2) for t in (b, c))
    y = torch.zeros_like(x)
    for r, (first, end, at) in enumerate(zip(s["positions"][:, 0].tolist(), s["lengths"].tolist(), s["row_ids"].tolist())):
        if first < 0:
            continue
        h = state[at] * (first > 0)
        for t in range(end - first):
            if case["kind"] == "tokens":
                h = h * (step[r, t, :, None] * rate).exp() + torch.outer(step[r, t] * x[r, t], b[r, t])
                y[r, t] = (h @ c[r, t] + d * x[r, t]) * gate[r, t]
            else:
                h = h * (step[r, t, :, None, None] * rate).exp() + step[r, t, :, None, None] * x[r, t, :, :, None] * b[r, t, :, None]
                y[r, t] = torch.einsum("hpn,hn->hp", h, c[r, t]) + d[:, None] * x[r, t]
        state[at] = h
    return {"y": y if case["kind"] == "tokens" else y.flatten(2), "state": state}


def _exact_norm(s):
    x, z, w, dy = (s[n].detach().double() for n in ("x", "z", "w", "dy"))
    gate = torch.sigmoid(z)
    u = x * z * gate
    r = 1 / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + EPS)
    y = u * r * w
    if not s["backward"]:
        return y
    g = dy * w * r
    du = g - u * r * r * (g * u).mean(-1, keepdim=True)
    return {"y": y, "dx": du * z * gate, "dz": du * x * gate * (1 + z * (1 - gate)), "dw": (dy * u * r).sum(0)}


def _exact_scan(s):
    x, dt, a, b, c, dy = (s[n].detach().double() for n in ("x", "dt", "a", "b", "c", "dy"))
    d, z, initial = (None if s[n] is None else s[n].detach().double() for n in ("d", "z", "initial"))
    T = x.shape[1]
    step = torch.nn.functional.softplus(dt, threshold=200)
    hs = [torch.zeros(x.shape[0], *a.shape, dtype=torch.float64, device=x.device) if initial is None else initial]
    ys = []
    for t in range(T):
        hs.append(hs[-1] * (step[:, t, :, None] * a).exp() + (step[:, t] * x[:, t])[..., None] * b[:, t, None])
        ys.append((hs[-1] @ c[:, t, :, None])[..., 0])
    y = torch.stack(ys, 1) + (0 if d is None else d * x)
    sig = None if z is None else torch.sigmoid(z)
    out = {"y": y if z is None else y * z * sig, "last": hs[-1]}
    if not s["backward"]:
        return out
    inner = dy if z is None else dy * z * sig                                  # the gradient of what the gate multiplies
    dh, da = s["dlast"].double(), torch.zeros_like(a)
    dx, dstep, db, dc = (torch.empty_like(t) for t in (x, dt, b, c))
    for t in reversed(range(T)):
        dh = dh + inner[:, t, :, None] * c[:, t, None]
        dc[:, t] = (inner[:, t, :, None] * hs[t + 1]).sum(1)
        decay = (step[:, t, :, None] * a).exp()
        through = dh * decay * hs[t]                                           # the gradient of step times a
        db[:, t] = ((step[:, t] * x[:, t])[..., None] * dh).sum(1)
        into = (dh @ b[:, t, :, None])[..., 0]
        dx[:, t] = into * step[:, t]
        dstep[:, t] = into * x[:, t] + (through * a).sum(-1)
        da += (through * step[:, t, :, None]).sum(0)
        dh = dh * decay
    grads = {"dx": dx if d is None else dx + inner * d, "ddt": dstep * torch.sigmoid(dt), "da": da, "db": db, "dc": dc}
    if d is not None:
        grads["dd"] = (inner * x).sum((0, 1))
    if z is not None:
        grads["dz"] = dy * y * sig * (1 + z * (1 - sig))
    if initial is not None:
        grads["dinitial"] = dh
    return {**out, **grads}
