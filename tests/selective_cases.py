"""The selective state space scan token by token in 64 bits, forward and backward, and what 32 bits may lose of it."""
import pytest
import torch

STEP = 2.0 ** -21        # of one token: the step (softplus, four units of 2^-24), its product with the rate and log2 e (three roundings), the exponential (2^-22), two multiply-adds


@pytest.fixture(autouse=True)
def draws_of_its_own():
    """What a test draws without a generator depends on no other test, nor does what another draws on it."""
    with torch.random.fork_rng(devices=list(range(torch.cuda.device_count()))):
        torch.manual_seed(0)
        yield


def softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


def scan(x, dt, a, b, c, d=None, z=None, initial=None, *, steps=False, dy=None, dlast=None):
    """``steps``: dt are the logits of the steps.  -> dict of y, last and, with ``dy`` (and ``dlast``), every gradient."""
    f = lambda t: None if t is None else t.detach().double()
    x, dt, a, b, c, d, z, initial, dy, dlast = (f(t) for t in (x, dt, a, b, c, d, z, initial, dy, dlast))
    return _scan(x, dt, softplus(dt) if steps else dt, torch.sigmoid(dt) if steps else torch.ones_like(dt), a, b, c, d, z, initial, dy, dlast,
                 None if z is None else z * torch.sigmoid(z), None if z is None else torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z))))


def _scan(x, dt, s, slope, a, b, c, d, z, initial, dy, dlast, gate, gate_slope, signed=True):
    B, T, C = x.shape
    rate = a if signed else -a                               # (the companion's rates are their absolute values; decays stay decays)
    h = [x.new_zeros(B, *a.shape) if initial is None else initial]
    for t in range(T):
        h.append(torch.exp(s[:, t, :, None] * rate) * h[-1] + (s[:, t] * x[:, t])[..., None] * b[:, t, None])
    inner = torch.stack([(h[t + 1] * c[:, t, None]).sum(-1) for t in range(T)], 1) + (0 if d is None else d * x)
    out = {"y": inner if z is None else inner * gate, "last": h[-1]}
    if dy is None:
        return out
    w = dy if z is None else dy * gate
    g = torch.zeros_like(h[0]) if dlast is None else dlast
    dx, ds, db, dc, da = torch.empty_like(x), torch.empty_like(x), torch.empty_like(b), torch.empty_like(c), torch.zeros_like(a)
    for t in reversed(range(T)):
        g = g + w[:, t, :, None] * c[:, t, None]
        decay = torch.exp(s[:, t, :, None] * rate)
        q = g * decay * h[t]
        into = (g * b[:, t, None]).sum(-1)
        dc[:, t], db[:, t] = (w[:, t, :, None] * h[t + 1]).sum(1), ((s[:, t] * x[:, t])[..., None] * g).sum(1)
        dx[:, t], ds[:, t] = s[:, t] * into, x[:, t] * into + (q * a).sum(-1)
        da += (q * s[:, t, :, None]).sum(0)
        g = g * decay
    out.update(dx=dx if d is None else dx + d * w, ddt=ds * slope, da=da, db=db, dc=dc)
    if d is not None:
        out["dd"] = (w * x).sum((0, 1))
    if z is not None:
        out["dz"] = dy * inner * gate_slope
    if initial is not None:
        out["dinitial"] = g
    return out


def companion(x, dt, a, b, c, d=None, z=None, initial=None, *, steps=False, dy=None, dlast=None):
    """The same sums with every term's absolute value: each rounding of the scan in 32 bits moves a result by a share of this."""
    m = lambda t: None if t is None else t.detach().double().abs()
    step = softplus(dt.detach().double()) if steps else dt.detach().double().abs()
    gate = None if z is None else m(z)                       # |silu(z)| <= |z|, its slope is below 1.1, and both are off by shares of |z| + 1
    return _scan(m(x), None, step, torch.ones_like(step), m(a), m(b), m(c), m(d), m(z), m(initial), m(dy), m(dlast), gate, None if z is None else 1.1 + gate, signed=False)


def bounds(got, want, size, T, C, N, most):
    """What each result may be off by: ``most`` is the largest product of a step and a rate.  A term passes up to 2 T decays, each off by (most + 2) STEP, and sums of up to N, T and C
    terms; bf16 results are rounded by half a step more."""
    share = (2 * T + N + C / 8 + 8) * (most + 2) * STEP      # (a sum of C terms loses up to C 2^-24)
    return {n: share * size[n] + (torch.finfo(torch.bfloat16).eps / 2 * 1.01 * want[n].abs() if got[n].dtype is torch.bfloat16 else 0) + 1e-30 for n in want}


def check(got, want, size, T, C, N, most):
    for n, bound in bounds(got, want, size, T, C, N, most).items():
        off = (got[n].detach().double() - want[n]).abs()
        assert got[n].shape == want[n].shape and bool((off <= bound).all()), (n, float((off / bound).max()), float(off.max()))


NAMES = ("x", "dt", "a", "b", "c", "d", "z", "initial")


def inputs(B, T, C, N, dtype, device, seed, gate=True, skip=True, initial=False, steps=True, strided=False, dt_type=None):
    g = torch.Generator(device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)
    wide = (lambda *s: r(*s[:-1], 2 * s[-1] + 3)[..., 3:3 + s[-1]]) if strided else r
    dt = r(B, T, C) - 3
    return dict(x=wide(B, T, C).to(dtype), dt=(dt if steps else softplus(dt)).to(dt_type or dtype), a=-torch.exp(r(C, N)), b=wide(B, T, N).to(dtype), c=wide(B, T, N).to(dtype),
                d=r(C) if skip else None, z=wide(B, T, C).to(dtype) if gate else None, initial=r(B, C, N) if initial else None)


def rows(first, lengths, S, row_ids, device):
    """``first``: the position of each row's first token, below 0 for a row that rests; ``lengths``: its tokens of the call's ``S``."""
    from dew_b200.ops.token_mix import Rows
    at = torch.arange(S)
    pos = torch.stack([torch.where(at < n, at + f, -torch.ones_like(at)) if f >= 0 else -torch.ones_like(at) for f, n in zip(first, lengths)]).to(torch.int32)
    ends = torch.tensor([f + n if f >= 0 else 0 for f, n in zip(first, lengths)], dtype=torch.int32)
    ids = None if row_ids is None else torch.tensor(row_ids, dtype=torch.int32, device=device)
    return Rows(pos.to(device), ends.to(device), ids)
