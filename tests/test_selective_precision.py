"""32 bits all through: steps and gates of far logits, and scans whose bounds do not grow with the row.  In units of 2^-24 of a result (or of the sum of its terms' absolute values)."""
import pytest
import torch

from dew_b200 import ops
from dew_b200.ops import library as L
from dew_b200.ops import scan, selective
from selective_cases import NAMES, companion, draws_of_its_own, rows  # noqa: F401
from selective_cases import scan as oracle
from selective_cases import softplus

pytestmark = pytest.mark.gpu
DEV, UNIT = "cuda", 2.0 ** -24
# The exponential 4 (2^-22) and its correction 1, 1 + t or 2 + t 1, the reciprocal 2, their product 1, the series 2, the last step 1: 12 for a softplus, 10 for a sigmoid; then
# one for every product that follows.
FAR = 12


def logits(n=4096):
    return torch.linspace(-86.0, 80.0, n, device=DEV)


def off(got, want, size=None):
    return float(((got.double() - want).abs() / (want.abs() if size is None else size)).max()) / UNIT


def test_far_steps_and_gates_of_whole_rows():
    """One token of one state: y is the step; with C of nothing and D of one, y is the gate.  Their gradients are the slopes."""
    t, one = logits(), torch.ones(1, 1, 1, device=DEV)
    x = torch.ones(1, 1, len(t), device=DEV)
    dt = t[None, None].clone().requires_grad_()
    y, last = scan.selective_scan(x, dt, -torch.ones(len(t), 1, device=DEV), one, one, softplus=True)
    slope, = torch.autograd.grad(y.sum(), dt)
    s = softplus(t.double())
    assert off(y[0, 0], s) <= FAR + 2 and off(last[0, :, 0], s) <= FAR + 2 and off(slope[0, 0], torch.sigmoid(t.double())) <= FAR + 3
    z = t[None, None].clone().requires_grad_()
    y, _ = scan.selective_scan(x, torch.zeros_like(x), -torch.ones(len(t), 1, device=DEV), one, 0 * one, torch.ones(len(t), device=DEV), z)
    slope, = torch.autograd.grad(y.sum(), z)
    d = t.double()
    sig = torch.sigmoid(d)
    assert off(y[0, 0], d * sig) <= FAR + 3
    # (two terms of opposite signs; 1 - sig is off by what sig is)
    assert off(slope[0, 0], sig * (1 + d * (1 - sig)), sig * (1 + d.abs() * (1 - sig)) + sig * d.abs() * sig) <= 2 * FAR


@pytest.mark.parametrize("S", [1, 3])
def test_far_steps_and_gates_of_a_calls_rows(S):
    t = logits()
    n, one = len(t), torch.ones(1, S, 1, device=DEV)
    at = rows([2], [S], S, None, DEV)
    state = torch.zeros(1, n, 1, device=DEV)
    far = lambda: torch.full((n, 1), 8.0, device=DEV)        # (rates of -e^8: nothing of a token is left at the next, but for steps that are next to nothing themselves)
    x = torch.ones(1, S, n, device=DEV)
    x[:, :-1] = 0
    y = selective.selective_tokens(x, t.expand(1, S, n).contiguous(), far(), one, one, None, None, at, state)
    s = softplus(t.double())
    assert off(y[0, -1], s) <= FAR + 2 and off(state[0, :, 0], s) <= FAR + 2
    y = selective.selective_tokens(x, torch.zeros_like(x), far(), one, 0 * one, torch.ones(n, device=DEV), t.expand(1, S, n).contiguous(), at, state)
    assert off(y[0, -1], t.double() * torch.sigmoid(t.double())) <= FAR + 3
    state = torch.zeros(1, n, 1, 1, device=DEV)
    y = selective.ssd_tokens(x, t.expand(1, S, n).contiguous(), None, torch.full((n,), 8.0, device=DEV), one, one, None, n, 1, at, state)
    assert off(y[0, -1], s) <= FAR + 2 and off(state[0, :, 0, 0], s) <= FAR + 2


@pytest.mark.parametrize("d", [8, 1024, 1031])
def test_far_gates_of_the_norm(d):
    """A far gate beside near ones, whose squares are the mean: all positive, so the mean is off by d / 2 roundings at most, its root by half of that."""
    t = logits(512)
    z, x = torch.full((512, d), 1.5, device=DEV), torch.ones(512, d, device=DEV)
    z[:, 0] = t
    leaves = [v.requires_grad_() for v in (x, z, torch.ones(d, device=DEV))]
    y = ops.gated_rms_norm(*leaves, 1e-5, gate_first=True)
    ins = [v.detach().double().requires_grad_() for v in leaves]
    u = ins[0] * ins[1] * torch.sigmoid(ins[1])
    want = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + 1e-5) * ins[2]
    assert off(y.detach(), want.detach()) <= FAR + 6 + d / 4
    # dy of one column alone: dx there is its gate times r (and next to nothing from the mean, where the gate is far below 0)
    dy = torch.zeros_like(y)
    dy[:, 0] = 1
    near = t < -20
    got, exact = torch.autograd.grad(y, leaves[0], dy)[0][near, 0], torch.autograd.grad(want, ins[0], dy.double())[0][near, 0]
    assert off(got, exact) <= FAR + 8 + d / 4


SCANS = [(2, 200, 40, 16), (1, 333, 70, 5), (1, 160, 33, 64), (1, 90, 20, 128)]


def positive(B, T, C, N):
    """Every number positive but the rates, between 3/4 and 5/4; decays of e^-1.56 to e^-2.5.  Of terms that differ by factors of up to 1.14 (5/3)^2 those that passed k decays make up at most
    3.2 e^-1.56k of what they add up to, so what decays are off by counts 3.2 sum k e^-1.56k / sum e^-1.56k = 0.84 times in a state; 1.4 times in a state's gradient (5.3 for 3.2: dy, gate, C)."""
    g = torch.Generator(DEV).manual_seed(T)
    r = lambda *s: torch.rand(*s, generator=g, device=DEV) / 2 + 0.75
    return dict(x=r(B, T, C), dt=1 + r(B, T, C) / 3, a=-(r(C, N) + 0.5), b=r(B, T, N), c=r(B, T, N), d=r(C), z=r(B, T, C), initial=r(B, C, N)), r(B, T, C), r(B, C, N)


# A decay is off by 4 (the exponential) and by 3 for each unit of its exponent (rate, constant, product), 12 in all; a term by that, FAR for its gate and one for each product and join (8); a
# sum of n positive terms by n more.  dA has the decays of both directions and its own: 3.3 times 12, FAR and 8 are below 2 TERM.
TERM = 16 + FAR + 8


@pytest.mark.parametrize("pieces", [1, 3])
@pytest.mark.parametrize("B,T,C,N", SCANS)
def test_scans_in_32_bits(B, T, C, N, pieces, monkeypatch):
    whole = selective._split
    if pieces > 1:
        monkeypatch.setattr(selective, "_split", lambda R, T, *a, **k: (max(16, T // pieces // 16 * 16), whole(R, T, *a, **k)[1]))
    t, dy, dlast = positive(B, T, C, N)
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
    out = scan.selective_scan(*leaves.values())
    grads = torch.autograd.grad(out, list(leaves.values()), (dy, dlast))
    L.check_status()
    want, size = oracle(**t, dy=dy, dlast=dlast), companion(**t, dy=dy, dlast=dlast)
    terms = dict(y=N, last=0, dx=N, ddt=2 * N, dz=N, db=C, dc=C, da=B * T, dd=B * T, dinitial=0)
    for n, v in dict(y=out[0], last=out[1], **{f"d{n}": v for n, v in zip(NAMES, grads)}).items():
        assert off(v.detach(), want[n], size[n]) <= 2 * TERM + terms[n], n        # (twice: what a gradient goes through backwards)


@pytest.mark.parametrize("H,P,N,S", [(4, 24, 16, 100), (2, 64, 128, 70), (3, 20, 200, 40), (2, 64, 128, 1), (3, 33, 30, 1)])
def test_heads_in_32_bits(H, P, N, S):
    g = torch.Generator(DEV).manual_seed(S + N)
    r = lambda *s: torch.rand(*s, generator=g, device=DEV) / 2 + 0.75
    x, dt, b, c, d, a, state = r(1, S, H * P), r(1, S, H), r(1, S, N), r(1, S, N), r(H), r(H), r(1, H, P, N)
    before = state.clone()
    y = selective.ssd_tokens(x, dt, None, a.log(), b, c, d, H, 1, rows([3], [S], S, None, DEV), state)
    for h in range(H):
        cols = slice(h * P, h * P + P)
        one = dict(x=x[..., cols], dt=dt[..., h:h + 1].expand(1, S, P), a=-a[h].log().double().exp().expand(P, N), b=b, c=c, d=d[h].expand(P), initial=before[:, h])
        want, size = oracle(**one, steps=True), companion(**one, steps=True)
        # (decays of e^-0.85 and less, 2.8 times as above with terms that differ by 3.7; steps from a softplus and rates from an exponential: FAR and 3 more of each exponent, up to 1.9)
        bound = 2.8 * (12 + 2 * (FAR + 3)) + TERM + FAR
        assert off(y[..., cols], want["y"], size["y"]) <= bound + N and off(state[:, h], want["last"], size["last"]) <= bound


@pytest.mark.parametrize("logit,a_log", [(0.0, 0.0), (5.0, 2.77), (2.0, 5.0)])
def test_states_of_chunks_in_32_bits(logit, a_log):
    """Also behind decays that are many times what is left of a row: 64 tokens of 80 each, then ends of every length."""
    g = torch.Generator(DEV).manual_seed(7)
    r = lambda *s: torch.rand(*s, generator=g, device=DEV) / 2 + 0.75
    S, H, P, N = 150, 2, 64, 128
    lengths = [150, 129, 131, 137, 64, 65, 100, 33]
    R = len(lengths)
    x, dt, b, c, state = r(R, S, H * P).bfloat16(), (r(R, S, H) + logit - 1).bfloat16(), r(R, S, N).bfloat16(), r(R, S, N).bfloat16(), r(R, H, P, N)
    rates, before = torch.full((H,), a_log, device=DEV), state.clone()
    assert selective._suits_chunks(x, H, 1, N, state)
    y = selective.ssd_tokens(x, dt, None, rates, b, c, None, H, 1, rows([1] * R, lengths, S, None, DEV), state)
    for i, n in enumerate(lengths):
        for h in range(H):
            one = dict(x=x[i:i + 1, :n, h * P:h * P + P], dt=dt[i:i + 1, :n, h:h + 1].expand(1, n, P), a=-rates[h].double().exp().expand(P, N), b=b[i:i + 1, :n], c=c[i:i + 1, :n],
                       initial=before[i:i + 1, h])
            want, size = oracle(**one, steps=True), companion(**one, steps=True)
            # A token's share: its step FAR, products 8, the decay behind it 4 and the roundings of its exponent (steps FAR, rates 4, a sum of 64 in 8 levels: 24 of each unit) where it is
            # up to 12; smaller shares than e^-12 are off by less than the sum's own roundings, 3 terms of 64 tokens.
            assert off(state[i:i + 1, h], want["last"], size["last"]) <= FAR + 8 + 4 + 24 * 12 + 3 * 64
            # y: half a step of bf16 for a weight, a state and itself; weights are of differences of sums: up to 2^-24 of 64 decays, twice
            most = 64 * float(softplus(dt.double()).max() * rates.double().exp().max())
            assert off(y[i:i + 1, :n, h * P:h * P + P], want["y"], size["y"]) <= 2.1 * 2 ** 16 + 4 * most


def forgetting(t):
    """Rates of minus infinity among the others, and what the definition makes of them: decays of 0."""
    a = t["a"].clone()
    a[::3, ::2] = -float("inf")
    a[-1] = -float("inf")
    return dict(t, a=a), dict(t, a=a.clamp_min(-1e30))


@pytest.mark.parametrize("pieces", [1, 3])
@pytest.mark.parametrize("B,T,C,N", [(1, 1, 7, 4), (2, 5, 7, 4), (1, 70, 40, 16), (2, 67, 20, 33), (1, 49, 9, 100)])
def test_states_without_memory(B, T, C, N, pieces, monkeypatch):
    whole = selective._split
    if pieces > 1:
        monkeypatch.setattr(selective, "_split", lambda R, T, *a, **k: (max(16, T // pieces // 16 * 16), whole(R, T, *a, **k)[1]))
    t, dy, dlast = positive(B, T, C, N)
    t, exact = forgetting(t)
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
    out = scan.selective_scan(*leaves.values())
    grads = torch.autograd.grad(out, list(leaves.values()), (dy, dlast))
    want, size = oracle(**exact, dy=dy, dlast=dlast), companion(**exact, dy=dy, dlast=dlast)
    terms = dict(y=N, last=0, dx=N, ddt=2 * N, dz=N, db=C, dc=C, da=B * T, dd=B * T, dinitial=0)
    for n, v in dict(y=out[0], last=out[1], **{f"d{n}": v for n, v in zip(NAMES, grads)}).items():
        assert v.isfinite().all() and off(v.detach(), want[n], size[n] + 1e-30) <= 2 * TERM + terms[n], n
    at = rows([5] * B, [T] * B, T, None, DEV)
    state = t["initial"].clone()
    logits = torch.log(torch.expm1(t["dt"].double())).float()
    y = selective.selective_tokens(t["x"], logits, torch.log(-t["a"]), t["b"], t["c"], t["d"], t["z"], at, state)
    # (steps and rates through a logarithm and back: FAR and 3 more of each exponent, up to 2.5, 1.84 times over; and of the step itself)
    more = TERM + 2 * 2.5 * (FAR + 3) + FAR
    assert off(y, want["y"], size["y"]) <= more + N and off(state, want["last"], size["last"] + 1e-30) <= more


@pytest.mark.parametrize("far", [95.0, float("inf")])
@pytest.mark.parametrize("S,P,N,dtype", [(1, 24, 16, torch.float32), (21, 24, 16, torch.float32), (70, 64, 128, torch.float32), (70, 64, 128, torch.bfloat16), (128, 64, 128, torch.bfloat16)])
def test_heads_without_memory(S, P, N, dtype, far):
    g, H = torch.Generator(DEV).manual_seed(S), 4
    r = lambda *s: torch.rand(*s, generator=g, device=DEV) / 2 + 0.75
    x, dt, b, c, d, a_log, state = r(2, S, H * P).to(dtype), r(2, S, H).to(dtype), r(2, S, N).to(dtype), r(2, S, N).to(dtype), r(H), torch.zeros(H, device=DEV), r(2, H, P, N)
    a_log[1::2] = far
    before = state.clone()
    y = selective.ssd_tokens(x, dt, None, a_log, b, c, d, H, 1, rows([3, 0], [S, max(1, S - 3)], S, None, DEV), state)
    assert y.isfinite().all() and state.isfinite().all()
    for i, (first, n) in enumerate(((3, S), (0, max(1, S - 3)))):
        for h in range(H):
            cols = slice(h * P, h * P + P)
            one = dict(x=x[i:i + 1, :n, cols], dt=dt[i:i + 1, :n, h:h + 1].expand(1, n, P), a=torch.full((P, N), -1e30 if h % 2 else -1.0, device=DEV, dtype=torch.float64), b=b[i:i + 1, :n],
                       c=c[i:i + 1, :n], d=d[h].expand(P), initial=before[i:i + 1, h] if first else None)
            want, size = oracle(**one, steps=True), companion(**one, steps=True)
            # (as above; in chunks a state's share is a sum of 64 tokens' three terms on the tensor cores, a rounding toward zero each; bf16: half a step of states, weights and y)
            bound = 2.8 * (12 + 2 * (FAR + 3)) + TERM + FAR + (2 * 3 * 64 if dtype is torch.bfloat16 else 0)
            assert off(state[i:i + 1, h], want["last"], size["last"]) <= bound
            assert off(y[i:i + 1, :n, cols], want["y"], size["y"]) <= (2.1 * 2.0 ** 16 if dtype is torch.bfloat16 else bound + N)
