"""The selective scan's plain forms against the scan token by token in 64 bits, and what its calls refuse."""
import pytest
import torch

from dew_b200.ops import scan, selective
from selective_cases import NAMES, check, companion, draws_of_its_own, inputs, rows  # noqa: F401
from selective_cases import scan as oracle
from selective_cases import softplus


def most(t):
    return float(softplus(t["dt"].detach().double()).amax() * t["a"].detach().abs().amax())


@pytest.mark.parametrize("B,T,C,N,more", [(1, 1, 1, 1, {}), (2, 70, 6, 4, dict(initial=True)), (1, 65, 9, 17, dict(gate=False, skip=False))])
def test_chunked_form_takes_logits(B, T, C, N, more):
    t = inputs(B, T, C, N, torch.float32, "cpu", 1, **more)
    leaves = {n: None if v is None else v.requires_grad_() for n, v in t.items()}
    out = scan.selective_scan(*leaves.values(), softplus=True)
    dy, dlast = torch.randn_like(out[0]), torch.randn_like(out[1])
    given = [n for n in NAMES if t[n] is not None]
    grads = torch.autograd.grad(out, [leaves[n] for n in given], (dy, dlast))
    got = dict(y=out[0], last=out[1], **{f"d{n}": v for n, v in zip(given, grads)})
    # (its chunks' decays are products of decays: as many factors as there are tokens between)
    check(got, oracle(**t, steps=True, dy=dy, dlast=dlast), companion(**t, steps=True, dy=dy, dlast=dlast), T, C, N, 4 * most(t) + 4)


def test_the_oracle_against_differences():
    t = {n: v.double().requires_grad_() for n, v in inputs(1, 4, 2, 3, torch.float32, "cpu", 2, initial=True).items()}
    dy, dlast = torch.randn(1, 4, 2, dtype=torch.float64), torch.randn(1, 2, 3, dtype=torch.float64)
    value = lambda: (lambda o: float((o["y"] * dy).sum() + (o["last"] * dlast).sum()))(oracle(**t, steps=True))
    want = oracle(**t, steps=True, dy=dy, dlast=dlast)
    for n, v in t.items():
        flat = v.detach().view(-1)
        for i in range(len(flat)):
            old, h = float(flat[i]), 1e-5
            flat[i] = old + h
            up = value()
            flat[i] = old - h
            down = value()
            flat[i] = old
            assert abs((up - down) / (2 * h) - float(want[f"d{n}"].reshape(-1)[i])) < 1e-7 * max(1.0, abs(up)), n


def test_tokens_against_whole_rows():
    """Rows that start, go on and rest, in one call; the same rows' tokens in two."""
    t = inputs(3, 20, 5, 4, torch.float32, "cpu", 3)
    a_log, state = torch.log(-t["a"]), torch.randn(4, 5, 4)
    before = state.clone()
    args = lambda i, j: (t["x"][:, i:j], t["dt"][:, i:j], a_log, t["b"][:, i:j], t["c"][:, i:j], t["d"], t["z"][:, i:j])
    y = selective.selective_tokens(*args(0, 20), rows([0, 7, -1], [20, 11, 0], 20, [2, 0, 1], "cpu"), state)
    assert not y[2].any() and not y[1, 11:].any() and torch.equal(state[[1, 3]], before[[1, 3]])
    for i, (n, at) in enumerate(((20, 2), (11, 0))):
        one = {k: v[i:i + 1, :n] if k in ("x", "dt", "b", "c", "z") else v for k, v in t.items()}
        one["initial"] = before[at:at + 1] if i else None
        check(dict(y=y[i:i + 1, :n], last=state[at:at + 1]), oracle(**one, steps=True), companion(**one, steps=True), n, 5, 4, 2 * most(t))
    again = torch.full_like(before, float("nan"))
    again[0] = before[0]
    first = selective.selective_tokens(*args(0, 8), rows([0, 7, -1], [8, 8, 0], 8, [2, 0, 1], "cpu"), again)
    second = selective.selective_tokens(*args(8, 20), rows([8, 15, -1], [12, 3, 0], 12, [2, 0, 1], "cpu"), again)
    assert torch.allclose(torch.cat([first, second], 1), y, atol=1e-5) and torch.allclose(again[[0, 2]], state[[0, 2]], atol=1e-5)


def test_heads_are_channels_of_one_rate():
    R, S, H, G, P, N = 2, 6, 4, 2, 3, 5
    x, dt, b, c = torch.randn(R, S, H * P), torch.randn(R, S, H), torch.randn(R, S, G * N), torch.randn(R, S, G * N)
    bias, a_log, d, state = torch.randn(H), torch.randn(H), torch.randn(H), torch.randn(R, H, P, N)
    r, before = rows([3, 0], [6, 4], S, None, "cpu"), state.clone()
    y = selective.ssd_tokens(x, dt, bias, a_log, b, c, d, H, G, r, state)
    for h in range(H):
        g, cols, kept = h // 2, slice(h * P, h * P + P), before[:, h].clone()
        want = selective.selective_tokens(x[..., cols], (dt[..., h:h + 1] + bias[h]).expand(R, S, P).contiguous(), a_log[h].expand(P, N), b[..., g * N:g * N + N], c[..., g * N:g * N + N],
                                          d[h].expand(P), None, r, kept)
        assert torch.allclose(y[..., cols], want, atol=1e-5) and torch.allclose(state[:, h], kept, atol=1e-5)


def test_gradients_pass_the_plain_form():
    t = inputs(2, 5, 3, 4, torch.float32, "cpu", 5)
    leaves = [t["x"].requires_grad_(), t["dt"].requires_grad_(), torch.log(-t["a"]).requires_grad_()]
    y = selective.selective_tokens(*leaves, t["b"], t["c"], t["d"], t["z"])
    want = scan.selective_scan(leaves[0], leaves[1], -torch.exp(leaves[2]), t["b"], t["c"], t["d"], t["z"], softplus=True)[0]
    for a, b in zip(torch.autograd.grad(y.sum(), leaves), torch.autograd.grad(want.sum(), leaves)):
        assert torch.allclose(a, b, atol=1e-4, rtol=1e-4)


def refused(kind, what, change):
    t = inputs(2, 3, 8, 4, torch.float32, "cpu", 6)
    call = dict(x=t["x"], dt=t["dt"], A_log=torch.log(-t["a"]), Bm=t["b"], Cm=t["c"], D=t["d"], z=t["z"], rows=rows([0, 4], [3, 2], 3, [1, 0], "cpu"), state=torch.zeros(2, 8, 4))
    if kind == "heads":
        call = dict(x=t["x"], dt=t["dt"][..., :2], dt_bias=torch.zeros(2), A_log=torch.zeros(2), Bm=t["b"], Cm=t["c"], D=torch.zeros(2), H=2, G=2, rows=call["rows"],
                    state=torch.zeros(2, 2, 4, 2))
    fn = selective.ssd_tokens if kind == "heads" else selective.selective_tokens
    fn(**call)
    call.update(change(call))
    with pytest.raises(what):
        fn(**call)


REFUSALS = [("tokens", ValueError, lambda c: dict(x=c["x"][0])), ("tokens", ValueError, lambda c: dict(dt=c["dt"][..., :4])), ("tokens", ValueError, lambda c: dict(Bm=c["Bm"][:, :2])),
            ("tokens", ValueError, lambda c: dict(z=c["z"][:1])), ("tokens", ValueError, lambda c: dict(D=c["D"][:3])), ("tokens", ValueError, lambda c: dict(A_log=c["A_log"][:3])),
            ("tokens", TypeError, lambda c: dict(x=c["x"].half())), ("tokens", TypeError, lambda c: dict(Cm=c["Cm"].bfloat16())), ("tokens", TypeError, lambda c: dict(dt=c["dt"].double())),
            ("tokens", TypeError, lambda c: dict(rows=c["rows"]._replace(positions=c["rows"].positions.long()))), ("tokens", ValueError, lambda c: dict(state=c["state"].double())),
            ("tokens", ValueError, lambda c: dict(rows=c["rows"]._replace(lengths=c["rows"].lengths[:1]))), ("tokens", ValueError, lambda c: dict(state=c["state"][:, :, :2])),
            ("tokens", ValueError, lambda c: dict(state=c["state"][:1], rows=c["rows"]._replace(row_ids=None))), ("tokens", ValueError, lambda c: dict(state=c["state"].transpose(0, 1))),
            ("heads", ValueError, lambda c: dict(H=3)), ("heads", ValueError, lambda c: dict(G=4)), ("heads", ValueError, lambda c: dict(A_log=torch.zeros(3))),
            ("heads", ValueError, lambda c: dict(dt_bias=torch.zeros(1))), ("heads", ValueError, lambda c: dict(dt=c["dt"][..., :1])), ("heads", ValueError, lambda c: dict(state=c["state"][:, :1])),
            ("heads", TypeError, lambda c: dict(Bm=c["Bm"].bfloat16()))]
# what lies elsewhere
REFUSALS += [("tokens", ValueError, lambda c, n=n: {n: c[n].to("meta")}) for n in ("dt", "Cm", "z", "A_log", "D", "state")]
REFUSALS += [("heads", ValueError, lambda c, n=n: {n: c[n].to("meta")}) for n in ("Bm", "A_log", "dt_bias", "D", "state")]
REFUSALS += [("tokens", ValueError, lambda c: dict(rows=c["rows"]._replace(row_ids=c["rows"].row_ids.to("meta"))))]


@pytest.mark.parametrize("kind,what,change", REFUSALS)
def test_refusals(kind, what, change):
    refused(kind, what, change)


def test_the_size_of_what_the_launchers_are_given():
    """What the kernels' sources assert of their structures."""
    assert selective._ARGS.size == 280 and selective._GRAD.size == 120


def test_empty_calls():
    t = inputs(2, 3, 8, 4, torch.float32, "cpu", 7)
    y = selective.selective_tokens(t["x"][:0], t["dt"][:0], torch.log(-t["a"]), t["b"][:0], t["c"][:0], t["d"], t["z"][:0])
    assert y.shape == (0, 3, 8)
    none = selective.selective_tokens(t["x"], t["dt"], torch.zeros(8, 0), t["b"][..., :0], t["c"][..., :0], t["d"])
    assert torch.equal(none, t["x"] * t["d"])
