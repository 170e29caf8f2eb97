"""The selective scan's kernels against the scan token by token in 64 bits: whole rows with every gradient, and a call's rows with the states of a store."""
import pytest
import torch

from dew_b200.ops import library as L
from dew_b200.ops import scan, selective
from selective_cases import NAMES, check, companion, draws_of_its_own, inputs, rows  # noqa: F401
from selective_cases import scan as oracle
from selective_cases import softplus

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def most(t, steps=True):
    s = softplus(t["dt"].double()) if steps else t["dt"].double()
    return float(s.amax() * t["a"].abs().amax())


def split(pieces, monkeypatch):
    """How rows are cut and states dealt: by the rule, or as given."""
    if pieces != "rule":
        n, each = pieces
        monkeypatch.setattr(selective, "_split", lambda R, T, C, N, groups, heads=0, backward=False, fp32=False: (
            max(16, T // n // 16 * 16), (max(2, each) if not fp32 else 2) if backward and N <= 16 else each if N <= 16 and not heads else 4))


# one token, a tile and its neighbours, segments; channels of a warp, of a block and odd ones; every width of the lanes over the states; rows of a wider tensor
SCANS = [(1, 1, 1, 1, FP32, {}), (2, 15, 3, 4, FP32, dict(gate=False)), (1, 16, 32, 16, BF16, {}), (3, 17, 129, 16, BF16, dict(initial=True)), (2, 130, 31, 17, FP32, dict(strided=True)),
         (1, 300, 64, 24, BF16, dict(strided=True, skip=False)), (2, 70, 20, 33, FP32, dict(initial=True)), (1, 33, 24, 64, BF16, dict(gate=False, skip=False)),
         (2, 40, 12, 100, FP32, dict(initial=True)), (1, 150, 17, 128, BF16, dict(initial=True)), (2, 200, 520, 16, FP32, dict(steps=False, initial=True)),
         (1, 96, 64, 16, BF16, dict(dt_type=FP32, steps=False))]


@pytest.mark.parametrize("pieces", ["rule", (1, 4), (3, 2), (5, 1)])
@pytest.mark.parametrize("B,T,C,N,dtype,more", SCANS)
def test_scan_and_gradients(B, T, C, N, dtype, more, pieces, monkeypatch):
    split(pieces, monkeypatch)
    steps = more.get("steps", True)
    t = inputs(B, T, C, N, dtype, DEV, T + C, **more)
    with torch.no_grad():
        y, last = scan.selective_scan(*t.values(), softplus=steps)
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out = scan.selective_scan(*leaves.values(), softplus=steps)
    assert torch.equal(out[0], y) and torch.equal(out[1], last)
    g = torch.Generator(DEV).manual_seed(5)
    dy, dlast = torch.randn(B, T, C, generator=g, device=DEV).to(dtype), torch.randn(B, C, N, generator=g, device=DEV)
    given = [n for n in NAMES if t[n] is not None]
    grads = torch.autograd.grad(out, [leaves[n] for n in given], (dy, dlast))
    L.check_status()
    got = dict(y=y, last=last, **{f"d{n}": v for n, v in zip(given, grads)})
    assert all(got[f"d{n}"].dtype is t[n].dtype for n in given)
    check(got, oracle(**t, steps=steps, dy=dy, dlast=dlast), companion(**t, steps=steps, dy=dy, dlast=dlast), T, C, N, most(t, steps))


def test_gradients_that_are_missing():
    """A gradient of one result alone; leaves that need none."""
    t = inputs(2, 50, 24, 16, FP32, DEV, 3, initial=True)
    for which in ("y", "last"):
        leaves = {n: v.detach().requires_grad_(n in ("x", "a", "initial")) for n, v in t.items()}
        y, last = scan.selective_scan(*leaves.values(), softplus=True)
        w = torch.randn_like(y if which == "y" else last)
        grads = torch.autograd.grad(y if which == "y" else last, [leaves[n] for n in ("x", "a", "initial")], w)
        given = dict(dy=w) if which == "y" else dict(dy=torch.zeros_like(y), dlast=w)
        want, size = oracle(**t, steps=True, **given), companion(**t, steps=True, **given)
        got = {f"d{n}": g for n, g in zip(("x", "a", "initial"), grads)}
        check(got, {n: want[n] for n in got}, size, 50, 24, 16, most(t))


def call(R, S, C, N, dtype, seed, first, lengths, ids, strided=False):
    t = inputs(R, S, C, N, dtype, DEV, seed, strided=strided)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    store = (R if ids is None else max(ids) + 1) + 2
    return t, rows(first, lengths, S, ids, DEV), torch.randn(store, C, N, generator=g, device=DEV)


TOKENS = [(1, 1, 64, 16, BF16, [9], [1], None), (4, 1, 130, 16, BF16, [3, 0, -1, 70], [1] * 4, [5, 1, 0, 2]), (3, 1, 7, 5, FP32, [0, 2, 9], [1] * 3, None),
          (2, 1, 33, 24, FP32, [4, 4], [1, 1], [1, 0]), (5, 1, 40, 128, BF16, [1] * 5, [1] * 5, None), (3, 1, 100, 10, BF16, [8, 0, 3], [1] * 3, [4, 2, 0]),
          (4, 40, 72, 16, BF16, [0, 5, -1, 30], [40, 1, 0, 17], [3, 0, 1, 6]), (2, 300, 33, 16, FP32, [0, 64], [131, 300], None), (3, 150, 20, 100, FP32, [7, 0, 1], [150, 3, 64], [2, 1, 0]),
          (1, 256, 512, 16, BF16, [512], [256], [1])]


@pytest.mark.parametrize("pieces", ["rule", (1, 4), (3, 2), (5, 1)])
@pytest.mark.parametrize("R,S,C,N,dtype,first,lengths,ids", TOKENS)
def test_tokens_with_states(R, S, C, N, dtype, first, lengths, ids, pieces, monkeypatch):
    split(pieces, monkeypatch)
    t, r, state = call(R, S, C, N, dtype, S + C, first, lengths, ids, strided=C % 2 == 0)
    before = state.clone()
    a_log = torch.log(-t["a"])
    y = selective.selective_tokens(t["x"], t["dt"], a_log, t["b"], t["c"], t["d"], t["z"], r, state)
    L.check_status()
    untouched = torch.ones(len(state), dtype=torch.bool)
    for i, (f, n) in enumerate(zip(first, lengths)):
        at = i if ids is None else ids[i]
        if f < 0:
            assert not y[i].any()
            continue
        untouched[at] = False
        assert not y[i, n:].any()
        one = {k: None if v is None else v[i:i + 1, :n] if v.dim() == 3 else v for k, v in t.items()}
        one["initial"] = before[at:at + 1] if f > 0 else None
        check(dict(y=y[i:i + 1, :n], last=state[at:at + 1]), oracle(**one, steps=True), companion(**one, steps=True), n, C, N, 2 * most(t))
    assert torch.equal(state[untouched], before[untouched])


def test_whole_rows_and_rows_in_two_calls():
    """Rows without a store are whole rows; a row's tokens in two calls and one by one are its tokens in one."""
    t, r, state = call(2, 96, 48, 16, FP32, 4, [0, 0], [96, 96], None)
    a_log, per = torch.log(-t["a"]), ("x", "dt", "b", "c", "z")
    run = lambda lo, hi, r, s: selective.selective_tokens(*(t[n][:, lo:hi] if n in per else a_log if n == "a" else t[n] for n in ("x", "dt", "a", "b", "c", "d", "z")), r, s)
    want = run(0, 96, None, None)
    assert torch.equal(want, run(0, 96, r, state))
    again = torch.full_like(state, float("nan"))
    parts = [run(0, 64, rows([0, 0], [64, 64], 64, None, DEV), again)] + [run(i, i + 1, rows([i, i], [1, 1], 1, None, DEV), again) for i in range(64, 96)]
    got = torch.cat(parts, 1)
    one = dict(t, initial=None)
    check(dict(y=got, last=again[:2]), oracle(**one, steps=True), companion(**one, steps=True), 96, 48, 16, most(t))
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)


def heads(R, S, H, G, P, N, dtype, seed, first, lengths, ids):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    wide = r(R, S, H * P + 2 * G * N + 1).to(dtype)
    t = dict(x=wide[..., 1:1 + H * P], dt=(r(R, S, H) - 3).to(dtype), dt_bias=r(H), a_log=r(H), b=wide[..., 1 + H * P:1 + H * P + G * N], c=wide[..., 1 + H * P + G * N:], d=r(H))
    store = (R if ids is None else max(ids) + 1) + 1
    return t, rows(first, lengths, S, ids, DEV), r(store, H, P, N)


HEADS = [(1, 1, 4, 1, 64, 128, BF16, [5], [1], None), (3, 1, 6, 2, 48, 80, BF16, [0, 7, -1], [1] * 3, [2, 0, 3]), (2, 1, 3, 1, 5, 7, FP32, [1, 2], [1, 1], None),
         (2, 1, 2, 1, 16, 256, BF16, [3, 0], [1, 1], [1, 0]), (2, 1, 4, 4, 100, 16, FP32, [3, 9], [1, 1], None), (1, 1, 2, 1, 33, 30, BF16, [6], [1], None),
         (3, 50, 4, 2, 32, 16, BF16, [0, 9, -1], [50, 13, 0], [1, 0, 3]), (2, 140, 2, 1, 64, 128, BF16, [0, 3], [140, 70], None), (2, 33, 3, 3, 20, 33, FP32, [0, 4], [1, 33], [2, 1]),
         (1, 200, 2, 1, 48, 200, FP32, [2], [200], None)]


@pytest.mark.parametrize("pieces", ["rule", (1, 4), (3, 2), (5, 1)])
@pytest.mark.parametrize("R,S,H,G,P,N,dtype,first,lengths,ids", HEADS)
def test_heads_with_states(R, S, H, G, P, N, dtype, first, lengths, ids, pieces, monkeypatch):
    """A decay per head is a rate per channel and state that is one number in each head.  Token by token (chunks: below)."""
    monkeypatch.setattr(selective, "CHUNKED_TOKENS", 1 << 30)
    split(pieces, monkeypatch)
    t, r, state = heads(R, S, H, G, P, N, dtype, S + H, first, lengths, ids)
    before = state.clone()
    y = selective.ssd_tokens(t["x"], t["dt"], t["dt_bias"], t["a_log"], t["b"], t["c"], t["d"], H, G, r, state)
    L.check_status()
    untouched = torch.ones(len(state), dtype=torch.bool)
    for i, (f, n) in enumerate(zip(first, lengths)):
        at = i if ids is None else ids[i]
        if f < 0:
            assert not y[i].any()
            continue
        untouched[at] = False
        assert not y[i, n:].any()
        for h in range(H):
            g, cols = h // (H // G), slice(h * P, (h + 1) * P)
            one = dict(x=t["x"][i:i + 1, :n, cols], dt=(t["dt"][i:i + 1, :n, h:h + 1].double() + t["dt_bias"][h].double()).expand(-1, -1, P), a=-t["a_log"][h].double().exp().expand(P, N),
                       b=t["b"][i:i + 1, :n, g * N:(g + 1) * N], c=t["c"][i:i + 1, :n, g * N:(g + 1) * N], d=t["d"][h].expand(P), initial=before[at:at + 1, h] if f > 0 else None)
            check(dict(y=y[i:i + 1, :n, cols], last=state[at:at + 1, h]), oracle(**one, steps=True), companion(**one, steps=True), n, P, N, 2 * most(one))
    assert torch.equal(state[untouched], before[untouched])


CHUNKS = [(1, 32, 2, 1, [0], [32], None), (3, 65, 4, 2, [0, 9, -1], [65, 13, 0], [1, 0, 3]), (2, 200, 8, 1, [5, 0], [200, 64], [3, 0]), (4, 100, 2, 1, [1, 0, 700, 3], [1, 2, 100, 63], None)]


@pytest.mark.parametrize("R,S,H,G,first,lengths,ids", CHUNKS)
def test_heads_in_chunks(R, S, H, G, first, lengths, ids):
    """Heads of 64 over 128 states in bf16: the states as exact as token by token; y of states and weights that were rounded to bf16 once."""
    P, N = 64, 128
    t, r, state = heads(R, S, H, G, P, N, BF16, S + H, first, lengths, ids)
    assert selective._suits_chunks(t["x"], H, G, N)
    for n in ("x", "b", "c", "dt"):                   # (nothing behind a row's end is read)
        t[n] = t[n].clone()
        for i, m in enumerate(lengths):
            t[n][i, m:] = float("nan")
    before = state.clone()
    y = selective.ssd_tokens(t["x"], t["dt"], t["dt_bias"], t["a_log"], t["b"], t["c"], t["d"], H, G, r, state)
    L.check_status()
    untouched = torch.ones(len(state), dtype=torch.bool)
    for i, (f, n) in enumerate(zip(first, lengths)):
        at = i if ids is None else ids[i]
        assert not y[i, max(n, 0):].any()
        if f < 0:
            continue
        untouched[at] = False
        for h in range(H):
            g, cols = h // (H // G), slice(h * P, (h + 1) * P)
            one = dict(x=t["x"][i:i + 1, :n, cols], dt=(t["dt"][i:i + 1, :n, h:h + 1].double() + t["dt_bias"][h].double()).expand(-1, -1, P), a=-t["a_log"][h].double().exp().expand(P, N),
                       b=t["b"][i:i + 1, :n, g * N:(g + 1) * N], c=t["c"][i:i + 1, :n, g * N:(g + 1) * N], d=t["d"][h].expand(P), initial=before[at:at + 1, h] if f > 0 else None)
            want, size = oracle(**one, steps=True), companion(**one, steps=True)
            check(dict(last=state[at:at + 1, h]), {"last": want["last"]}, size, n, P, N, 2 * most(one))
            # a term of y is off by half a step of bf16 for its state or weight, and the sum by half a step of its own
            off = (y[i:i + 1, :n, cols].double() - want["y"]).abs()
            assert bool((off <= 2.0 ** -8 * 1.05 * (size["y"] + want["y"].abs())).all())
    assert torch.equal(state[untouched], before[untouched])


def test_a_long_row_in_many_calls():
    """Chunks, tokens one after another and single tokens go on from one another's states."""
    t, r, state = heads(1, 300, 2, 1, 64, 128, BF16, 3, [0], [300], None)
    run = lambda lo, hi, s: selective.ssd_tokens(t["x"][:, lo:hi], t["dt"][:, lo:hi], t["dt_bias"], t["a_log"], t["b"][:, lo:hi], t["c"][:, lo:hi], t["d"], 2, 1,
                                                 rows([lo], [hi - lo], hi - lo, None, DEV), s)
    whole = state.clone()
    want = run(0, 300, whole)
    parts = torch.cat([run(lo, hi, state) for lo, hi in ((0, 130), (130, 131), (131, 150), (150, 299), (299, 300))], 1)
    far = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    assert far(state[0], whole[0]) < 1e-5 and far(parts, want) < 2.0 ** -7      # (the states' roundings to bf16 fall elsewhere)


@pytest.mark.parametrize("S,dtype", [(20, BF16), (100, BF16), (100, FP32)])
def test_padding_behind_a_state_that_overflowed(S, dtype):
    t, r, state = heads(2, S, 2, 1, 64, 128, dtype, 3, [4, 0], [S - 5, S], None)
    state[0] = float("inf")
    y = selective.ssd_tokens(t["x"], t["dt"], t["dt_bias"], t["a_log"], t["b"], t["c"], t["d"], 2, 1, r, state)
    assert not y[0, S - 5:].any() and not y[0, :S - 5].isfinite().all() and y[1].isfinite().all() and state[1].isfinite().all()


def test_rows_outside_the_store_are_reported():
    t, r, state = call(3, 1, 16, 16, BF16, 1, [1, 1, 1], [1] * 3, [0, 1, 2])
    before = state.clone()
    for S, bad in ((1, 5), (1, -1), (40, 5)):
        t, _, _ = call(3, S, 16, 16, BF16, 1, [1, 1, 1], [S] * 3, [0, 1, 2])
        r = rows([1, 1, 1], [S] * 3, S, [0, bad, 2], DEV)
        y = selective.selective_tokens(t["x"], t["dt"], torch.log(-t["a"]), t["b"], t["c"], t["d"], t["z"], r, state)
        with pytest.raises(L.KernelError, match="bad argument"):
            L.check_status()
        assert not y[1].any() and y[0].any() and torch.equal(state[3:], before[3:])
    # a step of so many rows that a block has several, and one that is cut into chunks
    t, _, _ = call(1600, 1, 16, 16, BF16, 1, [1] * 1600, [1] * 1600, None)
    state, ids = torch.randn(1600, 16, 16, device=DEV), list(range(1600))
    ids[801] = 1600
    r = rows([1] * 1600, [1] * 1600, 1, ids, DEV)
    y = selective.selective_tokens(t["x"], t["dt"], torch.log(-t["a"]), t["b"], t["c"], t["d"], t["z"], r, state)
    with pytest.raises(L.KernelError, match="bad argument"):
        L.check_status()
    assert not y[801].any() and y[800].any() and y[802].any()
    t, r, state = heads(2, 40, 2, 1, 64, 128, BF16, 1, [1, 1], [40, 40], [0, 1])
    r.row_ids[1] = 7
    before = state.clone()
    y = selective.ssd_tokens(t["x"], t["dt"], t["dt_bias"], t["a_log"], t["b"], t["c"], t["d"], 2, 1, r, state)
    with pytest.raises(L.KernelError, match="bad argument"):
        L.check_status()
    assert not y[1].any() and y[0].any() and torch.equal(state[1:], before[1:])
