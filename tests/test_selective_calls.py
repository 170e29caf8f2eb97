"""Which calls of the selective scans the kernels take, and that the others find their plain form: shapes that broadcast, empty ones, other types, autograd's view of a state."""
import pytest
import torch

from dew_b200.ops import library as L
from dew_b200.ops import scan, selective
from selective_cases import draws_of_its_own, inputs, rows  # noqa: F401


def call(device="cpu", B=2, T=9, C=8, N=4):
    t = inputs(B, T, C, N, torch.float32, device, 1, initial=True)
    return [t[n] for n in ("x", "dt", "a", "b", "c", "d", "z", "initial")]


# what broadcasts in the plain form, by its place among the arguments
SHAPES = [(5, lambda d: d[None, None]), (5, lambda d: d[None]), (5, lambda d: d.expand(9, 8).contiguous()), (5, lambda d: d.expand(2, 1, 8).contiguous()), (5, lambda d: d[0]),
          (6, lambda z: z[0, 0]), (6, lambda z: z[:1]), (6, lambda z: z[..., :1]), (1, lambda dt: dt[..., :1]), (2, lambda a: a[:1]), (3, lambda b: b[:1])]


@pytest.mark.parametrize("at,change", SHAPES)
def test_which_shapes_the_kernels_take(at, change):
    """All that expand to their size; a D of one row is a D."""
    args = call()
    args[at] = change(args[at])
    fits = selective.fits(*args)
    assert fits == (at != 5 or args[5].dim() < 2)
    assert selective.fits(*args[:5], None, None, None) or at in (5, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("at,change", SHAPES)
def test_what_broadcasts(at, change):
    args = call("cuda")
    args[at] = change(args[at])
    leaves = [t.detach().clone().requires_grad_() for t in args]
    got = scan.selective_scan(*leaves, softplus=True)
    plain = [t.detach().cpu().clone().requires_grad_() for t in args]
    want = scan.selective_scan_chunked(*plain, softplus=True)
    grads = torch.autograd.grad(got[0].square().sum() + got[1].sum(), leaves)
    for a, b in zip((*(t.detach() for t in got), *grads), (*(t.detach() for t in want), *torch.autograd.grad(want[0].square().sum() + want[1].sum(), plain))):
        assert a.shape == b.shape and torch.allclose(a.cpu(), b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


def empty_calls_have_gradients(device):
    for B, T, C in ((0, 5, 4), (2, 0, 4), (2, 5, 0), (0, 0, 0)):
        leaves = [t.requires_grad_() for t in call(device, B, T, C, 3)]
        y, last = scan.selective_scan(*leaves)
        assert y.shape == (B, T, C) and last.shape == (B, C, 3) and torch.equal(last, leaves[7]) == (T == 0 or 0 in (B, C))
        if T > 0:
            assert all(g is not None and not g.any() for g in torch.autograd.grad(y.sum() + last.sum(), leaves))
        else:
            dx, dlast = torch.autograd.grad(y.sum() + 2 * last.sum(), [leaves[0], leaves[7]])
            assert dx.shape == (B, T, C) and bool((dlast == 2).all())


def test_empty_calls_have_gradients():
    empty_calls_have_gradients("cpu")


@pytest.mark.gpu
def test_empty_calls_have_gradients_on_a_gpu():
    empty_calls_have_gradients("cuda")


FNS = {"channels": (selective.selective_tokens, lambda t: dict(x=t["x"], dt=t["dt"], A_log=torch.log(-t["a"]), Bm=t["b"], Cm=t["c"], D=t["d"], z=t["z"]), (8, 4)),
       "heads": (selective.ssd_tokens, lambda t: dict(x=t["x"], dt=t["dt"][..., :2], dt_bias=t["d"][:2], A_log=t["d"][2:4], Bm=t["b"], Cm=t["c"], D=t["d"][4:6], H=2, G=2), (2, 4, 2))}


def other_types(kind, dtype, device):
    """fp16 and fp64 in one type take the plain form, as the other recurrences leave them to theirs; the state stays fp32."""
    fn, make, shape = FNS[kind]
    t = inputs(3, 6, 8, 4, torch.float32, device, 2)
    one = make(t)
    cast = {k: v.to(dtype) if torch.is_tensor(v) and k not in ("A_log", "D", "dt_bias") else v for k, v in one.items()}
    wide = {k: v.float() if torch.is_tensor(v) else v for k, v in cast.items()}
    at = rows([0, 5, -1], [6, 4, 0], 6, [2, 0, 1], device)
    state = torch.randn(4, *shape, device=device)
    want_state = state.clone()
    y, want = fn(**cast, rows=at, state=state), fn(**wide, rows=at, state=want_state)
    assert y.dtype is dtype and torch.allclose(state, want_state, atol=1e-5)
    # (half a step of fp16, where the results are rounded to it)
    assert torch.allclose(y.float(), want, rtol=1e-5 + (2.0 ** -11 if dtype is torch.float16 else 0), atol=1e-5)
    with pytest.raises(TypeError):
        fn(**dict(cast, Bm=cast["Bm"].float()), rows=at, state=state)
    with pytest.raises(TypeError):
        fn(**dict(cast, dt=cast["dt"].bfloat16()), rows=at, state=state)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_other_types(kind, dtype):
    other_types(kind, dtype, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_other_types_on_a_gpu(kind, dtype):
    other_types(kind, dtype, "cuda")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("kind", ["mamba", "mamba2"])
def test_models_of_other_types_generate(kind, dtype):
    from dew_b200.sampling.text import Sampling, generate
    from test_state_space_models import model, prompts
    m, asked = model(kind).to(dtype), prompts(2)
    out = generate(m, None, asked, 4, sampling=Sampling(temperature=0.0))
    for r, p in enumerate(asked):
        row = out.tokens[r, :len(p) + 4]
        with torch.no_grad():
            logits = m(row[None])[0, len(p) - 1:-1].float()
        # (near to the whole row's best: in fp16 two tokens may come as near as its roundings)
        taken = logits.gather(1, row[len(p):, None])[:, 0]
        assert bool((logits.amax(1) - taken <= (2.0 ** -5 if dtype is torch.float16 else 1e-4)).all())


@pytest.mark.parametrize("bad", [-1, 4, 1 << 30])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_rows_outside_the_store_in_the_plain_form(kind, bad):
    """Nothing is read or written there: an error on the CPU, but for a row that rests."""
    fn, make, shape = FNS[kind]
    t = inputs(3, 6, 8, 4, torch.float32, "cpu", 2)
    state = torch.randn(4, *shape)
    before = state.clone()
    with pytest.raises(IndexError, match="store"):
        fn(**make(t), rows=rows([2, 5, 1], [6, 4, 6], 6, [2, bad, 1], "cpu"), state=state)
    assert torch.equal(state, before)
    y = fn(**make(t), rows=rows([2, -1, 1], [6, 0, 6], 6, [2, bad, 1], "cpu"), state=state)
    assert not y[1].any() and y[0].any() and torch.equal(state[[0, 3]], before[[0, 3]])


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["gradients", "fp16"])
@pytest.mark.parametrize("bad", [-1, 4, 1 << 30])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_rows_outside_the_store_in_the_plain_form_on_a_gpu(kind, bad, how):
    """Calls that the kernels leave to the plain form: such a row is reported and gives zeros there as well."""
    fn, make, shape = FNS[kind]
    one = make(inputs(3, 6, 8, 4, torch.float32, "cuda", 2))
    if how == "fp16":
        one = {k: v.half() if torch.is_tensor(v) and k not in ("A_log", "D", "dt_bias") else v for k, v in one.items()}
    else:
        one["D"].requires_grad_()
    state = torch.randn(4, *shape, device="cuda")
    before = state.clone()
    y = fn(**one, rows=rows([2, 5, 1], [6, 4, 6], 6, [2, bad, 1], "cuda"), state=state)
    with pytest.raises(L.KernelError, match="bad argument"):
        L.check_status()
    assert not y[1].any() and y[0].any() and torch.equal(state[[0, 3]], before[[0, 3]]) and not torch.equal(state[2], before[2])
    L.check_status()


def state_that_autograd_holds(kind, S, device, dtype=torch.float32):
    """A state that a call moves on is another value to autograd."""
    fn, make, shape = FNS[kind]
    one = {k: v.to(dtype) if torch.is_tensor(v) and k not in ("A_log", "D", "dt_bias") else v for k, v in make(inputs(2, S, 8, 4, torch.float32, device, 3)).items()}
    state, w = torch.randn(2, *shape, device=device), torch.ones((), device=device, requires_grad=True)
    held, version = (w * state).sum(), state._version
    with torch.no_grad():
        fn(**one, rows=rows([1, 0], [S, S], S, None, device), state=state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()
    with torch.inference_mode():
        again = torch.zeros(2, *shape, device=device)
        fn(**one, rows=rows([1, 0], [S, S], S, None, device), state=again)
        fn(**one)
    version = state._version
    with torch.no_grad():
        fn(**one)                                            # (no state: nothing moves)
    assert state._version == version


@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_autograd_sees_that_a_state_moved_on(kind, S):
    state_that_autograd_holds(kind, S, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("kind", sorted(FNS))
def test_autograd_sees_that_a_state_moved_on_on_a_gpu(kind, S):
    state_that_autograd_holds(kind, S, "cuda")


@pytest.mark.gpu
def test_autograd_sees_that_a_state_of_chunks_moved_on():
    r = lambda *s: torch.randn(*s, device="cuda")
    state = r(2, 2, 64, 128)
    version = state._version
    with torch.no_grad():
        selective.ssd_tokens(r(2, 40, 128).bfloat16(), r(2, 40, 2).bfloat16(), None, r(2), r(2, 40, 128).bfloat16(), r(2, 40, 128).bfloat16(), None, 2, 1, rows([0, 3], [40, 7], 40, None, "cuda"), state)
    assert state._version > version


# leaves that one of the two results does not depend on, alone and together
LEAVES = [("c",), ("d",), ("z",), ("c", "d", "z"), ("initial",), ("c", "x")]


@pytest.mark.parametrize("which", ["y", "last", "both"])
@pytest.mark.parametrize("names", LEAVES)
def test_gradients_to_be_differentiated_of_some_leaves(names, which):
    """What the node gives where its gradients keep a history, from the plain form."""
    all_names = ("x", "dt", "a", "b", "c", "d", "z", "initial")
    ins = [t.requires_grad_(n in names) for n, t in zip(all_names, call())]
    y, last = scan.selective_scan_chunked(*ins, softplus=True)
    dy, dlast = torch.randn_like(y) if which != "last" else None, torch.randn_like(last) if which != "y" else None
    got = selective._plain_gradients(ins, True, dy, dlast, [n in names for n in all_names])
    for n, t, g in zip(all_names, ins, got):
        if n not in names:
            assert g is None
            continue
        sees = [(o, d) for o, d in ((y, dy), (last, dlast)) if d is not None and o.requires_grad]
        want = torch.autograd.grad([o for o, _ in sees], t, [d for _, d in sees], retain_graph=True, allow_unused=True)[0] if sees else None
        # (with a history a gate's slope is formed of other products: sig (1 + z (1 - sig)), some six roundings either way, of terms up to 2 |dz|'s factors)
        assert (want is None and g is None) or torch.allclose(g, want, rtol=2.0 ** -20, atol=2.0 ** -20 * float(want.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("names", LEAVES)
def test_gradients_to_be_differentiated_of_some_leaves_on_a_gpu(names):
    """Through the kernels' node: with a history and without one."""
    all_names = ("x", "dt", "a", "b", "c", "d", "z", "initial")
    ins = [t.requires_grad_(n in names) for n, t in zip(all_names, call("cuda"))]
    y, last = scan.selective_scan(*ins, softplus=True)
    leaves, loss = [t for t in ins if t.requires_grad], y.square().sum() + last.square().sum()
    kept = torch.autograd.grad(loss, leaves, create_graph=True)
    for a, b in zip(kept, torch.autograd.grad(loss, leaves, retain_graph=True)):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))
    assert all(g.isfinite().all() for g in torch.autograd.grad(sum(g.square().sum() for g in kept), leaves))
