"""Which calls of the selective scans the kernels take, and that the others find their plain form: shapes that broadcast, empty ones, other types, autograd's view of a state."""
import pytest
import torch

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
    for a, b in zip((*got, *grads), (*want, *torch.autograd.grad(want[0].square().sum() + want[1].sum(), plain))):
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
