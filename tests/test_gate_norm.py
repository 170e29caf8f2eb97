"""The norm behind a gate against its formula in 64 bits, and its gradients against the formula's and against differences."""
import pytest
import torch

from dew_b200 import ops
from dew_b200.ops import gate_norm as K
from dew_b200.ops import library as L
from selective_cases import draws_of_its_own  # noqa: F401

EPS = 1e-5


def formula(x, z, w, dy):
    x, z, w, dy = (t.detach().double() for t in (x, z, w, dy))
    sig = torch.sigmoid(z)
    u = x * z * sig
    r = 1 / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + EPS)
    du = dy * w * r - u * r ** 3 * (dy * w * u).mean(-1, keepdim=True)
    big = (dy * w).abs() * r + u.abs() * r ** 3 * (dy * w * u).abs().mean(-1, keepdim=True)          # what the two terms of du are off by shares of
    lead = tuple(range(x.dim() - 1))
    want = dict(y=u * r * w, x=du * z * sig, z=du * x * sig * (1 + z * (1 - sig)), w=(dy * u * r).sum(lead))
    size = dict(y=want["y"].abs(), x=big * z.abs(), z=big * x.abs() * (1.1 + z.abs()), w=(dy * u * r).abs().sum(lead))
    return want, size


def check(got, want, size, d, rows):
    # 32 bits: the sigmoid and the gate 2^-21, a sum of d squares d / 2 roundings at worst and its root half of that, the sum over rows one a row; then half a step of bf16
    for n, t in got.items():
        bound = (d / 4 + 32 + (rows if n == "w" else 0)) * 2.0 ** -22 * size[n] + (2.0 ** -8 * 1.01 * want[n].abs() if t.dtype is torch.bfloat16 else 0) + 1e-30
        off = (t.detach().double() - want[n]).abs()
        assert t.shape == want[n].shape and bool((off <= bound).all()), (n, float((off / bound).max()))


def case(shape, dtype, device, seed=0, w_type=None, strided=False):
    g = torch.Generator(device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)
    z = r(*shape[:-1], 2 * shape[-1])[..., shape[-1]:] if strided else r(*shape)
    return r(*shape).to(dtype), z.to(dtype), (1 + 0.1 * r(shape[-1])).to(w_type or dtype), r(*shape).to(dtype)


def run(x, z, w, dy):
    with torch.no_grad():
        alone = ops.gated_rms_norm(x, z, w, EPS, gate_first=True)
    leaves = [t.detach().requires_grad_() for t in (x, z, w)]
    y = ops.gated_rms_norm(*leaves, EPS, gate_first=True)
    assert torch.equal(alone, y)
    return dict(zip(("y", "x", "z", "w"), (y, *torch.autograd.grad(y, leaves, dy))))


@pytest.mark.parametrize("shape", [(3, 8), (2, 5, 40), (1, 1), (7, 33)])
def test_plain_form(shape):
    x, z, w, dy = case(shape, torch.float32, "cpu")
    check(run(x, z, w, dy), *formula(x, z, w, dy), shape[-1], x.numel() // shape[-1])
    ins = [t.double().requires_grad_() for t in (x, z, w)]
    assert torch.autograd.gradcheck(lambda *t: ops.gated_rms_norm(*t, EPS, gate_first=True), ins)


# a warp's rows, a block's, rows that are read twice, odd ones; one row and more than there are blocks
@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype,w_type,strided", [((1, 8), torch.bfloat16, None, False), ((5, 7, 256), torch.bfloat16, torch.float32, True), ((700, 512), torch.bfloat16, None, True),
                                                       ((9, 1000), torch.bfloat16, torch.float32, False), ((3, 2048), torch.bfloat16, None, True), ((1201, 4096), torch.bfloat16, None, False),
                                                       ((20, 8192), torch.bfloat16, None, True), ((11, 16392), torch.bfloat16, None, False), ((13, 333), torch.bfloat16, None, True),
                                                       ((4, 100), torch.float32, None, False), ((30, 1024), torch.float32, None, True), ((600, 4096), torch.float32, None, True),
                                                       ((3, 5000), torch.float32, None, False), ((17, 31), torch.float32, None, True)])
def test_kernels(shape, dtype, w_type, strided):
    x, z, w, dy = case(shape, dtype, "cuda", sum(shape), w_type, strided)
    assert K.kernel_available(x, z, w)
    check(run(x, z, w, dy), *formula(x, z, w, dy), shape[-1], x.numel() // shape[-1])


@pytest.mark.gpu
def test_what_the_kernels_leave_to_the_plain_form():
    x, z, w, dy = case((4, 64), torch.float32, "cuda")
    leaves = [t.requires_grad_() for t in (x, z, w)]
    first = torch.autograd.grad(ops.gated_rms_norm(*leaves, EPS, gate_first=True), leaves, dy, create_graph=True)
    again = torch.autograd.grad(sum(g.sum() for g in first), leaves)
    ins = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(sum(g.sum() for g in torch.autograd.grad(K.plain(*ins, EPS), ins, dy.double(), create_graph=True)), ins)
    for a, b in zip(again, want):
        assert torch.allclose(a.double(), b, rtol=1e-4, atol=1e-4)
    assert not K.kernel_available(x.half(), z.half(), w.half())
    assert ops.gated_rms_norm(x[:0], z[:0], w, EPS, gate_first=True).shape == (0, 64)


@pytest.mark.gpu
def test_backward_in_a_graph():
    x, z, w, dy = case((40, 256), torch.bfloat16, "cuda")
    out = [torch.empty_like(t) for t in (x, z, w)]

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, z, w)]
        for o, g in zip(out, torch.autograd.grad(ops.gated_rms_norm(*leaves, EPS, gate_first=True), leaves, dy)):
            o.copy_(g)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x.copy_(torch.randn_like(x))
    graph.replay()
    got = [t.clone() for t in out]
    step()
    assert all(torch.equal(a, b) for a, b in zip(got, out))
    L.check_status()
