"""The selective scan's kernels where a call is unusual: captured, on another stream, with types that differ, differentiated twice, past 32 bits, with what is no number in places that do not
count."""
import pytest
import torch

from dew_b200 import ops
from dew_b200.ops import library as L
from dew_b200.ops import scan, selective
from selective_cases import NAMES, check, companion, draws_of_its_own, inputs, rows  # noqa: F401
from selective_cases import scan as oracle
from selective_cases import softplus

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def most(t):
    return float(softplus(t["dt"].double()).amax() * t["a"].abs().amax())


def captured(step):
    """``step`` on a side stream once, then recorded."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    return graph


def gradients(t, dy, dlast):
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out = scan.selective_scan(*leaves.values(), softplus=True)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [v for v in leaves.values() if v is not None], (dy, dlast)))


@pytest.mark.parametrize("B,T,C,dtype", [(2, 200, 96, BF16), (1, 40, 33, FP32)])
def test_a_captured_training_step(B, T, C, dtype):
    """Replayed on other inputs, the same bits as eagerly; twice the same bits."""
    t = inputs(B, T, C, 16, dtype, DEV, 1, initial=True)
    dy, dlast = torch.randn(B, T, C, device=DEV).to(dtype), torch.randn(B, C, 16, device=DEV)
    held = gradients(t, dy, dlast)
    out = [torch.empty_like(v) for v in held]

    def step():
        for o, v in zip(out, gradients(t, dy, dlast)):
            o.copy_(v)
    graph = captured(step)
    for seed in (2, 3):
        for v, w in zip(t.values(), inputs(B, T, C, 16, dtype, DEV, seed, initial=True).values()):
            v.copy_(w)
        graph.replay()
        want = gradients(t, dy, dlast)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(want, gradients(t, dy, dlast)))
    L.check_status()


def heads_of(R, S, H, P, N, seed, dtype=BF16):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return dict(x=r(R, S, H * P).to(dtype), dt=(r(R, S, H) - 3).to(dtype), dt_bias=r(H), A_log=r(H), Bm=r(R, S, N).to(dtype), Cm=r(R, S, N).to(dtype), D=r(H), H=H, G=1)


def tokens_of(R, S, C, N, seed, dtype=BF16):
    t = inputs(R, S, C, N, dtype, DEV, seed)
    return dict(x=t["x"], dt=t["dt"], A_log=torch.log(-t["a"]), Bm=t["b"], Cm=t["c"], D=t["d"], z=t["z"])


KINDS = {"channels": (selective.selective_tokens, lambda R, S, seed, dtype=BF16: tokens_of(R, S, 72, 16, seed, dtype), (72, 16)),
         "heads": (selective.ssd_tokens, lambda R, S, seed, dtype=BF16: heads_of(R, S, 3, 24, 40, seed, dtype), (3, 24, 40))}


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("S", [1, 150])
def test_a_captured_call_with_states(kind, S):
    """Positions, rows and states that change between replays."""
    fn, make, shape = KINDS[kind]
    call, state = make(3, S, 1), torch.randn(6, *shape, device=DEV)
    r = rows([4, 0, 9], [S, S, max(1, S - 7)], S, [5, 0, 2], DEV)
    start, out = state.clone(), torch.empty_like(call["x"])

    def step():
        state.copy_(start)
        out.copy_(fn(**call, rows=r, state=state))
    graph = captured(step)
    for first, lengths, ids in (([4, 0, 9], [S, S, max(1, S - 7)], [5, 0, 2]), ([0, -1, 3], [1, 0, S], [1, 2, 4])):
        now = rows(first, lengths, S, ids, DEV)
        for a, b in zip(r, now):
            a.copy_(b)
        start.normal_()
        graph.replay()
        again = start.clone()
        want = fn(**call, rows=now, state=again)
        assert torch.equal(out, want) and torch.equal(state, again)
    L.check_status()


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_two_graphs_and_a_side_stream(kind):
    """Calls that have scratch of their own do not see one another's."""
    fn, make, shape = KINDS[kind]
    calls, states = [make(2, 300, s) for s in (1, 2)], [torch.randn(2, *shape, device=DEV) for _ in range(2)]
    want = [fn(**c, state=s.clone()) for c, s in zip(calls, states)]
    outs = [torch.empty_like(w) for w in want]
    graphs = [captured(lambda c=c, s=s, o=o: o.copy_(fn(**c, state=s.clone()))) for c, s, o in zip(calls, states, outs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("S", [1, 40])
def test_what_is_no_number_where_nothing_counts(kind, dtype, S):
    """Padding, rows that rest, store rows that nobody has, states of rows that start."""
    fn, make, shape = KINDS[kind]
    call, state = make(4, S, 3, dtype), torch.randn(6, *shape, device=DEV)
    first, lengths, ids = [0, 5, -1, 7], [max(1, S - 3), S, 0, 1], [4, 0, 2, 3]
    want_state = state.clone()
    want = fn(**call, rows=rows(first, lengths, S, ids, DEV), state=want_state)
    spoilt = {k: v.clone() if torch.is_tensor(v) else v for k, v in call.items()}
    for name in ("x", "dt", "Bm", "Cm", "z"):
        if name in spoilt:
            for i, (f, n) in enumerate(zip(first, lengths)):
                spoilt[name][i, (n if f >= 0 else 0):] = float("nan") if i % 2 else float("inf")
    bad = state.clone()
    bad[[1, 2, 5]] = float("nan")                     # rows that rest or belong to nobody
    bad[4] = float("inf")                             # a row that starts
    got = fn(**spoilt, rows=rows(first, lengths, S, ids, DEV), state=bad)
    assert torch.equal(got, want) and torch.equal(bad[[0, 3, 4]], want_state[[0, 3, 4]])


def test_types_that_differ_and_what_broadcasts():
    t = inputs(2, 37, 24, 16, FP32, DEV, 5, initial=True)
    mixed = dict(t, x=t["x"].bfloat16(), b=t["b"].half(), z=t["z"].bfloat16(), d=t["d"].bfloat16())
    leaves = {n: v.detach().requires_grad_() for n, v in mixed.items()}
    out = scan.selective_scan(*leaves.values(), softplus=True)
    dy, dlast = torch.randn_like(out[0]), torch.randn_like(out[1])
    grads = torch.autograd.grad(out, list(leaves.values()), (dy, dlast))
    assert out[0].dtype is BF16 and all(g.dtype is v.dtype and g.shape == v.shape for g, v in zip(grads, leaves.values()))
    want, size = oracle(**mixed, steps=True, dy=dy, dlast=dlast), companion(**mixed, steps=True, dy=dy, dlast=dlast)
    got = dict(y=out[0], last=out[1], **{f"d{n}": g for n, g in zip(NAMES, grads)})
    got["db"], want["db"] = got["db"].float(), want["db"].half().double()        # (half: rounded to 11 bits, compared behind one more rounding)
    size["db"] = size["db"] + want["db"].abs() * 2.0 ** -10 / (2.0 ** -21)
    check(got, want, size, 37, 24, 16, most(mixed))
    # one step for all channels, one set of rates, one D, one state for all rows
    small = [t["x"], t["dt"][..., :1], t["a"][:1], t["b"][:1], t["c"], t["d"][:1], t["z"], t["initial"][:1]]
    leaves = [v.detach().clone().requires_grad_() for v in small]
    out = scan.selective_scan(*leaves, softplus=True)
    whole = dict(zip(NAMES, (t["x"], t["dt"][..., :1].expand(2, 37, 24), t["a"][:1].expand(24, 16), t["b"][:1].expand(2, 37, 16), t["c"], t["d"][:1].expand(24), t["z"],
                             t["initial"][:1].expand(2, 24, 16))))
    dy, dlast = dy.float(), dlast
    want, size = oracle(**whole, steps=True, dy=dy, dlast=dlast), companion(**whole, steps=True, dy=dy, dlast=dlast)
    grads = torch.autograd.grad(out, leaves, (dy, dlast))
    fit = lambda d: {k: d[k].sum_to_size(v.shape) if k in ("ddt", "da", "db", "dd", "dinitial") else d[k] for k, v in got.items()}
    got = dict(y=out[0], last=out[1], **{f"d{n}": g for n, g in zip(NAMES, grads)})
    check(got, fit(want), fit(size), 37, 24, 24 * 8, most(whole))                # (sums of 24 more terms)


def test_a_number_of_the_cpu_among_the_tensors():
    """A tensor of no dimensions broadcasts from wherever it lies, as in the plain operators; it has its gradient there."""
    t = inputs(2, 20, 16, 8, FP32, DEV, 6, initial=True)
    number = torch.tensor(0.75, requires_grad=True)
    y, _ = scan.selective_scan(t["x"], t["dt"], t["a"], t["b"], t["c"], number, t["z"], softplus=True)
    same = number.detach().to(DEV).expand(16).contiguous().requires_grad_()
    want, _ = scan.selective_scan(t["x"], t["dt"], t["a"], t["b"], t["c"], same, t["z"], softplus=True)
    y.sum().backward(), want.sum().backward()
    assert torch.equal(y, want) and number.grad.device == number.device
    assert torch.allclose(number.grad, same.grad.sum().cpu(), rtol=16 * 2.0 ** -24, atol=16 * 2.0 ** -24 * float(same.grad.abs().sum()))
    bare = scan.selective_scan(t["x"], torch.tensor(0.5), t["a"], t["b"], t["c"])[0]
    assert torch.equal(bare, scan.selective_scan(t["x"], torch.full_like(t["dt"], 0.5), t["a"], t["b"], t["c"])[0])


def test_layouts():
    """Columns of wider rows, tokens in front of rows, a batch of one at any stride: the same bits."""
    t = inputs(3, 50, 36, 16, BF16, DEV, 7)
    want = scan.selective_scan(*t.values(), softplus=True)
    turned = {n: v.transpose(0, 1).contiguous().transpose(0, 1) if n in ("x", "dt", "b", "c", "z") else v for n, v in t.items()}
    wide = {n: torch.cat([v, v], -1)[..., v.shape[-1]:] if n in ("x", "dt", "b", "c", "z") else v for n, v in t.items()}
    apart = {n: v.transpose(1, 2).contiguous().transpose(1, 2) if n in ("x", "dt", "b", "c", "z") else v for n, v in t.items()}
    for other in (turned, wide, apart):
        got = scan.selective_scan(*other.values(), softplus=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_gradient_that_is_differentiated_again_and_a_tangent():
    t = inputs(1, 12, 8, 4, FP32, DEV, 9, initial=True)

    def second(fn, t):
        leaves = [v.detach().clone().requires_grad_() for v in t.values()]
        y, last = fn(*leaves, softplus=True)
        first = torch.autograd.grad((y.square().sum() + last.sum(),), leaves, create_graph=True)
        return torch.autograd.grad(sum(g.square().sum() for g in first), leaves)
    for a, b in zip(second(scan.selective_scan, t), second(scan.selective_scan_chunked, {n: v.cpu() for n, v in t.items()})):
        assert torch.allclose(a.cpu(), b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))
    rest = list(t.values())[1:]
    _, got = torch.func.jvp(lambda x: scan.selective_scan(x, *rest, softplus=True)[0], (t["x"],), (torch.ones_like(t["x"]),))
    want = scan.selective_scan(torch.ones_like(t["x"]), *rest[:-1], torch.zeros_like(t["initial"]), softplus=True)[0]         # (the scan is linear in x)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)


def test_empty_calls():
    t = inputs(2, 5, 8, 4, FP32, DEV, 1, initial=True)
    y, last = scan.selective_scan(t["x"][:, :0], t["dt"][:, :0], t["a"], t["b"][:, :0], t["c"][:, :0], t["d"], t["z"][:, :0], t["initial"])
    assert y.shape == (2, 0, 8) and torch.equal(last, t["initial"])
    fn, make, shape = KINDS["heads"]
    call = make(2, 3, 1)
    assert fn(**{k: v[:0] if torch.is_tensor(v) and v.dim() == 3 else v for k, v in call.items()}).shape == (0, 3, 72)


def test_elements_past_32_bits():
    """More than 2^31 tokens times channels, forward and backward, against the last tokens alone: with steps of about 0.7 and rates of 1 and more, what is 128 tokens away counts for
    less than e^-80."""
    T, C, tail = 524_800, 4096, 256
    g = torch.Generator(DEV).manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=BF16)
    x, z, dy = (make(1, T, C) for _ in range(3))
    dt = torch.zeros(1, T, 1, device=DEV, dtype=BF16).expand(1, T, C).contiguous()
    b, c = make(1, T, 16), make(1, T, 16)
    a = -torch.arange(1, 17, device=DEV, dtype=FP32).repeat(C, 1)
    leaves = [v.requires_grad_() for v in (x, dt, z)]
    y, last = scan.selective_scan(x, dt, a, b, c, None, z, softplus=True)
    grads = torch.autograd.grad(y, leaves, dy)
    L.check_status()
    cut = lambda v: v.detach()[:, -tail:, -64:]
    small = dict(x=cut(x), dt=cut(dt), a=a[-64:], b=b[:, -tail:], c=c[:, -tail:], z=cut(z))
    want, size = oracle(**small, steps=True, dy=cut(dy)), companion(**small, steps=True, dy=cut(dy))
    got = dict(y=cut(y), last=last[:, -64:], **{f"d{n}": cut(v) for n, v in zip(("x", "dt", "z"), grads)})
    half = lambda d: {k: (d[k][:, tail // 2:] if k != "last" else d[k]) for k in got}
    check(half(got), half(want), half(size), tail, 64, 16, 16 * 0.7)


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("S", [1, 20])
def test_stores_past_32_bits(kind, S):
    fn, make, shape = KINDS[kind]
    each = torch.Size(shape).numel()
    far = (1 << 31) // each + 5
    state = torch.empty(far + 1, *shape, device=DEV)
    call = make(2, S, 4)
    state[far], state[3] = torch.randn(shape, device=DEV), torch.randn(shape, device=DEV)
    near = torch.stack([state[far], state[3]])
    want = fn(**call, rows=rows([2, 5], [S, S], S, None, DEV), state=near)
    got = fn(**call, rows=rows([2, 5], [S, S], S, [far, 3], DEV), state=state)
    L.check_status()
    assert torch.equal(got, want) and torch.equal(state[far], near[0]) and torch.equal(state[3], near[1])


def test_a_layer_of_states_in_sequence():
    """The operators together, as a layer of Mamba-2 calls them: a prompt in two pieces and two steps, against the layer over the whole row."""
    from dew_b200.nn.kv_cache import CacheSlot, KVCache, KVStore
    from dew_b200.nn.layers import reset_all
    from dew_b200.nn.mamba2 import Mamba2
    layer = Mamba2(128, state_dim=32, head_dim=32, groups=2).to(DEV).eval()
    reset_all(layer, 0)
    x = torch.randn(2, 70, 128, device=DEV)
    store = KVStore(KVCache(page_size=64), 1, 3, 128, 0, 0, FP32, DEV, slots=[layer.cache_slot()])
    assert isinstance(layer.cache_slot(), CacheSlot)
    at = torch.arange(70, device=DEV)[None].expand(2, -1)
    with torch.no_grad():
        want = layer(x)
        store.select(torch.tensor([2, 0], device=DEV))
        got = torch.cat([layer(x[:, lo:hi], cache=store, positions=at[:, lo:hi].contiguous()) for lo, hi in ((0, 40), (40, 68), (68, 69), (69, 70))], 1)
    assert torch.allclose(got, want, atol=2e-4 * float(want.abs().max()))


def test_norm_behind_a_gate_takes_rows_of_a_projection():
    wide = torch.randn(4, 6, 300, device=DEV).bfloat16()
    z, y, w = wide[..., :128], torch.randn(4, 6, 128, device=DEV).bfloat16(), torch.rand(128, device=DEV).bfloat16()
    assert torch.equal(ops.gated_rms_norm(y, z, w, gate_first=True), ops.gated_rms_norm(y, z.contiguous(), w, gate_first=True))
