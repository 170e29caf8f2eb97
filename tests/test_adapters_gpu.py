"""The adapters' kernels against the formula in 64 bits."""
import pytest
import torch

from adapters_cases import allowed, batch, truth
from dew_b200.ops import library as L
from dew_b200.ops.adapters import Bank, adapted_linear, add_adapters

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def check(a, bias=None):
    L.check_status()
    found = truth(a, bias)
    got = adapted_linear(**a, bias=bias)
    L.check_status()
    over = float(((got.double().cpu().reshape(found[0].shape) - found[0]).abs() / allowed(a, found)).max())
    assert over <= 1.0, over
    return got


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens", [1, 2, 17, 64, 130, 300])
@pytest.mark.parametrize("n, rank, width, out", [(1, 1, 8, 8), (3, 8, 64, 40), (5, 5, 104, 72), (4, 16, 1024, 512), (7, 13, 200, 136), (2, 64, 520, 1000), (3, 100, 256, 264),
                                                 (70, 16, 256, 128), (2, 200, 136, 256)])
def test_shapes(dtype, tokens, n, rank, width, out):
    check(batch(tokens, n, rank, width, out, dtype, device=DEV, seed=tokens))


@pytest.mark.parametrize("dtype, width, out", [(FP32, 33, 17), (FP32, 1, 1), (BF16, 33, 17), (BF16, 12, 20), (BF16, 264, 9)])
@pytest.mark.parametrize("tokens", [1, 50, 270])
def test_odd_widths(dtype, width, out, tokens):
    check(batch(tokens, 6, 5, width, out, dtype, device=DEV))


@pytest.mark.parametrize("tokens, used, runs", [(1024, 3, True), (1500, 12, True), (1500, 12, False), (4096, 1, True), (2000, 64, False)])
@pytest.mark.parametrize("without", [0.0, 0.3, 1.0])
def test_prompts(tokens, used, runs, without):
    check(batch(tokens, 64, 32, 512, 768, BF16, device=DEV, used=used, runs=runs, without=without))


@pytest.mark.parametrize("n, rank, width, out", [(3, 8, 72, 136), (5, 5, 200, 1000), (2, 13, 520, 72), (40, 72, 136, 264), (2, 200, 264, 392), (4, 16, 33, 17), (3, 24, 64, 130), (600, 4, 128, 128)])
@pytest.mark.parametrize("tokens, runs", [(513, True), (900, False)])
def test_prompts_of_odd_sizes(n, rank, width, out, tokens, runs):
    check(batch(tokens, n, rank, width, out, BF16, device=DEV, runs=runs))


def test_prompts_of_one_token_each_and_of_one_adapter():
    a = batch(700, 700, 8, 64, 128, BF16, device=DEV, without=0.0)
    a["ids"] = torch.randperm(700, device=DEV, dtype=torch.int32)
    for t in a["bank"]:
        t.copy_(torch.randn_like(t) * 0.3)
    check(a)
    check({**a, "ids": torch.full_like(a["ids"], 5)})
    check({**a, "ids": torch.where(torch.arange(700, device=DEV) == 650, 3, -1).to(torch.int32)})


def test_layouts_bias_and_streams():
    a = batch(96, 5, 16, 256, 384, BF16, device=DEV)
    bias = torch.randn(384, device=DEV).to(BF16)
    want = check(a, bias)
    wide = torch.randn(96, 512, device=DEV).to(BF16)
    wide[:, 128:384] = a["x"]
    assert torch.equal(check({**a, "x": wide[:, 128:384]}, bias), want)
    odd = torch.randn(96, 259, device=DEV).to(BF16)                      # rows that do not begin at 16 bytes
    odd[:, 3:] = a["x"]
    check({**a, "x": odd[:, 3:]}, bias)
    assert torch.equal(adapted_linear(a["x"].view(4, 24, 256), a["weight"], a["bank"], a["ids"].view(4, 24), bias).view(96, 384), want)
    every_other = torch.stack([a["ids"], a["ids"]], 1)[:, 0]
    assert torch.equal(adapted_linear(a["x"], a["weight"], a["bank"], every_other, bias), want)
    raw = torch.empty(5 * 16 * 256 + 1, device=DEV, dtype=BF16)          # adapters that do not begin at 16 bytes
    raw[1:] = a["bank"].a.reshape(-1)
    check({**a, "bank": a["bank"]._replace(a=raw[1:].view(5, 16, 256))}, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = adapted_linear(**a, bias=bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


@pytest.mark.parametrize("tokens", [1, 64, 600])
def test_captured_calls_follow_ids_and_adapters(tokens):
    a = batch(tokens, 5, 16, 256, 384, BF16, device=DEV, without=0.0)
    ids = a["ids"].clone()
    live = {**a, "ids": torch.full_like(ids, -1), "bank": Bank(*(t.clone() for t in a["bank"]))}
    adapted_linear(**live)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(adapted_linear(**live))
    live["ids"].copy_(ids)
    live["bank"].scale.mul_(2.0)
    for g in graphs + graphs:
        g.replay()
    found = truth(live)
    for o in outs:
        assert bool(((o.double().cpu() - found[0]).abs() <= allowed(live, found)).all())
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("tokens", [3, 700])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_ids_past_the_last_adapter_are_reported_and_add_nothing(tokens, dtype):
    a = batch(tokens, 5, 16, 256, 384, dtype, device=DEV)
    base = adapted_linear(a["x"], a["weight"], a["bank"], torch.full_like(a["ids"], -7))
    for past in (5, 1 << 30):
        y = base.clone()
        add_adapters(y, a["x"], a["bank"], torch.full_like(a["ids"], past))
        with pytest.raises(L.KernelError):
            L.check_status()
        assert torch.equal(y, base)
    check(a)


def test_the_same_bits_again():
    a = batch(200, 9, 24, 1024, 640, BF16, device=DEV)
    want = check(a)
    assert all(torch.equal(adapted_linear(**a), want) for _ in range(5))


@pytest.mark.parametrize("tokens", [60, 900])
@pytest.mark.parametrize("n, rank", [(3500, 8), (3501, 8), (4, 512), (3, 513)])
def test_the_largest_banks_and_ranks(n, rank, tokens):
    check(batch(tokens, n, rank, 64, 72, BF16, device=DEV, used=min(n, 200), seed=tokens))


@pytest.mark.parametrize("tokens", [40, 600])
def test_rows_that_overlap_or_are_one(tokens):
    a = batch(tokens, 3, 8, 64, 40, BF16, device=DEV)
    one = a["x"][:1]
    want = adapted_linear(**{**a, "x": one.expand(tokens, -1).contiguous()})
    assert torch.equal(adapted_linear(**{**a, "x": one.expand(tokens, -1)}), want)
    flat = a["x"].flatten()[:tokens * 8 + 64]
    windows = flat.as_strided((tokens, 64), (8, 1))
    assert torch.equal(adapted_linear(**{**a, "x": windows}), adapted_linear(**{**a, "x": windows.contiguous()}))


@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("tokens, n, rank, width, out", [(8000, 12, 64, 1024, 2048), (500, 48, 32, 2048, 1536), (2000, 5, 24, 512, 1000)])
def test_the_same_bits_from_memory(tokens, n, rank, width, out, runs):
    """Operands that come late (nothing of them is in the cache), on all SMs."""
    a = batch(tokens, n, rank, width, out, BF16, device=DEV, runs=runs)
    want, flush = check(a), torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    for i in range(20):
        if i % 3:
            flush.zero_()
        assert torch.equal(adapted_linear(**a), want), i
    L.check_status()


@pytest.mark.parametrize("runs", [False, True])
def test_layouts_of_prompts(runs):
    a = batch(640, 5, 16, 256, 384, BF16, device=DEV, runs=runs)
    want = check(a)
    wide = torch.randn(640, 512, device=DEV).to(BF16)
    wide[:, 128:384] = a["x"]
    assert torch.equal(check({**a, "x": wide[:, 128:384]}), want)
    odd = torch.randn(640, 259, device=DEV).to(BF16)                     # rows that do not begin at 16 bytes
    odd[:, 3:] = a["x"]
    check({**a, "x": odd[:, 3:]})
    for name, shape in (("a", (5, 16, 256)), ("b", (5, 384, 16))):       # adapters that do not begin at 16 bytes
        raw = torch.empty(a["bank"].a.numel() * 2 + 1, device=DEV, dtype=BF16)
        part = getattr(a["bank"], name)
        raw[1:1 + part.numel()] = part.reshape(-1)
        check({**a, "bank": a["bank"]._replace(**{name: raw[1:1 + part.numel()].view(shape)})})
    y = torch.empty(640 * 384 + 1, device=DEV, dtype=BF16)[1:].view(640, 384)
    base = adapted_linear(a["x"], a["weight"], a["bank"], torch.full_like(a["ids"], -1))
    assert torch.equal(add_adapters(y.copy_(base), a["x"], a["bank"], a["ids"]), add_adapters(base.clone(), a["x"], a["bank"], a["ids"]))
    assert torch.equal(adapted_linear(a["x"].view(4, 160, 256), a["weight"], a["bank"], a["ids"].view(4, 160)).view(640, 384), want)
