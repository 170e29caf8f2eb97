"""The kernels of a decode step over shared prefixes against the formula in 64 bits."""
import pytest
import torch

from dew_b200.ops import library as L
from dew_b200.ops.prefix import Shared, shared_decode
from prefix_cases import allowed, batch, truth

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def check(a, window=None, softcap=0.0, sinks=None):
    L.check_status()
    found = truth(a, window, softcap, sinks)
    got = shared_decode(**a, window=window, softcap=softcap, sinks=sinks)
    L.check_status()
    over = ((got.double().cpu() - found[0]).abs() / allowed(a, found)).max()
    assert float(over) <= 1.0 and not got[a["lengths"] == 0].any(), float(over)
    return got


# (shared tokens, own tokens of each row)
SHAPES = {
    "one row": [(0, [1])],
    "one long row": [(0, [700])],
    "two rows": [(64, [1, 2])],
    "a key each": [(0, [1] * 5)],
    "several": [(130, [1, 64, 65, 200]), (0, [33]), (16, [2, 2, 2]), (512, [1, 1])],
    "wide": [(257, [1 + i % 7 for i in range(40)]), (300, [5] * 9)],
    "long": [(2100, [3, 100, 900])],
}


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("heads, kv, dim, page, dtype, pool", [
    (8, 2, 128, 64, BF16, None), (8, 8, 64, 16, BF16, None), (6, 2, 128, 48, BF16, None), (5, 1, 64, 128, BF16, None), (32, 2, 128, 16, BF16, None), (40, 2, 64, 32, BF16, None),
    (4, 2, 80, 16, BF16, None), (6, 3, 40, 16, FP32, None), (4, 4, 256, 16, FP32, None), (2, 1, 256, 64, BF16, None), (4, 2, 128, 64, BF16, torch.int8),
    (4, 2, 64, 16, BF16, torch.float8_e4m3fn), (3, 3, 33, 5, FP32, torch.int8), (36, 2, 16, 7, FP32, None)])
def test_shapes(name, heads, kv, dim, page, dtype, pool):
    check(batch(SHAPES[name], heads, kv, dim, page, dtype, pool, device=DEV))


@pytest.mark.parametrize("heads, kv, dim, page, dtype", [(8, 2, 128, 64, BF16), (5, 1, 64, 16, BF16), (6, 2, 80, 16, FP32)])
@pytest.mark.parametrize("window, softcap, sinks", [(1, 0.0, False), (30, 0.0, True), (100, 0.0, False), (150, 7.0, False), (5000, 0.0, False), (None, 30.0, True), (None, 0.0, True)])
@pytest.mark.parametrize("resting", [(), (0,), (1, 2, 4), tuple(range(10))])
def test_variants_and_resting_rows(heads, kv, dim, page, dtype, window, softcap, sinks, resting):
    a = batch([(130, [1, 64, 65, 200]), (0, [33]), (96, [2, 30, 60]), (512, [1, 1])], heads, kv, dim, page, dtype, device=DEV, resting=resting)
    check(a, window, softcap, torch.randn(heads, device=DEV) * 3 if sinks else None)


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
def test_rows_of_other_tensors_and_streams(dtype, dim):
    a = batch([(130, [1, 64, 65, 200]), (64, [3, 4])], 4, 2, dim, 16, dtype, device=DEV)
    want = check(a)
    packed = torch.randn(6, 9, dim, device=DEV).to(dtype)                 # a packed projection: the queries are its first heads
    packed[:, :4] = a["q"]
    assert torch.equal(check({**a, "q": packed[:, :4]}), want)
    turned = a["q"].transpose(0, 1).contiguous().transpose(0, 1)          # heads apart
    assert torch.equal(check({**a, "q": turned}), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = shared_decode(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    assert torch.equal(shared_decode(**a), want)                          # the same bits again


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (BF16, 64), (FP32, 48)])
def test_grouping_changes_no_more_than_rounding(dtype, dim):
    a = batch([(130, [1, 64, 65, 200]), (64, [3, 4, 5])], 4, 2, dim, 16, dtype, device=DEV)
    R = a["q"].shape[0]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    check({**a, "shared": Shared(ints(range(R)), ints(range(R + 1)), ints([0] * R))})                  # nobody shares
    s = a["shared"]
    check({**a, "shared": Shared(s.order, s.first, s.tokens // 2)})                                    # less than there is
    check({**a, "shared": Shared(s.order, ints(s.first.tolist() + [R] * 3), ints(s.tokens.tolist() + [0] * 3))})      # empty groups behind the last
    check({**a, "shared": Shared(s.order, ints([0] + s.first.tolist()), ints([64] + s.tokens.tolist()))})             # and in front of the first


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
def test_captured_steps_follow_lengths_and_groups(dtype, dim):
    a = batch([(130, [1, 64, 65, 200]), (64, [3, 4, 5])], 4, 2, dim, 16, dtype, device=DEV)
    b = {**a, "lengths": torch.zeros_like(a["lengths"]), "shared": Shared(*(t.clone() for t in a["shared"]))}
    shared_decode(**b)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]                   # two captured steps of the same buffers
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(shared_decode(**b))
    want = check(a)
    b["lengths"].copy_(a["lengths"])
    for g in graphs + graphs[::-1]:
        g.replay()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    b["shared"].tokens.zero_()
    b["lengths"][2] = 0
    graphs[0].replay()
    found = truth({**b, "shared": None})
    assert bool(((outs[0].double().cpu() - found[0]).abs() <= allowed(b, found)).all()) and not outs[0][2].any()


def test_pages_and_rows_outside_are_reported_and_not_read():
    a = batch([(64, [3, 4, 5])], 4, 2, 128, 16, BF16, device=DEV)
    table = a["table"].clone()
    table[1, -1] = 1 << 30
    lengths = torch.full_like(a["lengths"], a["table"].shape[1] * 16)
    for change in (dict(table=table), dict(table=-table), dict(lengths=lengths + 1), dict(shared=a["shared"]._replace(order=a["shared"].order + 1)),
                   dict(shared=a["shared"]._replace(order=a["shared"].order - 1))):
        L.check_status()
        shared_decode(**{**a, "lengths": lengths, **change})
        with pytest.raises(L.KernelError):
            L.check_status()
    check(a)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_large_scores_and_values(dtype):
    """Scores in the hundreds, one key that takes all the weight, equal keys."""
    a = batch([(130, [1, 64, 65, 200]), (64, [3, 4, 5])], 4, 2, 128, 16, dtype, device=DEV)
    check({**a, "scale": 3.0})
    check({**a, "scale": 0.0})
    check({**a, "k": a["k"] * 1e4, "q": a["q"] * 1e-4})
    check({**a, "v": a["v"] * 2.0 ** 60})


# enough work for every SM, lists that begin in one place and end in another, values that come late (nothing of the pools is in the cache): rows of 50 to 400 own keys
def _many(rows, *shared):
    per = rows // len(shared)
    return [(n, [50 + (i * 37 + 11 * g) % 350 for i in range(per)]) for g, n in enumerate(shared)]


@pytest.mark.parametrize("groups, heads, kv, dim, page, window, softcap, sinks", [
    (_many(96, 2500), 16, 4, 128, 64, None, 0.0, False),                       # queries of many rows
    (_many(96, *[600 + 64 * i for i in range(12)]), 16, 4, 128, 16, None, 0.0, True),      # of eight
    (_many(90, 1000, 64, 2100), 40, 8, 64, 16, None, 30.0, True),
    (_many(80, *[320] * 40), 32, 8, 64, 64, 500, 0.0, False),                  # of two, keys that a window ends
    (_many(64, 1500, 700), 8, 2, 256, 32, None, 0.0, False),
    ([(0, [200 + 13 * i]) for i in range(70)], 32, 8, 128, 64, None, 0.0, False),
    (_many(400, 100, 300), 8, 8, 64, 16, None, 0.0, False)])
def test_all_engines_and_late_values(groups, heads, kv, dim, page, window, softcap, sinks):
    a = batch(groups, heads, kv, dim, page, BF16, device=DEV)
    sinks = torch.randn(heads, device=DEV) * 3 if sinks else None
    want = check(a, window, softcap, sinks)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    for i in range(30):
        if i % 3:
            flush.zero_()
        assert torch.equal(shared_decode(**a, window=window, softcap=softcap, sinks=sinks), want), i
    L.check_status()


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
def test_a_row_named_twice_is_reported(dtype, dim):
    a = batch([(64, [3, 4, 5]), (0, [9])], 4, 2, dim, 16, dtype, device=DEV)
    order = a["shared"].order.clone()
    order[1] = order[0]
    L.check_status()
    shared_decode(**{**a, "shared": a["shared"]._replace(order=order)})
    with pytest.raises(L.KernelError):
        L.check_status()
    check(a)
