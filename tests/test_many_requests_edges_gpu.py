"""The kernels of a server of many requests at their edges: groups that leave rows out, numbers that are none, packed prompts, captured calls."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, PackedRows
from dew_b200.nn.lora import AdapterBank
from dew_b200.ops import library as L
from dew_b200.ops.adapters import Bank, add_adapters
from dew_b200.ops.pages import move_pages
from dew_b200.ops.prefix import Shared, shared_decode
from dew_b200.sampling.text import RowBatch, generate
from dew_b200.utils.trees import module_variables, tree_map
from prefix_cases import allowed, batch, numbers_that_are_none, truth

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def reported(a, **kw):
    L.check_status()
    out = shared_decode(**a, **kw)
    with pytest.raises(L.KernelError):
        L.check_status()
    return out


# ---------------------------------------------------------------------------------------------------------- groups that do not hold every row once
@pytest.mark.parametrize("dtype, heads, kv, dim, page", [(BF16, 8, 2, 128, 16), (BF16, 64, 2, 64, 64), (FP32, 8, 2, 48, 16)])
@pytest.mark.parametrize("held", [0, 2, 5])
def test_rows_that_no_group_holds_are_reported_and_give_zeros(dtype, heads, kv, dim, page, held):
    a = batch([(2048, [1 + i % 40 for i in range(30)])], heads, kv, dim, page, dtype, device=DEV)
    order, R = a["shared"].order, a["q"].shape[0]
    out = reported({**a, "shared": Shared(order, ints([0, held]), a["shared"].tokens[:1].contiguous())})
    left = order.long()[held:]
    assert left.numel() == R - held and not out[left].any()
    got = shared_decode(**a)                                  # (the word is clear again)
    L.check_status()
    found = truth(a)
    assert bool(((got.double().cpu() - found[0]).abs() <= allowed(a, found)).all())


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
@pytest.mark.parametrize("first", [[0, 4, 2, 6], [0, 6, 3, 6], [3, 0, 6, 6]])
def test_groups_that_begin_behind_their_end_are_reported(dtype, dim, first):
    a = batch([(64, [3, 4, 5, 6, 7, 8])], 4, 2, dim, 16, dtype, device=DEV)
    reported({**a, "shared": Shared(a["shared"].order, ints(first), ints([64, 64, 64]))})


# ---------------------------------------------------------------------------------------------------------- adapters
CONFIG = dict(vocab_size=96, emb_features=128, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64, mlp_features=256, max_seq_len=512, tie_embeddings=False)
TARGETS = ("qkv_proj", "o_proj", "gate_up_proj", "down_proj")


def banked(dtype=BF16, seed=0):
    torch.manual_seed(seed)
    m = CausalTransformer(**CONFIG).eval().to(DEV, dtype)
    bank = AdapterBank(m, TARGETS, slots=3, rank=8)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for layer in bank.layers.values():
        for t in (layer.a, layer.b):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV) * 0.1)
        layer.scale.fill_(1.0)
    return m, bank


def test_rows_of_prompts_behind_one_another_keep_their_adapters(monkeypatch):
    m, bank = banked()
    prompts = [[1 + (i * 7 + j) % 90 for j in range(n)] for i, n in enumerate((300, 20, 150, 9))]
    packed, plain = [], RowBatch._prefill_packed
    monkeypatch.setattr(RowBatch, "_prefill_packed", lambda *a: packed.append(1) or plain(*a))
    generate(m, None, prompts, 2)
    assert packed                                             # (what such prompts take without adapters)
    with bank.using(ints([0, -1, 2, 1])):
        got = generate(m, None, prompts, 4)
        monkeypatch.setattr(PackedRows, "pays", staticmethod(lambda *a: False))
        want = generate(m, None, prompts, 4)
    assert len(packed) == 1 and torch.equal(got.tokens, want.tokens)
    L.check_status()


def test_captured_calls_of_several_tokens_follow_their_ids():
    m, bank = banked()
    tokens = torch.randint(96, (3, 7), device=DEV)
    ids, later = ints([0, -1, 1]), ints([2, 0, -1])
    with torch.no_grad():
        with bank.using(later):
            want = m(tokens)
        with bank.using(ids):
            eager = m(tokens)                                 # (a warm-up, and calls between and behind captures)
            graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
            outs = []
            for g in graphs:
                with torch.cuda.graph(g):
                    outs.append(m(tokens))
                assert torch.equal(m(tokens), eager)
            ids.copy_(later)
            graphs[1].replay()
            assert torch.equal(outs[1], want) and torch.equal(m(tokens), want)
            graphs[0].replay()
            assert torch.equal(outs[0], want)
    L.check_status()


# ---------------------------------------------------------------------------------------------------------- scores that are no numbers
@pytest.mark.parametrize("groups", [[(130, [1, 64, 65, 200]), (0, [33]), (512, [1, 1])], [(257, [1 + i % 7 for i in range(40)]), (300, [5] * 9)], [(0, [300])] * 2])
@pytest.mark.parametrize("heads, kv, dim, page, dtype", [(8, 2, 128, 64, BF16), (16, 2, 64, 16, BF16), (4, 2, 256, 16, BF16), (6, 2, 80, 16, BF16), (8, 2, 48, 16, FP32)])
@pytest.mark.parametrize("sinks", [False, True])
def test_scores_that_are_no_numbers_show(groups, heads, kv, dim, page, dtype, sinks):
    a = batch(groups, heads, kv, dim, page, dtype, device=DEV, resting=(len(groups[0][1]),) if len(groups) > 2 else ())
    s = torch.randn(heads, device=DEV) if sinks else None
    live = [r for r, n in enumerate(a["lengths"].tolist()) if n]
    b, nan, zero, same = numbers_that_are_none(a, live[0], live[1])
    L.check_status()
    got = shared_decode(**b, sinks=s).cpu()
    L.check_status()
    found = truth(a, None, 0.0, s)
    assert bool(got[nan].isnan().all()) and not got[zero].any()
    assert bool(((got.double() - found[0]).abs() <= allowed(a, found))[same].all())


# ---------------------------------------------------------------------------------------------------------- what is written in place
def test_autograd_knows_what_was_written_in_place():
    x, ids = torch.randn(5, 64, device=DEV), ints([0, -1, 1, 0, 1])
    bank = Bank(torch.randn(2, 8, 64, device=DEV), torch.randn(2, 48, 8, device=DEV), torch.ones(2, device=DEV))
    for by in (x, x.bfloat16()):
        y, p = torch.randn(5, 48, device=DEV).to(by.dtype), torch.ones(48, device=DEV, dtype=by.dtype, requires_grad=True)
        z = (y * p).sum()                                     # (keeps y)
        add_adapters(y, by, Bank(bank.a.to(by.dtype), bank.b.to(by.dtype), bank.scale), ids)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    pools, table = [torch.randn(2, 6, 4, device=DEV), torch.randn(1, 6, 9, device=DEV)], ints([[0, 1], [2, 3]])
    before = [t._version for t in (*pools, table)]
    move_pages(pools, [0], [1], table, [(0, 0, [5])])
    assert all(t._version > v for t, v in zip((*pools, table), before))
    with torch.inference_mode():
        y = torch.randn(5, 48, device=DEV)
        add_adapters(y, x, bank, ids)
        move_pages([torch.zeros(2, 6, 4, device=DEV)], [0], [1])


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
def test_a_window_past_32_bits_is_none(dtype, dim):
    a = batch([(130, [1, 64, 65, 200]), (64, [3, 4, 5])], 4, 2, dim, 16, dtype, device=DEV)
    want = shared_decode(**a)
    for window in ((1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        assert torch.equal(shared_decode(**a, window=window), want)
    L.check_status()


# ---------------------------------------------------------------------------------------------------------- servers
def small(seed, dtype=FP32):
    torch.manual_seed(seed)
    return CausalTransformer(**CONFIG).eval().to(DEV, dtype)


def alone(m, prompts, new=8):
    return [Server(m, slots=1, capacity=256, kv_cache=KVCache(page_size=16), prefix_cache=False)([p], new)[0] for p in prompts]


@pytest.mark.parametrize("graph", [False, True])
def test_variables_and_reloads_beside_a_bank(graph):
    prompts = [[1 + i % 90 for i in range(70)], [5, 4, 3], [1 + i % 90 for i in range(70)]]
    want, old = alone(small(7), prompts), alone(small(0), prompts)
    assert want != old
    m = small(0)
    bank = AdapterBank(m, TARGETS, slots=2, rank=8)
    theirs = tree_map(lambda t: t.detach().clone(), module_variables(small(7)))
    server = Server(m, theirs, slots=3, capacity=256, kv_cache=KVCache(page_size=16), cuda_graph=graph, shared_prefix=True, adapters=bank)
    assert server(prompts, 8) == want
    server.reload(tree_map(lambda t: t.detach().clone(), module_variables(small(0))))
    assert server(prompts, 8) == old
    server.reload(theirs)
    assert server(prompts, 8) == want
    L.check_status()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_pools_of_other_sizes_between_requests(graph, dtype):
    m = small(3, dtype)
    long, prompts = [1 + i % 90 for i in range(200)], [[1 + i % 60 for i in range(70)], [2 + i % 50 for i in range(33)]]

    def run(resize):
        server = Server(m, slots=2, capacity=256, kv_cache=KVCache(page_size=16), chunk=32, cuda_graph=graph, shared_prefix=True)
        server([long, long[3:]], 6)
        out = []
        for pages in (12, 9, 40):
            if resize:
                server.resize(pages)
                assert int(server.store.page_table.max()) < pages and server.store.k.shape[1] == pages + 1
            out.append(server(prompts, 6))                    # unequal prompts in chunks
            row = server.submit(prompts[1], 6)                # a step beside an idle row
            server.run()
            out.append(row.result())
        L.check_status()
        return out
    assert run(True) == run(False)
