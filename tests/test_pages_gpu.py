"""The kernel that moves pages and writes tables against plain indexing, and a server whose rows fork and whose pool is compacted."""
import random

import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, KVStore
from dew_b200.ops import library as L
from dew_b200.ops.pages import move_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pools_of(shapes, dtype, pages, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    out = []
    for layers, *page in shapes:
        raw = torch.randint(0, 256, (layers, pages, *page, torch.empty((), dtype=dtype).element_size()), generator=g, device=DEV, dtype=torch.uint8)
        out.append(raw.view(dtype).squeeze(-1) if raw.shape[-1] > 1 else raw.squeeze(-1).view(dtype))
    return out


def as_bytes(t):
    return t.contiguous().view(torch.uint8)


def plain(pools, src, dst, table, tables):
    out = [p.clone() for p in pools]
    for w, p in zip(out, pools):
        if len(src):
            s, d = torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV)
            as_bytes_w, as_bytes_p = w.view(torch.uint8) if w.dim() else w, p.view(torch.uint8)
            as_bytes_w[:, d] = as_bytes_p[:, s]
    t = table.clone()
    for row, first, ps in tables:
        t[row, first:first + len(ps)] = torch.tensor(ps, dtype=torch.int32, device=DEV)
    return out, t


def moves(pages, copies, seed, spans=0, rows=7, columns=11):
    rng = random.Random(seed)
    order = rng.sample(range(pages), pages)
    src, dst = [rng.choice(order[copies:]) for _ in range(copies)], order[:copies]
    tables = []
    for row in rng.sample(range(rows), min(spans, rows)):
        n = rng.randint(0, columns)
        tables.append((row, rng.randint(0, columns - n), [rng.randrange(pages) for _ in range(n)]))
    return src, dst, tables


def same(pools, table, want):
    assert all(torch.equal(as_bytes(p), as_bytes(w)) for p, w in zip(pools, want[0])) and torch.equal(table, want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (2, 16, 2, 64), (5, 7, 1, 5), (3, 48, 3, 80), (4, 2)])
@pytest.mark.parametrize("copies", [0, 1, 9])
def test_moves(dtype, shape, copies):
    pools = pools_of([shape, (shape[0] + 1, 5)], dtype, 31)
    table = torch.arange(77, device=DEV, dtype=torch.int32).view(7, 11) % 31
    src, dst, tables = moves(31, copies, copies, spans=5)
    want = plain(pools, src, dst, table, tables)
    before = L.LAUNCHES
    move_pages(pools, src, dst, table, tables)
    same(pools, table, want)
    assert L.LAUNCHES - before == 1
    move_pages(pools, src, dst)                                                # the sources are as they were: the same again
    same(pools, table, want)


@pytest.mark.parametrize("pages, copies, rows, columns", [(9000, 4000, 300, 40), (20000, 9001, 3, 20000), (60, 3, 2000, 9)])
def test_lists_of_several_launches(pages, copies, rows, columns):
    pools = pools_of([(2, 6), (1, 16)], torch.bfloat16, pages)
    table = torch.zeros(rows, columns, device=DEV, dtype=torch.int32)
    src, dst, tables = moves(pages, copies, 3, spans=rows, rows=rows, columns=columns)
    want = plain(pools, src, dst, table, tables)
    move_pages(pools, src, dst, table, tables)
    same(pools, table, want)


def test_many_pools_and_layers_apart():
    whole = torch.randn(6, 20, 4, 8, device=DEV)
    pools = [whole[::2, :17], *pools_of([(1, 3)] * 70, torch.float32, 17)]
    src, dst, tables = moves(17, 6, 1, spans=4)
    table = torch.zeros(7, 11, device=DEV, dtype=torch.int32)
    untouched = whole.clone()
    want = [p.clone() for p in pools]
    for w, p in zip(want, pools):
        w[:, dst] = p[:, src]
    move_pages(pools, src, dst, table, tables)
    assert all(torch.equal(as_bytes(p), as_bytes(w)) for p, w in zip(pools, want))
    assert torch.equal(whole[1::2], untouched[1::2]) and torch.equal(whole[:, 17:], untouched[:, 17:])


def test_refusals_write_nothing():
    from test_pages_cpu import REFUSED
    pool, table = torch.randn(2, 9, 3, device=DEV), torch.zeros(3, 4, dtype=torch.int32, device=DEV)
    before = pool.clone()
    for src, dst, tables in REFUSED:
        with pytest.raises(ValueError):
            move_pages([pool], src, dst, table, tables)
    with pytest.raises(ValueError):
        move_pages([pool, pool.cpu()], [0], [1])
    with pytest.raises(ValueError):
        move_pages([pool], [0], [1], table.cpu(), [(0, 0, [1])])
    assert torch.equal(pool, before) and not table.any()


def test_on_another_stream_and_captured():
    pools = pools_of([(4, 64, 8)], torch.bfloat16, 40)
    table = torch.zeros(7, 11, device=DEV, dtype=torch.int32)
    src, dst, tables = moves(40, 11, 5, spans=7)
    fresh = [p.clone() for p in pools]
    want = plain(pools, src, dst, table, tables)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        move_pages(pools, src, dst, table, tables)
    torch.cuda.current_stream().wait_stream(side)
    same(pools, table, want)
    pools[0].copy_(fresh[0])
    table.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        move_pages(pools, src, dst, table, tables)
    src.clear()                                                                # the lists have been read
    graph.replay()
    same(pools, table, want)


def model():
    torch.manual_seed(0)
    return CausalTransformer(vocab_size=512, emb_features=256, num_layers=3, num_heads=4, num_kv_heads=2, head_dim=64, mlp_features=256, max_seq_len=512, dtype=torch.bfloat16).to(DEV).eval()


@pytest.mark.parametrize("page, quantized", [(16, None), (64, None), (64, "int8")])
def test_forks_leave_their_parent_alone(page, quantized):
    store = KVStore(KVCache(quantized, page, 40), 3, 4, 256, 2, 64, device=DEV)
    for t in (store.k, store.v):
        t.copy_(torch.randint(-100, 100, t.shape, device=DEV))
    from dew_b200.inference.pages import PageLedger
    led = PageLedger(40, page)
    tokens = page + 5
    row = led.seat(list(range(tokens)), tokens + 20).pages
    store.move_pages([], [], [(0, 0, row)])
    forks = [led.fork(row, tokens, tokens + 20) for _ in range(3)]
    store.move_pages([p for f in forks for p in f.src], [p for f in forks for p in f.dst], [(i + 1, 0, f.pages) for i, f in enumerate(forks)])
    held = [t.clone() for t in store.gather(1, tokens)]
    for t in held:
        assert all(torch.equal(t[0], t[i]) for i in (1, 2, 3))
    # each row's next token is its own
    pos = torch.full((4, 1), tokens, device=DEV)
    store.write(1, torch.arange(4, device=DEV, dtype=torch.bfloat16).view(4, 1, 1, 1).expand(4, 1, 2, 64).contiguous(),
                torch.ones(4, 1, 2, 64, device=DEV, dtype=torch.bfloat16), pos)
    after = store.gather(1, tokens + 1)
    assert torch.equal(after[0][:, :tokens], held[0]) and [float(after[0][i, tokens, 0, 0]) for i in range(4)] == pytest.approx([0, 1, 2, 3], rel=2 ** -8)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_a_served_group_and_compaction(graph, page):
    m, prompt = model(), list(range(5, 155))
    # a row's products do not depend on the rows beside it where as many rows are decoded: six slots in both
    alone = Server(m, slots=6, capacity=256, kv_cache=KVCache(page_size=page), prefix_cache=False)
    want = alone([prompt] * 4, 24)
    server = Server(m, slots=6, capacity=256, kv_cache=KVCache(page_size=page, pages=6 * (256 // page)), cuda_graph=graph)
    first = server.submit([3] * 40, 4)
    got = server.submit_group(prompt, 4, 24)
    moved = 0
    while server.busy:
        server.step()
        if server.steps in (6, 9):
            moved += server.compact()
        if server.steps == 12:
            server.resize(len(server.ledger.refs) + 3)
    assert len(first.result()) == 4 and moved > 0
    assert all(t.result() == got[0].result() for t in got)
    agree = sum(a == b for a, b in zip(got[0].result(), want[0]))
    assert got[0].result()[0] == want[0][0] and agree >= 1


@pytest.mark.parametrize("runs", [[1], [2], [7], [5, 1, 1, 9], [1, 1, 1], [3] * 40, [1, 2] * 60, [4000], [3000, 1, 2500], [2, 1] * 900 + [5000]])
@pytest.mark.parametrize("dtype, page", [(torch.bfloat16, 8), (torch.int8, 5), (torch.float32, 3)])
def test_copies_of_one_page_that_follow_one_another(runs, dtype, page):
    """A source's copies side by side are made from one load; the runs may be cut between two launches."""
    n, copies = len(runs), sum(runs)
    g = torch.Generator().manual_seed(copies)
    order = torch.randperm(n + copies + 3, generator=g).tolist()
    src = [s for s, k in zip(order, runs) for _ in range(k)]
    dst = order[n:n + copies]
    pools = [torch.randint(-100, 100, (2, len(order), page, 3), generator=g).to(dtype).to(DEV) for _ in range(2)]
    table = torch.zeros(4, 9, dtype=torch.int32, device=DEV)
    tables = [(1, 2, dst[:3]), (3, 0, src[:1])]
    want = plain(pools, src, dst, table, tables)
    move_pages(pools, src, dst, table, tables)
    same(pools, table, want)
