"""Pages that move: copies and table pieces, the ledger's forks and compaction, samples that fork from one prompt."""
import ctypes
import random

import pytest
import torch

from dew_b200.inference.pages import OutOfPages, PageLedger
from dew_b200.inference.rollouts import NativeRolloutServer
from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import CacheSlot, KVCache, KVStore
from dew_b200.ops import library as L
from dew_b200.ops.pages import move_pages
from dew_b200.sampling.text import Sampling


def model(**kw):
    torch.manual_seed(0)
    return CausalTransformer(**{**dict(vocab_size=64, emb_features=32, num_layers=2, num_heads=2, num_kv_heads=1, head_dim=16, mlp_features=48, max_seq_len=96), **kw}).eval()


def test_copies_and_table_pieces():
    pools = [torch.randn(3, 9, 4, 2), torch.randint(-100, 100, (1, 9, 5), dtype=torch.int8)]
    table = torch.arange(12, dtype=torch.int32).view(3, 4) % 9
    want = [p.clone() for p in pools]
    for w in want:
        w[:, 1], w[:, 2], w[:, 8] = w[:, 5].clone(), w[:, 5].clone(), w[:, 0].clone()
    move_pages(pools, [5, 5, 0], [1, 2, 8], table, [(2, 1, [7, 8]), (0, 0, [3]), (1, 4, [])])
    assert all(torch.equal(p, w) for p, w in zip(pools, want))
    assert table.tolist() == [[3, 1, 2, 3], [4, 5, 6, 7], [8, 7, 8, 2]]
    move_pages(pools, [], [])
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


REFUSED = [([0], [9], []), ([-1], [1], []), ([0, 1], [2, 2], []), ([0, 1], [1, 2], []), ([3], [3], []), ([], [], [(3, 0, [1])]), ([], [], [(-1, 0, [1])]),
           ([], [], [(0, 3, [1, 2])]), ([], [], [(0, -1, [1])]), ([], [], [(0, 0, [9])]), ([], [], [(0, 0, [-1])]), ([], [], [(1, 0, [1, 2]), (0, 0, [1]), (1, 1, [3])])]


@pytest.mark.parametrize("src, dst, tables", REFUSED)
def test_refusals_write_nothing(src, dst, tables):
    pool, table = torch.randn(2, 9, 3), torch.zeros(3, 4, dtype=torch.int32)
    before = pool.clone()
    with pytest.raises(ValueError):
        move_pages([pool], src, dst, table, tables)
    assert torch.equal(pool, before) and not table.any()


def test_refusals_of_layouts():
    pool, table = torch.randn(2, 9, 3, 4), torch.zeros(3, 4, dtype=torch.int32)
    for pools, src, t, tables in [([], [0], table, []), ([pool, pool[:, :8]], [0], table, []), ([pool.transpose(2, 3)], [0], table, []), ([pool[:, ::2]], [0], table, []),
                                  ([pool], [0, 1], table, []), ([pool], [0], None, [(0, 0, [1])]), ([pool], [0], table.long(), [(0, 0, [1])]), ([pool], [0], table.T, [(0, 0, [1])])]:
        with pytest.raises(ValueError):
            move_pages(pools, src, [1], t, tables)


def _native(src, dst, pages, columns, rows, tables):
    """What the launcher's own look at the lists says (host code: it runs without a GPU)."""
    if not L.exists():
        pytest.skip("the library is not built")
    ints = lambda x: (ctypes.c_int * max(1, len(x)))(*x)
    at = lambda x: ctypes.addressof(x)
    lists = [ints(x) for x in (src, dst, [t[0] for t in tables], [t[1] for t in tables], [len(t[2]) for t in tables], [p for t in tables for p in t[2]])]
    return L.load().dewb_check_moves(at(lists[0]), at(lists[1]), len(src), pages, *map(at, lists[2:]), len(tables), rows, columns)


def test_the_launchers_look():
    assert _native([5, 5, 0], [1, 2, 8], 9, 4, 3, [(2, 1, [7, 8]), (0, 0, [3]), (1, 4, []), (1, 0, [1])]) == 0
    assert _native([], [], 9, 4, 3, []) == 0
    codes = [_native(src, dst, 9, 4, 3, tables) for src, dst, tables in REFUSED]
    assert codes == [-11, -11, -12, -13, -13, -14, -14, -14, -14, -11, -11, -16]


def test_a_fork_shares_whole_pages_and_copies_the_last():
    led = PageLedger(pages=12, page_size=4)
    row = led.seat(list(range(10)), 14).pages
    fork = led.fork(row, 10, 18)
    assert fork.pages[:2] == row[:2] and len(fork.pages) == 5 and not set(fork.pages[2:]) & set(row) and (fork.src, fork.dst) == ([row[2]], [fork.pages[2]])
    even = led.fork(row, 8, 8)
    assert even.pages == row[:2] and not even.src and not even.dst
    assert led.refs[row[0]] == 3 and led.available() == 12 - 4 - 3
    with pytest.raises(OutOfPages):
        led.fork(row, 10, 40)
    assert led.refs[row[0]] == 3 and led.available() == 5                     # a refused fork holds nothing
    for bad in ((17, 17), (-1, 4), (10, 9)):
        with pytest.raises(ValueError):
            led.fork(row, *bad)
    led.release(row)
    led.release(even.pages)
    assert led.truncate(fork.pages, 5) and len(fork.pages) == 2 and led.available() == 10
    led.release(fork.pages)
    assert led.available() == 12 and not led.refs
    with pytest.raises(ValueError):
        led.fork(row, 10, 18)                                                  # given back: another row's by now


def test_compaction_renames_what_is_held():
    rng = random.Random(0)
    led = PageLedger(pages=40, page_size=4)
    prompts = [[rng.randrange(50) for _ in range(rng.randint(1, 18))] for _ in range(6)]
    rows = [led.seat(p, len(p) + 6) for p in prompts]
    for p, r in zip(prompts, rows):
        led.publish(p, r.pages)
    for r in rows[:3]:
        led.release(r.pages)
    before = {h: p for h, p in led.page_of.items()}
    refs, idle = dict(led.refs), list(led.idle)
    moved = led.compact()
    name = lambda p: moved.get(p, p)
    held = len(refs) + len(idle)
    assert moved and set(moved).isdisjoint(moved.values()) and max(led.refs) < held and max(led.idle, default=0) < held
    assert led.refs == {name(p): n for p, n in refs.items()} and list(led.idle) == [name(p) for p in idle]
    assert led.page_of == {h: name(p) for h, p in before.items()} and all(led.page_of[h] == p for p, h in led.name_of.items())
    assert sorted(led.free) == list(range(held, 40)) and led.compact() == {}
    with pytest.raises(ValueError):
        led.resize(held - 1)
    led.evict(held - 1)
    assert len(led.idle) == len(idle) - 1 and len(led.free) == 40 - held + 1
    led.evict(len(led.refs))
    led.compact()
    led.resize(len(led.refs))
    assert not led.free and led.available() == 0


@pytest.mark.parametrize("quantized", [None, "int8"])
def test_a_store_moves_every_layer_and_scale(quantized):
    store = KVStore(KVCache(quantized, 4, 6), 3, 2, 16, 2, 8, dtype=torch.float32)
    for t in (store.k, store.v, store.k_scale, store.v_scale):
        if t is not None:
            t.copy_(torch.randn(t.shape) * 50)
    want = [t.clone() for t in store.pools()]
    store.move_pages([2, 3], [0, 5], [(1, 0, [5, 0])])
    for got, w in zip(store.pools(), want):
        assert torch.equal(got[:, 0], w[:, 2]) and torch.equal(got[:, 5], w[:, 3]) and torch.equal(got[:, 1:5], w[:, 1:5])
    assert store.page_table[1, :2].tolist() == [5, 0] and len(store.pools()) == (4 if quantized else 2)
    with pytest.raises(ValueError):
        store.move_pages([0], [6])                                             # the spare page is nobody's
    store.resize(8)
    assert all(torch.equal(got[:, 5], w[:, 3]) and got.shape[1] == 8 for got, w in zip(store.pools(), want))
    store.resize(2)
    assert store.k.shape[1] == 3 and store.pages == 2
    with pytest.raises(ValueError):
        store.resize(0)


def test_slots_of_several_kinds():
    slots = [CacheSlot(2, 8, 8), CacheSlot(state=(3,), more=(("conv", (2, 2)),)), CacheSlot(2, 8, 8, source=0), CacheSlot(1, 16, 8, latent=True)]
    store = KVStore(KVCache(page_size=4, pages=5), 4, 3, 8, 2, 8, dtype=torch.float32, slots=slots)
    assert len(store.pools()) == 3                                             # keys and values of slot 0, the latent rows of slot 3
    store.states[1].copy_(torch.randn(3, 3))
    store.more[1]["conv"].copy_(torch.randn(3, 2, 2))
    state, conv = store.states[1].clone(), store.more[1]["conv"].clone()
    store.fork_rows([1, 1], [0, 2])
    assert torch.equal(store.states[1], state[[1, 1, 1]]) and torch.equal(store.more[1]["conv"], conv[[1, 1, 1]])
    for bad in (([0], [3]), ([-1], [0])):
        with pytest.raises(ValueError):
            store.fork_rows(*bad)
    store.k[0].copy_(torch.randn(store.k[0].shape))
    kept = store.k[0].clone()
    store.resize(3)
    assert store.k[2] is store.k[0] and store.v[3] is store.k[3] and torch.equal(store.k[0][:3], kept[:3]) and store.k[0].shape[0] == 4


def _tokens(tickets):
    return [t.result() for t in tickets]


@pytest.mark.parametrize("prompt_len", [1, 7, 8, 19])
@pytest.mark.parametrize("greedy", [True, False])
def test_samples_of_one_prompt_are_those_of_requests_of_their_own(prompt_len, greedy):
    m, prompt = model(), list(range(3, 3 + prompt_len))
    sampling = Sampling(temperature=0.0 if greedy else 1.0)
    alone = Server(m, slots=6, capacity=48, kv_cache=KVCache(page_size=8), prefix_cache=False, sampling=sampling)
    want = [alone.submit(prompt, 9, key=k) for k in (5, 6, 7, 8)]
    alone.run()
    server = Server(m, slots=6, capacity=48, kv_cache=KVCache(page_size=8), sampling=sampling)
    other = server.submit([9, 8, 7, 6, 5], 12, key=1)
    got = server.submit_group(prompt, 4, 9, keys=(5, 6, 7, 8))
    server.run()
    assert _tokens(got) == _tokens(want) and len(other.result()) == 12 and not server.ledger.refs
    alone_too = Server(m, slots=1, capacity=48, kv_cache=KVCache(page_size=8), sampling=sampling)
    expected = alone_too.submit([9, 8, 7, 6, 5], 12, key=1)
    alone_too.run()
    assert other.result() == expected.result()


def test_samples_without_a_slot_wait_like_other_requests():
    m = model()
    server = Server(m, slots=2, capacity=32, kv_cache=KVCache(page_size=4, pages=11))      # room for one sample beside the first
    got = server.submit_group(list(range(10)), 5, 6)
    server.run()
    alone = Server(m, slots=1, capacity=32, kv_cache=KVCache(page_size=4))
    want = [alone.submit(list(range(10)), 6, key=k) for k in range(5)]
    alone.run()
    assert _tokens(got) == _tokens(want)
    for bad in (dict(n=0), dict(n=2, keys=[1])):
        with pytest.raises(ValueError):
            server.submit_group([1, 2], max_new_tokens=2, **bad)
    with pytest.raises(ValueError):
        server.submit_group([], 2, 2)
    assert not server.queue
    waiting = server.submit_group([1, 2, 3], 3, 2)
    server.fail(RuntimeError("stopped"))
    assert all(t.done and isinstance(t.error, RuntimeError) for t in waiting)


@pytest.mark.parametrize("kw", [dict(), dict(layer_types=("gdn", "attention"))])
def test_a_recurrent_state_forks_with_its_row(kw):
    try:
        m = model(**kw)
    except TypeError:
        pytest.skip("no such layers")
    prompt = list(range(2, 13))
    alone = Server(m, slots=1, capacity=32, kv_cache=KVCache(page_size=8), prefix_cache=False)
    want = alone([prompt], 6)
    server = Server(m, slots=4, capacity=32, kv_cache=KVCache(page_size=8))
    got = server.submit_group(prompt, 3, 6)
    server.run()
    assert _tokens(got) == want * 3


def test_compaction_between_steps_changes_no_token():
    m = model()
    prompts = [list(range(i, i + 5 + 3 * i)) for i in range(5)]
    want = Server(m, slots=5, capacity=48, kv_cache=KVCache(page_size=4), prefix_cache=False)(prompts, 12)
    server = Server(m, slots=3, capacity=48, kv_cache=KVCache(page_size=4, pages=40))
    tickets = [server.submit(p, 12) for p in prompts]
    moved, sizes = 0, []
    while server.busy:
        server.step()
        moved += server.compact()
        if server.steps % 5 == 0:
            server.resize(len(server.ledger.refs) + 17)
            sizes.append(server.store.k.shape[1] - 1)
    assert _tokens(tickets) == want and moved > 0 and len(set(sizes)) > 1
    with pytest.raises(OutOfPages):
        server.submit(prompts[4], 12)
        server.step()
        server.resize(1)


def test_a_group_of_rollouts_reads_its_prompt_once():
    m = model()
    direct = Server(m, slots=4, capacity=32, sampling=Sampling(temperature=1.0))
    want = [direct.submit([1, 2, 3], 6, key=k) for k in (3, 4, 5)]
    direct.run()
    server = Server(m, slots=4, capacity=32, sampling=Sampling(temperature=1.0))
    with NativeRolloutServer(server) as rs:
        draws = [f.result(timeout=120) for f in rs.submit_group([1, 2, 3], 3, 6, keys=(3, 4, 5))]
        for bad in (dict(n=0), dict(n=2, keys=[1])):
            with pytest.raises(ValueError):
                rs.submit_group([1], max_new_tokens=2, **bad)
        with pytest.raises(ValueError):
            rs.submit_group([], 2, 2)
    assert [d.tokens for d in draws] == _tokens(want)
