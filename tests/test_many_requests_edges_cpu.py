"""Where a server of many requests meets the rest of the framework: pools that change their size, weights given as variables, threads, layouts that nobody has in mind."""
import copy
import itertools
import math
import random
import sys
import threading
import time
from contextlib import nullcontext
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad
from torch.overrides import TorchFunctionMode

import prefix_cases
from dew_b200.inference.serving import Server
from dew_b200.inference.tasks import TextGeneration
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import CacheSlot, KVCache, KVStore, PackedRows
from dew_b200.nn.layers import reset_all
from dew_b200.nn.lora import AdapterBank, apply_lora, lora_state, merge_all
from dew_b200.nn.quantization import Quantization, convert_qat, prepare_qat, quantize_model
from dew_b200.ops.adapters import Bank, adapted_linear, add_adapters
from dew_b200.ops.pages import move_pages
from dew_b200.ops.prefix import group_rows, shared_decode
from dew_b200.sampling.text import Sampling
from dew_b200.utils.trees import flatten, module_variables, tree_map

CONFIG = dict(vocab_size=64, emb_features=32, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, mlp_features=48, max_seq_len=160, tie_embeddings=False)


def model(seed=0, **kw):
    torch.manual_seed(seed)
    return CausalTransformer(**{**CONFIG, **kw}).eval()


# ---------------------------------------------------------------------------------------------------------- pools of another size
def test_a_smaller_pool_leaves_no_name_of_a_page_that_is_gone():
    m = model()
    prompts = [[i % 60 for i in range(49)], [i % 50 for i in range(18)]]
    want = [Server(m, slots=1, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False)([p], 6)[0] for p in prompts]
    server = Server(m, slots=2, capacity=160, kv_cache=KVCache(page_size=8), chunk=16)
    server([[1 + i % 50 for i in range(140)], [2 + i % 50 for i in range(130)]], 8)       # names of pages all over the pool
    server.resize(20)
    assert int(server.store.page_table.max()) < 20
    assert server(prompts, 6) == want                         # unequal prompts in several chunks
    server.resize(9)
    short = server.submit(prompts[1], 6)                      # a decode step beside an idle row
    server.run()
    assert short.result() == want[1] and int(server.store.page_table.max()) < 9


def test_a_row_that_lives_through_a_smaller_pool_keeps_its_own_names():
    m, prompt = model(), list(range(3, 30))
    want = Server(m, slots=1, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False)([prompt], 20)[0]
    server = Server(m, slots=3, capacity=160, kv_cache=KVCache(page_size=8), chunk=16)
    server([[1 + i % 50 for i in range(140)]] * 3, 8)
    row = server.submit(prompt, 20)
    for _ in range(6):
        server.step()
    before = server.store.page_table.data_ptr()
    server.resize(12)
    assert int(server.store.page_table.max()) < 12 and server.store.page_table.data_ptr() == before
    server.run()
    assert row.result() == want
    server.resize(40)
    assert server([prompt], 20) == [want]


def test_a_store_takes_names_past_its_end_out_of_the_table():
    store = KVStore(KVCache(page_size=8, pages=20), 1, 2, 64, 1, 16, dtype=torch.float32)
    store.page_table.copy_(torch.arange(16, dtype=torch.int32).view(2, 8) + 4)
    store.resize(10)
    assert store.page_table.tolist() == [[4, 5, 6, 7, 8, 9, 0, 0], [0] * 8]
    store.gather(0, 64)


def _stores():
    slots = [CacheSlot(1, 8, 8), CacheSlot(2, 16, 16), CacheSlot(1, 8, 8, source=0)]
    return [KVStore(KVCache(page_size=4, pages=12), 2, 2, 24, 1, 8, dtype=torch.float32), KVStore(KVCache("int8", 4, 12), 2, 2, 24, 1, 8, dtype=torch.float32),
            KVStore(KVCache(page_size=4, pages=12), 3, 2, 24, 1, 8, dtype=torch.float32, slots=slots)]


def _filled(store):
    for i, t in enumerate(store.pools()):
        t.copy_((torch.arange(t.numel(), dtype=torch.float32) * (i + 1) % 100).view(t.shape))
    return [t.clone() for t in store.pools()]


class ShortOfMemory(TorchFunctionMode):
    """The device has no room for a pool from the ``after``-th one asked for on, ``times`` times."""

    def __init__(self, after, times=100):
        super().__init__()
        self.made, self.after, self.times = 0, after, times

    def __torch_function__(self, func, types, args=(), kwargs=None):
        if func in (torch.zeros, torch.ones, torch.empty, torch.full, torch.Tensor.new_zeros, torch.Tensor.new_ones, torch.Tensor.new_empty, torch.Tensor.new_full):
            self.made += 1
            if self.after < self.made <= self.after + self.times:
                raise torch.OutOfMemoryError("no room")
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("after", [0, 1])
def test_a_pool_that_cannot_grow_stays_as_it_is(which, after):
    store = _stores()[which]
    held = _filled(store)
    with pytest.raises(torch.OutOfMemoryError), ShortOfMemory(after):
        store.resize(30)
    assert store.pages == 12 and all(torch.equal(a, b) for a, b in zip(store.pools(), held)) and len(store.pools()) == len(held)
    assert {t.shape[1 if store.slots is None else 0] for t in _all(store)} == {13}
    store.resize(30)
    assert store.pages == 30 and all(torch.equal(a[:, :12], b) for a, b in zip(store.pools(), held)) and len(store.pools()) == len(held)


def _all(store):
    return [t for t in ([store.k, store.v, store.k_scale, store.v_scale] if store.slots is None else [*store.k, *store.v]) if t is not None]


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("after", [0, 1])
def test_a_pool_shrinks_where_there_is_no_room_for_both(which, after):
    store = _stores()[which]
    held = _filled(store)
    with ShortOfMemory(after, 1):                             # (there is room once the old one is gone)
        store.resize(5)
    assert store.pages == 5 and all(torch.equal(a, b[:, :5]) for a, b in zip(store.pools(), held))
    if store.slots is not None:
        assert store.k[2] is store.k[0] and store.v[2] is store.v[0]


# ---------------------------------------------------------------------------------------------------------- weights given as variables
PROMPTS = [list(range(3, 25)), [9, 8, 7]]


def variables_of(m):
    return tree_map(lambda t: t.detach().clone(), module_variables(m))


def alone(m, prompt, variables=None, new=8):
    return Server(m, variables, slots=1, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False)([prompt], new)[0]


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.02])
def test_variables_reach_the_head(tied, temperature):
    def tokens(m, variables=None, reloaded=None):
        server = Server(m, variables, slots=2, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False, sampling=Sampling(temperature=temperature))
        if reloaded is not None:
            server.reload(reloaded)
        return server(PROMPTS, 8)
    ours, theirs = model(0, tie_embeddings=tied), model(7, tie_embeddings=tied)
    for m in (ours, theirs):
        m.embed.weight.data.mul_(0.05)                        # (a tied head repeats its input otherwise)
    want = tokens(theirs)
    assert want != tokens(ours)
    assert tokens(ours, variables_of(theirs)) == want
    assert tokens(ours, None, variables_of(theirs)) == want


# ---------------------------------------------------------------------------------------------------------- a bank of adapters and the model's weights
TARGETS = ("qkv_proj", "o_proj", "down_proj")


def adapter(seed, rank=4, base=0):
    """An adapter as training leaves it on ``model(base)``, and the model that has it merged into its weights."""
    m = model(base)
    apply_lora(m, TARGETS, rank=rank, alpha=2.0 * rank)
    g = torch.Generator().manual_seed(seed)
    for n, p in m.named_parameters():
        if ".lora_b" in n:
            p.data.normal_(0.0, 0.2, generator=g)
    state = lora_state(m)
    merge_all(m)
    return state, m


def test_variables_reach_the_layers_of_a_bank():
    want = [alone(model(7), p) for p in PROMPTS]
    assert want != [alone(model(0), p) for p in PROMPTS]
    state, merged = adapter(1, base=7)
    m = model(0)
    bank = AdapterBank(m, TARGETS, slots=2, rank=4)
    bank.load("one", state, alpha=8.0)
    make = dict(slots=3, capacity=160, kv_cache=KVCache(page_size=8), adapters=bank)
    for server in (Server(m, variables_of(model(7)), **make), Server.from_task(TextGeneration(m, variables_of(model(7))), **make)):
        plain, adapted = [server.submit(p, 8) for p in PROMPTS], server.submit(PROMPTS[0], 8, adapter="one")
        server.run()
        assert [t.result() for t in plain] == want and adapted.result() == alone(merged, PROMPTS[0])
    server = Server(m, **make)
    assert server(PROMPTS, 8) == [alone(model(0), p) for p in PROMPTS]
    server = Server(m, prefix_cache=False, **make)
    server.reload(variables_of(model(7)))
    assert server(PROMPTS, 8) == want


def test_a_bank_changes_no_name_of_the_model():
    m, plain = model(), model()
    AdapterBank(m, TARGETS, slots=2, rank=4)
    assert [n for n, _ in m.named_parameters()] == [n for n, _ in plain.named_parameters()] and list(m.state_dict()) == list(plain.state_dict())
    m.load_state_dict(model(7).state_dict())
    assert alone(m, PROMPTS[0]) == alone(model(7), PROMPTS[0])
    other = model(3)
    AdapterBank(other, TARGETS, slots=1, rank=2)
    reset_all(other, 5), reset_all(plain, 5)
    assert all(torch.equal(a, b) for a, b in zip(other.parameters(), plain.parameters()))


def test_layers_of_a_bank_can_still_be_quantised_and_watched():
    state, merged = adapter(1)
    m, plain = model(), model()
    seen = []
    m.layers[0].mixer.qkv_proj.register_forward_hook(lambda mod, args, out: seen.append(out.shape))
    bank = AdapterBank(m, TARGETS, slots=2, rank=4)
    bank.load("one", state, alpha=8.0)
    q = Quantization("int8", min_size=0, skip=("embed",))
    assert quantize_model(m, q) == quantize_model(plain, q)
    ids = torch.tensor([[1, 2, 3, 4]])
    with torch.no_grad():
        want = plain(ids)
        assert torch.equal(m(ids), want) and seen
        with bank.using(torch.tensor([0], dtype=torch.int32)):
            got = m(ids)
    assert not torch.allclose(got, want, atol=1e-2) and torch.allclose(got, merged(ids), atol=0.2)
    assert m.layers[0].mixer.qkv_proj.weight.shape == plain.layers[0].mixer.qkv_proj.weight.shape
    m = model()
    AdapterBank(m, TARGETS, slots=2, rank=4)
    assert prepare_qat(m, q) == prepare_qat(model(), q)
    with torch.no_grad():
        m(ids)
    assert convert_qat(m) == convert_qat(_qat(q))


def _qat(q):
    m = model()
    prepare_qat(m, q)
    return m


@pytest.mark.parametrize("host_pages", [0, 8])
def test_pages_of_other_weights_are_no_prefix(host_pages):
    prompts = [list(range(3, 25)), list(range(3, 45)), list(range(3, 25))]
    want = [alone(model(7), p) for p in prompts]
    server = Server(model(0), slots=2, capacity=160, kv_cache=KVCache(page_size=8, pages=9 if host_pages else None), chunk=16, host_pages=host_pages)
    server(prompts[:1], 8)
    late = server.submit(prompts[1], 8)
    server.step()                                             # a prompt half way through when the weights change: its pages are of both
    server.reload(variables_of(model(7)))
    server.run()
    hits = server.ledger.hits
    assert [server([p], 8)[0] for p in prompts] == want and len(late.result()) == 8
    assert server.ledger.hits == hits + 2 + 2                 # the two whole pages that all three begin with, of the new weights


def test_variables_bring_no_adapters_along():
    """What stands in a bank is the bank's: a copy of the model's variables, taken earlier, says nothing about it."""
    state, merged = adapter(1)
    m = model()
    bank = AdapterBank(m, TARGETS, slots=2, rank=4)
    early = variables_of(m)
    bank.load("one", state, alpha=8.0)
    server = Server(m, early, slots=1, capacity=160, kv_cache=KVCache(page_size=8), adapters=bank)
    ticket = server.submit(PROMPTS[0], 8, adapter="one")
    server.run()
    assert ticket.result() == alone(merged, PROMPTS[0])
    assert set(flatten(early)) == set(flatten(variables_of(model())))


def test_a_bank_moves_with_its_model():
    state, _ = adapter(1)
    m = model()
    bank = AdapterBank(m, TARGETS, slots=2, rank=4)
    bank.load("one", state, alpha=8.1)
    layer = bank.layers["layers.0.mixer.qkv_proj"]
    scale = layer.scale
    m.to(torch.bfloat16)
    assert layer.a.dtype == layer.b.dtype == torch.bfloat16 and torch.equal(layer.scale, scale) and layer.scale.dtype == torch.float32 and layer.a.any()
    with torch.no_grad(), bank.using(torch.tensor([0], dtype=torch.int32)):
        m(torch.tensor([[1, 2, 3]]))
    m.to("meta")
    assert layer.a.device.type == layer.b.device.type == layer.scale.device.type == "meta"


def test_prompts_behind_one_another_are_not_for_rows_with_adapters():
    store = SimpleNamespace(slots=None, kind=0, dtype=torch.bfloat16, device=torch.device("cuda"), row_ids=None, head_dim=16 * 4, kv_heads=2)
    m = model(head_dim=64)
    assert PackedRows.suits(store, m)
    bank = AdapterBank(m, TARGETS, slots=2, rank=4)
    assert PackedRows.suits(store, m)
    with bank.using(torch.tensor([0, -1, 1], dtype=torch.int32)):
        assert not PackedRows.suits(store, m)
        with bank.using(None):
            assert PackedRows.suits(store, m)


def random_bank(m, slots=2):
    bank, g = AdapterBank(m, TARGETS, slots=slots, rank=4), torch.Generator().manual_seed(2)
    for layer in bank.layers.values():
        for t in (layer.a, layer.b):
            t.copy_(torch.randn(t.shape, generator=g) * 0.2)
        layer.scale.fill_(1.0)
    return bank


def test_every_thread_has_its_own_rows():
    m = model()
    bank = random_bank(m)
    calls = [(torch.tensor(ids, dtype=torch.int32), torch.randint(60, (len(ids), 5), generator=torch.Generator().manual_seed(i))) for i, ids in enumerate(([0, 1], [1, 0], [-1, 1, 0]))]

    def one(ids, tokens):
        with torch.no_grad(), bank.using(ids):
            return m(tokens)
    want = [one(*c) for c in calls]
    with torch.no_grad():
        plain = m(calls[2][1])
    together, got = threading.Barrier(4, timeout=20), [None] * 4

    def work(i):
        with torch.no_grad(), bank.using(calls[i][0]) if i < 3 else nullcontext():
            together.wait()                                   # all are inside
            got[i] = m(calls[min(i, 2)][1])
            together.wait()
    threads = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert all(x is not None and torch.equal(x, w) for x, w in zip(got, want + [plain]))


def test_holds_of_many_threads_are_counted():
    bank = AdapterBank(model(), TARGETS, slots=2, rank=4)
    bank.load("x", adapter(1)[0], alpha=8.0)
    was = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        def work():
            for _ in range(20000):
                bank.acquire("x")
                bank.release("x")
        threads = [threading.Thread(target=work, daemon=True) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
    finally:
        sys.setswitchinterval(was)
    assert bank.holds["x"] == 0


def test_a_model_with_a_bank_is_copied_with_it():
    m = model()
    random_bank(m)
    other = copy.deepcopy(m)
    theirs = other.layers[0].mixer.qkv_proj._of[0]
    assert theirs.layers["layers.0.mixer.qkv_proj"] is other.layers[0].mixer.qkv_proj
    ids = torch.tensor([0], dtype=torch.int32)
    with torch.no_grad(), theirs.using(ids), m.layers[0].mixer.qkv_proj._of[0].using(ids):
        assert torch.equal(other(torch.tensor([[1, 2, 3]])), m(torch.tensor([[1, 2, 3]])))


def test_ids_are_read_when_the_calls_run():
    m = model()
    bank, ids, tokens = random_bank(m), torch.tensor([0, -1], dtype=torch.int32), torch.tensor([[1, 2, 3], [4, 5, 6]])
    other = torch.tensor([1, 0], dtype=torch.int32)
    with torch.no_grad():
        with bank.using(other):
            want = m(tokens)
        with bank.using(ids):
            first = m(tokens)
            ids.copy_(other)
            assert torch.equal(m(tokens), want) and not torch.equal(first, want)
    with torch.inference_mode():
        ids = torch.tensor([0, -1], dtype=torch.int32)        # (which counts no versions)
        with bank.using(ids):
            m(tokens)
            ids.copy_(other)
            assert torch.equal(m(tokens), want)


def test_layers_whose_weight_the_model_takes_itself_are_refused():
    """The head's weight, the latent attention's up-projection: what stands beside such a layer would be passed over."""
    ids, tokens = torch.tensor([0], dtype=torch.int32), torch.tensor([[1, 2, 3]])
    for m, targets in ((model(), ("head",)), (model(layer_types=("mla", "mla"), mixer_options=dict(kv_latent=16, nope_dim=8, rope_dim=8, v_dim=8)), ("kv_up", "o_proj"))):
        plain = m(tokens)
        bank = AdapterBank(m, targets, slots=1, rank=4)
        server = Server(m, slots=1, capacity=160, kv_cache=KVCache(page_size=8), adapters=bank)
        layer = next(iter(bank.layers.values()))
        bank.load("x", {f"{path}.lora_{n}": torch.ones(*s) for path, x in bank.layers.items() for n, s in (("a", (1, x.in_features)), ("b", (x.out_features, 1)))}, alpha=1.0)
        server.submit([1, 2, 3], 4, adapter="x")
        with pytest.raises(RuntimeError, match="itself"):
            server.run()
        assert layer.weight.shape == (layer.out_features, layer.in_features) and torch.equal(m(tokens), plain)


def test_a_bank_of_another_model_is_refused():
    m, other = model(), model()
    bank = AdapterBank(other, TARGETS, slots=1, rank=4)
    with pytest.raises(ValueError, match="bank"):
        Server(m, slots=1, capacity=32, adapters=bank)
    Server(other, slots=1, capacity=32, adapters=bank)


# ---------------------------------------------------------------------------------------------------------- which rows share what
def groups_of(tables, page=16, least=1):
    order, first, tokens = group_rows(tables, page, least)
    R = len(tables)
    assert sorted(order) == list(range(R)) and len(first) == R + 1 and len(tokens) == R and first[0] == 0 and first[-1] == R and first == sorted(first)
    found = {tuple(order[a:b]): n for a, b, n in zip(first, first[1:], tokens) if a < b}
    for rows, n in found.items():
        assert n % page == 0 and (n == 0 if len(rows) == 1 else n >= max(1, least))
        assert len({tuple(tables[r][:n // page]) if n else r for r in rows}) == (1 if n else len(rows)) and all(len(tables[r] or ()) * page >= n for r in rows)
    return found


def saved(found):
    return sum((len(rows) - 1) * n for rows, n in found.items())


def best(tables, page, least):
    """Most tokens that any grouping saves, by trying all of them."""
    def part(rows):
        if not rows:
            return 0
        head, rest = rows[0], rows[1:]
        most = 0
        for mask in range(1 << len(rest)):
            group = [head] + [r for i, r in enumerate(rest) if mask >> i & 1]
            common = 0
            for column in zip(*(tables[r] or () for r in group)):
                if len(set(column)) > 1:
                    break
                common += 1
            n = common * page if len(group) > 1 and common * page >= max(1, least) else 0
            if n or len(group) == 1:
                most = max(most, (len(group) - 1) * n + part([r for r in rest if r not in group]))
        return most
    return part(list(range(len(tables))))


def test_groups_behind_a_common_start_share_their_own_prefixes():
    # prompts behind one template of a page: four groups of eight that share 64 pages each
    tables = [[1] + [100 * g + i for i in range(63)] + [10000 + 8 * g + r] for g in range(4) for r in range(8)]
    assert groups_of(tables, least=512) == {tuple(range(8 * g, 8 * g + 8)): 1024 for g in range(4)}
    # one row that leaves early does not end what the others share
    assert groups_of(tables[:8] + [[1, 7, 8]], least=512) == {tuple(range(8)): 1024, (8,): 0}
    assert groups_of([[1, 2, 3, 4], [1, 2, 3, 5], [1, 9, 8, 7], [1, 9, 8, 6]], least=32) == {(0, 1): 48, (2, 3): 48}
    # a long start that many rows have is worth more than what two of them have beyond it, and less than what most of them have
    start = list(range(40))
    assert groups_of([start + [50 + i] for i in range(6)] + [start + [99, 7], start + [99, 8]]) == {tuple(range(8)): 640}
    deep = start + list(range(200, 300))
    assert groups_of([start + [50], start + [51]] + [deep + [60 + i] for i in range(6)]) == {(0, 1): 640, tuple(range(2, 8)): 2240}
    assert groups_of([[1, 2], (1, 2), [1, 2, 3]]) == {(0, 1, 2): 32}


@pytest.mark.parametrize("seed", range(40))
def test_no_grouping_saves_more(seed):
    rng = random.Random(seed)
    names, tables = itertools.count(), []
    for _ in range(rng.randint(1, 7)):
        kind = rng.random()
        if kind < 0.1:
            tables.append(rng.choice((None, [])))
            continue
        t = list(rng.choice(tables) or ()) if tables and kind < 0.85 else []
        t = t[:rng.randint(0, len(t))]
        tables.append(t + [next(names) for _ in range(rng.randint(0 if t else 1, 4))])
    for least in (1, 17, 33):
        assert saved(groups_of(tables, 16, least)) == best(tables, 16, least)


def test_many_rows_are_grouped_quickly():
    tables = [list(range(i + 1)) + [1000 + i] for i in range(448)]                # each leaves the others one page later
    start = time.perf_counter()
    groups_of(tables)
    assert time.perf_counter() - start < 5.0


def test_a_server_shares_what_groups_behind_a_template_have(monkeypatch):
    from dew_b200.inference import serving
    monkeypatch.setattr(serving, "SHARED_LEAST", 32)
    template, told = list(range(1, 9)), []
    plain = KVStore.share
    monkeypatch.setattr(KVStore, "share", lambda self, *a: plain(self, *a) or told.append(sorted(self.shared.tokens.tolist())[-2:]))
    server = Server(model(), slots=8, capacity=160, kv_cache=KVCache(page_size=8), shared_prefix=True)
    got = [server.submit_group(template + [10 + 20 * g + i % 20 for i in range(41)], 3, 6) for g in range(2)]
    server.run()
    want = [alone(model(), template + [10 + 20 * g + i % 20 for i in range(41)], new=6) for g in range(2)]
    assert [t.result() for ts in got for t in ts] == [w for w in want for _ in range(3)] and [48, 48] in told


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sinks", [False, True])
def test_scores_that_are_no_numbers_show(dtype, sinks):
    a = prefix_cases.batch([(32, [1, 9, 17]), (0, [5]), (50, [3, 3])], 6, 2, 24, 16, dtype, resting=(1,))
    s = torch.randn(6, generator=torch.Generator().manual_seed(1)) if sinks else None
    live = [r for r, n in enumerate(a["lengths"].tolist()) if n]
    b, nan, zero, same = prefix_cases.numbers_that_are_none(a, live[0], live[1])
    got, was = shared_decode(**b, sinks=s), shared_decode(**a, sinks=s)
    assert bool(got[nan].isnan().all()) and not got[zero].any() and torch.equal(got[same], was[same])


# ---------------------------------------------------------------------------------------------------------- what the operators refuse
def adapter_call():
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=g)
    return make(5, 8), make(6, 8), Bank(make(2, 3, 8), make(2, 6, 3), torch.ones(2)), torch.tensor([0, -1, 1, 0, 1], dtype=torch.int32)


def test_tangents_and_transforms_are_refused():
    x, w, bank, ids = adapter_call()
    a = prefix_cases.batch([(16, [1, 2])], 4, 2, 16, 16, torch.float32)
    calls = [lambda t: adapted_linear(t(x), w, bank, ids), lambda t: adapted_linear(x, t(w), bank, ids), lambda t: adapted_linear(x, w, bank._replace(b=t(bank.b)), ids),
             lambda t: add_adapters(t(torch.zeros(5, 6)), x, bank, ids), lambda t: add_adapters(torch.zeros(5, 6), t(x), bank, ids),
             lambda t: shared_decode(**{**a, "q": t(a["q"])}), lambda t: shared_decode(**{**a, "v": t(a["v"])}), lambda t: shared_decode(**a, sinks=t(torch.zeros(4))),
             lambda t: move_pages([t(torch.zeros(2, 4, 3))], [0], [1])]
    for call in calls:
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
            call(lambda t: t)                                 # (nothing here has a tangent)
        with pytest.raises(NotImplementedError):
            torch.func.vmap(lambda by: call(lambda t: t * by))(torch.ones(2))
        with pytest.raises(NotImplementedError):
            torch.func.grad(lambda by: torch.as_tensor(call(lambda t: t * by)).sum())(torch.ones(()))
    with pytest.raises(NotImplementedError):
        move_pages([torch.zeros(2, 4, 3, requires_grad=True)], [0], [1])
    with torch.no_grad():
        move_pages([torch.zeros(2, 4, 3, requires_grad=True)], [0], [1])


def test_a_store_reads_rows_apart_under_a_tangent():
    store = KVStore(KVCache(page_size=8, pages=8), 1, 2, 32, 1, 16, dtype=torch.float32)
    store.share([[0, 1], [0, 2]])
    q, lengths = torch.randn(2, 2, 16), torch.tensor([9, 10], dtype=torch.int32)
    with torch.no_grad(), forward_ad.dual_level():
        assert store.decode_attention(0, forward_ad.make_dual(q, torch.ones_like(q)), lengths).shape == q.shape


def test_a_result_that_lies_over_what_is_read_is_refused():
    x, w, bank, ids = adapter_call()
    room = torch.zeros(200)

    def at(offset, *shape):
        return room[offset:offset + math.prod(shape)].view(shape)
    for y, mine in ((at(0, 5, 6), at(0, 5, 8)), (at(20, 5, 6), at(0, 5, 8)), (at(0, 5, 6), at(29, 5, 8)), (at(39, 5, 6), at(0, 5, 8)),
                    (at(0, 5, 6), torch.as_strided(room, (5, 8), (20, 1), 10))):
        with pytest.raises(ValueError, match="over"):
            add_adapters(y, mine, bank, ids)
    for y, mine in ((at(40, 5, 6), at(0, 5, 8)), (at(0, 5, 6), at(30, 5, 8)), (at(0, 5, 6), torch.as_strided(room, (5, 8), (20, 1), 30)), (at(0, 5, 6), at(30, 1, 8).expand(5, 8)),
                    (at(0, 0, 6), at(0, 0, 8))):
        add_adapters(y, mine, bank, ids[:len(y)])
    y = torch.zeros(5, 6)
    for i, shape in enumerate(((2, 3, 8), (2, 6, 3), (2,))):
        with pytest.raises(ValueError, match="over"):
            add_adapters(at(10, 5, 6), x, bank._replace(**{bank._fields[i]: at(39, *shape)}), ids)
    with pytest.raises(ValueError, match="over"):
        add_adapters(y, x, bank, y.view(torch.int32)[0, :5])


def test_pools_and_tables_without_a_page_are_refused():
    a = prefix_cases.batch([(16, [1, 2])], 4, 2, 16, 16, torch.float32)
    for changed in (dict(table=a["table"][:, :0].contiguous()), dict(k=a["k"][:0], v=a["v"][:0]), dict(k=a["k"][:, :0].contiguous(), v=a["v"][:, :0].contiguous())):
        with pytest.raises(ValueError, match="page"):
            shared_decode(**{**a, **changed})
        with pytest.raises(ValueError, match="page"):
            shared_decode(**{**a, **changed, "lengths": torch.zeros_like(a["lengths"])})


def test_requests_that_fail_give_their_pages_back():
    server = Server(model(), slots=4, capacity=48, kv_cache=KVCache(page_size=8))
    for _ in range(3):
        server.submit_group(PROMPTS[0], 3, 8), server.submit(PROMPTS[1], 8)
        server.step()
        server.fail(RuntimeError("stopped"))
        assert not server.ledger.refs and server.ledger.available() == server.ledger.pages
    assert server([PROMPTS[0]], 8) == [alone(model(), PROMPTS[0])]


# ---------------------------------------------------------------------------------------------------------- pages of every type
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8, torch.uint8, torch.bool, torch.float16, torch.bfloat16, torch.float64, torch.int64])
def test_pages_of_any_type_move(dtype):
    pool = (torch.arange(2 * 6 * 5).view(2, 6, 5) % 7).to(dtype)
    want = [pool[:, p].clone() for p in (0, 0, 4, 3, 4, 5)]
    move_pages([pool], [0, 4], [1, 2])
    assert all(torch.equal(pool[:, i].float(), w.float()) for i, w in enumerate(want))


def test_samples_fork_in_caches_of_every_kind():
    for kind in (None, "int8", "float8_e4m3fn"):
        server = Server(model(), slots=3, capacity=48, kv_cache=KVCache(kind, 8))
        got = server.submit_group(PROMPTS[0], 3, 6)
        while server.busy:
            server.step()
            server.compact()
        assert len({tuple(t.result()) for t in got}) == 1
        assert got[0].result() == Server(model(), slots=1, capacity=48, kv_cache=KVCache(kind, 8))([PROMPTS[0]], 6)[0]


def test_a_copy_made_inside_using_is_not_in_use():
    m = model()
    bank = random_bank(m)
    with bank.using(torch.tensor([0], dtype=torch.int32)):
        other = copy.deepcopy(m)
    assert not other.layers[0].mixer.qkv_proj.in_use
    with torch.no_grad():
        assert torch.equal(other(torch.tensor([[1, 2], [3, 4]])), m(torch.tensor([[1, 2], [3, 4]])))
