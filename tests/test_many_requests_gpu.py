"""A server of many requests on the GPU: prefixes that decode steps read once, an adapter for each request, rows that fork, with and without a captured step."""
import pytest
import torch

from dew_b200.inference import serving
from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, KVStore
from dew_b200.nn.lora import AdapterBank, apply_lora, lora_state, merge_all
from dew_b200.ops import adapters, library as L, prefix
from prefix_cases import allowed, truth

pytestmark = pytest.mark.gpu
DEV = "cuda"
CONFIG = dict(vocab_size=96, emb_features=128, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64, mlp_features=256, max_seq_len=256)
TARGETS = ("qkv_proj", "o_proj", "down_proj")


def model(dtype):
    torch.manual_seed(0)
    return CausalTransformer(**CONFIG).eval().to(DEV, dtype)


def adapter(seed, rank, dtype):
    """An adapter as training leaves it, and the model that has it merged into its weights."""
    m = model(torch.float32)
    apply_lora(m, TARGETS, rank=rank, alpha=2.0 * rank)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for n, p in m.named_parameters():
        if ".lora_b" in n:
            p.data.normal_(0.0, 0.1, generator=g)
    state = lora_state(m)
    merge_all(m)
    return {k: v.to(dtype) for k, v in state.items()}, m.to(dtype)


SYSTEM = [5 + i % 80 for i in range(75)]


def run(m, bank, graph, calls=None, page=16):
    """Requests that come, fork, compact and go; their tokens."""
    server = Server(m, slots=9, capacity=256, kv_cache=KVCache(page_size=page), cuda_graph=graph, shared_prefix=True, adapters=bank)
    first = server.submit(SYSTEM + [1, 2], 14, adapter="one")
    for _ in range(3):
        server.step()
    rest = [server.submit(SYSTEM + [3 + i], 12, adapter=n) for i, n in enumerate(("one", None, "two"))] + server.submit_group(SYSTEM + [9], 3, 10, adapter="one")
    steps = 0
    while server.busy:
        server.step()
        steps += 1
        if steps % 5 == 0:
            server.compact()
    L.check_status()
    return [t.result() for t in (first, *rest)]


@pytest.mark.parametrize("graph", [False, True])
def test_tokens_are_those_of_requests_alone(monkeypatch, graph):
    monkeypatch.setattr(serving, "SHARED_LEAST", 32)
    dtype = torch.float32
    (one, merged_one), (two, merged_two) = adapter(1, 8, dtype), adapter(2, 4, dtype)
    m, plain = model(dtype), model(dtype)
    bank = AdapterBank(m, TARGETS, slots=3, rank=8)
    bank.load("one", one, alpha=16.0)
    bank.load("two", two, alpha=8.0)

    def alone(x, prompt, n):
        return Server(x, slots=1, capacity=256, kv_cache=KVCache(page_size=16), prefix_cache=False)([prompt], n)[0]
    want = [alone(merged_one, SYSTEM + [1, 2], 14)] + [alone(x, SYSTEM + [3 + i], 12) for i, x in enumerate((merged_one, plain, merged_two))] + [alone(merged_one, SYSTEM + [9], 10)] * 3
    assert run(m, bank, graph) == want


def test_a_captured_step_is_the_eager_one(monkeypatch):
    """In bf16, where the tensor cores' kernels run: the same kernels on the same numbers."""
    monkeypatch.setattr(serving, "SHARED_LEAST", 32)
    dtype = torch.bfloat16
    (one, _), (two, _) = adapter(1, 8, dtype), adapter(2, 4, dtype)
    m = model(dtype)
    bank = AdapterBank(m, TARGETS, slots=3, rank=8)
    bank.load("one", one, alpha=16.0)
    bank.load("two", two, alpha=8.0)
    shared, added = [], []
    plain, plain_add = prefix.shared_decode, adapters._add
    monkeypatch.setattr(prefix, "shared_decode", lambda *a, **k: shared.append(prefix.on_tensor_cores(a[0], a[1], a[2], a[3].shape[1], 9)) or plain(*a, **k))
    monkeypatch.setattr(adapters, "_add", lambda *a: added.append(1) or plain_add(*a))
    eager = run(m, bank, False)
    assert shared and all(shared) and added
    assert run(m, bank, True) == eager == run(m, bank, False)


@pytest.mark.parametrize("quantized, page, dim, taken", [(None, 16, 64, True), (None, 64, 128, True), ("int8", 16, 64, False), (None, 8, 64, False), (None, 16, 80, False)])
def test_a_store_reads_shared_pages_once_where_that_is_sooner(monkeypatch, quantized, page, dim, taken):
    rows, G, H, n = 5, 2, 4, 160
    store = KVStore(KVCache(quantized, page, pages=rows * 256 // page), 2, rows, 256, G, dim, dtype=torch.bfloat16, device=DEV)
    each = 256 // page
    tables = [list(range(r * each, (r + 1) * each)) for r in range(rows)]
    tables[1][:96 // page] = tables[0][:96 // page]
    tables[3][:96 // page] = tables[0][:96 // page]
    store.page_table.copy_(torch.tensor(tables, dtype=torch.int32))
    g = torch.Generator(device=DEV).manual_seed(3)
    for t in (store.k, store.v):
        t.copy_(torch.randn(t.shape, device=DEV, generator=g) * (20 if quantized else 1))
    if quantized:
        store.k_scale.fill_(0.05), store.v_scale.fill_(0.05)
    q = torch.randn(rows, H, dim, device=DEV, generator=g).bfloat16()
    lengths = torch.tensor([n, 97, 0, 130, 40], device=DEV, dtype=torch.int32)
    calls, plain = [], prefix.shared_decode
    monkeypatch.setattr(prefix, "shared_decode", lambda *a, **k: calls.append(1) or plain(*a, **k))
    with torch.no_grad():
        apart = store.decode_attention(1, q, lengths)
        assert not calls
        store.share(tables, 64)
        got = store.decode_attention(1, q, lengths)
    assert bool(calls) == taken
    if not taken:
        assert torch.equal(got, apart)
        return
    a = dict(q=q, k=store.k[1], v=store.v[1], table=store.page_table, lengths=lengths, shared=store.shared, scale=dim ** -0.5)
    found = truth(a, None, 0.0, None)
    assert float(((got.double().cpu() - found[0]).abs() / allowed(a, found)).max()) <= 1.0
    L.check_status()


def test_two_streams_and_two_graphs_at_once():
    """Two captured steps of one model's operators, replayed side by side on two streams, give what each gives alone: no scratch is shared."""
    g = torch.Generator(device=DEV).manual_seed(5)
    T, n, rank, width, out = 700, 6, 16, 256, 512
    bank = adapters.Bank(torch.randn(n, rank, width, device=DEV, generator=g).bfloat16() * 0.1, torch.randn(n, out, rank, device=DEV, generator=g).bfloat16() * 0.1, torch.ones(n, device=DEV))
    w = torch.randn(out, width, device=DEV, generator=g).bfloat16() * 0.05
    rows, H, G, D, page = 40, 8, 2, 128, 64
    k, v = (torch.randn(200, page, G, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    table = torch.arange(rows, device=DEV, dtype=torch.int32)[:, None] * 4 + torch.arange(4, device=DEV, dtype=torch.int32)
    table[:, :2] = table[0, :2]
    order, first, tokens = prefix.group_rows(table.tolist(), page)
    shared = prefix.Shared(*(torch.tensor(x, device=DEV, dtype=torch.int32) for x in (order, first, tokens)))
    lengths = torch.randint(130, 256, (rows,), device=DEV, generator=g).int()
    sides = []
    for _ in range(2):
        x, ids = torch.randn(T, width, device=DEV, generator=g).bfloat16(), torch.randint(-1, n, (T,), device=DEV, generator=g).int()
        q = torch.randn(rows, H, D, device=DEV, generator=g).bfloat16()

        def step(x=x, ids=ids, q=q):
            return [adapters.adapted_linear(x, w, bank, ids), adapters.adapted_linear(x[:30], w, bank, ids[:30]),
                    prefix.shared_decode(q, k, v, table, lengths, shared, D ** -0.5)]
        with torch.no_grad():
            want = [t.clone() for t in step()]
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step()
        sides.append((want, graph, got, torch.cuda.Stream(), step))          # (which holds the inputs)
    for _ in range(5):
        for _, graph, _, stream, _ in sides:
            with torch.cuda.stream(stream):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for want, _, got, _, _ in sides:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    L.check_status()
