"""A server of many requests: prefixes that decode steps read once, an adapter for each request, both with rows that fork."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, KVStore
from dew_b200.nn.lora import AdaptedLinear, AdapterBank, apply_lora, lora_state, merge_all
from dew_b200.sampling.text import Sampling

CONFIG = dict(vocab_size=64, emb_features=32, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, mlp_features=48, max_seq_len=160)


def model(**kw):
    torch.manual_seed(0)
    return CausalTransformer(**{**CONFIG, **kw}).eval()


def adapter(seed, rank, targets=("qkv_proj", "o_proj", "down_proj")):
    """An adapter as training leaves it, and the model that has it merged into its weights."""
    m = model()
    apply_lora(m, targets, rank=rank, alpha=2.0 * rank)
    g = torch.Generator().manual_seed(seed)
    for n, p in m.named_parameters():
        if ".lora_b" in n:
            p.data.normal_(0.0, 0.2, generator=g)
    state = lora_state(m)
    merge_all(m)
    return state, m


def served(m, prompts, new=8, **kw):
    return Server(m, slots=len(prompts), capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False, **kw)(prompts, new)


@pytest.mark.parametrize("quantized", [None, "int8"])
@pytest.mark.parametrize("window", [None, 20])
def test_shared_prefixes_change_no_token(monkeypatch, quantized, window):
    from dew_b200.inference import serving
    from dew_b200.ops import prefix
    monkeypatch.setattr(serving, "SHARED_LEAST", 8)
    calls, plain = [], prefix.shared_decode
    monkeypatch.setattr(prefix, "shared_decode", lambda *a, **k: calls.append(a[5].tokens.max().item()) or plain(*a, **k))
    m = model(**({} if window is None else dict(window=window, layer_types=("local", "attention"))))
    system = list(range(1, 40))
    prompts = [system + [40 + i, 41] for i in range(3)] + [[5, 6, 7]]

    def run(**kw):
        server = Server(m, slots=5, capacity=160, kv_cache=KVCache(quantized, 8), **kw)
        first = server.submit(prompts[0], 10)
        for _ in range(3):
            server.step()
        tickets = [first] + [server.submit(p, 10) for p in prompts[1:]] + server.submit_group(system + [50], 3, 6)
        server.run()
        return [t.result() for t in tickets]
    want = run()
    assert not calls
    assert run(shared_prefix=True) == want and max(calls) >= 32


def test_a_store_knows_its_groups():
    store = KVStore(KVCache(page_size=8, pages=20), 1, 4, 64, 1, 16, dtype=torch.float32)
    store.share([[1, 2, 3], None, [1, 2, 4], [5]])
    order, first, tokens = (t.tolist() for t in store.shared)
    assert order[:2] == [0, 2] and first[:2] == [0, 2] and tokens[0] == 16
    before = store.shared.tokens.data_ptr()
    store.share([None] * 4)
    assert store.shared.tokens.data_ptr() == before and not store.shared.tokens.any()
    with pytest.raises(ValueError):
        store.share([None])
    store.share(None)
    assert store.shared is None


def test_every_request_has_its_adapter():
    (one, merged_one), (two, merged_two) = adapter(1, 4), adapter(2, 3, ("qkv_proj",))
    m = model()
    plain = model()
    bank = AdapterBank(m, ("qkv_proj", "o_proj", "down_proj"), slots=3, rank=4)
    assert len(bank.layers) == 6 and all(isinstance(x, AdaptedLinear) for x in bank.layers.values())
    bank.load("one", one, alpha=8.0)
    bank.load("two", two, alpha=6.0)
    prompts = [list(range(3, 25)), list(range(3, 25)), [9, 8, 7], [1, 2, 3, 4]]
    names = ["one", "two", None, "one"]
    want = [served(x, [p])[0] for x, p in zip((merged_one, merged_two, plain, merged_one), prompts)]
    server = Server(m, slots=3, capacity=160, kv_cache=KVCache(page_size=8), adapters=bank)
    tickets = [server.submit(p, 8, adapter=n) for p, n in zip(prompts, names)]
    assert bank.holds["one"] == 2
    with pytest.raises(RuntimeError):
        bank.load("one", two, alpha=1.0)
    with pytest.raises(RuntimeError):
        bank.remove("two")
    server.run()
    assert [t.result() for t in tickets] == want and not any(bank.holds.values())
    # the same prompt again: pages of another adapter, or of none, are not its prefix
    hits = server.ledger.hits
    again = [server.submit(prompts[0], 8, adapter=n) for n in ("two", None)]
    server.run()
    assert again[0].result() == want[1] and again[1].result() == served(plain, [prompts[0]])[0] and server.ledger.hits == hits + 2
    # an adapter that takes a name over has pages of its own
    bank.load("one", two, alpha=6.0)
    other = server.submit(prompts[0], 8, adapter="one")
    server.run()
    assert other.result() == want[1] and server.ledger.hits == hits + 2
    bank.remove("one")
    with pytest.raises(KeyError):
        server.submit(prompts[0], 8, adapter="one")
    group = server.submit_group(prompts[0], 3, 8, adapter="two")
    assert bank.holds["two"] == 3
    server.run()
    assert [t.result() for t in group] == [want[1]] * 3 and not bank.holds["two"]
    waiting = server.submit_group([1, 2, 3], 3, 2, adapter="two")
    server.fail(RuntimeError("stopped"))
    assert not bank.holds["two"] and all(t.done for t in waiting)
    with pytest.raises(ValueError):
        Server(plain, slots=1, capacity=32).submit([1, 2], 2, adapter="one")


def test_what_a_bank_refuses():
    state, _ = adapter(1, 4)
    m = model()
    with pytest.raises(ValueError):
        AdapterBank(m, ("nothing",))
    for bad in (dict(slots=0), dict(rank=0)):
        with pytest.raises(ValueError):
            AdapterBank(model(), **bad)
    bank = AdapterBank(m, ("qkv_proj", "o_proj", "down_proj"), slots=1, rank=4)
    with pytest.raises(KeyError):
        bank.load("x", {"layers.9.mixer.qkv_proj.lora_a": torch.zeros(4, 32)}, 1.0)
    with pytest.raises(KeyError):
        bank.load("x", {k.replace("lora_b", "magnitude"): v for k, v in state.items()}, 1.0)
    key = next(k for k in state if k.endswith("lora_a"))
    for bad in (state[key][:, :8], torch.zeros(5, state[key].shape[1]), state[key][0]):
        with pytest.raises(ValueError):
            bank.load("x", {**state, key: bad}, 1.0)
    with pytest.raises(ValueError):
        bank.load("x", {k: v for k, v in state.items() if k != key}, 1.0)
    assert not bank.names and all(not layer.a.any() for layer in bank.layers.values())
    assert bank.load("x", state, 1.0, rs=True) == 0 and float(next(iter(bank.layers.values())).scale[0]) == 0.5
    with pytest.raises(RuntimeError):
        bank.load("y", state, 1.0)
    with pytest.raises(TypeError):
        with bank.using(torch.zeros(2)):
            pass
    with bank.using(torch.tensor([0, -1], dtype=torch.int32)), torch.no_grad():
        got = m(torch.tensor([[1, 2, 3], [1, 2, 3]]))
        with pytest.raises(ValueError):
            m(torch.tensor([[1, 2, 3]]))
    with torch.no_grad():
        base = m(torch.tensor([[1, 2, 3]]))[0]
        assert torch.allclose(got[1], base, atol=1e-6) and not torch.allclose(got[0], base, atol=1e-3)
    with bank.using(torch.tensor([0, -1], dtype=torch.int32)):
        with pytest.raises(NotImplementedError):
            m(torch.tensor([[1, 2, 3], [1, 2, 3]]))


def test_samples_with_adapters_over_shared_prefixes(monkeypatch):
    from dew_b200.inference import serving
    monkeypatch.setattr(serving, "SHARED_LEAST", 8)
    state, merged = adapter(3, 4)
    m = model()
    bank = AdapterBank(m, ("qkv_proj", "o_proj", "down_proj"), slots=2, rank=4)
    bank.load("x", state, alpha=8.0)
    prompt, sampling = list(range(2, 33)), Sampling(temperature=1.0)
    alone = Server(merged, slots=4, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False, sampling=sampling)
    want = [alone.submit(prompt, 9, key=k) for k in range(4)]
    alone.run()
    server = Server(m, slots=6, capacity=160, kv_cache=KVCache(page_size=8), sampling=sampling, shared_prefix=True, adapters=bank)
    other = server.submit(prompt, 5, key=7)
    got = server.submit_group(prompt, 4, 9, adapter="x")
    while server.busy:
        server.step()
        server.compact()
    assert [t.result() for t in got] == [t.result() for t in want] and len(other.result()) == 5


def test_a_later_chunk_may_end_in_padding():
    """A chunk behind a cached prefix, padded as a server pads it: its tokens see what they see without the padding."""
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn(2, 30, n, 16, generator=g) for n in (2, 2, 4))

    def chunks(pad):
        store = KVStore(KVCache(page_size=8), 1, 2, 64, 2, 16, dtype=torch.float32)
        out = []
        for a, b in ((0, 17), (17, 30)):
            x = [torch.cat([t[:, a:b], torch.randn(2, pad, *t.shape[2:], generator=g)], 1) for t in (q, k, v)]
            pos = torch.cat([torch.arange(a, b), torch.full((pad,), -1)])[None].expand(2, -1)
            store.chunk_span = (a, b)
            out.append(store.attend(0, *x, pos)[:, :b - a])
        return torch.cat(out, 1)
    want = chunks(0)
    assert torch.allclose(chunks(5), want, atol=1e-6) and torch.allclose(chunks(40), want, atol=1e-6)
