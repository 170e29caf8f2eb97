"""Decoders of state space layers where a call is unusual: caches in pieces, caches without a place for a state, packed documents, other types, options of a store."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, KVStore
from dew_b200.nn.linear_attention import RecurrentCache, ShortConv
from dew_b200.ops import scan
from dew_b200.sampling.text import RowBatch, Sampling, generate, make_cache
from selective_cases import draws_of_its_own  # noqa: F401
from test_state_space_models import OPTIONS, greedy, model, prompts


# a piece in front and behind, pieces shorter than the three inputs that a convolution of four taps keeps, single tokens between them
@pytest.mark.parametrize("pieces", [(20, 20), (6, 6, 28), (1, 2, 2, 1, 34), (2, 1, 3, 4, 30), (39, 1)])
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_the_plain_cache_in_pieces(kind, pieces):
    m = model(kind)
    tokens = torch.randint(1, 97, (2, 40))
    cache, got, at = RecurrentCache(make_cache(m, 2, 64)), [], 0
    with torch.no_grad():
        want = m(tokens)
        for n in pieces:
            got.append(m(tokens[:, at:at + n], positions=torch.arange(at, at + n)[None].expand(2, n), cache=cache))
            at += n
    assert torch.allclose(torch.cat(got, 1), want, atol=1e-4)


@pytest.mark.parametrize("taps", [1, 2, 4, 7])
def test_a_convolution_goes_on_from_its_last_inputs(taps):
    conv, x = ShortConv(6, taps, bias=True), torch.randn(2, 30, 6)
    with torch.no_grad():
        want, kept, got = conv(x), torch.zeros(2, taps - 1, 6), []
        for lo, hi in ((0, 9), (9, 10), (10, 12), (12, 15), (15, 30)):
            got.append(conv(x[:, lo:hi], cache=kept))
            assert torch.equal(kept, torch.cat([torch.zeros(2, taps, 6), x[:, :hi]], 1)[:, taps + hi - (taps - 1):])
        assert torch.allclose(torch.cat(got, 1), want, atol=1e-6)
        # documents packed into a row: what was kept belongs to the first of them
        segments = torch.tensor([[0] * 5 + [1] * 10] * 2)
        again = conv(x[:, 15:], segments, x[:, 15 - (taps - 1):15].clone())
        assert torch.allclose(again, torch.cat([conv(x[:, :20])[:, 15:], conv(x[:, 20:])], 1), atol=1e-6)


def beside(left, right):
    """Two mixers in every layer."""
    sides = {"mamba2": ("mamba2", dict(mixer_options=OPTIONS["mamba2"])), "mamba": ("mamba", dict(mixer_options=OPTIONS["mamba"])), "nope": ("nope", {})}
    return CausalTransformer(vocab_size=97, emb_features=64, num_layers=2, num_heads=4, num_kv_heads=2, max_seq_len=512, mlp_features=96, layer_types=("pair",), fp32_residual=True,
                             mixer_options=dict(left=sides[left], right=sides[right]), dtype=torch.float32).eval()


@pytest.mark.parametrize("left,right", [("mamba2", "nope"), ("nope", "mamba2"), ("mamba2", "mamba"), ("nope", "nope")])
def test_keys_beside_states_are_asked_for_in_the_type_that_they_are_kept_in(left, right):
    """Keys in fewer bits are refused wherever there are keys, on either side of a layer; where there are none, nobody misses them."""
    m = beside(left, right)
    assert make_cache(m, 2, 64).pools() or "nope" not in (left, right)
    for kind in ("int8", "float8_e4m3fn"):
        if "nope" in (left, right):
            with pytest.raises(NotImplementedError, match="quantised"):
                make_cache(m, 2, 64, KVCache(quantized=kind))
        else:
            assert not make_cache(m, 2, 64, KVCache(quantized=kind)).pools()


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_packed_documents_and_a_state_are_refused(kind):
    """A slot's state stands for one row: it would run from a document into the next."""
    m = model(kind)
    layer, store, x = m.layers[0].mixer, make_cache(m, 2, 64), torch.randn(2, 9, 64)
    at, segments = torch.arange(9)[None].expand(2, 9), torch.tensor([[0] * 4 + [1] * 5] * 2)
    before = [t.clone() for t in store.kept_states()]
    with pytest.raises(NotImplementedError, match="packed"):
        layer(x, segments, store, 0, positions=at)
    assert all(torch.equal(a, b) for a, b in zip(before, store.kept_states()))
    with torch.no_grad():
        assert torch.allclose(layer(x, None, store, 0, positions=at), layer(x), atol=1e-5)


def between_attention(kind, device="cpu", **more):
    """State space layers between attention layers that turn by the model's tables: one shape of keys for all, states beside."""
    return model(kind, device, **{**dict(num_heads=4, num_kv_heads=2, layer_types=(kind, "attention", kind), layer_mlp=None, mlp_features=96, num_layers=3), **more})


def generates(m):
    """As the whole row again for every token: in one batch, through a server's chunks, slots that are used again and forks."""
    asked = prompts()
    want = [greedy(m, p, 6) for p in asked]
    assert m.cache_slots() is None
    store = make_cache(m, 2, 64)
    assert store.keeps_state and [store.holds(i) for i in range(4)] == [True, False, True, False] and len(store.kept_states()) == 4
    out = generate(m, None, asked, 6, sampling=Sampling(temperature=0.0))
    assert [out.tokens[r, len(p):len(p) + 6].tolist() for r, p in enumerate(asked)] == want
    for spec in (None, KVCache(page_size=16)):
        server = Server(m, slots=2, capacity=256, chunk=32, kv_cache=spec, sampling=Sampling(temperature=0.0))
        assert server(asked, 6) == want and server(asked[::-1], 6) == want[::-1]
        group = server.submit_group(asked[0], 2, 6)
        server.run()
        assert [t.result() for t in group] == [want[0], want[0]]


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_between_attention_layers(kind):
    generates(between_attention(kind))


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_pieces_between_attention_layers(kind):
    """Prompts of their own lengths, then a token at a time with rows that rest; chunks that begin together; from the first token on also without positions."""
    m = between_attention(kind)
    tokens = torch.randint(1, 97, (3, 24))
    batch, at = RowBatch(m, 3, 64), [7, 12, 1]
    with torch.no_grad():
        want = m(tokens)
        got = batch.prefill(tokens[:, :12], torch.tensor(at))
        assert torch.allclose(got, want[[0, 1, 2], [6, 11, 0]], atol=1e-4)
        for step in [(1, 0, 1), (1, 1, 1), (0, 1, 0), (1, 1, 1)]:
            pos = torch.tensor([a if n else -1 for a, n in zip(at, step)])
            out = batch.forward(tokens.gather(1, pos.clamp_min(0)[:, None]), pos[:, None])[:, 0]
            for r, n in enumerate(step):
                assert not n or torch.allclose(out[r], want[r, at[r]], atol=1e-4), (r, at[r])
                at[r] += n
        store = make_cache(m, 3, 64)
        assert torch.allclose(m(tokens[:, :11], cache=store), want[:, :11], atol=1e-4)
        for lo, hi in ((11, 18), (18, 20), (20, 21), (21, 24)):
            assert torch.allclose(m(tokens[:, lo:hi], positions=torch.arange(lo, hi)[None].expand(3, hi - lo), cache=store), want[:, lo:hi], atol=1e-4)


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_a_cache_without_a_place_for_a_state_is_refused(kind):
    """A store of keys alone.  A cache of states around it serves such a stack, in any pieces."""
    m = between_attention(kind)
    bare = KVStore(KVCache(), 3, 2, 64, 2, 16, torch.float32, "cpu")
    tokens = torch.randint(1, 97, (2, 20))
    with pytest.raises(NotImplementedError, match="no place for its state"):
        m(tokens, positions=torch.arange(20)[None].expand(2, 20), cache=bare)
    cache, got = RecurrentCache(bare), []
    with torch.no_grad():
        for lo, hi in ((0, 9), (9, 16), (16, 17), (17, 20)):
            got.append(m(tokens[:, lo:hi], positions=torch.arange(lo, hi)[None].expand(2, hi - lo), cache=cache))
        assert torch.allclose(torch.cat(got, 1), m(tokens), atol=1e-4)


def test_states_without_memory_in_the_plain_form():
    """Rates of minus infinity: what a token leaves is gone at the next."""
    x, dt, b, c = torch.randn(2, 70, 5), torch.rand(2, 70, 5) + 0.1, torch.randn(2, 70, 3), torch.randn(2, 70, 3)
    a, initial = torch.full((5, 3), -float("inf")), torch.randn(2, 5, 3)
    leaves = [t.requires_grad_() for t in (x, dt, a, b, c)]
    y, last = scan.selective_scan(*leaves, initial_state=initial)
    state = (dt * x).unsqueeze(-1) * b.unsqueeze(2)
    assert torch.allclose(y, (state * c.unsqueeze(2)).sum(-1), atol=1e-5) and torch.allclose(last, state[:, -1], atol=1e-6)
    assert all(g.isfinite().all() for g in torch.autograd.grad(y.sum() + last.sum(), leaves))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_between_attention_layers_on_a_gpu(kind):
    """fp32 weights, the same tokens as on the CPU."""
    m, asked = between_attention(kind), prompts()
    want = [greedy(m, p, 8) for p in asked]
    m = m.cuda()
    out = generate(m, None, asked, 8, sampling=Sampling(temperature=0.0))
    assert [out.tokens[r, len(p):len(p) + 8].tolist() for r, p in enumerate(asked)] == want
    server = Server(m, slots=3, capacity=256, chunk=64, kv_cache=KVCache(page_size=64), sampling=Sampling(temperature=0.0))
    assert server(asked, 8) == want and server(asked[::-1], 8) == want[::-1]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_steps_between_attention_layers_in_bf16(kind):
    """Widths that the kernels of attention and of chunks take: as near to fp32 as the whole row in bf16 is; a server's captured steps are its steps."""
    more = dict(emb_features=256, num_heads=4, num_kv_heads=2, mixer_options=dict(state_dim=128, head_dim=64, groups=1) if kind == "mamba2" else {})
    m32, m = between_attention(kind, "cuda", **more), between_attention(kind, "cuda", **more).to(torch.bfloat16)
    m32.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    rows = torch.randint(1, 97, (3, 160), device="cuda")
    batch, pos = RowBatch(m, 3, 256), torch.arange(160, device="cuda")[None].expand(3, -1)
    with torch.no_grad():
        exact, whole = m32(rows), m(rows).float()
        steps = torch.cat([batch.forward(rows[:, :128], pos[:, :128], (0, 128))] + [batch.forward(rows[:, t:t + 1], pos[:, t:t + 1]) for t in range(128, 160)], 1).float()
    far = lambda a: float((a - exact).norm() / exact.norm())
    assert far(steps) < 2 * far(whole) + 1e-3 and far(whole) < 0.1
    plain, graph = (Server(m, slots=2, capacity=256, chunk=64, kv_cache=KVCache(page_size=64), sampling=Sampling(temperature=0.0), cuda_graph=g)(prompts(), 8) for g in (False, True))
    assert plain == graph


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_the_plain_cache_in_pieces_in_bf16(kind):
    """As near to fp32 as the whole row in bf16 is."""
    more = dict(mixer_options=dict(state_dim=128, head_dim=64, groups=1)) if kind == "mamba2" else {}
    m32, m = model(kind, "cuda", **more), model(kind, "cuda", **more).to(torch.bfloat16)
    m32.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    tokens = torch.randint(1, 97, (3, 160), device="cuda")
    cache, got, at = RecurrentCache(make_cache(m, 3, 256)), [], 0
    with torch.no_grad():
        exact, whole = m32(tokens), m(tokens).float()
        for n in (70, 2, 1, 67, 20):
            got.append(m(tokens[:, at:at + n], positions=torch.arange(at, at + n, device="cuda")[None].expand(3, n), cache=cache).float())
            at += n
    far = lambda a: float((a - exact).norm() / exact.norm())
    assert far(torch.cat(got, 1)) < 2 * far(whole) + 1e-3 and far(whole) < 0.1
