"""Decoders of state space layers where a call is unusual: caches in pieces, caches without a place for a state, packed documents, other types, options of a store."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache
from dew_b200.nn.linear_attention import RecurrentCache, ShortConv
from dew_b200.ops import scan
from dew_b200.sampling.text import Sampling, generate, make_cache
from selective_cases import draws_of_its_own  # noqa: F401
from test_state_space_models import OPTIONS, model


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


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_a_cache_without_a_place_for_a_state_is_refused(kind):
    """State space layers between attention layers that turn by the model's tables: their store has keys alone.  A cache of states around it serves them."""
    m = model(kind, num_heads=4, layer_types=(kind, "attention"), layer_mlp=None, mlp_features=96, num_layers=2)
    assert m.cache_slots() is None
    with pytest.raises(NotImplementedError, match="no place for its state"):
        generate(m, None, [[3, 4, 5]], 4, sampling=Sampling(temperature=0.0))
    with pytest.raises(NotImplementedError, match="no place for its state"):
        Server(m, slots=2, capacity=64, sampling=Sampling(temperature=0.0))([[3, 4, 5]], 4)
    tokens = torch.randint(1, 97, (2, 20))
    cache, got = RecurrentCache(make_cache(m, 2, 64)), []
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
