"""Decoders of state space layers: a prompt and its tokens one by one against the whole row, generation, the server with forks and a captured step, training."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache
from dew_b200.nn.linear_attention import RecurrentCache
from dew_b200.ops import token_mix
from dew_b200.sampling.text import RowBatch, Sampling, generate, make_cache
from selective_cases import draws_of_its_own  # noqa: F401

OPTIONS = {"mamba": dict(state_dim=16), "mamba2": dict(state_dim=16, head_dim=16, groups=2)}


def model(kind, device="cpu", dtype=torch.float32, seed=0, **more):
    torch.manual_seed(seed)
    options = dict(OPTIONS[kind], **more.pop("mixer_options", {}))
    m = CausalTransformer(**{**dict(vocab_size=97, emb_features=64, num_layers=3, num_heads=1, max_seq_len=512, layer_types=(kind,), layer_mlp=(False,), mixer_options=options), **more},
                          dtype=dtype).eval()
    for n, p in m.named_parameters():
        if p.dim() == 1 or "conv" in n:
            p.data.add_(0.1 * torch.randn_like(p))
    return m.to(device)


def prompts(n=3, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, 97, (k,), generator=g).tolist() for k in (17, 5, 140)[:n]]


def greedy(m, prompt, n):
    """The whole row again for every token."""
    ids = list(prompt)
    device = next(m.parameters()).device
    with torch.no_grad():
        for _ in range(n):
            ids.append(int(m(torch.tensor([ids], device=device))[0, -1].float().argmax()))
    return ids[len(prompt):]


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_pieces_of_rows_are_the_rows(kind):
    """Rows that come in pieces of their own lengths, one that rests, one that is released and starts anew."""
    m = model(kind)
    batch = RowBatch(m, 3, 64)
    assert batch.store.slots is not None and batch.store.keeps_state and not batch.store.pools()
    rows = [torch.randint(1, 97, (30,)).tolist() for _ in range(3)]
    pieces = [(7, 0, 1), (1, 12, 1), (1, 1, 0), (20, 1, 9)]
    at, got = [0, 0, 0], [[], [], []]
    for piece in pieces:
        out = batch.feed([rows[r][at[r]:at[r] + n] for r, n in enumerate(piece)], [list(range(n)) for n in piece])
        for r, n in enumerate(piece):
            got[r].append(out[:n])
            out = out[n:]
            at[r] += n
    with torch.no_grad():
        for r in range(3):
            want = m(torch.tensor([rows[r][:at[r]]]))[0]
            assert torch.allclose(torch.cat(got[r]), want, atol=1e-4), r
    batch.release(1)
    again = batch.feed([[], rows[1][:4], []], [[], [0, 1, 2, 3], []])
    assert torch.allclose(again, got[1][1][:4], atol=1e-4)


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_generation_and_server(kind):
    m = model(kind)
    asked = prompts()
    want = [greedy(m, p, 6) for p in asked]
    out = generate(m, None, asked, 6, sampling=Sampling(temperature=0.0))
    assert [out.tokens[r, len(p):len(p) + 6].tolist() for r, p in enumerate(asked)] == want
    server = Server(m, slots=2, capacity=256, chunk=32, sampling=Sampling(temperature=0.0))
    assert server(asked, 6) == want                          # (three requests on two slots: a slot's state starts from nothing again)
    group = server.submit_group(asked[0], 2, 6)
    server.run()
    assert [t.result() for t in group] == [want[0], want[0]]


def test_options_that_concern_pages_alone():
    """A server of states has no pages to quantise, share or keep on the host; it is asked for them all the same, as one of keys would be."""
    m = model("mamba")
    asked = prompts(2)
    server = Server(m, slots=2, capacity=256, kv_cache=KVCache(quantized="int8", page_size=16), host_pages=8, shared_prefix=True, sampling=Sampling(temperature=0.0))
    assert server(asked, 4) == [greedy(m, p, 4) for p in asked]
    server.compact()
    server.resize(40)
    assert server(asked, 4) == [greedy(m, p, 4) for p in asked]


@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_the_plain_cache_of_recurrent_layers(kind):
    m = model(kind)
    tokens = torch.randint(1, 97, (2, 12))
    with torch.no_grad():
        want = m(tokens)
        cache = RecurrentCache(make_cache(m, 2, 32))
        got = [m(tokens[:, :8], positions=torch.arange(8)[None].expand(2, 8), cache=cache)]
        got += [m(tokens[:, t:t + 1], positions=torch.full((2, 1), t), cache=cache) for t in range(8, 12)]
    assert torch.allclose(torch.cat(got, 1), want, atol=1e-4)


def test_beside_attention_over_an_fp32_residual():
    """State space layers between attention layers that carry their own rotation."""
    m = model("mamba2", num_heads=4, num_kv_heads=2, layer_types=("mamba2", "mamba2", "attention"), layer_mlp=None, mlp_features=96, fp32_residual=True,
              rotation=dict(dims=16))
    rows = [torch.randint(1, 97, (20,)).tolist() for _ in range(2)]
    batch = RowBatch(m, 2, 64)
    out = [batch.feed([r[:9] for r in rows], [[8], [8]])] + [batch.feed([[r[t]] for r in rows], [[0], [0]]) for t in range(9, 20)]
    with torch.no_grad():
        want = m(torch.tensor(rows))[:, 8:].transpose(0, 1)
    assert torch.allclose(torch.stack(out), want, atol=2e-4)


def test_positions_are_counted_where_none_are_given():
    m = model("mamba")
    tokens = torch.randint(1, 97, (2, 9))
    store = make_cache(m, 2, 32)
    with torch.no_grad():
        got, want = m(tokens, cache=store), m(tokens)
        more = m(tokens[:, :1], positions=torch.full((2, 1), 9), cache=store)
        assert torch.allclose(got, want, atol=1e-4) and torch.allclose(more, m(torch.cat([tokens, tokens[:, :1]], 1))[:, -1:], atol=1e-4)


@pytest.mark.parametrize("silu", [False, True])
def test_convolution_with_an_offset(silu, device="cpu", dtype=torch.float32):
    x, w, b, add = (torch.randn(*s, device=device).to(dtype) for s in ((2, 9, 8), (8, 4), (8,), (8,)))
    got = token_mix.conv_tokens(x, w, b, silu, None, None, add)
    state = torch.zeros(2, 8, 3, device=device)
    whole = token_mix.whole(2, 9, device)
    parts = [token_mix.conv_tokens(x[:, lo:hi], w, b, silu, token_mix.Rows(whole.positions[:, lo:hi].contiguous(), torch.full_like(whole.lengths, hi)), state, add)
             for lo, hi in ((0, 5), (5, 6), (6, 9))]
    u = torch.nn.functional.pad((x + b).double(), (0, 0, 3, 0))
    want = sum(u[:, j:j + 9] * w[:, j].double() for j in range(4)) + add.double()
    want = want * torch.sigmoid(want) if silu else want
    close = dict(atol=1e-5, rtol=1e-5) if dtype is torch.float32 else dict(atol=0.05, rtol=2.0 ** -7)      # (x + b is rounded to bf16 in the formula here, by up to 2^-7 at 4)
    assert torch.allclose(got.double(), want, **close) and torch.allclose(torch.cat(parts, 1).double(), want, **close)


@pytest.mark.parametrize("add", [torch.zeros(7), torch.zeros(1, 8), torch.zeros(8, device="meta")])
def test_offsets_that_a_convolution_refuses(add):
    with pytest.raises(ValueError, match="offset"):
        token_mix.conv_tokens(torch.zeros(2, 9, 8), torch.zeros(8, 4), None, False, None, None, add)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_convolution_with_an_offset_gpu(dtype):
    for silu in (False, True):
        test_convolution_with_an_offset(silu, "cuda", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_server_on_a_gpu(kind, graph):
    """fp32 weights: the same tokens as the whole row on the CPU, through prompts in chunks, forks and (captured) steps."""
    m = model(kind)
    asked = prompts()
    want = [greedy(m, p, 8) for p in asked]
    server = Server(m.cuda(), slots=3, capacity=256, chunk=64, kv_cache=KVCache(page_size=64), sampling=Sampling(temperature=0.0), cuda_graph=graph)
    assert server(asked, 8) == want
    group = server.submit_group(asked[1], 2, 8)
    server.run()
    assert [t.result() for t in group] == [want[1], want[1]] and server(asked[::-1], 8) == want[::-1]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_steps_in_bf16(kind):
    """A prompt and its tokens one by one in bf16 give the whole row's logits as near as the whole row is to fp32's."""
    more = dict(mixer_options=dict(state_dim=128, head_dim=64, groups=1)) if kind == "mamba2" else {}
    m32 = model(kind, "cuda", **more)
    m = model(kind, "cuda", **more).to(torch.bfloat16)
    m32.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    rows = torch.randint(1, 97, (3, 160), device="cuda")
    batch = RowBatch(m, 3, 256)
    pos = torch.arange(160, device="cuda")[None].expand(3, -1)
    with torch.no_grad():
        exact, whole = m32(rows), m(rows).float()
        steps = torch.cat([batch.forward(rows[:, :128], pos[:, :128], (0, 128))] + [batch.forward(rows[:, t:t + 1], pos[:, t:t + 1]) for t in range(128, 160)], 1).float()
    far = lambda a: float((a - exact).norm() / exact.norm())
    assert far(steps) < 2 * far(whole) + 1e-3 and far(whole) < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(OPTIONS))
def test_gradients_of_a_model(kind):
    """On the kernels and on the CPU, in fp32."""
    m = model(kind)
    tokens = torch.randint(1, 97, (2, 70))
    grads = []
    for device in ("cpu", "cuda"):
        m = m.to(device)
        m.zero_grad()
        m(tokens.to(device)).float().log_softmax(-1)[..., 5].mean().backward()
        grads.append({n: p.grad.detach().cpu().clone() for n, p in m.named_parameters()})
    for n, g in grads[0].items():
        assert float((g - grads[1][n]).norm()) <= 2e-3 * float(g.norm()) + 1e-7, n      # (fp32 products on the tensor cores' fp32 path of the library, 70 tokens of three layers)
