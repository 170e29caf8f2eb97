"""Where states lie and how many rows a call has, of the scans with a decay per head.  The chunks read and write states in pairs of floats: those that begin on an odd one go token by token
or lie elsewhere first."""
import ctypes

import pytest
import torch

from dew_b200.ops import library as L
from dew_b200.ops import scan, selective
from dew_b200.ops import ssd as chunks
from selective_cases import draws_of_its_own, rows  # noqa: F401


def odd(t):
    """The same numbers from an odd float on, in one piece."""
    room = t.new_empty(t.numel() + 1)[1:].view(t.shape).copy_(t)
    assert room.is_contiguous() and room.data_ptr() % 8 == 4
    return room


class Library:
    dewb_ssd_rows = None


def test_which_states_the_chunks_take(monkeypatch):
    monkeypatch.setattr(L, "load", lambda: Library)
    x, state = torch.zeros(2, 32, 256, dtype=torch.bfloat16), torch.zeros(2, 4, 64, 128)
    assert selective._suits_chunks(x, 4, 2, 128, state) and selective._suits_chunks(x, 4, 2, 128, None)
    assert not selective._suits_chunks(x, 4, 2, 128, odd(state)) and not selective._suits_chunks(x[:, :31], 4, 2, 128, state)


@pytest.mark.skipif(not L.exists(), reason="the library is not built")
def test_the_launcher_looks():
    """(Refused before anything is launched: the addresses are the host's.)"""
    room = torch.zeros(64, dtype=torch.float64)
    at, strides = room.data_ptr() + (-room.data_ptr()) % 16, (ctypes.c_longlong * 6)()
    for off in (1, 2, 4, 12):
        assert L.load().dewb_ssd_rows(at, at, at, at, at, at, at + off, at, at, at, at, at, 1, 64, 2, 1, ctypes.addressof(strides), 0) == -3
    assert L.load().dewb_ssd_rows(at, at, at, at, at, at, 0, at, at, 0, at, at, 1, 64, 2, 1, ctypes.addressof(strides), 0) == -3      # (no lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 31, 32, 100])
def test_states_from_an_odd_float_on(S, monkeypatch):
    """The same bits as from an even one, token by token."""
    g = torch.Generator("cuda").manual_seed(S)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    call = dict(x=r(2, S, 256).bfloat16(), dt=(r(2, S, 4) - 3).bfloat16(), dt_bias=r(4), A_log=r(4), Bm=r(2, S, 256).bfloat16(), Cm=r(2, S, 256).bfloat16(), D=r(4), H=4, G=2,
                rows=rows([3, 0], [S, max(1, S - 5)], S, [2, 0], "cuda"))
    start = r(3, 4, 64, 128)
    state, beside = odd(start), start.clone()
    y = selective.ssd_tokens(**call, state=state)
    monkeypatch.setattr(selective, "CHUNKED_TOKENS", 1 << 30)
    want = selective.ssd_tokens(**call, state=beside)
    L.check_status()
    assert torch.equal(y, want) and torch.equal(state, beside)


@pytest.mark.skipif(not L.exists(), reason="the library is not built")
def test_the_launchers_of_whole_rows_look():
    room = torch.zeros(64, dtype=torch.float64)
    at, strides = room.data_ptr() + (-room.data_ptr()) % 16, (ctypes.c_longlong * 6)()
    p, i = ctypes.c_void_p, ctypes.c_int
    sizes = (i(1), i(64), i(2), i(1), strides, p(0))
    for initial, last in ((4, 0), (0, 12)):
        assert L.load().dewb_ssd_fwd(*(p(at),) * 6, p(at + initial), p(at), p(at), p(at + last), *sizes) == -3
    for initial, dlast, dinitial in ((4, 0, 0), (0, 4, 0), (0, 0, 4)):
        assert L.load().dewb_ssd_bwd(*(p(at),) * 6, p(at + initial), p(at), p(at + dlast), *(p(at),) * 6, *(p(at),) * 6, p(at + dinitial), *sizes) == -3


def test_what_the_kernels_are_given_of_states():
    state = torch.randn(2, 2, 64, 128)
    assert chunks._even(None) is None and chunks._even(state) is state
    moved = chunks._even(odd(state))
    assert torch.equal(moved, state) and moved.data_ptr() % 8 == 0


@pytest.mark.gpu
def test_whole_rows_from_states_and_gradients_on_odd_floats():
    """The state that rows begin with, and the gradient of the one that they end with."""
    g = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, b, c, dt, a = r(2, 70, 2, 64).bfloat16(), r(2, 70, 1, 128).bfloat16(), r(2, 70, 1, 128).bfloat16(), torch.nn.functional.softplus(r(2, 70, 2) - 3), -torch.exp(r(2))
    initial, dy, dlast = r(2, 2, 64, 128), r(2, 70, 2, 64).bfloat16(), r(2, 2, 64, 128)

    def run(initial, dlast):
        leaves = [t.detach().requires_grad_() for t in (x, dt, a, b, c, initial)]
        out = scan.ssd(*leaves[:5], None, leaves[5])
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (dy, dlast)))
    want, got = run(initial, dlast), run(odd(initial), odd(dlast))
    L.check_status()
    assert all(torch.equal(u, v) for u, v in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("R", [65535, 65537, 200_001])
def test_a_token_of_many_rows(R):
    """The rows of one call are the rows of several."""
    g = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    call = dict(x=r(R, 1, 6), dt=r(R, 1, 3) - 3, Bm=r(R, 1, 5), Cm=r(R, 1, 5))
    heads = dict(dt_bias=r(3), A_log=r(3), D=r(3), H=3, G=1)
    at = rows([4], [1], 1, None, "cuda")
    many = at._replace(positions=at.positions.expand(R, 1).contiguous(), lengths=at.lengths.expand(R).contiguous())
    start = r(R, 3, 2, 5)
    state, parts = start.clone(), []
    y = selective.ssd_tokens(**call, **heads, rows=many, state=state)
    for lo in range(0, R, 30_000):
        hi = min(R, lo + 30_000)
        parts.append(selective.ssd_tokens(**{k: v[lo:hi] for k, v in call.items()}, **heads, rows=at._replace(positions=many.positions[lo:hi], lengths=many.lengths[lo:hi]), state=start[lo:hi]))
    L.check_status()
    assert torch.equal(y, torch.cat(parts)) and torch.equal(state, start)
