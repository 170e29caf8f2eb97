"""Attention of rows that share prefixes: the plain form, how rows are grouped, what is refused."""
import pytest
import torch

from dew_b200.ops.prefix import Shared, group_rows, shared_decode
from prefix_cases import allowed, batch, truth


@pytest.mark.parametrize("window, softcap, sinks", [(None, 0.0, False), (9, 0.0, False), (None, 5.0, True), (40, 3.0, True)])
@pytest.mark.parametrize("dtype, pool", [(torch.float32, None), (torch.bfloat16, None), (torch.float32, torch.int8), (torch.bfloat16, torch.float8_e4m3fn)])
def test_the_plain_form(window, softcap, sinks, dtype, pool):
    a = batch([(32, [1, 9, 17]), (0, [5]), (50, [3, 3])], 6, 2, 24, 16, dtype, pool, resting=(1,))
    s = torch.randn(6) if sinks else None
    found = truth(a, window, softcap, s)
    got = shared_decode(**a, window=window, softcap=softcap, sinks=s).double()
    assert bool(((got - found[0]).abs() <= allowed(a, found)).all())
    assert not got[a["lengths"] == 0].any()


def test_rows_group_by_their_first_pages():
    order, first, tokens = group_rows([[5, 6, 7], [1, 2], [5, 6, 9], None, [5, 6], [1, 3], []], 16)
    groups = {tuple(order[a:b]): n for a, b, n in zip(first, first[1:], tokens) if a < b}
    assert groups == {(0, 2, 4): 32, (1, 5): 16, (3,): 0, (6,): 0}
    assert len(first) == 8 and len(tokens) == 7 and first[-1] == 7 and sorted(order) == list(range(7))
    order, first, tokens = group_rows([[5, 6, 7], [1, 2], [5, 6, 9], [1, 3]], 16, least=32)
    assert {tuple(order[a:b]): n for a, b, n in zip(first, first[1:], tokens) if a < b} == {(0, 2): 32, (1,): 0, (3,): 0}
    assert group_rows([], 16) == ([], [0], [])


def test_no_rows():
    a = batch([(16, [1, 2])], 4, 2, 16, 16)
    none = {n: a[n][:0].contiguous() for n in ("q", "table", "lengths")}
    shared = Shared(a["shared"].order[:0], torch.zeros(1, dtype=torch.int32), a["shared"].tokens[:0])
    assert shared_decode(**{**a, **none, "shared": shared}).shape == (0, 4, 16)


def _refused(a, error, **changed):
    with pytest.raises(error):
        shared_decode(**{**a, **changed})


def test_refusals():
    a = batch([(16, [1, 2]), (0, [3])], 4, 2, 16, 16, torch.float32)
    s = a["shared"]
    _refused(a, ValueError, q=a["q"][:, :3])                              # heads that the key heads do not divide
    _refused(a, ValueError, q=a["q"][..., :8])
    _refused(a, ValueError, q=a["q"][:2])
    _refused(a, ValueError, v=a["v"][:, :8])
    _refused(a, TypeError, q=a["q"].half())
    _refused(a, TypeError, k=a["k"].bfloat16())
    _refused(a, TypeError, k=a["k"].bfloat16(), v=a["v"].bfloat16())
    _refused(a, TypeError, table=a["table"].long())
    _refused(a, TypeError, lengths=a["lengths"].long())
    _refused(a, TypeError, table=a["table"].T.contiguous().T)
    _refused(a, ValueError, table=a["table"][:2])
    _refused(a, ValueError, lengths=a["lengths"][:2])
    _refused(a, ValueError, shared=Shared(s.order[:2], s.first, s.tokens))
    _refused(a, ValueError, shared=Shared(s.order, s.first[:2], s.tokens))
    _refused(a, ValueError, k=a["k"].transpose(0, 1).contiguous().transpose(0, 1))
    _refused(a, ValueError, window=0)
    _refused(a, ValueError, softcap=-1.0)
    _refused(a, ValueError, sinks=torch.zeros(2))
    _refused(a, ValueError, sinks=torch.zeros(4, dtype=torch.bfloat16))
    _refused(a, ValueError, k_scale=torch.ones(a["k"].shape[:3]))
    _refused(a, ValueError, q=a["q"].to("meta"))
    _refused(a, NotImplementedError, q=a["q"].clone().requires_grad_())
    b = batch([(16, [1, 2])], 4, 2, 16, 16, torch.float32, torch.int8)
    _refused(b, ValueError, k_scale=None)
    _refused(b, ValueError, k_scale=b["k_scale"][:, :8])
    wide = batch([(16, [1, 2])], 1, 1, 264, 16, torch.float32)
    _refused(wide, ValueError)
    with torch.no_grad():
        shared_decode(**{**a, "q": a["q"].clone().requires_grad_()})
