"""Low-rank adapters of many requests beside one projection: the plain form and what is refused."""
import pytest
import torch

from adapters_cases import allowed, batch, truth
from dew_b200.ops.adapters import Bank, adapted_linear, add_adapters


@pytest.mark.parametrize("tokens, n, rank, width, out", [(1, 1, 1, 3, 2), (9, 4, 5, 24, 17), (40, 3, 8, 16, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_the_plain_form(tokens, n, rank, width, out, dtype, bias):
    a = batch(tokens, n, rank, width, out, dtype)
    b = torch.randn(out).to(dtype) if bias else None
    found = truth(a, b)
    got = adapted_linear(**a, bias=b)
    assert got.dtype == dtype and bool(((got.double() - found[0]).abs() <= allowed(a, found)).all())
    three = adapted_linear(a["x"].view(1, tokens, 1, width), a["weight"], a["bank"], a["ids"].view(1, tokens, 1), b)
    assert torch.equal(three.view(tokens, out), got)


def test_tokens_without_an_adapter_are_the_projections():
    a = batch(6, 3, 4, 16, 8)
    none = torch.full_like(a["ids"], -1)
    assert torch.equal(adapted_linear(a["x"], a["weight"], a["bank"], none), torch.nn.functional.linear(a["x"], a["weight"]))
    empty = Bank(*(t[:0] for t in a["bank"]))
    assert torch.equal(adapted_linear(a["x"], a["weight"], empty, none), torch.nn.functional.linear(a["x"], a["weight"]))
    assert adapted_linear(a["x"][:0], a["weight"], a["bank"], none[:0]).shape == (0, 8)


def test_refusals():
    a = batch(6, 3, 4, 16, 8, torch.float32)
    x, w, bank, ids = a["x"], a["weight"], a["bank"], a["ids"]
    cases = [(ValueError, x[:, :8], w, bank, ids), (ValueError, x, w[:4], bank, ids), (ValueError, x, w, bank, ids[:5]), (TypeError, x, w, bank, ids.long()),
             (TypeError, x.half(), w, bank, ids), (TypeError, x.bfloat16(), w.bfloat16(), bank, ids), (TypeError, x, w, bank._replace(scale=bank.scale.double()), ids),
             (ValueError, x, w, bank._replace(scale=bank.scale[:2]), ids), (ValueError, x, w, bank._replace(b=bank.b[:2]), ids),
             (ValueError, x, w, bank._replace(a=bank.a.transpose(1, 2).contiguous().transpose(1, 2)), ids), (ValueError, x, w, bank, ids.to("meta")),
             (NotImplementedError, x.clone().requires_grad_(), w, bank, ids), (NotImplementedError, x, w, bank._replace(a=bank.a.clone().requires_grad_()), ids)]
    for error, *call in cases:
        with pytest.raises(error):
            adapted_linear(*call)
    y = torch.zeros(6, 8)
    for bad in (y[:5], y.double(), torch.zeros(8, 6).T):
        with pytest.raises(ValueError):
            add_adapters(bad, x, bank, ids)


def test_the_result_may_not_be_the_tokens():
    a = batch(6, 3, 4, 16, 16, torch.float32)
    with pytest.raises(ValueError):
        add_adapters(a["x"], a["x"], a["bank"], a["ids"])
