"""The kernels of a server of many requests at their edges: groups that leave rows out, numbers that are none, packed prompts, captured calls."""
import math

import pytest
import torch

from dew_b200.ops import library as L
from dew_b200.ops.prefix import Shared, shared_decode
from prefix_cases import allowed, batch, truth

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def reported(a, **kw):
    L.check_status()
    out = shared_decode(**a, **kw)
    with pytest.raises(L.KernelError):
        L.check_status()
    return out


# ---------------------------------------------------------------------------------------------------------- groups that do not hold every row once
@pytest.mark.parametrize("dtype, heads, kv, dim, page", [(BF16, 8, 2, 128, 16), (BF16, 64, 2, 64, 64), (FP32, 8, 2, 48, 16)])
@pytest.mark.parametrize("held", [0, 2, 5])
def test_rows_that_no_group_holds_are_reported_and_give_zeros(dtype, heads, kv, dim, page, held):
    a = batch([(2048, [1 + i % 40 for i in range(30)])], heads, kv, dim, page, dtype, device=DEV)
    order, R = a["shared"].order, a["q"].shape[0]
    out = reported({**a, "shared": Shared(order, ints([0, held]), a["shared"].tokens[:1].contiguous())})
    left = order.long()[held:]
    assert left.numel() == R - held and not out[left].any()
    got = shared_decode(**a)                                  # (the word is clear again)
    L.check_status()
    found = truth(a)
    assert bool(((got.double().cpu() - found[0]).abs() <= allowed(a, found)).all())


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (FP32, 48)])
@pytest.mark.parametrize("first", [[0, 4, 2, 6], [0, 6, 3, 6], [3, 0, 6, 6]])
def test_groups_that_begin_behind_their_end_are_reported(dtype, dim, first):
    a = batch([(64, [3, 4, 5, 6, 7, 8])], 4, 2, dim, 16, dtype, device=DEV)
    reported({**a, "shared": Shared(a["shared"].order, ints(first), ints([64, 64, 64]))})
