"""Tokens of many requests with adapters, and the formula in 64 bits."""
import math

import torch

from dew_b200.ops.adapters import Bank


def batch(tokens, n, rank, width, out, dtype=torch.bfloat16, seed=0, device="cpu", used=None, without=0.2, runs=False):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dtype).to(device)
    names = torch.randperm(n, generator=g)[:used or n]
    ids = names[torch.randint(len(names), (tokens,), generator=g)] if len(names) else torch.full((tokens,), -1)
    ids = torch.where(torch.rand(tokens, generator=g) < without, -1, ids)
    if runs:
        ids = ids.sort().values
    bank = Bank(make(n, rank, width, by=width ** -0.5), make(n, out, rank, by=max(1, rank) ** -0.5), (torch.rand(n, generator=g) + 0.5).to(device))
    for i in set(range(n)) - set(ids.tolist()):                          # nobody's: not read
        bank.a[i], bank.b[i], bank.scale[i] = math.nan, math.nan, math.nan
    return dict(x=make(tokens, width), weight=make(out, width, by=width ** -0.5), bank=bank, ids=ids.to(device, torch.int32))


def truth(a, bias=None):
    """``(y, what its roundings are of)`` in 64 bits: |projection| and the adapters' sum |low b|."""
    x, w, (A, B, s) = a["x"].double().cpu(), a["weight"].double().cpu(), (t.double().cpu() for t in a["bank"])
    ids = a["ids"].cpu().reshape(-1)
    x = x.reshape(-1, x.shape[-1])
    base = x @ w.T + (0 if bias is None else bias.double().cpu())
    y, size, low_size = base.clone(), torch.zeros_like(base), torch.zeros_like(base)
    for i in set(ids.tolist()) - {-1}:
        at = (ids == i).nonzero()[:, 0]
        low = x[at] @ A[i].T * s[i]
        y[at] += low @ B[i].T
        size[at] = low.abs() @ B[i].abs().T
        low_size[at] = (x[at].abs() @ A[i].abs().T * s[i].abs()) @ B[i].abs().T
    return y, base, size, (x.abs() @ w.abs().T) + low_size


def allowed(a, found):
    """The projection's rounding and the result's (half a step each); in bf16 the rank's values are rounded for the second product; sums in fp32 of everything."""
    y, base, size, everything = found
    half = torch.finfo(a["x"].dtype).eps / 2
    bf16 = a["x"].dtype == torch.bfloat16
    n = a["x"].shape[-1] + a["bank"].a.shape[1]
    return half * 1.01 * (base.abs() + y.abs()) + (half * 1.01 * size if bf16 else 0) + everything * (n + 4) * 2.0 ** -24 + 1e-30
