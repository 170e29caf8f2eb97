"""Low-rank adapters of many requests beside one projection (``csrc/kernels/adapters.cu``): the projection's weight is read once for all tokens, each adapter once for its own."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import library as L


class Bank(NamedTuple):
    """The adapters of one projection: ``a [n, rank, in]``, ``b [n, out, rank]``, ``scale [n]`` (fp32).  Adapters of lower rank have zeros behind."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor


SCANNED = 512            # tokens whose ids every CTA looks through; more are grouped by a kernel of their own


def on_tensor_cores(x: torch.Tensor, n: int, rank: int) -> bool:
    return x.dtype == torch.bfloat16 and n <= 4096 and rank <= 512


def _splits(tiles: int, rank: int, width: int) -> int:
    """Parts of a prompt's width that are summed apart: two CTAs an SM, each with four slots' worth of columns at least."""
    return max(1, min(8, width // 256, 296 // (tiles * -(-rank // 64))))


def _check(x, bank: Bank, ids, out: int, weight_device) -> None:
    a, b, scale = bank
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or scale.shape != a.shape[:1]:
        raise ValueError(f"adapters: a [n, rank, in], b [n, out, rank] and scale [n], got {tuple(a.shape)}, {tuple(b.shape)}, {tuple(scale.shape)}")
    if x.shape[-1] != a.shape[2] or out != b.shape[1]:
        raise ValueError(f"adapters: of {a.shape[2]} to {b.shape[1]} beside a projection of {x.shape[-1]} to {out}")
    if ids.shape != x.shape[:-1]:
        raise ValueError(f"adapters: one id a token, {tuple(x.shape[:-1])}, got {tuple(ids.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32) or a.dtype != x.dtype or b.dtype != x.dtype or scale.dtype != torch.float32 or ids.dtype != torch.int32:
        raise TypeError(f"adapters: bf16 or fp32 tokens and adapters of one type, fp32 scales and int32 ids, got {x.dtype}, {a.dtype}, {b.dtype}, {scale.dtype}, {ids.dtype}")
    if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous()):
        raise ValueError("adapters: a, b and scale in one piece each")
    if any(t.device != x.device for t in (a, b, scale, ids)) or weight_device != x.device:
        raise ValueError("adapters: tensors of one device")


def add_adapters_reference(y: torch.Tensor, x: torch.Tensor, bank: Bank, ids: torch.Tensor) -> torch.Tensor:
    flat, x2, out = ids.reshape(-1), x.reshape(-1, x.shape[-1]).float(), y.view(-1, y.shape[-1])
    for i in sorted(set(flat.tolist())):
        if i < 0:
            continue
        at = (flat == i).nonzero()[:, 0]
        out[at] = (out[at].float() + (x2[at] @ bank.a[i].float().T * bank.scale[i]) @ bank.b[i].float().T).to(y.dtype)
    return y


def add_adapters(y: torch.Tensor, x: torch.Tensor, bank: Bank, ids: torch.Tensor) -> torch.Tensor:
    """``y [..., out] += scale[i] (x [..., in] a[i]^T) b[i]^T`` in place, ``i = ids [...]`` (int32; below 0: the token has none) -> ``y``.  The rank's values and the sum are fp32."""
    _check(x, bank, ids, y.shape[-1], y.device)
    if y.dtype != x.dtype or y.shape[:-1] != x.shape[:-1] or not y.is_contiguous():
        raise ValueError("add_adapters: the projection's result in one piece, of the tokens' type and count")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (y, x, *bank)):
        raise NotImplementedError("add_adapters has no gradient: it serves adapters that were trained alone (nn.lora)")
    if bank.a.shape[0] == 0 or bank.a.shape[1] == 0 or y.numel() == 0 or x.shape[-1] == 0:
        return y
    if not L.use_cuda(x):
        return add_adapters_reference(y, x, bank, ids)
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    ids = ids.contiguous()
    n, rank, width = bank.a.shape
    tokens, out = x2.shape[0], y.shape[-1]
    err = L.status(x.device).data_ptr()
    with L.on_device_of(x) as stream:
        if on_tensor_cores(x, n, rank):
            # one piece of scratch a call: the rank's values by parts of the width, the tokens by adapter, their tiles
            grouped = tokens > SCANNED
            splits, order, tiles, scratch = 1, 0, 0, None
            if grouped:
                splits = _splits(tokens // 128 + 1, rank, width)
                values, numbers = -(-splits * tokens * rank // 4) * 4, -(-tokens // 4) * 4
                scratch = torch.empty(values + numbers + 4 * (tokens // 128 + min(n, tokens) + 2), dtype=torch.float32, device=x.device)
                order = scratch.data_ptr() + 4 * values
                tiles = order + 4 * numbers
            L.check(L.load().dewb_add_adapters_mma(x2.data_ptr(), x2.stride(0), bank.a.data_ptr(), bank.b.data_ptr(), bank.scale.data_ptr(), ids.data_ptr(), order, tiles, L.at(scratch),
                                                   y.data_ptr(), tokens, n, rank, width, out, splits, err, stream), "add_adapters_mma")
            L.count_launches(3 if grouped else 1)
            return y
        splits = max(1, min(16, width // 256, 592 // tokens))
        low = torch.empty(splits * tokens * rank, dtype=torch.float32, device=x.device)
        L.check(L.load().dewb_add_adapters(x2.data_ptr(), x2.stride(0), bank.a.data_ptr(), bank.b.data_ptr(), bank.scale.data_ptr(), ids.data_ptr(), low.data_ptr(), y.data_ptr(),
                                           tokens, n, rank, width, out, splits, int(x.dtype == torch.float32), err, stream), "add_adapters")
    L.count_launches(2)
    return y


def adapted_linear(x: torch.Tensor, weight: torch.Tensor, bank: Bank, ids: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``ops.linear(x, weight, bias)`` plus each token's adapter (``add_adapters``): ``x [..., in]``, ``weight [out, in]``, ``ids [...]`` int32."""
    from .functional import linear
    _check(x, bank, ids, weight.shape[0], weight.device)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, *bank)):
        raise NotImplementedError("adapted_linear has no gradient: it serves adapters that were trained alone (nn.lora)")
    return add_adapters(linear(x, weight, bias), x, bank, ids)
