"""Low-rank adapters of many requests beside one projection (``csrc/kernels/adapters.cu``): the projection's weight is read once for all tokens, each adapter once for its own."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import library as L
from .functional import linear


class Bank(NamedTuple):
    """The adapters of one projection: ``a [n, rank, in]``, ``b [n, out, rank]``, ``scale [n]`` (fp32).  Adapters of lower rank have zeros behind."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor


SCANNED = 512            # tokens whose ids every CTA looks through; more are grouped by a kernel of their own (512 against 520 tokens, beside 4096 x 4096: one adapter 12 and 15 us,
                         # four of rank 64 19 and 26, 48 of rank 32 17 and 35)


def on_tensor_cores(x: torch.Tensor, n: int, rank: int) -> bool:
    return x.dtype == torch.bfloat16 and n <= 3500 and rank <= 512


def _splits(tiles: int, rank: int, width: int) -> int:
    """Parts of a prompt's width that are summed apart: two CTAs an SM, each with four slots' worth of columns at least; a cluster of 1, 2, 4 or 8.
    (1, 2, 4, 8 parts: 8192 tokens of rank 64, 4096 to 4096: 67, 57, 57, 65 us; 2048 of rank 16: 35, 25, 20, 18.5; 1024 of rank 64, 14336 to 4096: 80, 47, 32, 24.)"""
    parts = max(1, min(8, width // 256, 296 // (tiles * -(-rank // 64))))
    return 1 << parts.bit_length() - 1


def _check(x, bank: Bank, ids, out: int, device) -> None:
    a, b, scale = bank
    a_shape, b_shape, x_shape = a.shape, b.shape, x.shape
    if len(a_shape) != 3 or len(b_shape) != 3 or a_shape[0] != b_shape[0] or a_shape[1] != b_shape[2] or scale.shape != a_shape[:1]:
        raise ValueError(f"adapters: a [n, rank, in], b [n, out, rank] and scale [n], got {tuple(a.shape)}, {tuple(b.shape)}, {tuple(scale.shape)}")
    if not x_shape or x_shape[-1] != a_shape[2] or out != b_shape[1]:
        raise ValueError(f"adapters: of {a_shape[2]} to {b_shape[1]} beside a projection of {x_shape[-1:]} to {out}")
    if ids.shape != x_shape[:-1]:
        raise ValueError(f"adapters: one id a token, {tuple(x.shape[:-1])}, got {tuple(ids.shape)}")
    own = x.dtype
    if (own is not torch.bfloat16 and own is not torch.float32) or a.dtype is not own or b.dtype is not own or scale.dtype is not torch.float32 or ids.dtype is not torch.int32:
        raise TypeError(f"adapters: bf16 or fp32 tokens and adapters of one type, fp32 scales and int32 ids, got {x.dtype}, {a.dtype}, {b.dtype}, {scale.dtype}, {ids.dtype}")
    if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous()):
        raise ValueError("adapters: a, b and scale in one piece each")
    if x.is_cuda and type(device) is int:                # (the quicker question)
        apart = a.get_device() != device or b.get_device() != device or scale.get_device() != device or ids.get_device() != device or x.get_device() != device
    else:
        apart = a.device != device or b.device != device or scale.device != device or ids.device != device or x.device != device
    if apart:
        raise ValueError("adapters: tensors of one device")


def _end(t: torch.Tensor, at: int) -> int:
    """The address behind a tensor's last element."""
    return at + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else at


def add_adapters_reference(y: torch.Tensor, x: torch.Tensor, bank: Bank, ids: torch.Tensor) -> torch.Tensor:
    flat, x2, out = ids.reshape(-1), x.reshape(-1, x.shape[-1]).float(), y.view(-1, y.shape[-1])
    for i in sorted(set(flat.tolist())):
        if i < 0:
            continue
        at = (flat == i).nonzero()[:, 0]
        out[at] = (out[at].float() + (x2[at] @ bank.a[i].float().T * bank.scale[i]) @ bank.b[i].float().T).to(y.dtype)
    return y


def add_adapters(y: torch.Tensor, x: torch.Tensor, bank: Bank, ids: torch.Tensor) -> torch.Tensor:
    """``y [..., out] += scale[i] (x [..., in] a[i]^T) b[i]^T`` in place, ``i = ids [...]`` (int32; below 0: the token has none) -> ``y``.  Sums are fp32; in bf16 the rank's
    values, with their scale, are rounded once between the two products.  ``y`` lies over nothing that is read."""
    _check(x, bank, ids, y.shape[-1] if y.dim() else 0, y.get_device() if y.is_cuda else y.device)
    if y.dtype is not x.dtype or y.shape[:-1] != x.shape[:-1] or not y.is_contiguous():
        raise ValueError("add_adapters: the projection's result in one piece, of the tokens' type and count")
    if L.transformed(y, x, *bank) or (torch.is_grad_enabled() and any(t.requires_grad for t in (y, x, *bank))):
        raise NotImplementedError("add_adapters has no gradient: it serves adapters that were trained alone (nn.lora)")
    if y.numel():                                       # (tokens are read and results written in no order)
        first = y.data_ptr()
        end = first + y.numel() * y.element_size()
        for t in (x, *bank, ids):
            at = t.data_ptr()
            if at < end and _end(t, at) > first:
                raise ValueError("add_adapters: the projection's result lies over what is read")
    _add(y, x, bank, ids)
    if y.is_cuda:                                       # (autograd is to know, as it does of what torch writes)
        torch.autograd.graph.increment_version(y)
    return y


def _add(y: torch.Tensor, x: torch.Tensor, bank: Bank, ids: torch.Tensor) -> torch.Tensor:
    a, b, scale = bank
    (n, rank, width), out, tokens = a.shape, b.shape[1], ids.numel()
    if n == 0 or rank == 0 or tokens == 0 or out == 0 or width == 0:
        return y
    if not L.use_cuda(x):
        return add_adapters_reference(y, x, bank, ids)
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _add(y, x, bank, ids)
    x2 = x if x.dim() == 2 else x.reshape(-1, width)
    stride, step = x2.stride()
    if step != 1 or stride < width:                     # (rows that overlap, or are one)
        x2 = x2.contiguous()
        stride = width
    if not ids.is_contiguous():
        ids = ids.contiguous()
    lib, err, stream = L.load(), L.status(x.device).data_ptr(), L.stream()
    if on_tensor_cores(x, n, rank):
        # one piece of scratch a prompt: the rank's values in bf16, the tokens by adapter, their tiles
        grouped = tokens > SCANNED
        splits, low, order, tiles = 1, 0, 0, 0
        if grouped:
            splits = _splits(tokens // 128 + 1, rank, width)
            values, numbers = tokens * -(-rank // 64) * 32, -(-tokens // 4) * 4
            scratch = torch.empty(values + numbers + 4 * (tokens // 128 + min(n, tokens) + 2), dtype=torch.float32, device=x.device)
            low = scratch.data_ptr()
            order = low + 4 * values
            tiles = order + 4 * numbers
        L.check(lib.dewb_add_adapters_mma(x2.data_ptr(), stride, a.data_ptr(), b.data_ptr(), scale.data_ptr(), ids.data_ptr(), order, tiles, low, y.data_ptr(),
                                          tokens, n, rank, width, out, splits, err, stream), "add_adapters_mma")
        L.count_launches(3 if grouped else 1)
        return y
    splits = max(1, min(16, width // 256, 592 // tokens))
    low = torch.empty(splits * tokens * rank, dtype=torch.float32, device=x.device)
    L.check(lib.dewb_add_adapters(x2.data_ptr(), stride, a.data_ptr(), b.data_ptr(), scale.data_ptr(), ids.data_ptr(), low.data_ptr(), y.data_ptr(),
                                  tokens, n, rank, width, out, splits, int(x.dtype is torch.float32), err, stream), "add_adapters")
    L.count_launches(2)
    return y


def adapted_linear(x: torch.Tensor, weight: torch.Tensor, bank: Bank, ids: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``ops.linear(x, weight, bias)`` plus each token's adapter (``add_adapters``): ``x [..., in]``, ``weight [out, in]``, ``ids [...]`` int32."""
    _check(x, bank, ids, weight.shape[0], weight.get_device() if weight.is_cuda else weight.device)
    if L.transformed(x, weight, bias, *bank) or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, *bank))):
        raise NotImplementedError("adapted_linear has no gradient: it serves adapters that were trained alone (nn.lora)")
    y = linear(x, weight, bias)
    return _add(y if y.is_contiguous() else y.contiguous(), x, bank, ids)
