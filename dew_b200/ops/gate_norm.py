"""The norm behind a gate, ``norm(x silu(z)) w`` (``csrc/kernels/gate_norm.cu``), forward and backward: launchers and autograd node."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import library as L


def _blocks(rows: int, row_bytes: int) -> int:
    """Blocks that walk the rows of a backward: as many as an SM holds of them (8192 rows of 1024 bf16 values: 148, 296, 592, 1184 blocks 64, 39, 29, 34 us with the sum of their parts)."""
    if row_bytes <= 1024:                  # a row a warp
        return max(1, min(148, -(-rows // 8)))
    return min(rows, 148 * (4 if row_bytes <= 4096 or row_bytes > 16384 else 2 if row_bytes <= 8192 else 1))


def plain(x, z, w, eps: float) -> torch.Tensor:
    f = torch.float64 if x.dtype is torch.float64 else torch.float32
    u = x.to(f) * F.silu(z.to(f))
    return (u * torch.rsqrt(u.pow(2).mean(-1, keepdim=True) + eps) * w.to(f)).to(x.dtype)


def kernel_available(x: torch.Tensor, z: torch.Tensor, w: torch.Tensor) -> bool:
    return (x.is_cuda and x.dtype in (torch.bfloat16, torch.float32) and z.dtype is x.dtype and w.dtype in (x.dtype, torch.float32) and w.dim() == 1 and x.dim() > 0 and x.numel() > 0
            and z.shape == x.shape and w.shape[0] == x.shape[-1] and z.device == w.device == x.device and not L.transformed(x, z, w) and L.use_cuda(x))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t [..., d]`` as rows, each in one piece (a view of a wider tensor is one already)."""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _forward(x, z, w, eps: float) -> torch.Tensor:
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _forward(x, z, w, eps)
    x2, z2, w = _rows(x), _rows(z), w.contiguous()
    rows, d = x2.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    L.check(L.load().dewb_gate_norm_fwd(x2.data_ptr(), x2.stride(0), z2.data_ptr(), z2.stride(0), w.data_ptr(), y.data_ptr(), rows, d, eps, int(x.dtype is torch.float32),
                                        int(w.dtype is torch.float32), L.stream()), "gate_norm_fwd")
    L.count_launches()
    return y


def _backward(x, z, w, eps: float, dy):
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _backward(x, z, w, eps, dy)
    L.ensure_device(x)                                       # (a thread of autograd's may come here first)
    x2, z2, w, dy2 = _rows(x), _rows(z), w.contiguous(), _rows(dy.to(x.dtype))
    rows, d = x2.shape
    dx, dz, dw = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (x, z, w))
    blocks = _blocks(rows, d * x.element_size())
    parts = torch.empty(blocks, d, dtype=torch.float32, device=x.device)
    L.check(L.load().dewb_gate_norm_bwd(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), z2.data_ptr(), z2.stride(0), w.data_ptr(), dx.data_ptr(), dz.data_ptr(),
                                        dw.data_ptr(), parts.data_ptr(), blocks, rows, d, eps, int(x.dtype is torch.float32), int(w.dtype is torch.float32), L.stream()), "gate_norm_bwd")
    L.count_launches(2)
    return dx, dz, dw


class _GateNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, w, eps):
        ctx.save_for_backward(x, z, w)
        ctx.eps = eps
        return _forward(x, z, w, eps)

    @staticmethod
    def backward(ctx, dy):
        x, z, w = ctx.saved_tensors
        if torch.is_grad_enabled():                          # (create_graph: the kernel's results would have no history)
            at = [i for i, t in enumerate((x, z, w)) if ctx.needs_input_grad[i]]
            grads = torch.autograd.grad(plain(x, z, w, ctx.eps), [(x, z, w)[i] for i in at], dy, create_graph=True)
            return (*(grads[at.index(i)] if i in at else None for i in range(3)), None)
        return (*_backward(x, z, w, ctx.eps, dy), None)


def gate_norm(x: torch.Tensor, z: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    if not kernel_available(x, z, w):
        return plain(x, z, w, eps)
    return _forward(x, z, w, eps) if L.unrecorded(x, z, w) else _GateNorm.apply(x, z, w, eps)
