"""Mamba-1 block: input projection to (x, z), short causal conv + SiLU, input-dependent (dt, B, C), selective scan, gate,
output projection; a row of a cache keeps the convolution's last inputs and the scan's state.  Reference: src/dew/nn/mixers/mamba.py (450 lines)."""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from ..ops import scan, selective, token_mix
from .layers import Linear, declare
from .linear_attention import ShortConv, in_slot, kept_state


class Mamba(nn.Module):
    def __init__(self, features: int, state_dim: int = 16, expand: int = 2, conv_size: int = 4, dt_rank: int | None = None, dtype=None, device=None):
        super().__init__()
        inner = expand * features
        self.inner, self.n = inner, state_dim
        self.dt_rank = dt_rank or math.ceil(features / 16)
        kw = dict(dtype=dtype, device=device)
        self.in_proj = Linear(features, 2 * inner, **kw)
        self.conv = ShortConv(inner, conv_size, bias=True, activation=True, **kw)
        self.x_proj = Linear(inner, self.dt_rank + 2 * state_dim, **kw)
        self.dt_proj = Linear(self.dt_rank, inner, bias=True, **kw)
        self.A_log = declare(nn.Parameter(torch.log(torch.arange(1, state_dim + 1, dtype=torch.float32, device=device)).repeat(inner, 1)), ("mlp", None), "A_log")
        self.D = declare(nn.Parameter(torch.ones(inner, dtype=torch.float32, device=device)), ("mlp",), "scale")
        self.out_proj = Linear(inner, features, **kw)

    def fresh_state(self, batch: int) -> dict:
        p = self.out_proj.weight
        return {"conv": torch.zeros(batch, self.conv.kernel_size - 1, self.inner, dtype=p.dtype, device=p.device),
                "S": torch.zeros(batch, self.inner, self.n, dtype=torch.float32, device=p.device)}

    def cache_slot(self):
        from .kv_cache import CacheSlot
        conv = (("conv", (self.inner, self.conv.kernel_size - 1)),) if self.conv.kernel_size > 1 else ()
        return CacheSlot(state=(self.inner, self.n), more=conv)

    def _narrow(self, xi):
        """The step's logits, B and C of every token."""
        p = self.x_proj(xi)
        return self.dt_proj(p[..., :self.dt_rank]), p[..., self.dt_rank:self.dt_rank + self.n], p[..., self.dt_rank + self.n:]

    def _in_slot(self, x, cache, slot: int, positions):
        """A call's tokens with the state in the cache's slot."""
        rows, state, more = cache.call(positions).rows, cache.states[slot], cache.more[slot]
        xz = self.in_proj(x)
        xi = token_mix.conv_tokens(xz[..., :self.inner], self.conv.weight, None, self.conv.activation, rows, more.get("conv"), self.conv.bias)
        dt, Bm, Cm = self._narrow(xi)
        return self.out_proj(selective.selective_tokens(xi, dt, self.A_log, Bm, Cm, self.D, xz[..., self.inner:], rows, state))

    def forward(self, x, segment_ids=None, cache=None, layer: int = 0, chunked: bool = True, positions=None):
        if in_slot(cache, layer):
            if segment_ids is not None:
                raise NotImplementedError("a state in a cache's slot runs over rows without packed segments")
            return self._in_slot(x, cache, layer, positions)
        xz = self.in_proj(x)
        xi, z = xz[..., :self.inner], xz[..., self.inner:]
        state = kept_state(cache, layer, x.shape[0], self)
        xi = self.conv(xi, segment_ids, state["conv"] if state is not None else None)
        dt, Bm, Cm = self._narrow(xi)
        fn = scan.selective_scan if chunked else scan.selective_scan_reference
        y, S = fn(xi, dt, -torch.exp(self.A_log.float()), Bm, Cm, self.D, z, initial_state=None if state is None else state["S"], softplus=True)
        if state is not None:
            state["S"].copy_(S)
        return self.out_proj(y.to(x.dtype))
