"""LoRA adapters: wrap chosen ``Linear`` layers with a frozen base weight plus a trainable low-rank update
``W + (alpha / r) B A``; merge / unmerge; adapter-only state for checkpoints (reference: src/dew/lora.py)."""
from __future__ import annotations

import math
import re
import threading
from typing import Dict, Iterable, List, Optional

import torch
import torch.nn as nn

from .. import ops
from ..ops import adapters
from .layers import Linear, declare


class LoRALinear(nn.Module):
    def __init__(self, base: Linear, rank: int = 8, alpha: float = 16.0, dropout: float = 0.0):
        super().__init__()
        self.base, self.rank, self.scale = base, rank, alpha / rank
        self.base.weight.requires_grad_(False)
        dt, dev = base.weight.dtype, base.weight.device
        self.lora_a = declare(nn.Parameter(torch.empty(rank, base.in_features, dtype=dt, device=dev)), ("lora", "embed"), "kernel")
        self.lora_b = declare(nn.Parameter(torch.zeros(base.out_features, rank, dtype=dt, device=dev)), ("mlp", "lora"), "kernel")
        self.dropout = nn.Dropout(dropout) if dropout else None
        self.merged = False
        self.reset_parameters()

    def reset_parameters(self, generator=None):
        with torch.no_grad():
            self.lora_a.normal_(0.0, 1.0 / math.sqrt(self.base.in_features), generator=generator)
            self.lora_b.zero_()

    @property
    def weight(self):
        return self.base.weight

    @property
    def in_features(self):
        return self.base.in_features

    @property
    def out_features(self):
        return self.base.out_features

    def forward(self, x):
        y = self.base(x)
        if self.merged:
            return y
        h = self.dropout(x) if self.dropout is not None else x
        return y + ops.linear(ops.linear(h, self.lora_a), self.lora_b) * self.scale

    def merge(self):
        if not self.merged:
            with torch.no_grad():
                self.base.weight.add_((self.lora_b.float() @ self.lora_a.float() * self.scale).to(self.base.weight.dtype))
            self.merged = True

    def unmerge(self):
        if self.merged:
            with torch.no_grad():
                self.base.weight.sub_((self.lora_b.float() @ self.lora_a.float() * self.scale).to(self.base.weight.dtype))
            self.merged = False


def apply_lora(model: nn.Module, targets: Iterable[str] = ("qkv_proj", "o_proj"), rank: int = 8, alpha: float = 16.0,
               dropout: float = 0.0, freeze_rest: bool = True) -> List[str]:
    """Replace every ``Linear`` whose attribute name matches one of ``targets`` (regexes); returns the wrapped paths."""
    pats = [re.compile(t) for t in targets]
    wrapped = []
    if freeze_rest:
        for p in model.parameters():
            p.requires_grad_(False)
    for path, module in list(model.named_modules()):
        for name, child in list(module.named_children()):
            if isinstance(child, Linear) and not isinstance(child, AdaptedLinear) and any(p.search(name) for p in pats):
                setattr(module, name, LoRALinear(child, rank, alpha, dropout))
                wrapped.append(f"{path}.{name}" if path else name)
    return wrapped


def lora_state(model: nn.Module) -> Dict[str, torch.Tensor]:
    return {n: p.detach().clone() for n, p in model.named_parameters() if ".lora_a" in n or ".lora_b" in n}


def merge_all(model: nn.Module) -> None:
    for m in model.modules():
        if isinstance(m, LoRALinear):
            m.merge()


# ---------------------------------------------------------------------------------------------------------------
# Configuration, variants and adapter files
from dataclasses import dataclass, field  # noqa: E402
from contextlib import contextmanager  # noqa: E402
from typing import Mapping, Sequence, Tuple  # noqa: E402


@dataclass(frozen=True)
class LoRAConfig:
    """Which layers get adapters and of what shape.

    ``targets``       regexes matched against the attribute name of each ``Linear`` (``qkv_proj``, ``down_proj`` ...)
    ``rank`` / ``alpha`` / ``dropout``  the usual; ``rank_pattern`` maps a regex over the module *path* to another rank
    ``rs``            rank-stabilised scaling ``alpha / sqrt(r)`` instead of ``alpha / r`` (rsLoRA)
    ``dora``          weight-decomposed adaptation: the adapted weight's direction comes from ``W + s B A`` and a trainable
                      per-output-row magnitude replaces its row norms (DoRA)
    ``quantize_base`` keep the frozen base weight in a quantised form (``int8`` / ``float8_e4m3fn`` / ``nvfp4``) and
                      de-quantise it for the product: adapter training over a base that costs a quarter to a half of bf16
    """
    targets: Tuple[str, ...] = ("qkv_proj", "o_proj")
    rank: int = 8
    alpha: float = 16.0
    dropout: float = 0.0
    rank_pattern: Mapping[str, int] = field(default_factory=dict)
    rs: bool = False
    dora: bool = False
    quantize_base: Optional[str] = None
    freeze_rest: bool = True


class DoRALinear(LoRALinear):
    """``y = m * (W + s B A) x / ||W + s B A||_row``: direction from the adapted weight, magnitude ``m`` trainable (initialised
    to the base weight's row norms, so the layer starts as the base)."""

    def __init__(self, base: Linear, rank: int = 8, alpha: float = 16.0, dropout: float = 0.0):
        super().__init__(base, rank, alpha, dropout)
        with torch.no_grad():
            m = base.weight.float().norm(dim=1)
        self.magnitude = declare(nn.Parameter(m.to(base.weight.dtype)), ("mlp",), "scale")

    def forward(self, x):
        if self.merged:
            return self.base(x)
        w = self.base.weight.float() + self.scale * (self.lora_b.float() @ self.lora_a.float())
        norm = w.norm(dim=1).detach()                       # the norm is treated as a constant in the backward (the DoRA paper's choice)
        h = self.dropout(x) if self.dropout is not None else x
        y = self.base(x) + ops.linear(ops.linear(h, self.lora_a), self.lora_b) * self.scale
        if self.base.bias is not None:
            y = y - self.base.bias
        y = y * (self.magnitude.float() / norm).to(y.dtype)
        return y if self.base.bias is None else y + self.base.bias

    def merge(self):
        if not self.merged:
            with torch.no_grad():
                w = self.base.weight.float() + self.scale * (self.lora_b.float() @ self.lora_a.float())
                self._kept = self.base.weight.detach().clone()
                self.base.weight.copy_((w * (self.magnitude.float() / w.norm(dim=1))[:, None]).to(self.base.weight.dtype))
            self.merged = True

    def unmerge(self):
        if self.merged:
            with torch.no_grad():
                self.base.weight.copy_(self._kept)
            self.merged = False


class _QuantizedBase(nn.Module):
    """A frozen ``Linear`` whose weight is held quantised (see ``nn.quantization``) and de-quantised per call."""

    def __init__(self, base: Linear, kind: str):
        super().__init__()
        from .quantization import quantize_weight
        self.kind, self.in_features, self.out_features = kind, base.in_features, base.out_features
        self.dtype = base.weight.dtype
        for k, v in quantize_weight(base.weight.detach(), kind).items():
            self.register_buffer(f"q_{k}", v)
        self.bias = base.bias

    @property
    def weight(self):
        from .quantization import dequantize_weight
        stored = {k[2:]: v for k, v in self._buffers.items() if k.startswith("q_")}
        return dequantize_weight(stored, self.kind, self.dtype)

    def forward(self, x):
        return ops.linear(x, self.weight, self.bias)


def apply_lora_config(model: nn.Module, cfg: LoRAConfig) -> List[str]:
    """``apply_lora`` driven by a ``LoRAConfig`` (rank patterns, rsLoRA, DoRA, quantised base)."""
    pats = [re.compile(t) for t in cfg.targets]
    wrapped = []
    if cfg.freeze_rest:
        for p in model.parameters():
            p.requires_grad_(False)
    for path, module in list(model.named_modules()):
        for name, child in list(module.named_children()):
            if not isinstance(child, Linear) or isinstance(child, AdaptedLinear) or not any(p.search(name) for p in pats):
                continue
            full = f"{path}.{name}" if path else name
            rank = next((r for pat, r in cfg.rank_pattern.items() if re.search(pat, full)), cfg.rank)
            alpha = cfg.alpha * (math.sqrt(rank) if cfg.rs else 1.0)        # alpha / r * sqrt(r) = alpha / sqrt(r)
            cls = DoRALinear if cfg.dora else LoRALinear
            layer = cls(child, rank, alpha, cfg.dropout)
            if cfg.quantize_base:
                layer.base = _QuantizedBase(child, cfg.quantize_base)
            setattr(module, name, layer)
            wrapped.append(full)
    if not wrapped:
        raise ValueError(f"no Linear matches {list(cfg.targets)}; attribute names seen: "
                         f"{sorted({n for _, m in model.named_modules() for n, c in m.named_children() if isinstance(c, Linear)})}")
    return wrapped


@contextmanager
def adapters_disabled(model: nn.Module):
    """Run the base model: every adapter's update is switched off inside the block (the reference policy of DPO-style
    objectives over a LoRA-tuned model needs no second copy of the weights)."""
    layers = [m for m in model.modules() if isinstance(m, LoRALinear)]
    for m in layers:
        m._forward_kept = m.forward
        m.forward = m.base.forward if not m.merged else m._forward_kept
    try:
        yield model
    finally:
        for m in layers:
            m.forward = m._forward_kept
            del m._forward_kept


def load_lora_state(model: nn.Module, state: Mapping[str, torch.Tensor], strict: bool = True) -> None:
    own = {n: p for n, p in model.named_parameters() if ".lora_a" in n or ".lora_b" in n or n.endswith(".magnitude")}
    missing = [k for k in own if k not in state]
    extra = [k for k in state if k not in own]
    if strict and (missing or extra):
        raise KeyError(f"adapter state does not match the model: missing {missing[:4]}, unexpected {extra[:4]}")
    with torch.no_grad():
        for k, p in own.items():
            if k in state:
                p.copy_(state[k].to(p.dtype))


def to_peft_state(model: nn.Module) -> Dict[str, torch.Tensor]:
    """Adapter tensors under the key names the PEFT library writes (``base_model.model.<path>.lora_A.weight`` ...), so an
    adapter trained here loads there."""
    out = {}
    for n, p in model.named_parameters():
        if n.endswith(".lora_a"):
            out[f"base_model.model.{n[:-len('.lora_a')]}.lora_A.weight"] = p.detach().clone()
        elif n.endswith(".lora_b"):
            out[f"base_model.model.{n[:-len('.lora_b')]}.lora_B.weight"] = p.detach().clone()
        elif n.endswith(".magnitude"):
            out[f"base_model.model.{n[:-len('.magnitude')]}.lora_magnitude_vector"] = p.detach().clone()
    return out


def from_peft_state(state: Mapping[str, torch.Tensor]) -> Dict[str, torch.Tensor]:
    out = {}
    for k, v in state.items():
        k = k[len("base_model.model."):] if k.startswith("base_model.model.") else k
        for src, dst in ((".lora_A.weight", ".lora_a"), (".lora_B.weight", ".lora_b"), (".lora_magnitude_vector", ".magnitude"),
                         (".lora_A.default.weight", ".lora_a"), (".lora_B.default.weight", ".lora_b")):
            if k.endswith(src):
                out[k[:-len(src)] + dst] = v
    return out


# ---------------------------------------------------------------------------------------------------------------
# Serving: adapters of many requests beside one copy of the weights


class AdaptedLinear(Linear):
    """A ``Linear`` beside which every token may have an adapter of its own, as ``bank.using`` says; without it, the ``Linear``.  It stands in for ``base`` with the same
    parameters under the same names (and the same hooks): variables, checkpoints and optimisers of the model without a bank are those of the model with one."""

    def __init__(self, base: Linear, bank: "AdapterBank"):
        if "forward" in base.__dict__:
            raise ValueError("a Linear whose forward has been replaced cannot have adapters beside it")
        self.__dict__.update(base.__dict__)
        self._of = (bank,)                                 # (not a module of this one)
        w = base.weight
        rank = -(-bank.rank // 8) * 8 if w.dtype == torch.bfloat16 else bank.rank            # (rows of b that begin at 16 bytes are fetched as blocks)
        # (the bank's, not the model's: no buffers, which variables would take along)
        self.a = torch.zeros(bank.slots, rank, self.in_features, dtype=w.dtype, device=w.device)
        self.b = torch.zeros(bank.slots, self.out_features, rank, dtype=w.dtype, device=w.device)
        self.scale = torch.zeros(bank.slots, dtype=torch.float32, device=w.device)

    def _apply(self, fn, recurse=True):
        """``to`` and its like: the scales stay as they are, in fp32."""
        super()._apply(fn, recurse)
        self.a, self.b, self.scale = fn(self.a), fn(self.b), self.scale.to(fn(self.scale).device)
        return self

    @property
    def in_use(self) -> bool:
        """Whether the calls of now have adapters (``AdapterBank.using``)."""
        return self._of[0]._now()[0] is not None

    def opened(self) -> Tuple[nn.Module, str, Linear]:
        """``(module, name, layer)`` of a ``Linear`` of its own that holds the parameters from here on, for what replaces layers by others (``nn.quantization``)."""
        if "base" not in self._modules:
            base = Linear.__new__(Linear)
            nn.Module.__init__(base)
            base.in_features, base.out_features, base.init_std, base.zero_init = self.in_features, self.out_features, self.init_std, self.zero_init
            base._parameters, self._parameters = self._parameters, {}
            if "bias" in self.__dict__:                    # (None: not among the parameters)
                base.bias = self.__dict__.pop("bias")
            base.training = self.training
            self.base = base
        return self, "base", self.base

    def __getattr__(self, name):
        if name == "weight" and self.in_use:
            raise RuntimeError("the model multiplies with this layer's weight itself: adapters beside it would be passed over, so it cannot be a target of theirs")
        if name in ("weight", "bias") and "base" in self.__dict__["_modules"]:
            return getattr(self.base, name)
        return super().__getattr__(name)

    def reset_parameters(self, generator: Optional[torch.Generator] = None):
        if "base" not in self._modules:
            super().reset_parameters(generator)

    def forward(self, x):
        ids, base = self._of[0].ids_for(x.shape[:-1]), self._modules.get("base")
        bank = adapters.Bank(self.a, self.b, self.scale)
        if base is None:
            w = self._parameters["weight"]
            return ops.linear(x, w, self.bias) if ids is None else adapters.adapted_linear(x, w, bank, ids, self.bias)
        y = base(x)
        return y if ids is None else adapters.add_adapters(y, x, bank, ids)


_BANKS = threading.RLock()       # what stands in banks, and who holds it, changes by one thread at a time


class AdapterBank:
    """Room for ``slots`` adapters of rank up to ``rank`` beside the ``targets`` of ``model`` (regexes over the attribute names of its ``Linear`` layers, which are replaced).
    ``load`` takes what ``lora_state`` (or ``from_peft_state``) gives; ``using`` says which adapter each row of the calls inside it has.  For generation: the adapters take no
    gradient."""

    def __init__(self, model: nn.Module, targets: Iterable[str] = ("qkv_proj", "o_proj"), slots: int = 8, rank: int = 16):
        if slots < 1 or rank < 1:
            raise ValueError(f"a bank of {slots} adapters of rank {rank}")
        self.slots, self.rank = slots, rank
        pats = [re.compile(t) for t in targets]
        self.layers: Dict[str, AdaptedLinear] = {}
        for path, module in list(model.named_modules()):
            for name, child in list(module.named_children()):
                if type(child) is Linear and any(p.search(name) for p in pats):
                    layer = AdaptedLinear(child, self)
                    setattr(module, name, layer)
                    self.layers[f"{path}.{name}" if path else name] = layer
        if not self.layers:
            raise ValueError(f"no Linear matches {list(targets)}")
        self.names: Dict[str, int] = {}                    # adapter -> slot
        self.version: Dict[str, int] = {}                  # how often something was loaded under that name
        self.holds: Dict[str, int] = {}                    # requests in flight
        self._calls: Dict[int, Tuple[Optional[torch.Tensor], Dict]] = {}      # thread -> the ids of its calls, and those spread over tokens

    def __getstate__(self):
        return {**self.__dict__, "_calls": {}}             # (a copy is in nobody's use)

    def _now(self) -> Tuple[Optional[torch.Tensor], Dict]:
        return self._calls.get(threading.get_ident(), (None, {}))

    def load(self, name: str, state: Mapping[str, torch.Tensor], alpha: float, rs: bool = False) -> int:
        """Put an adapter under ``name`` (in place of one that is not in use); returns its slot.  Its scale is ``alpha / rank``, or ``alpha / sqrt(rank)`` with ``rs``, by each
        layer's own rank; layers that it does not name are left as the model has them."""
        found = {}
        for key, t in state.items():
            path, _, part = key.rpartition(".")
            if part not in ("lora_a", "lora_b") or path not in self.layers:
                raise KeyError(f"adapter {name!r}: {key} belongs to no layer of the bank (their parts are lora_a and lora_b; a layer's magnitude cannot be served beside it)")
            found.setdefault(path, {})[part] = t
        for path, parts in found.items():
            layer, a, b = self.layers[path], parts.get("lora_a"), parts.get("lora_b")
            if a is None or b is None or a.dim() != 2 or b.shape != (layer.out_features, a.shape[0]) or a.shape[1] != layer.in_features or not 0 < a.shape[0] <= self.rank:
                raise ValueError(f"adapter {name!r}, {path}: lora_a [rank, {layer.in_features}] and lora_b [{layer.out_features}, rank] of rank up to {self.rank}")
        with _BANKS:
            self._free(name)
            slot = self.names.get(name)
            if slot is None:
                taken = set(self.names.values())
                slot = next((i for i in range(self.slots) if i not in taken), None)
                if slot is None:
                    raise RuntimeError(f"the bank's {self.slots} slots are taken: {sorted(self.names)}")
            with torch.no_grad():
                for path, layer in self.layers.items():
                    parts = found.get(path)
                    layer.a[slot].zero_()
                    layer.b[slot].zero_()
                    layer.scale[slot] = 0.0
                    if parts is not None:
                        r = parts["lora_a"].shape[0]
                        layer.a[slot, :r] = parts["lora_a"].to(layer.a)
                        layer.b[slot, :, :r] = parts["lora_b"].to(layer.b)
                        layer.scale[slot] = alpha / (math.sqrt(r) if rs else r)
            self.names[name] = slot
            self.version[name] = self.version.get(name, 0) + 1
            return slot

    def remove(self, name: str) -> None:
        with _BANKS:
            self._free(name)
            del self.names[name]

    def _free(self, name: str) -> None:
        if self.holds.get(name):
            raise RuntimeError(f"adapter {name!r} is in use by {self.holds[name]} requests")

    def acquire(self, name: str) -> int:
        """The adapter's slot, held for a request until ``release``."""
        with _BANKS:
            if name not in self.names:
                raise KeyError(f"no adapter {name!r}; loaded: {sorted(self.names)}")
            self.holds[name] = self.holds.get(name, 0) + 1
            return self.names[name]

    def release(self, name: str) -> None:
        with _BANKS:
            self.holds[name] -= 1

    @contextmanager
    def using(self, ids: Optional[torch.Tensor]):
        """Rows' adapters (int32 ``[rows]`` on the model's device, below 0: none) for this thread's calls inside.  The tensor is read when they run: a captured call follows its
        values."""
        if ids is not None and (ids.dtype != torch.int32 or ids.dim() != 1):
            raise TypeError(f"one int32 id a row, got {ids.dtype} {tuple(ids.shape)}")
        thread = threading.get_ident()
        before = self._calls.get(thread)
        self._calls[thread] = (ids, {})
        try:
            yield self
        finally:
            if before is None:
                del self._calls[thread]
            else:
                self._calls[thread] = before

    def ids_for(self, shape) -> Optional[torch.Tensor]:
        """The ids of tokens ``[rows, ...]``."""
        ids, wide = self._now()
        if ids is None:
            return None
        shape = tuple(shape)
        if not shape or shape[0] != ids.shape[0]:
            raise ValueError(f"adapters of {ids.shape[0]} rows in a call of {shape}")
        spread = ids.view(-1, *(1,) * (len(shape) - 1)).expand(shape)
        if spread.numel() == ids.numel():
            return ids.view(shape)
        # what the layers of one call share: not once the ids have changed, not across streams, and a captured call makes its own
        if ids.is_inference() or (ids.is_cuda and torch.cuda.is_current_stream_capturing()):
            return spread.contiguous()
        key = (shape, ids._version, torch.cuda.current_stream(ids.device).cuda_stream if ids.is_cuda else 0)
        if key not in wide:
            wide.clear()
            wide[key] = spread.contiguous()
        return wide[key]
