"""Frozen layers under adapters: an nn.Linear held in 8 bits, and the gated projection of a feed-forward block.

LyCORIS trains adapters on layers that never change, and it takes any nn.Linear subclass for a quantised one (bypass mode: the base weight
is never read, lycoris/modules/base.py:162-177).  ``Int8Linear`` is such a layer on ops.int8_linear, ``GatedLinear`` the block
`value * act(gate)` behind one projection on ops.gated_linear, with the adapters of the projection inside its kernel.  Replace the layers
first (``quantize_frozen``), then create the network: the adapters find the layers under the names they had.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops


def _stock(layer, forward):
    """is `forward` the class's own, on this layer?  (a layer whose adapter was restored keeps it as an instance attribute)"""
    return getattr(forward, "__func__", None) is type(layer).forward and getattr(forward, "__self__", None) is layer


def _hooked(layer):
    """does calling the layer do more than its forward?"""
    return any(getattr(layer, n, None) for n in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks"))


class Int8Linear(nn.Linear):
    """nn.Linear with its weight as 8-bit integers and one scale an output channel; frozen.

    ``weight_q`` [out, pitch] (rows padded to a pitch of 128 with zeros) and ``weight_scale`` [out] are buffers, the bias stays a
    parameter without a gradient.  ``weight`` is the weight as it is held, expanded to the layer's dtype on every access: for shapes, norms
    and export, not for writing (adapters cannot be merged into it)."""

    def __init__(self, in_features, out_features, bias=True, device=None, dtype=None):
        nn.Module.__init__(self)  # not nn.Linear's: there is no weight parameter
        self.in_features, self.out_features = in_features, out_features
        self.dtype = dtype or torch.get_default_dtype()
        self.register_buffer("weight_q", torch.zeros(out_features, (in_features + 127) // 128 * 128, dtype=torch.int8, device=device))
        self.register_buffer("weight_scale", torch.zeros(out_features, device=device))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=self.dtype), requires_grad=False) if bias else None

    @classmethod
    def from_linear(cls, layer: nn.Linear) -> "Int8Linear":
        """the layer `layer` is, with its weight quantised row by row (ops.int8_quantize)"""
        if type(layer) is not nn.Linear:
            raise TypeError(f"Int8Linear.from_linear takes a plain nn.Linear, got {type(layer).__name__}")
        w = layer.weight.detach()
        new = cls(layer.in_features, layer.out_features, bias=layer.bias is not None, device=w.device, dtype=w.dtype)
        q, scale = ops.int8_quantize(w)
        new.weight_q[:, :layer.in_features].copy_(q)
        new.weight_scale.copy_(scale)
        if layer.bias is not None:
            new.bias.data.copy_(layer.bias.detach())
        return new.train(layer.training)

    @property
    def wq(self):
        return self.weight_q[:, :self.in_features]

    @property
    def weight(self):
        return (self.wq.float() * self.weight_scale[:, None]).to(self.dtype)

    def _apply(self, fn, recurse=True):
        # .half() / .to(dtype) set the dtype the layer stands for; the scales stay the fp32 they were
        scale = self.weight_scale
        super()._apply(fn, recurse)
        self.dtype = fn(torch.zeros((), dtype=self.dtype, device=self.weight_q.device)).dtype
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def reset_parameters(self):
        raise NotImplementedError("Int8Linear is frozen")

    def forward(self, x):
        return ops.int8_linear(x, self.wq, self.weight_scale, self.bias)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, int8"


class GatedLinear(nn.Module):
    """value * act(gate) of the halves of `proj(x)`: the first half of a gated feed-forward block, in one kernel.

    ``proj`` is an nn.Linear or Int8Linear with 2 F outputs; the value half comes first unless ``gate_first``.  Adapters on ``proj`` (it
    keeps that name, which is also diffusers') are evaluated as its `base` operand when they are plain -- no dropout active, no weight
    decomposition, no hooks on proj -- and by calling proj itself otherwise; the result is the same function."""

    def __init__(self, proj: nn.Linear, act: str = "gelu", gate_first: bool = False):
        super().__init__()
        if not isinstance(proj, nn.Linear) or proj.out_features % 2:
            raise TypeError("GatedLinear takes a linear projection with an even number of outputs")
        if act not in ops.ACTIVATIONS:
            raise ValueError(f"act must be one of {sorted(ops.ACTIVATIONS)}, got {act!r}")
        self.proj, self.act, self.gate_first = proj, act, gate_first

    def _adapters(self):
        """the adapters on proj when their sum can be taken beside the projection, else None"""
        from .base import _ORIG, _STACK
        stack = getattr(self.proj, _STACK, [])
        if not stack:
            return [] if _stock(self.proj, self.proj.forward) else None
        if not _stock(self.proj, getattr(self.proj, _ORIG)) or self.proj.forward != stack[-1].forward:
            return None
        for a in stack:
            if not getattr(a, "additive", bool)():  # bool() is False: another package's adapter
                return None
        return stack

    def forward(self, x):
        proj, held = self.proj, isinstance(self.proj, Int8Linear)
        plain = type(proj) in (nn.Linear, Int8Linear) and not _hooked(proj) and not getattr(proj, "parametrizations", None)
        adapters = self._adapters() if plain else None
        if adapters is None:
            first, second = proj(x).chunk(2, -1)
            value, gate = (second, first) if self.gate_first else (first, second)
            a = nn.functional.silu(gate) if self.act == "silu" else nn.functional.gelu(gate, approximate="tanh" if self.act == "gelu_tanh" else "none")
            return value * a
        base = None
        for a in adapters:
            delta = a.bypass_forward_diff(x, scale=a.multiplier)
            base = delta if base is None else base + delta
        return ops.gated_linear(x, proj.wq if held else proj.weight, proj.bias, base, act=self.act, gate_first=self.gate_first,
                                weight_scale=proj.weight_scale if held else None)


def quantize_frozen(model: nn.Module, where=None) -> list:
    """Replace every plain nn.Linear of `model` (those for which ``where(name, layer)`` holds) by the Int8Linear it becomes; returns the
    names.  To be called before the network's adapters are created; a layer that already carries one, or hooks, is refused."""
    from .base import _STACK
    found = [(name, layer) for name, layer in model.named_modules() if name and type(layer) is nn.Linear and (where is None or where(name, layer))]
    for name, layer in found:
        if hasattr(layer, _STACK) or not _stock(layer, layer.forward) or getattr(layer, "parametrizations", None):
            raise RuntimeError(f"quantize_frozen: {name} already carries an adapter; quantise the model before the network is created")
        if _hooked(layer):
            raise RuntimeError(f"quantize_frozen: {name} carries hooks, which its replacement would lose; register them afterwards")
    made = {}  # a layer shared under several names stays shared
    for name, layer in found:
        made.setdefault(id(layer), None)
        if made[id(layer)] is None:
            made[id(layer)] = Int8Linear.from_linear(layer)
    for parent in list(model.modules()):
        for child, layer in list(parent._modules.items()):
            if layer is not None and id(layer) in made:
                parent._modules[child] = made[id(layer)]
    return [name for name, _ in found]
