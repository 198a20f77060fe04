"""The workspace branch's linear layers in 8-bit integers, for inference.

``quantize_branches(model)`` replaces qkv, proj, w12 and w3 (local_thc.py:213-269) of every branch of a model by
``Int8Linear``: weights in 8 bits with a scale for each channel, laid out once; activations in 8 bits with a scale for each
token, formed on the way.  A branch whose layers have that form runs the 8-bit operators where its elementwise chains feed
them: its norms write 8-bit rows (``ops_int8.norm_quantize``), w12 with the activation is one product
(``ops_int8.int8_gated_linear``).  Everything around the branches stays as it is.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn
from torch import Tensor

from . import ops_int8


class QuantizedRows(NamedTuple):
    """8-bit rows with their scales, and the dtype of a layer's result on them."""

    values: Tensor
    scale: Tensor
    dtype: torch.dtype


def _dtype(x: Tensor) -> torch.dtype:
    """The dtype of a linear layer's result on x: autocast's in its region."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


@torch.no_grad()
def _weight_rows(weight: Tensor) -> tuple[Tensor, Tensor]:
    """(values, scales) of a linear layer's weight, the same on the CPU and on the GPU."""
    w = weight.detach()
    w = w if w.dtype in (torch.float32, torch.bfloat16, torch.float16) else w.float()
    return ops_int8.quantize_rows(w) if w.is_cuda else ops_int8.quantize_rows_eager(w)


class Int8Linear(nn.Module):
    """nn.Linear for inference on 8-bit rows: weight int8 [out, in rounded up to a multiple of 16], weight_scale and bias fp32.

    forward takes activations (quantised here) or QuantizedRows and returns the activations' dtype (autocast's in its
    region).  weight_scale and bias stay fp32 when the module is converted to another dtype.  A state dict holds the 8-bit
    values with their scales; a linear layer's is taken too, and its weight quantised."""

    def __init__(self, weight: Tensor, weight_scale: Tensor, bias: Tensor | None, in_features: int) -> None:
        super().__init__()
        self.in_features = in_features
        self.out_features = weight.shape[0]
        self.register_buffer("weight", ops_int8.whole_lines(weight))
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, layer: nn.Linear) -> Int8Linear:
        return cls(*_weight_rows(layer.weight), None if layer.bias is None else layer.bias.detach().float().clone(), layer.in_features)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs) -> None:
        """A linear layer's weight is quantised on the way; 8-bit values and their scales come together."""
        names = [prefix + n for n in ("weight", "weight_scale")]
        w, scale = (state_dict.get(n) for n in names)
        if isinstance(w, Tensor) and w.is_floating_point():
            if w.shape != (self.out_features, self.in_features):
                error_msgs.append(f"{names[0]}: [{self.out_features}, {self.in_features}] expected for a linear layer's weight, got {list(w.shape)}")
                return
            on = w.device if self.weight.is_meta else self.weight.device
            state_dict = {**state_dict, **dict(zip(names, _weight_rows(w.to(on))))}
            bias = state_dict.get(prefix + "bias")
            if bias is not None:
                state_dict[prefix + "bias"] = bias.float()
        elif (w is None) != (scale is None) or (w is not None and getattr(w, "dtype", None) != torch.int8):
            error_msgs.append(f"{names[0]}: a linear layer's weight, or int8 values with {names[1]}, expected")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

    def _apply(self, fn, recurse: bool = True):
        kept = {n: b for n, b in (("weight_scale", self.weight_scale), ("bias", self.bias)) if b is not None}
        super()._apply(fn, recurse)
        for n, b in kept.items():  # where fn only changed the dtype, the fp32 values themselves
            moved = getattr(self, n)
            if moved.dtype != torch.float32:
                setattr(self, n, b.to(moved.device))
        self.weight = ops_int8.whole_lines(self.weight)
        return self

    def rows(self, x: Tensor | QuantizedRows) -> QuantizedRows:
        if isinstance(x, QuantizedRows):
            return x
        # 8-bit rows are padded to multiples of 16, and so other widths would pass the product's own check
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"Int8Linear of {self.in_features} channels: [..., {self.in_features}] expected, got {list(x.shape)}")
        return QuantizedRows(*ops_int8.quantize_rows(x), _dtype(x))

    def forward(self, x: Tensor | QuantizedRows) -> Tensor:
        q, scale, dtype = self.rows(x)
        return ops_int8.int8_linear(q, scale, self.weight, self.weight_scale, self.bias, dtype)

    def gated(self, x: Tensor | QuantizedRows, activation: str) -> Tensor:
        """act(g) * u of this layer's two halves (g, u)."""
        q, scale, dtype = self.rows(x)
        return ops_int8.int8_gated_linear(q, scale, self.weight, self.weight_scale, self.bias, activation, dtype)


def norm_rows(
    norm: nn.Module, x: Tensor, shift: Tensor, scale: Tensor, residual: Tensor | None = None, gate: Tensor | None = None, keep: str = "none"
) -> tuple[Tensor, QuantizedRows]:
    """(kept, modulate(norm(residual + gate * x), shift, scale) as 8-bit rows): ops_int8.norm_quantize of an RMSNorm."""
    kept, q, s = ops_int8.norm_quantize(x, norm.weight, norm.eps, residual, gate, shift, scale, keep)
    return kept, QuantizedRows(q, s, _dtype(x))


def quantize_branches(model: nn.Module) -> nn.Module:
    """Replaces the linear layers of every workspace branch of `model` by Int8Linear, in place, and returns the model.

    For inference: call the model under torch.no_grad().  The state dict holds 8-bit weights afterwards; one of the model as it
    was is taken too (Int8Linear).  A layer that is not a plain linear layer (hooks, a parametrization, another class) is refused."""
    from .model import SwiGLUFFN, WorkspaceAttention, _plain_projection

    found = [(m, n) for m in model.modules() if isinstance(m, WorkspaceAttention) for n in ("qkv", "proj")]
    found += [(m, n) for m in model.modules() if isinstance(m, SwiGLUFFN) for n in ("w12", "w3")]
    if not found:
        raise ValueError("the model has no workspace branch")
    for m, n in found:
        layer = getattr(m, n)
        if not (type(layer) is Int8Linear or _plain_projection(layer)):
            raise ValueError(f"{type(m).__name__}.{n} is not a plain linear layer: {type(layer).__name__}")
    for m, n in found:
        layer = getattr(m, n)
        if type(layer) is not Int8Linear:
            setattr(m, n, Int8Linear.from_linear(layer))
    return model
