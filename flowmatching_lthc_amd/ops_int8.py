"""Inference of the workspace branch in 8-bit integers (gfx950 HIP kernels).

The branch's linear layers (qkv, proj, w12 and w3, local_thc.py:213-269) on rows of 8-bit integers with an fp32 scale
each, for activations (a token's row) and weights (a channel's row) alike:

* ``jit_thc::quantize_rows``, ``jit_thc::dequantize_rows``: rows in that form, and their values back;
* ``jit_thc::norm_quantize``: the branch's RMS norm with the residual's addition, its gate and its modulation
  (``gate_add_norm_modulate``, ``norm_modulate``), the output in that form;
* ``jit_thc::int8_linear``: a linear layer on such rows;
* ``jit_thc::int8_gated_linear``: both projections of a gated feed-forward, the activation and the product of the two.

They have no reference op.  Products are summed exactly in 32-bit integers; everything else is fp32, rounded once where a
result is stored.  Rounding to 8 bits has no gradient: a call that autograd would record raises.  ``quantized`` holds the
layers and the models' inference on them.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import ops_branch
from .ops import _fake, _refuse

TINY = 2.0**-126  # the smallest scale of a row


def padded(channels: int) -> int:
    """Elements of an 8-bit row of `channels` channels: a multiple of 16, the elements past the channels are zeros."""
    return -(-channels // 16) * 16


def _new_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """(q, scale) for the rows of x: rows of 512 elements and more begin at whole lines of memory, 128 bytes."""
    c = padded(x.shape[-1])
    q = x.new_empty((*x.shape[:-1], c if c < 512 else -(-c // 128) * 128), dtype=torch.int8)
    return q[..., :c], x.new_empty(x.shape[:-1], dtype=torch.float32)


def whole_lines(q: Tensor) -> Tensor:
    """8-bit rows [N, K] in the layout that quantize_rows gives them on the GPU: themselves, or a copy."""
    if not q.is_cuda or padded(q.shape[1]) != q.shape[1]:
        return q
    to, _ = _new_rows(q)
    return q if q.stride() == to.stride() else to.copy_(q)


# ---------------------------------------------------------------------------
# eager restatements: what the kernels' values are compared with
# ---------------------------------------------------------------------------
def quantize_rows_eager(x: Tensor) -> tuple[Tensor, Tensor]:
    x = x.float()
    top = x.abs().amax(-1)
    # by a tensor: a GPU tensor's quotient by a number is a product with the number's reciprocal
    scale = torch.where(top.isfinite(), (top / torch.full_like(top, 127)).clamp(min=TINY), torch.nan)
    q = torch.where(scale.isnan().unsqueeze(-1), 0, torch.round(x / scale.unsqueeze(-1)))
    return torch.nn.functional.pad(q, (0, padded(x.shape[-1]) - x.shape[-1])).to(torch.int8), scale


def norm_quantize_eager(
    x: Tensor, weight: Tensor, eps: float, residual: Tensor | None = None, gate: Tensor | None = None, shift: Tensor | None = None,
    scale: Tensor | None = None, keep: str = "none",
) -> tuple[Tensor, Tensor, Tensor]:
    row = lambda t: t.float().unsqueeze(1) if t.dim() == 2 else t.float()  # noqa: E731
    u = x.float() if gate is None else x.float() * row(gate)
    t = u if residual is None else u + residual.float()
    y = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    if scale is not None:
        y = y * (1 + row(scale)) + row(shift)
    kept = {"none": x.new_empty(0), "sum": t.to(x.dtype), "update": u.to(x.dtype)}[keep]
    return kept, *quantize_rows_eager(y)


def int8_linear_eager(q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None, dtype: torch.dtype) -> Tensor:
    y = (q.double() @ weight.double().t()).float() * q_scale.unsqueeze(-1) * weight_scale
    return (y if bias is None else y + bias.float()).to(dtype)


def int8_gated_linear_eager(
    q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None, activation: str, dtype: torch.dtype
) -> Tensor:
    g, u = int8_linear_eager(q, q_scale, weight, weight_scale, bias, torch.float32).chunk(2, dim=-1)
    return (ops_branch.ACTIVATIONS[activation](g) * u).to(dtype)


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
@torch.library.custom_op("jit_thc::quantize_rows", mutates_args=())
def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """(q, scale) of x [..., C], fp32, bf16 or fp16: scale = max(max |x| / 127, 2^-126) of each row, q = rint(x / scale) as
    int8 [..., padded(C)], zeros past C; rows of 512 elements and more lie a multiple of 128 apart.  Both quotients are
    fp32, ties go to the even integer.  A row with a NaN or an infinity has the scale NaN and q 0."""
    _refuse(x)


@_fake(quantize_rows)
def _(x):
    return _new_rows(x)


@torch.library.custom_op("jit_thc::dequantize_rows", mutates_args=())
def dequantize_rows(q: Tensor, scale: Tensor, channels: int, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The values q * scale of the first `channels` of int8 rows [..., K] in `dtype`, rounded once."""
    _refuse(q)


@_fake(dequantize_rows)
def _(q, scale, channels, dtype=torch.bfloat16):
    return q.new_empty((*q.shape[:-1], channels), dtype=dtype)


@torch.library.custom_op("jit_thc::norm_quantize", mutates_args=())
def norm_quantize(
    x: Tensor, weight: Tensor, eps: float, residual: Tensor | None = None, gate: Tensor | None = None, shift: Tensor | None = None,
    scale: Tensor | None = None, keep: str = "none",
) -> tuple[Tensor, Tensor, Tensor]:
    """(kept, q, scales) for x [..., C]: u = gate * x, t = residual + u, y = RMSNorm(t) * (1 + scale) + shift, (q, scales) =
    quantize_rows(y), one pass, nothing rounded in between.

    residual (x's shape and dtype), gate, and shift with scale are optional; gate, shift and scale are [C], or [B, C] for x
    [B, N, C], parts of wider rows among them.  kept is t (keep "sum"), u ("update") or empty ("none"), in x's dtype."""
    _refuse(x)


@_fake(norm_quantize)
def _(x, weight, eps, residual=None, gate=None, shift=None, scale=None, keep="none"):
    kept = x.new_empty((0,) if keep == "none" else x.shape)
    return kept, *_new_rows(x)


# ---------------------------------------------------------------------------
# linear layers
# ---------------------------------------------------------------------------
@torch.library.custom_op("jit_thc::int8_linear", mutates_args=())
def int8_linear(
    q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None = None, dtype: torch.dtype = torch.bfloat16
) -> Tensor:
    """(q weight^T) * q_scale * weight_scale + bias as `dtype` [..., N] for int8 rows q [..., K] and weight [N, K] with an fp32
    scale for each of their rows, as quantize_rows gives them: K a multiple of 16, up to 131056."""
    _refuse(q)


@_fake(int8_linear)
def _(q, q_scale, weight, weight_scale, bias=None, dtype=torch.bfloat16):
    return q.new_empty((*q.shape[:-1], weight.shape[0]), dtype=dtype)


@torch.library.custom_op("jit_thc::int8_gated_linear", mutates_args=())
def int8_gated_linear(
    q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None = None, activation: str = "silu",
    dtype: torch.dtype = torch.bfloat16,
) -> Tensor:
    """act(g) * u as `dtype` [..., F] for (g, u) = int8_linear with weight [2F, K], in fp32 up to the one rounding of the
    result; activation silu, gelu or gelu_tanh."""
    _refuse(q)


@_fake(int8_gated_linear)
def _(q, q_scale, weight, weight_scale, bias=None, activation="silu", dtype=torch.bfloat16):
    return q.new_empty((*q.shape[:-1], weight.shape[0] // 2), dtype=dtype)
