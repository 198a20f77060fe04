"""Operators of a transformer branch's inference in 8 bits, as cases that can be timed and checked.

* ``quant``: rows in 8-bit integers with a scale each, and their values back (``ops_int8.quantize_rows``,
  ``ops_int8.dequantize_rows``);
* ``norm``: RMS norm with the residual's addition, a gate and a modulation, its output in 8 bits with a scale for each token
  (``ops_int8.norm_quantize``);
* ``linear``: a matrix product in 8-bit integers with scales for each token and channel (``ops_int8.int8_linear``);
* ``gated``: both projections of a gated feed-forward as such a product, the activation and the product of the two
  (``ops_int8.int8_gated_linear``).

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits, rounded once at the end; where it is
true, it calls the package.  What is held in 8 bits is returned as the values it stands for, in 16 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
TINY = 2.0**-126  # the smallest scale


def listed() -> list[dict]:
    return [
        # one sample's conditioning vector before an 8-bit layer: latency of a single row
        {"name": "quant_one_row", "kind": "quant", "M": 1, "C": 768, "dtype": "bf16"},
        # the hidden activations of a sampler's batch (64 workspaces of 256 tokens) before the feed-forward's last layer
        {"name": "quant_hidden_b64", "kind": "quant", "M": 16384, "C": 2048, "dtype": "bf16"},
        # the fp32 weight of the 512-pixel configuration's feed-forward, whose hidden width no tile divides: once for each model
        {"name": "quant_weight_fp32", "kind": "quant", "M": 1024, "C": 2730, "dtype": "fp32"},
        # one token of each of three sequences, residual without gate or modulation, fp16
        {"name": "norm_one_token", "kind": "norm", "B": 3, "N": 1, "C": 768, "gate": False, "mod": False, "residual": True, "keep": "sum", "dtype": "fp16"},
        # the second pre-norm of LTHC-B/4's branch at a sampler's batch: gated residual and modulation for each sample
        {"name": "norm_b64", "kind": "norm", "B": 64, "N": 256, "C": 768, "gate": True, "mod": True, "residual": True, "keep": "update", "dtype": "bf16"},
        # odd lengths and channels, fp32, a modulation and no residual
        {"name": "norm_ragged_fp32", "kind": "norm", "B": 7, "N": 413, "C": 1219, "gate": False, "mod": True, "residual": False, "keep": "none", "dtype": "fp32"},
        # the AdaLN head of eight samples: 768 channels to six modulations
        {"name": "linear_few_rows", "kind": "linear", "M": 8, "K": 768, "N": 4608, "bias": True, "dtype": "bf16"},
        # the qkv projection of a sampler's batch
        {"name": "linear_qkv_b64", "kind": "linear", "M": 16384, "K": 768, "N": 2304, "bias": True, "dtype": "bf16"},
        # the last layer of the 512-pixel configuration's feed-forward: 32 workspaces of 1024 tokens, hidden width 2730 in rows of 2736
        {"name": "linear_512px", "kind": "linear", "M": 32768, "K": 2736, "N": 1024, "bias": True, "dtype": "bf16"},
        # one sample's vector through a feed-forward of LTHC-B/4's width
        {"name": "gated_one_row", "kind": "gated", "M": 1, "K": 768, "F": 2048, "act": "silu", "bias": True, "dtype": "bf16"},
        # a few hundred rows of widths that no tile divides, no bias, fp16
        {"name": "gated_ragged_fp16", "kind": "gated", "M": 413, "K": 464, "F": 1219, "act": "gelu", "bias": False, "dtype": "fp16"},
        # the feed-forward of the 512-pixel configuration
        {"name": "gated_512px", "kind": "gated", "M": 32768, "K": 1024, "F": 2730, "act": "silu", "bias": True, "dtype": "bf16"},
    ]  # fmt: skip


MOST_PRODUCTS = 32768 * 1024 * 5460
MOST_VALUES = 16384 * 2048


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["quant", "norm", "linear", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "quant":
        C = _log(rng, 1, 8192)
        return {"kind": kind, "M": _log(rng, 1, min(65536, MOST_VALUES // C)), "C": C, "dtype": dtype}
    if kind == "norm":
        C, B = _log(rng, 8, 4096), _log(rng, 1, 64)
        residual, gate = rng.random() < 0.6, rng.random() < 0.5
        return {
            "kind": kind,
            "B": B,
            "N": _log(rng, 1, max(1, min(4096, MOST_VALUES // 2 // (B * C)))),
            "C": C,
            "gate": gate,
            "mod": rng.random() < 0.6,
            "residual": residual,
            "keep": rng.choice(["none"] + ["sum"] * residual + ["update"] * gate),
            "dtype": dtype,
        }
    K = 16 * _log(rng, 1, 256)
    if kind == "linear":
        N = _log(rng, 1, 6144)
        return {"kind": kind, "M": _log(rng, 1, min(32768, MOST_PRODUCTS // (K * N))), "K": K, "N": N, "bias": rng.random() < 0.7, "dtype": dtype}
    F = _log(rng, 1, 2730)
    return {
        "kind": kind,
        "M": _log(rng, 1, min(32768, MOST_PRODUCTS // (2 * K * F))),
        "K": K,
        "F": F,
        "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh"]),
        "bias": rng.random() < 0.7,
        "dtype": dtype,
    }


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, shape, dtype=torch.float32, std: float = 1.0) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device=DEV).mul_(std).to(dtype)


def _channels(gen, C: int) -> torch.Tensor:
    """The sizes of a transformer's channels: most alike, a few several times larger."""
    return torch.exp(0.5 * torch.randn(C, generator=gen, device=DEV)).clamp_(max=6.0)


def _int8_rows(gen, R: int, K: int, std: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(int8 [R, K], fp32 scales [R]) of normally distributed rows."""
    x = _randn(gen, (R, K), std=std)
    s = x.abs().amax(1) / 127
    return torch.round(x / s[:, None]).to(torch.int8), s


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, dt = case["kind"], DT[case["dtype"]]
    s = {"case": case, "dt": dt}
    if kind == "quant":
        s["x"] = (_randn(gen, (case["M"], case["C"])) * _channels(gen, case["C"])).to(dt)
    elif kind == "norm":
        B, N, C = case["B"], case["N"], case["C"]
        s["x"] = (_randn(gen, (B, N, C)) * _channels(gen, C)).to(dt)
        s["residual"] = (_randn(gen, (B, N, C), std=2.0) * _channels(gen, C)).to(dt) if case["residual"] else None
        s["weight"] = 1 + _randn(gen, (C,), std=0.1)
        # gate, shift and scale of a sample are parts of one row, as an AdaLN head gives them
        rows = _randn(gen, (B, 3 * C), dt, 0.3)
        gate, shift, scale = rows.chunk(3, dim=-1)
        s["gate"] = gate if case["gate"] else None
        s["shift"], s["scale"] = (shift, scale) if case["mod"] else (None, None)
    else:
        R = case["N"] if kind == "linear" else 2 * case["F"]
        s["q"], s["qs"] = _int8_rows(gen, case["M"], case["K"], 1.0)
        s["w"], s["ws"] = _int8_rows(gen, R, case["K"], case["K"] ** -0.5)
        s["bias"] = _randn(gen, (R,), std=0.1) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _half(dt: torch.dtype) -> torch.dtype:
    """The type that 8-bit values are returned in."""
    return torch.bfloat16 if dt == torch.float32 else dt


def _rows_to_8bit(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(int8 values, scales) of fp32 rows."""
    s = (y.abs().amax(-1) / 127).clamp(min=TINY)
    return torch.round(y / s.unsqueeze(-1)).to(torch.int8), s


def _act(g: torch.Tensor, act: str) -> torch.Tensor:
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_norm(s: dict):
    case, u = s["case"], s["x"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float().unsqueeze(1)
    t = u if s["residual"] is None else u + s["residual"].float()
    y = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * s["weight"]
    if s["scale"] is not None:
        y = y * (1 + s["scale"].float().unsqueeze(1)) + s["shift"].float().unsqueeze(1)
    q, qs = _rows_to_8bit(y)
    out = {"values": (q.float() * qs.unsqueeze(-1)).to(_half(s["dt"])), "scales": qs}
    if case["keep"] != "none":
        out["kept"] = (t if case["keep"] == "sum" else u).to(s["dt"])
    return out


@torch.no_grad()
def _plain(s: dict):
    case = s["case"]
    if case["kind"] == "quant":
        q, qs = _rows_to_8bit(s["x"].float())
        return {"values": (q.float() * qs.unsqueeze(-1)).to(_half(s["dt"])), "scales": qs}
    if case["kind"] == "norm":
        return _plain_norm(s)
    h = (s["q"].float() @ s["w"].float().t()) * s["qs"].unsqueeze(-1) * s["ws"]
    if s["bias"] is not None:
        h = h + s["bias"]
    if case["kind"] == "linear":
        return h.to(s["dt"])
    g, u = h.chunk(2, -1)
    return (_act(g, case["act"]) * u).to(s["dt"])


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------
@torch.no_grad()
def _own(s: dict):
    from flowmatching_lthc_amd import ops_int8

    case = s["case"]
    if case["kind"] == "quant":
        q, qs = ops_int8.quantize_rows(s["x"])
        return {"values": ops_int8.dequantize_rows(q, qs, case["C"], _half(s["dt"])), "scales": qs}
    if case["kind"] == "norm":
        kept, q, qs = ops_int8.norm_quantize(s["x"], s["weight"], EPS, s["residual"], s["gate"], s["shift"], s["scale"], case["keep"])
        out = {"values": ops_int8.dequantize_rows(q, qs, case["C"], _half(s["dt"])), "scales": qs}
        if case["keep"] != "none":
            out["kept"] = kept
        return out
    if case["kind"] == "linear":
        return ops_int8.int8_linear(s["q"], s["qs"], s["w"], s["ws"], s["bias"], s["dt"])
    return ops_int8.int8_gated_linear(s["q"], s["qs"], s["w"], s["ws"], s["bias"], case["act"], s["dt"])


def run(state: dict):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(what the rows' 8-bit values stand for, their scales)."""
    largest = torch.maximum(y.max(-1, keepdim=True).values, -y.min(-1, keepdim=True).values)
    step = torch.clamp(largest / 127.0, min=TINY)
    return torch.round(y / step) * step, step[..., 0]


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f64 = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    kind = case["kind"]
    if kind == "quant":
        values, scales = _exact_rows(f64["x"])
        return {"values": values, "scales": scales}
    if kind == "norm":
        update = f64["x"] * f64["gate"][:, None, :] if case["gate"] else f64["x"]
        total = update + f64["residual"] if case["residual"] else update
        rms = torch.sqrt(torch.sum(total**2, dim=-1, keepdim=True) / case["C"] + EPS)
        y = total / rms * f64["weight"]
        if case["mod"]:
            y = y + y * f64["scale"][:, None, :] + f64["shift"][:, None, :]
        values, scales = _exact_rows(y)
        out = {"values": values, "scales": scales}
        if case["keep"] != "none":
            out["kept"] = total if case["keep"] == "sum" else update
        return out
    x, w = f64["q"] * f64["qs"][:, None], f64["w"] * f64["ws"][:, None]
    h = torch.matmul(x, w.t().contiguous())
    if case["bias"]:
        h += f64["bias"]
    if kind == "linear":
        return h
    F = case["F"]
    g, u = h[:, :F], h[:, F:]
    if case["act"] == "silu":
        a = g * torch.sigmoid(g)
    elif case["act"] == "gelu":
        a = g * 0.5 * torch.erfc(-g / math.sqrt(2.0))
    else:
        a = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g**3))
    return a * u


def work(case: dict) -> dict:
    e = 4 if case["dtype"] == "fp32" else 2
    kind = case["kind"]
    if kind == "quant":
        n = case["M"] * case["C"]
        return {"bytes": n * (e + 2) + 4 * case["M"], "flops": 3 * n}
    if kind == "norm":
        rows, C = case["B"] * case["N"], case["C"]
        n = rows * C
        moved = n * e * (1 + case["residual"] + (case["keep"] != "none")) + 2 * n + 4 * rows
        per_sample = case["gate"] + 2 * case["mod"]
        return {"bytes": moved + 4 * C + per_sample * case["B"] * C * e, "flops": 10 * n}
    M, K = case["M"], case["K"]
    N = case["N"] if kind == "linear" else 2 * case["F"]
    out = case["N"] if kind == "linear" else case["F"]
    bias = 4 * N if case["bias"] else 0
    return {"bytes": M * K + N * K + 4 * (M + N) + bias + M * out * e, "flops": 2 * M * N * K}
