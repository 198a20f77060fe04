"""Operators of a transformer branch's training step, as cases that can be timed and checked.

* ``gated_linear``: both projections of a gated feed-forward, the activation and the product (``ops_branch``);
* ``axial_rope``: rotary positions with several axes, on q and k (``ops_branch``);
* ``adamw``: an AdamW step over many tensors at once with clipping by the global norm, fp32 master weights and the
  moving average of the weights, its states in 32 or in 8 bits (``optim``).

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits, rounded once at the end
(angles of positions in 64 bits); where it is true, it calls the package.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
RUN = 256  # elements of an 8-bit state that share a scale


def listed() -> list[dict]:
    return [
        # one sample's conditioning vector through a feed-forward of LTHC-B/4's width: latency of a single row
        {"name": "ffn_one_row", "kind": "ffn", "M": 1, "C": 768, "F": 2048, "act": "silu", "bias": True, "dtype": "bf16", "train": False},
        # a few hundred rows of a width that no tile divides, no bias, fp16
        {"name": "ffn_ragged_fp16", "kind": "ffn", "M": 413, "C": 456, "F": 1219, "act": "gelu", "bias": False, "dtype": "fp16", "train": False},
        # a sampler's batch: 64 workspaces of 256 tokens
        {"name": "ffn_fwd_b64", "kind": "ffn", "M": 16384, "C": 768, "F": 2048, "act": "silu", "bias": True, "dtype": "bf16", "train": False},
        # a training step's batch on one GPU
        {"name": "ffn_train_b32", "kind": "ffn", "M": 8192, "C": 768, "F": 2048, "act": "silu", "bias": True, "dtype": "bf16", "train": True},
        # the 512-pixel configuration in training: 32 workspaces of 1024 tokens, 1024 channels, hidden width 2730
        {"name": "ffn_train_512px", "kind": "ffn", "M": 32768, "C": 1024, "F": 2730, "act": "silu", "bias": True, "dtype": "bf16", "train": True},
        # one new token for each of a few sequences, fewer key heads than query heads, a far position
        {"name": "rope_one_token", "kind": "rope", "B": 8, "N": 1, "Hq": 16, "Hk": 4, "D": 128, "sections": "32,48,48", "pairs": "interleaved", "layout": "bnhd", "pos": "far", "dtype": "bf16", "train": False},
        # LTHC-B/4's attention at its batch: rows and columns of the 16x16 workspace, q and k inside the qkv projection
        {"name": "rope_image_b64", "kind": "rope", "B": 64, "N": 256, "Hq": 12, "Hk": 12, "D": 64, "sections": "32,32", "pairs": "interleaved", "layout": "qkv", "pos": "grid", "dtype": "bf16", "train": False},
        # video tokens (time, height, width) in training, two clips of 16384 tokens
        {"name": "rope_video_train", "kind": "rope", "B": 2, "N": 16384, "Hq": 16, "Hk": 16, "D": 128, "sections": "32,48,48", "pairs": "interleaved", "layout": "bnhd", "pos": "video", "dtype": "bf16", "train": True},
        # an odd length, a partly rotated head of an odd width, halves, heads outside tokens, fractional positions
        {"name": "rope_ragged_fp32", "kind": "rope", "B": 3, "N": 1357, "Hq": 5, "Hk": 1, "D": 84, "sections": "20,26,18", "pairs": "halves", "layout": "bhnd", "pos": "fraction", "dtype": "fp32", "train": True},
        # fine-tuning a handful of small odd tensors: launches and calls count
        {"name": "adamw_small", "kind": "adamw", "sizes": "odd", "count": 40, "width": 96, "param": "fp32", "grad": "fp32", "bits": 32, "master": False, "ema": False, "clip": True},
        # LTHC-B/4's parameters: 12 blocks of 768 channels, fp32, with clipping and the moving average of the weights
        {"name": "adamw_b4", "kind": "adamw", "sizes": "model", "count": 12, "width": 768, "param": "fp32", "grad": "fp32", "bits": 32, "master": False, "ema": True, "clip": True},
        # the weight matrices of four blocks of 960 channels in bf16 with fp32 master weights, states in 8 bits
        {"name": "adamw_8bit", "kind": "adamw", "sizes": "matrices", "count": 4, "width": 960, "param": "bf16", "grad": "bf16", "bits": 8, "master": True, "ema": False, "clip": False},
    ]  # fmt: skip


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["ffn", "ffn", "rope", "rope", "adamw"])
    if kind == "ffn":
        C, F = 8 * _log(rng, 4, 144), _log(rng, 24, 2730)
        most = 32768 * 1024 * 2730 // (C * F)
        return {
            "kind": kind,
            "M": _log(rng, 1, min(32768, most)),
            "C": C,
            "F": F,
            "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh"]),
            "bias": rng.random() < 0.7,
            "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "train": rng.random() < 0.5,
        }
    if kind == "rope":
        axes = rng.randint(1, 4)
        sections = [2 * rng.randint(1, 16) for _ in range(axes)]
        Hq = rng.randint(1, 16)
        D = sum(sections) + 2 * rng.choice([0, 0, 0, 4, rng.randint(0, 12)])
        layout = rng.choice(["qkv", "bnhd", "bhnd"])
        most = 2 * 16384 * 16 * 128 // (Hq * D)
        B = _log(rng, 1, 64)
        return {
            "kind": kind,
            "B": B,
            "N": _log(rng, 1, max(1, min(16384, most // B))),
            "Hq": Hq,
            "Hk": Hq if layout == "qkv" else rng.randint(1, Hq),
            "D": D,
            "sections": ",".join(map(str, sections)),
            "pairs": rng.choice(["interleaved", "halves"]),
            "layout": layout,
            "pos": rng.choice(["video", "far", "fraction"]),
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "train": rng.random() < 0.5,
        }
    bits = rng.choice([32, 8])
    param = rng.choice(["fp32", "bf16", "fp16"])
    sizes = rng.choice(["odd", "matrices"] if bits == 8 else ["odd", "matrices", "model"])
    return {
        "kind": kind,
        "sizes": sizes,
        "count": rng.randint(1, 24) if sizes == "odd" else rng.randint(1, 6),
        "width": _log(rng, 8, 1024) if sizes == "odd" else 8 * _log(rng, 4, 128),
        "param": param,
        "grad": rng.choice([param, "fp32"]),
        "bits": bits,
        "master": param != "fp32" and rng.random() < 0.7,
        "ema": rng.random() < 0.5,
        "clip": rng.random() < 0.5,
    }


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, shape, dtype=torch.float32, std: float = 1.0) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device=DEV).mul_(std).to(dtype)


def _shapes(case: dict) -> list[int]:
    """Element counts of a case's tensors."""
    n, c = case["count"], case["width"]
    if case["sizes"] == "odd":  # vectors and matrices of unlike, odd sizes
        return [(i * 37 % c + 1) * (1 if i % 3 == 0 else 2 * i + 1) for i in range(n)]
    hidden = int(4 * c * 2 / 3)
    matrices = [3 * c * c, c * c, 2 * hidden * c, hidden * c]
    if case["sizes"] == "matrices":
        return matrices * n
    block = [c, 3 * c * c, 3 * c, 64, 64, c * c, c, c, 2 * hidden * c, 2 * hidden, hidden * c, c, 16 * c]
    return [48 * 128, 128 * c, c, 256 * c, c, c * c, c, 1001 * c, 6 * c * c, 6 * c, *(block * n), 2 * c * c, 2 * c, 48 * c, 48]


def _views(flat: torch.Tensor, sizes: list[int]) -> list[torch.Tensor]:
    return list(flat.split(sizes))


def _prepare_adamw(case: dict, gen) -> dict:
    sizes = _shapes(case)
    total = sum(sizes)
    pdt, gdt = DT[case["param"]], DT[case["grad"]]
    p = _randn(gen, total, std=0.02)
    s = {
        "sizes": sizes,
        "p": p.to(pdt),
        "g": _randn(gen, total, gdt, 1e-3),
        # a run's 1000th step, with a learning rate that moves the weights visibly within one pass
        "hyper": {"step": 1000, "lr": 1e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.05},
    }
    m, v = _randn(gen, total, std=3e-4), _randn(gen, total, std=1e-3).square_()
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        got = [_quantised(a, b) for a, b in zip(_views(m, sizes), _views(v, sizes))]
        s["m8"], s["v8"], s["scales"] = (list(t) for t in zip(*got))
    if case["master"]:
        s["master"] = p
    if case["ema"]:
        s["ema"] = p + _randn(gen, total, std=1e-4)
    s["max_norm"] = 1e-3 * math.sqrt(total) * 0.7  # the norm of these gradients is above it
    # what a training loop hands over: its tensors one by one, views of the flat buffers
    s["views"] = {k: _views(s[k], sizes) for k in ("p", "g", "m", "v", "master", "ema") if k in s}
    return s


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    if kind == "adamw":
        return {"case": case, **_prepare_adamw(case, gen)}
    dt = DT[case["dtype"]]
    if kind == "ffn":
        M, C, F = case["M"], case["C"], case["F"]
        s = {
            "case": case,
            "x": _randn(gen, (M, C), dt),
            "w": _randn(gen, (2 * F, C), dt, C**-0.5),
            "b": _randn(gen, (2 * F,), dt, 0.1) if case["bias"] else None,
        }
        if case["train"]:
            s["dy"] = _randn(gen, (M, F), dt, 1e-2)
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["w"], s["b"]) if t is not None]
        return s
    B, N, Hq, Hk, D = (case[k] for k in ("B", "N", "Hq", "Hk", "D"))
    sections = [int(t) for t in case["sections"].split(",")]
    A = len(sections)
    if case["layout"] == "qkv":
        qkv = _randn(gen, (B, N, 3, Hq, D), dt)
        q, k = qkv[:, :, 0], qkv[:, :, 1]
    elif case["layout"] == "bnhd":
        q, k = _randn(gen, (B, N, Hq, D), dt), _randn(gen, (B, N, Hk, D), dt)
    else:  # [B, H, N, D] in memory
        q, k = (_randn(gen, (B, H, N, D), dt).transpose(1, 2) for H in (Hq, Hk))
    token = torch.arange(N, device=DEV)
    if case["pos"] == "grid":  # one map for the batch: row and column of a square grid
        side = math.isqrt(N)
        positions = torch.stack([token // side, token % side], -1)
    elif case["pos"] == "video":  # one map for each sample: frames of 32 x 32 that begin at different times
        axes = torch.stack([token // 1024, token // 32 % 32, token % 32, token], -1)[:, :A]
        start = torch.randint(0, 4096, (B, 1, A), generator=gen, device=DEV)
        positions = axes + start
    elif case["pos"] == "far":
        positions = torch.randint(0, 1 << 20, (B, N, A), generator=gen, device=DEV)
    else:
        positions = torch.rand((N, A), generator=gen, device=DEV) * 100
    # the angles' speeds, as a module keeps them: theta^(-2 j / section) for each axis
    inv = [10000.0 ** (-2.0 * torch.arange(n // 2, dtype=torch.float64) / n) for n in sections]
    s = {"case": case, "q": q, "k": k, "positions": positions, "inv_freq": torch.cat(inv).to(DEV), "sections": sections}
    if case["train"]:
        s["dq"], s["dk"] = _randn(gen, q.shape, dt), _randn(gen, k.shape, dt)
        s["leaves"] = [q.requires_grad_(), k.requires_grad_()]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _act(g: torch.Tensor, act: str) -> tuple[torch.Tensor, torch.Tensor]:
    """The activation and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    a, c = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (g + c * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * c * g * g)


@torch.no_grad()
def _plain_ffn(s: dict):
    x, w = s["x"].float(), s["w"].float()
    h = x @ w.t()
    if s["b"] is not None:
        h = h + s["b"].float()
    g, u = h.chunk(2, -1)
    a, da = _act(g, s["case"]["act"])
    dt = s["x"].dtype
    y = (a * u).to(dt)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    dh = torch.cat([dy * u * da, dy * a], -1)
    out = [y, (dh @ w).to(dt), (dh.t() @ x).to(dt)]
    return out + ([dh.sum(0).to(dt)] if s["b"] is not None else [])


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, R: int, interleaved: bool) -> torch.Tensor:
    head = x[..., :R].float()
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = head[..., : R // 2], head[..., R // 2 :]
        out = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([out.to(x.dtype), x[..., R:]], -1)


@torch.no_grad()
def _plain_rope(s: dict):
    sections = s["sections"]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections) // 2).to(DEV)
    ang = s["positions"].double()[..., axis] * s["inv_freq"]  # [(B,) N, R / 2]
    cos, sin = ang.cos().float().unsqueeze(-2), ang.sin().float().unsqueeze(-2)
    R, inter = sum(sections), s["case"]["pairs"] == "interleaved"
    out = [_rotate(s[t], cos, sin, R, inter) for t in ("q", "k")]
    if s["case"]["train"]:
        out += [_rotate(s[t], cos, -sin, R, inter) for t in ("dq", "dk")]
    return out


def _blocks(t: torch.Tensor) -> torch.Tensor:
    """The values in runs that share a scale, the last one filled with zeros."""
    return torch.nn.functional.pad(t, (0, -t.numel() % RUN)).view(-1, RUN)


def _quantised(m: torch.Tensor, v: torch.Tensor):
    """(codes of m, codes of v, their scales [2, runs]): m = A c|c| / 127^2, v = B (c / 255)^4."""
    mb, vb = _blocks(m), _blocks(v)
    a, b = mb.abs().amax(1, keepdim=True), vb.amax(1, keepdim=True)
    rm = torch.where(a > 0, mb.abs() / a, 0.0)
    rv = torch.where(b > 0, vb / b, 0.0)
    cm = torch.round(torch.sqrt(rm) * 127.0) * torch.sign(mb)
    cv = torch.round(torch.sqrt(torch.sqrt(rv)) * 255.0)
    cv = torch.where(vb > 0, cv.clamp(min=1.0), 0.0)
    n = m.numel()
    return cm.to(torch.int8).view(-1)[:n].clone(), cv.to(torch.uint8).view(-1)[:n].clone(), torch.cat([a, b], 1).t().contiguous()


def _values(cm: torch.Tensor, cv: torch.Tensor, scales: torch.Tensor):
    n = cm.numel()
    t, r = _blocks(cm).float() * (1 / 127), _blocks(cv).float() * (1 / 255)
    m = scales[0, :, None] * (t * t.abs())
    r = r * r
    v = scales[1, :, None] * (r * r)
    return m.view(-1)[:n], v.view(-1)[:n]


def _adamw_update(p, g, m, v, hyper: dict, clip):
    """(p, m, v) after the step, in the operands' precision."""
    (b1, b2), lr, step = hyper["betas"], hyper["lr"], hyper["step"]
    if clip is not None:
        g = g * clip
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    denom = torch.sqrt(v) / math.sqrt(1 - b2**step) + hyper["eps"]
    p = p * (1 - lr * hyper["weight_decay"]) - (lr / (1 - b1**step)) * (m / denom)
    return p, m, v


EMA_DECAY = 0.999


@torch.no_grad()
def _plain_adamw(s: dict):
    case, sizes = s["case"], s["sizes"]
    g = s["g"].float()
    out, clip = {}, None
    if case["clip"]:
        norm = (g.double() * g.double()).sum().sqrt().float()
        clip = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        out["norm"] = norm
    if case["bits"] == 8:
        old = [_values(*t) for t in zip(s["m8"], s["v8"], s["scales"])]
        m, v = (torch.cat(t) for t in zip(*old))
    else:
        m, v = s["m"], s["v"]
    w = s["master"] if case["master"] else s["p"]
    p, m, v = _adamw_update(w.float(), g, m, v, s["hyper"], clip)
    s["p"].copy_(p)
    out["p"] = s["p"]
    if case["master"]:
        out["master"] = s["master"].copy_(p)
    if case["ema"]:
        out["ema"] = s["ema"].copy_(s["ema"] * EMA_DECAY + p * (1 - EMA_DECAY))
    if case["bits"] == 8:
        out["m"], out["v"] = [], []
        for a, b, *to in zip(_views(m, sizes), _views(v, sizes), s["m8"], s["v8"], s["scales"]):
            for dst, src in zip(to, _quantised(a, b)):
                dst.copy_(src)
            a, b = _values(*to)
            out["m"].append(a)
            out["v"].append(b)
    else:
        out["m"], out["v"] = s["m"].copy_(m), s["v"].copy_(v)
    return out


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own_ffn(s: dict):
    from flowmatching_lthc_amd import ops_branch

    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            return ops_branch.gated_linear(s["x"], s["w"], s["b"], case["act"])
    y = ops_branch.gated_linear(s["x"], s["w"], s["b"], case["act"])
    return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]


def _own_rope(s: dict):
    from flowmatching_lthc_amd import ops_branch

    args = (s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], s["case"]["pairs"] == "interleaved")
    if not s["case"]["train"]:
        with torch.no_grad():
            return list(ops_branch.axial_rope(*args))
    q, k = ops_branch.axial_rope(*args)
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"]))]


def _own_adamw(s: dict):
    from flowmatching_lthc_amd import optim

    case, views = s["case"], s["views"]
    out, more = {}, {}
    if case["clip"]:
        out["norm"] = optim.grad_norm(views["g"])
        more = {"grad_norm": out["norm"], "max_norm": s["max_norm"]}
    if case["master"]:
        more["masters"] = views["master"]
    if case["ema"]:
        more.update(emas=views["ema"], ema_decay=EMA_DECAY)
    if case["bits"] == 8:
        optim.adamw_step(views["p"], views["g"], s["m8"], s["v8"], scales=s["scales"], **s["hyper"], **more)
        out["m"], out["v"] = optim.state_values(s["m8"], s["v8"], s["scales"])
    else:
        optim.adamw_step(views["p"], views["g"], views["m"], views["v"], **s["hyper"], **more)
        out["m"], out["v"] = s["m"], s["v"]
    out["p"] = s["p"]
    for name in ("master", "ema"):
        if case[name]:
            out[name] = s[name]
    return out


def run(s: dict):
    kind = s["case"]["kind"]
    if kind == "ffn":
        return _own_ffn(s) if own else _plain_ffn(s)
    if kind == "rope":
        return _own_rope(s) if own else _plain_rope(s)
    return _own_adamw(s) if own else _plain_adamw(s)


# ---------------------------------------------------------------------------
# work and the definition in 64 bits
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "ffn":
        M, C, F, e = case["M"], case["C"], case["F"], size[case["dtype"]]
        b = 2 * F if case["bias"] else 0
        nbytes = (M * C + 2 * F * C + b + M * F) * e
        if case["train"]:  # dy read; dx, dW, db written
            nbytes += (M * F + M * C + 2 * F * C + b) * e
        return {"bytes": nbytes, "flops": (12 if case["train"] else 4) * M * F * C}
    if kind == "rope":
        elems = case["B"] * case["N"] * (case["Hq"] + case["Hk"]) * case["D"]
        axes = case["sections"].count(",") + 1
        shared = 1 if case["pos"] in ("grid", "fraction") else case["B"]
        nbytes = 2 * elems * size[case["dtype"]] * (2 if case["train"] else 1)
        return {"bytes": nbytes + 8 * shared * case["N"] * axes, "flops": 3 * elems * (2 if case["train"] else 1)}
    p, g = size[case["param"]], size[case["grad"]]
    each = g + (p + 8 if case["master"] else 2 * p)  # the gradient; the parameter, or master weights and its copy
    each += 16 if case["bits"] == 32 else 4 + 8  # the states, read and written; in 8 bits, their values too
    each += 8 if case["ema"] else 0
    each += g if case["clip"] else 0  # the norm comes before the step
    return {"bytes": each * sum(_shapes(case)), "flops": 20 * sum(_shapes(case))}


def _exact_ffn(s: dict):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    F = w.shape[0] // 2
    g, u = x @ w[:F].t(), x @ w[F:].t()
    if s["b"] is not None:
        g, u = g + s["b"].detach()[:F].double(), u + s["b"].detach()[F:].double()
    act = {
        "silu": torch.nn.functional.silu,
        "gelu": torch.nn.functional.gelu,
        "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"),
    }[s["case"]["act"]]
    if not s["case"]["train"]:
        return act(g) * u
    with torch.enable_grad():
        g.requires_grad_()
        a = act(g)
        (slope,) = torch.autograd.grad(a.sum(), g)
    dy, a = s["dy"].double(), a.detach()
    dg, du = dy * u * slope, dy * a
    out = [a * u, dg @ w[:F] + du @ w[F:], torch.cat([dg.t() @ x, du.t() @ x])]
    return out + ([torch.cat([dg.sum(0), du.sum(0)])] if s["b"] is not None else [])


def _exact_rope(s: dict):
    def turned(x, sign):
        """Each pair of channels as a complex number, times e^(i angle)."""
        R = sum(s["sections"])
        axis = [a for a, n in enumerate(s["sections"]) for _ in range(n // 2)]
        ang = torch.stack([s["positions"][..., a].double() * f for a, f in zip(axis, s["inv_freq"])], -1)
        ang = sign * (ang if ang.dim() == 3 else ang[None])[:, :, None]
        first, second = (slice(0, R, 2), slice(1, R, 2)) if s["case"]["pairs"] == "interleaved" else (slice(0, R // 2), slice(R // 2, R))
        x = x.detach().double()
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.polar(torch.ones_like(ang), ang)
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out = [turned(s["q"], 1), turned(s["k"], 1)]
    return out + ([turned(s["dq"], -1), turned(s["dk"], -1)] if s["case"]["train"] else [])


def _exact_adamw(s: dict):
    case, h = s["case"], s["hyper"]
    g = s["g"].double()
    out = {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, s["max_norm"] / (float(out["norm"]) + 1e-6))
    if case["bits"] == 8:
        old = []
        for cm, cv, scales in zip(s["m8"], s["v8"], s["scales"]):
            run = torch.arange(cm.numel(), device=DEV) // RUN
            cm, cv = cm.double() / 127, cv.double() / 255
            old.append((scales[0].double()[run] * cm * cm.abs(), scales[1].double()[run] * cv**4))
        m, v = (torch.cat(t) for t in zip(*old))
    else:
        m, v = s["m"].double(), s["v"].double()
    b1, b2 = h["betas"]
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    p = (s["master"] if case["master"] else s["p"]).double()
    step = (m / (1 - b1 ** h["step"])) / ((v / (1 - b2 ** h["step"])).sqrt() + h["eps"])
    p = p - h["lr"] * (h["weight_decay"] * p + step)
    out["p"] = p
    if case["master"]:
        out["master"] = p
    if case["ema"]:
        out["ema"] = torch.lerp(p, s["ema"].double(), EMA_DECAY)
    # a moment in 8 bits next to the border of two codes has either one's value: no exact one
    out["m"], out["v"] = (m, v) if case["bits"] == 32 else ([None] * len(s["m8"]), [None] * len(s["v8"]))
    return out


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"ffn": _exact_ffn, "rope": _exact_rope, "adamw": _exact_adamw}[case["kind"]](s)
