"""A branch's training step on the operators for it together: rotary positions on q and k, the gated feed-forward, their
gradients, the clipping norm and the AdamW update with master weights and the moving average."""

import functools
import math

import pytest
import torch
import torch.nn.functional as F

from flowmatching_lthc_amd import model as M
from flowmatching_lthc_amd import ops_branch as OB
from flowmatching_lthc_amd import optim

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
B, N, C, H, D, FH = 3, 70, 96, 4, 24, 200
SECTIONS = (8, 8, 4)  # three axes, the last 4 channels of a head as they are
HYPER = dict(lr=1e-2, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.1)


def randn(shape, seed, std=1.0, dtype=BF16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


@functools.cache
def positions():
    n = torch.arange(N)
    return torch.stack([n // 35, n // 7 % 5, n % 7], -1).to(DEV)


@functools.cache
def frequencies():
    return torch.cat([100.0 ** (-torch.arange(0, s, 2, dtype=torch.float64) / s) for s in SECTIONS]).to(DEV)


def parameters():
    shapes = [(3 * H * D, C), (2 * FH, C), (2 * FH,), (C, FH)]
    return [torch.nn.Parameter(randn(s, i, 0.1 if len(s) == 1 else s[-1] ** -0.5)) for i, s in enumerate(shapes)]


def rotate(x, pos, freq):
    """The rotation in x's precision, pairs adjacent."""
    axis = torch.repeat_interleave(torch.arange(len(SECTIONS), device=x.device), torch.tensor(SECTIONS, device=x.device) // 2)
    angle = (pos.double()[..., axis] * freq).to(x.dtype)[:, None]  # [N, 1, pairs]
    R = sum(SECTIONS)
    a, b = x[..., :R:2], x[..., 1:R:2]
    cos, sin = angle.cos(), angle.sin()
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., R:]], -1)


def branch(x, params, own):
    qkv_w, gate_w, gate_b, out_w = params
    q, k, v = F.linear(x, qkv_w).view(B, N, 3, H, D).unbind(2)
    if own:
        q, k = OB.axial_rope(q, k, positions(), frequencies(), SECTIONS)
    else:
        q, k = rotate(q, positions(), frequencies()), rotate(k, positions(), frequencies())
    wide = torch.float32 if own else x.dtype  # the attention itself: fp32 products of contiguous operands
    q, k, v = (t.to(wide).transpose(1, 2).contiguous() for t in (q, k, v))
    p = (torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)).softmax(-1)
    x = x + torch.matmul(p, v).transpose(1, 2).reshape(B, N, C).to(x.dtype)
    if own:
        h = OB.gated_linear(x, gate_w, gate_b, "gelu_tanh")
    else:
        g, u = F.linear(x, gate_w, gate_b).chunk(2, -1)
        h = F.gelu(g, approximate="tanh") * u
    return x + F.linear(h, out_w)


def test_steps_of_a_branch_match_64_bits():
    """Gradients against the branch's in 64 bits from the same parameters: 16 tensors on the longest way (forward 6, backward
    10) are rounded to 16 bits, by 2^-8 of a value at most, and each is carried on with a factor of about one in norm: 16 x
    2^-8.  The update against its own gradients in 64 bits: fp32 arithmetic, 32 steps of 2^-24 of |p| and of the move, which
    is at most lr times 1 / sqrt(1 - b2) (the ratio of m and sqrt(v) after any gradients), 0.04 here."""
    print("case training step", flush=True)
    params = parameters()
    opt = optim.AdamW(params, **HYPER, master_weights=True, ema_decay=0.5, max_norm=0.05)
    m64 = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    v64 = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    master = [p.detach().double() for p in params]
    ema = [t.clone() for t in master]
    for t in range(1, 4):
        x = randn((B, N, C), 10 + t)
        dy = randn((B, N, C), 20 + t, 0.05)
        opt.zero_grad()
        branch(x, params, True).backward(dy)
        leaves = [p.detach().double().requires_grad_() for p in params]
        want = torch.autograd.grad(branch(x.double(), leaves, False), leaves, dy.double())
        for p, w in zip(params, want):
            assert float((p.grad.double() - w).norm()) <= 16 * 2**-8 * float(w.norm()), tuple(p.shape)
        norm = torch.stack([p.grad.double().norm() for p in params]).norm()
        assert float(norm) > 0.05
        opt.step()
        assert abs(float(opt.last_grad_norm) - float(norm)) <= 2**-22 * float(norm)
        b1, b2 = HYPER["betas"]
        for i, p in enumerate(params):
            g = p.grad.double() * (0.05 / (norm + 1e-6))
            m64[i] = m64[i] * b1 + g * (1 - b1)
            v64[i] = v64[i] * b2 + g * g * (1 - b2)
            denom = (v64[i] / (1 - b2**t)).sqrt() + HYPER["eps"]
            master[i] = master[i] * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] / (1 - b1**t) * m64[i] / denom
            ema[i] = ema[i] * 0.5 + master[i] * 0.5
            state = opt.state[p]
            bound = t * 32 * 2**-24 * (master[i].abs() + 0.04)
            assert bool(((state["master"].double() - master[i]).abs() <= bound).all())
            assert bool(((state["ema"].double() - ema[i]).abs() <= bound).all())
            assert torch.equal(p.detach(), state["master"].to(BF16))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(bits):
    print("case captured training step", bits, flush=True)
    x, dy = randn((B, N, C), 1), randn((B, N, C), 2, 0.05)

    def make():
        params = parameters()
        return params, optim.AdamW(params, **HYPER, state_bits=bits, master_weights=True, max_norm=0.05, capturable=True)

    def step(params, opt):
        grads = torch.autograd.grad(branch(x, params, True), params, dy)
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()

    eager, captured = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*captured)  # lays out the states
    torch.cuda.current_stream().wait_stream(side)
    step(*eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*captured)
    for t in range(3):
        x.copy_(randn(x.shape, 30 + t))
        dy.copy_(randn(dy.shape, 40 + t, 0.05))
        graph.replay()
        torch.cuda.synchronize()
        step(*eager)
        torch.cuda.synchronize()
        for p, q in zip(captured[0], eager[0]):
            assert torch.equal(p, q), t
            for key, value in captured[1].state[p].items():
                assert torch.equal(torch.as_tensor(value), torch.as_tensor(eager[1].state[q][key])), (t, key)


def test_the_model_trains_on_them():
    """The model with its feed-forwards fused and this optimizer: the first step's gradients, from equal weights, differ from
    the eager sequence's by its roundings (a feed-forward's 3 of 2^-8, on at most 2 depths and there and back), and every
    parameter takes AdamW's step."""
    print("case model training step", flush=True)
    kw = dict(input_size=32, patch_size=4, hidden_size=128, depth=2, num_heads=2, num_classes=10, bottleneck_dim=16, workspace_grid=2)
    nets = [M.randomize_parameters(M.SharedReadLocalTHCSharedAdaLNJiT(**kw), seed=3).to(DEV) for _ in range(2)]
    x = randn((2, 3, 32, 32), 5, dtype=torch.float32)
    t = torch.tensor([0.2, 0.7], device=DEV)
    y = torch.tensor([1, 7], device=DEV)
    grads = []
    for net, on in zip(nets, (False, True)):
        for mod in net.modules():
            if isinstance(mod, M.SwiGLUFFN):
                mod.fused_projections = on
        with torch.autocast("cuda", dtype=BF16):
            out = net(x, t, y)
        out.float().backward(torch.ones_like(out, dtype=torch.float32) / out.numel())
        grads.append([p.grad for p in net.parameters()])
    whole = [torch.cat([g.flatten().double() for g in gs if g is not None]) for gs in grads]
    assert float((whole[0] - whole[1]).norm()) <= 12 * 2**-8 * float(whole[0].norm())
    assert not torch.equal(*whole)
    net = nets[1]
    opt = optim.AdamW(net.parameters(), lr=1e-3, weight_decay=0.0, eps=1e-30, ema_decay=0.9)
    before = [p.detach().clone() for p in net.parameters()]
    opt.step()
    for p, q, e in zip(net.parameters(), before, opt.ema_params()):
        if p.grad is None:
            assert torch.equal(p, q)
            continue
        # the first step moves by lr sign(g), where g^2 does not vanish in fp32
        moved = torch.where(p.grad.abs() > 1e-15, -1e-3 * p.grad.sign(), 0.0)
        some = p.grad.abs() > 1e-15
        assert bool((((p - q) - moved).abs() <= 2**-20 * q.abs() + 1e-3 * 2**-18)[some].all())
        assert bool(((e - (0.9 * q + 0.1 * p)).abs() <= 2**-22 * (q.abs() + 1e-3)).all())
