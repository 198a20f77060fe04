"""Activations of the gated linear layers over their whole range, relative to their own size: far below zero they are small,
and as exact as anywhere."""

import math

import pytest
import torch

from flowmatching_lthc_amd import ops_branch, ops_int8

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24  # a rounding to fp32


def gates(dtype):
    """Gates from -9 to 9, as `dtype` holds them."""
    g = torch.linspace(-9, 9, 3601, dtype=torch.float64)
    return torch.cat([g, torch.tensor([-5.0, -5.4, -5.7, -8.0, 0.0])]).to(dtype).to(DEV)


def act64(g, name):
    """(act, its slope, roundings of 2^-24 that act and the slope's two terms may be off by) in 64 bits.

    erfc((-g) sqrt(1/2)): the argument has two roundings, which its logarithm feels (1 + g^2)-fold; the function itself and
    the products around it are within 8.  exp(-g^2 / 2): three roundings, g^2 / 2-fold, and 4.  1 / (1 + exp(-p)): its
    argument's are felt |p|-fold, 2 for silu and up to 7 for the cubic; the power, the reciprocal and the products 8."""
    if name == "silu":
        s, p, dp, n = torch.sigmoid(g), g, 1.0, 2
    elif name == "gelu_tanh":
        k = 2 * math.sqrt(2 / math.pi)
        p, dp, n = k * (g + 0.044715 * g**3), k * (1 + 3 * 0.044715 * g * g), 7
        s = torch.sigmoid(p)
    else:
        c = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        t = g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        off = 8 + 2 * (1 + g * g)
        return g * c, c + t, (g * c).abs() * off, c * off + t.abs() * (4 + 3 * g * g / 2)
    off = 8 + n * p.abs()
    t = g * s * (1 - s) * dp
    # 1 - s is off by s's roundings where s is close to 1
    return g * s, s + t, (g * s).abs() * off, s * off + t.abs() * (2 * off + 8) + (g * s * dp).abs() * s * off


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half a step of fp16's subnormal numbers; bf16 and fp32 hold every value here."""
    return 2.0**-25 if dtype == torch.float16 else 0.0


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 20, 70, 700])
def test_int8_gated_linear(act, dtype, m):
    # with a weight of zeros the projections are the bias itself
    g = gates(torch.float32)
    bias = torch.cat([g, torch.full_like(g, 0.75)])
    q, w = (torch.zeros(r, 32, device=DEV, dtype=torch.int8) for r in (m, 2 * len(g)))
    y = ops_int8.int8_gated_linear(q, torch.ones(m, device=DEV), w, torch.ones(2 * len(g), device=DEV), bias, act, dtype)
    a, _, off, _ = act64(g.double(), act)
    want, bound = 0.75 * a, 0.75 * off * U
    bound = bound + half_step(dtype) * (want.abs() + bound) + least(dtype)
    assert bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 20, 70, 700])
def test_gated_linear_and_its_gradients(act, dtype, m):
    g = gates(dtype)
    f = len(g)
    bias = torch.cat([g, torch.full_like(g, 0.75)])
    x, w = torch.zeros(m, 64, device=DEV, dtype=dtype), torch.zeros(2 * f, 64, device=DEV, dtype=dtype)
    a, d, ea, ed = act64(g.double(), act)
    y = ops_branch.gated_linear(x, w, bias, act)
    rounded = lambda v, e: e + half_step(dtype) * (v.abs() + e) + least(dtype)  # noqa: E731
    assert bool(((y.double() - 0.75 * a).abs() <= rounded(0.75 * a, 0.75 * ea * U)).all())
    dy = torch.zeros(m, f, device=DEV, dtype=dtype)
    dy[m // 2] = 1
    db = ops_branch.gated_linear_backward(dy, x, w, bias, act, True, True, True)[2].double()
    for got, want, e in ((db[:f], 0.75 * d, 0.75 * ed), (db[f:], a, ea)):
        assert bool(((got - want).abs() <= rounded(want, e * U)).all())
