"""Rows in 8-bit integers: values between two steps go where the division sends them."""

import pytest
import torch

from flowmatching_lthc_amd import ops_int8

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# a row for 4, 16 or 64 lanes, for a block by each number of loads a lane has, and longer than registers
WIDTHS = [9, 60, 250, 500, 768, 1219, 2048, 2730, 4097, 8192, 16000, 20011]


def rows_with_ties(m, c, dtype, seed=0):
    """Rows whose values lie at or next to halves of their steps, as far as the dtype allows, among ordinary ones; row i's
    size goes through the dtype's range."""
    gen = torch.Generator().manual_seed(seed + c)
    x = torch.randn(m, c, generator=gen, dtype=torch.float64)
    top = x.abs().amax(1, keepdim=True)
    half = (torch.randint(-127, 127, (m, c), generator=gen) + 0.5) / 127 * top
    x = torch.where(torch.rand(m, c, generator=gen) < 0.5, half, x)
    x[:, c // 2] = top[:, 0]
    info = torch.finfo(dtype)
    low = -140.0 if dtype != torch.float16 else -20.0  # subnormal rows among them
    high = torch.log2(torch.tensor(info.max, dtype=torch.float64)).item() - 4
    sizes = 2.0 ** torch.linspace(low, high, m, dtype=torch.float64).round()
    x = (x * sizes.unsqueeze(1)).to(dtype)
    x[0] = x[0].sign() * x[0].abs().amax() / 2  # halves of the largest value: 63.5 steps
    x[0, 0] = x[0, 0] * 2
    return x


def divided(x):
    """(q, scale) by the divisions, on the CPU."""
    x = x.float()
    scale = (x.abs().amax(-1) / torch.full(x.shape[:-1], 127.0)).clamp(min=ops_int8.TINY)
    return torch.round(x / scale.unsqueeze(-1).expand_as(x)).to(torch.int8), scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", WIDTHS)
def test_quantize_rows_divides(dtype, c):
    x = rows_with_ties(71, c, dtype)
    q, s = ops_int8.quantize_rows(x.to(DEV))
    want, scale = divided(x)
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q[:, :c].cpu(), want) and not q[:, c:].any()
    # and so a weight has the same 8-bit values whichever device it is quantised on
    eager, same = ops_int8.quantize_rows_eager(x)
    assert torch.equal(q.cpu(), eager) and torch.equal(s.cpu(), same)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", WIDTHS)
def test_norm_quantize_divides(dtype, c):
    # with a weight of zeros the norm's output is the shift itself
    shift = rows_with_ties(17, c, dtype, seed=1)
    x = torch.ones(17, 3, c, device=DEV, dtype=dtype)
    sh = shift.to(DEV)
    _, q, s = ops_int8.norm_quantize(x, torch.zeros(c, device=DEV), 1e-6, shift=sh, scale=torch.zeros_like(sh))
    want, scale = divided(shift)
    assert torch.equal(s.cpu(), scale.unsqueeze(1).expand(17, 3))
    assert torch.equal(q[..., :c].cpu(), want.unsqueeze(1).expand(17, 3, c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [60, 768, 2730])
def test_the_eager_rows_are_the_same_on_either_device(dtype, c):
    x = rows_with_ties(200, c, dtype, seed=2)
    q, s = ops_int8.quantize_rows_eager(x.to(DEV))
    want, scale = ops_int8.quantize_rows_eager(x)
    assert torch.equal(q.cpu(), want) and torch.equal(s.cpu(), scale)
