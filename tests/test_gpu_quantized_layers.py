"""The branch's 8-bit layers on the GPU: loading, widths, hooks."""

import pytest
import torch

from flowmatching_lthc_amd import model as M
from flowmatching_lthc_amd.quantized import Int8Linear

pytestmark = pytest.mark.gpu

DEV = "cuda"


def linear(k, n, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    layer = M.CastLinear(k, n)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * k**-0.5)
    return layer.to(DEV, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("assign", [False, True])
@torch.no_grad()
def test_a_layer_takes_a_linear_layers_state(dtype, assign):
    layer = linear(2730, 40, dtype=dtype)
    want = Int8Linear.from_linear(layer)
    x = torch.randn(3, 2730, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    for state in (layer.state_dict(), {n: t.cpu() for n, t in layer.state_dict().items()}, want.state_dict()):
        q = Int8Linear.from_linear(linear(2730, 40, seed=5))
        q.load_state_dict(state, assign=assign)
        q = q.to(DEV)
        assert q.weight.dtype == torch.int8 and q.weight_scale.dtype == q.bias.dtype == torch.float32
        assert torch.equal(q(x), want(x))
