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


@pytest.mark.parametrize("k", [5, 768, 2730])
@torch.no_grad()
def test_a_layer_refuses_other_widths(k):
    layer = Int8Linear.from_linear(linear(k, 6))
    assert layer(torch.zeros(2, k, device=DEV)).shape == (2, 6) and layer.gated(torch.zeros(2, k, device=DEV), "silu").shape == (2, 3)
    for wrong in (k - 1, k + 1, layer.weight.shape[1] + 16):
        for call in (layer, lambda x: layer.gated(x, "silu")):
            with pytest.raises(ValueError, match=f"of {k} channels"):
                call(torch.zeros(2, wrong, device=DEV))
