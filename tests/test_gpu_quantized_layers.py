"""The branch's 8-bit layers on the GPU: loading, widths, hooks."""

import pytest
import torch

from flowmatching_lthc_amd import model as M
from flowmatching_lthc_amd.quantized import Int8Linear, quantize_branches

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


def branch(dim, heads, seed=1):
    torch.manual_seed(seed)
    b = M.WorkspaceSharedAdaLNBranch(dim, heads)
    with torch.no_grad():
        for n, p in b.named_parameters():
            p.copy_(1 + 0.1 * torch.randn_like(p) if "norm" in n else torch.randn_like(p) * (p.shape[-1] ** -0.5))
    return b.to(DEV).eval()


def doubled(norm, how):
    """Lets the norm's output be twice as large, by a hook or by a forward of its own."""
    if how == "hook":
        norm.register_forward_hook(lambda m, args, out: 2 * out)
    elif how == "pre-hook":  # sees what the norm takes
        seen = norm.__dict__.setdefault("seen", [])
        norm.register_forward_pre_hook(lambda m, args: seen.append(tuple(args[0].shape)))
    elif how == "forward":
        norm.forward = lambda x: 2 * M.RMSNorm.forward(norm, x)
    else:
        raise AssertionError(how)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("how", ["hook", "forward"])
@pytest.mark.parametrize("which", ["norm1", "norm2"])
@pytest.mark.parametrize("dim", [256, 2304])
@torch.no_grad()
def test_a_norm_that_is_hooked_or_replaced_runs(quantised, how, which, dim):
    got, want = (branch(dim, dim // 64) for _ in range(2))
    for b in (got, want):
        if quantised:
            quantize_branches(b)
        b.to(torch.bfloat16)
    rope = M.VisionRotaryEmbeddingFast(32, 8).to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    z = torch.randn(2, 64, dim, device=DEV, generator=gen).bfloat16()
    t6 = 0.3 * torch.randn(2, 6 * dim, device=DEV, generator=gen).bfloat16()
    plain = want(z, t6, rope)
    doubled(getattr(got, which), how)
    # the same sequence with twice the weight, every value but the weight's a power of two away: equal
    getattr(want, which).weight.mul_(2)
    doubled(getattr(want, which), "pre-hook")
    y = got(z, t6, rope)
    assert torch.equal(y, want(z, t6, rope)) and not torch.equal(y, plain)
    assert getattr(want, which).seen == [(2, 64, dim)]


@pytest.mark.parametrize("quantised", [False, True])
@torch.no_grad()
def test_a_norm_of_another_class_runs(quantised):
    b = branch(256, 4)
    if quantised:
        quantize_branches(b)
    b.norm1, b.norm2 = (torch.nn.LayerNorm(256, elementwise_affine=False) for _ in range(2))
    seen = []
    for n in (b.norm1, b.norm2):
        n.register_forward_hook(lambda m, args, out: seen.append(float(out.float().mean(-1).abs().max())))
    z, t6 = torch.randn(2, 64, 256, device=DEV) + 3, 0.3 * torch.randn(2, 6 * 256, device=DEV)
    assert b(z, t6, M.VisionRotaryEmbeddingFast(32, 8).to(DEV)).shape == z.shape
    assert len(seen) == 2 and max(seen) < 1e-5  # means are taken off


@pytest.mark.parametrize("quantised", [False, True])
@torch.no_grad()
def test_a_models_norms_that_are_hooked_run(quantised):
    torch.manual_seed(0)
    model = M.randomize_parameters(M.build_model("lthc_b4_velocity")).to(DEV).eval()
    if quantised:
        quantize_branches(model)
    gen = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.rand(s, generator=gen, device=DEV)  # noqa: E731
    x = r(2, 3, 256, 256) * 2 - 1, r(2), torch.randint(0, 1000, (2,), generator=gen, device=DEV)

    def call():
        with torch.autocast("cuda", torch.bfloat16):
            return model(*x).float()

    want = call()
    for which in ("norm1", "norm2"):
        norm = getattr(model.blocks[5].branch, which)
        seen = []
        handle = norm.register_forward_hook(lambda m, args, out: seen.append(out.shape))
        got = call()
        handle.remove()
        assert len(seen) == 1
        # the eager sequence rounds in other places: a few values pass to the next step of 8 or 16 bits
        assert float((got - want).norm()) <= 2.0**-6 * float(want.norm())
        handle = norm.register_forward_hook(lambda m, args, out: 0 * out)
        assert float((call() - want).norm()) > 2.0**-6 * float(want.norm())
        handle.remove()
    assert torch.equal(call(), want)
