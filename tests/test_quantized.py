"""The branch's 8-bit layers on the CPU: their weights, and loading them."""

import copy

import pytest
import torch

from flowmatching_lthc_amd import model as M
from flowmatching_lthc_amd import ops_int8
from flowmatching_lthc_amd.checkpoint import checkpoint_state, load_model_state
from flowmatching_lthc_amd.quantized import Int8Linear, quantize_branches

NAME = "lthc_b4_velocity"


def linear(k, n, seed=0, bias=True):
    gen = torch.Generator().manual_seed(seed)
    layer = M.CastLinear(k, n, bias=bias)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * k**-0.5)
    return layer


def numbers(module):
    return {n: t.clone() for n, t in module.state_dict().items()}


def assert_same(a, b):
    assert a.keys() == b.keys()
    for n in a:
        assert a[n].dtype == b[n].dtype and torch.equal(a[n], b[n]), n


@pytest.fixture(scope="module")
def models():
    """(a model, its 8-bit form, another model's 8-bit form)."""
    out = []
    for seed in (1, 2):
        torch.manual_seed(seed)
        out.append(M.randomize_parameters(M.build_model(NAME)))
    return out[0], quantize_branches(copy.deepcopy(out[0])), quantize_branches(out[1])


def test_every_layer_of_a_branch_holds_its_weight(models):
    plain, quantised, _ = models
    found = {n: m for n, m in quantised.named_modules() if isinstance(m, Int8Linear)}
    assert len(found) == 4 * len(plain.blocks)
    for n, m in found.items():
        w = plain.get_submodule(n).weight.double()
        s = m.weight_scale.double().unsqueeze(1)
        # the quotient's rounding to fp32 passes a tie by at most 127 2^-24
        assert bool(((m.weight[:, : w.shape[1]].double() * s - w).abs() <= s * (0.5 + 2.0**-17)).all())
        assert torch.equal(s.float().squeeze(1), (w.abs().amax(1) / 127).float())
        assert torch.equal(m.bias, plain.get_submodule(n).bias)


@pytest.mark.parametrize("key", ["model", "ema"])
def test_a_checkpoint_of_the_model_is_quantised_on_the_way_in(models, key):
    plain, want, other = models
    model = copy.deepcopy(other)
    ckpt = checkpoint_state(plain, None, [p.detach() for p in plain.parameters()], 1)
    kept = load_model_state(model, ckpt, key)
    assert not [n for n in kept if "weight" in n]
    assert_same(numbers(model), numbers(want))


@pytest.mark.parametrize("assign", [False, True])
def test_load_state_dict_takes_both_forms(models, assign):
    plain, want, other = models
    for strict in (True, False):
        for state in (plain.state_dict(), want.state_dict()):
            model = copy.deepcopy(other)
            missing, unexpected = model.load_state_dict(state, strict=strict, assign=assign)
            assert not missing and not unexpected
            assert_same(numbers(model), numbers(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("k", [16, 37])
def test_a_layer_takes_a_linear_layers_state(dtype, k):
    layer = linear(k, 5).to(dtype)
    want = Int8Linear.from_linear(layer)
    for assign in (False, True):
        q = Int8Linear.from_linear(linear(k, 5, seed=3))
        q.load_state_dict(layer.state_dict(), assign=assign)
        assert_same(numbers(q), numbers(want))
    assert q.bias.dtype == torch.float32 and q.weight.shape == (5, ops_int8.padded(k))


@pytest.mark.parametrize("strict", [True, False])
def test_a_state_that_would_mix_two_layers_is_refused(strict):
    mine, other = Int8Linear.from_linear(linear(48, 5)), Int8Linear.from_linear(linear(48, 5, seed=3))
    before, state = numbers(mine), numbers(other)
    wide = linear(40, 5).state_dict()  # as wide as 48 where both are padded
    bad = [
        {n: t for n, t in state.items() if n != "weight_scale"},
        {n: t for n, t in state.items() if n != "weight"},
        state | {"weight": state["weight"].int()},
        wide,
        {"weight": linear(48, 6).weight.detach()},
    ]
    for s in bad:
        with pytest.raises(RuntimeError, match="weight"):
            mine.load_state_dict(s, strict=strict)
        assert_same(numbers(mine), before)


def test_a_state_without_the_layer_leaves_it_as_it_is():
    mine = Int8Linear.from_linear(linear(48, 5))
    before = numbers(mine)
    missing, _ = mine.load_state_dict({}, strict=False)
    assert set(missing) == {"weight", "weight_scale", "bias"}
    assert_same(numbers(mine), before)
    with pytest.raises(RuntimeError, match="Missing"):
        mine.load_state_dict({})


@pytest.mark.parametrize("k,wrong", [(768, 767), (768, 753), (2730, 2731), (2730, 2736), (2730, 2721), (5, 16), (16, 32)])
def test_a_layer_refuses_other_widths(k, wrong):
    layer = Int8Linear.from_linear(linear(k, 6))
    for x in (torch.zeros(3, wrong), torch.zeros(wrong), torch.tensor(1.0)):
        with pytest.raises(ValueError, match=f"of {k} channels"):
            layer(x)
        with pytest.raises(ValueError, match=f"of {k} channels"):
            layer.gated(x, "silu")


@pytest.mark.parametrize("strict", [True, False])
def test_a_linear_layer_refuses_8_bit_values(models, strict):
    plain, quantised, _ = models
    model = copy.deepcopy(plain)
    before = numbers(model)
    with pytest.raises(RuntimeError, match="quantize_branches"):
        model.load_state_dict(quantised.state_dict(), strict=strict)
    with pytest.raises(RuntimeError, match="quantize_branches"):
        load_model_state(model, {"ema": quantised.state_dict()}, "ema")
    assert all(torch.equal(t, before[n]) for n, t in model.state_dict().items() if ".branch." in n)
