"""The autograd nodes of the gated linear layer and the rotary positions on CPU tensors: plain-torch kernels stand in for the
HIP ones while a test runs, so that what autograd sees of the nodes can be checked without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from flowmatching_lthc_amd import ops_branch as OB


def gated_backward(grad, x, weight, bias, activation, need_x, need_weight, need_bias):
    """Of silu."""
    g, u = torch.nn.functional.linear(x.float(), weight.float(), None if bias is None else bias.float()).chunk(2, -1)
    s, d = torch.sigmoid(g), grad.float()
    dh = torch.cat([d * u * s * (1 + g * (1 - s)), d * g * s], -1)
    rows, empty = dh.reshape(-1, dh.shape[-1]), x.new_empty
    gx = (dh @ weight.float()).to(x.dtype) if need_x else empty(0)
    gw = (rows.t() @ x.float().reshape(-1, x.shape[-1])).to(x.dtype) if need_weight else empty((0, x.shape[-1]))
    return gx, gw, rows.sum(0).to(x.dtype) if need_bias else empty(0)


def rotated(q, k, positions, inv_freq, sections, interleaved=True, inverse=False):
    """Of interleaved pairs and one axis."""
    angle = positions[:, :1].double() * inv_freq * (-1 if inverse else 1)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    return turn(q), turn(k)


@pytest.fixture(autouse=True)
def cpu_kernels():
    lib = torch.library.Library("jit_thc", "IMPL")
    lib.impl("gated_linear", OB.gated_linear_eager, "CPU")
    lib.impl("gated_linear_backward", gated_backward, "CPU")
    lib.impl("axial_rope", rotated, "CPU")
    yield
    lib._destroy()


def leaf(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).requires_grad_()


def gated(bias=True):
    leaves = [leaf((5, 8), 0), leaf((12, 8), 1), *([leaf((12,), 2)] if bias else [])]
    return leaves, [OB.gated_linear(*leaves)]


def rope():
    leaves = [leaf((2, 3, 4, 8), 0, torch.float32), leaf((2, 3, 1, 8), 1, torch.float32)]
    return leaves, list(OB.axial_rope(*leaves, torch.arange(3.0)[:, None], torch.tensor([1.0, 0.5, 0.2, 0.1]).double(), (8,)))


@pytest.mark.parametrize("bias", [True, False])
def test_a_traced_gated_backward_is_the_kernels(bias):
    """Its products stay the op's: no fp32 product of the eager sequence in the graph."""

    def step(grad, *leaves):
        leaves = [t.detach().requires_grad_() for t in leaves]
        return torch.autograd.grad(OB.gated_linear(*leaves), leaves, grad)

    leaves, (y,) = gated(bias)
    graph = make_fx(step, tracing_mode="fake")(torch.ones_like(y), *(t.detach() for t in leaves)).graph
    names = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    assert "jit_thc.gated_linear_backward.default" in names
    assert not {n for n in names if "mm" in n or "linear.default" in n.replace("gated_linear.default", "")}
    (out,) = [n for n in graph.nodes if n.op == "output"]
    assert [(n.meta["val"].shape, n.meta["val"].dtype) for n in out.args[0]] == [(t.shape, t.dtype) for t in leaves]


@pytest.mark.parametrize("node", [gated, rope])
def test_batched_gradients_are_those_of_each_sample(node):
    leaves, outs = node()
    grads = [leaf((3, *o.shape), 40 + i, o.dtype).detach() for i, o in enumerate(outs)]
    each = [torch.autograd.grad(outs, leaves, [g[i] for g in grads], retain_graph=True) for i in range(3)]
    for want in (slice(0, None), slice(0, 1), slice(1, 2)):
        got = torch.autograd.grad(outs, leaves[want], grads, is_grads_batched=True, retain_graph=True)
        vmapped = torch.vmap(lambda *g: torch.autograd.grad(outs, leaves[want], g, retain_graph=True))(*grads)
        for a, v, b in zip(got, vmapped, zip(*(e[want] for e in each))):
            assert torch.equal(a, torch.stack(b)) and torch.equal(v, a)


@pytest.mark.parametrize("recorded", [True, False])
@pytest.mark.parametrize("node", [gated, rope])
def test_forward_mode_is_refused(node, recorded):
    """A tangent is not lost without a word."""

    def call(*args):
        return OB.gated_linear(*args) if node is gated else OB.axial_rope(*args, torch.zeros(3, 1), torch.ones(4).double(), (8,))

    leaves, _ = node()
    for i in range(len(leaves)):
        args = [t.detach().requires_grad_(recorded) for t in leaves]
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*args[:i], dual, *args[i + 1 :])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: call(*args[:i], t, *args[i + 1 :]), (args[i].detach(),), (args[i].detach(),))
