"""jit_thc::gated_linear and its backward against the formulas in 64 bits (MI355X only)."""

from __future__ import annotations

import math

import pytest
import torch

from flowmatching_lthc_amd import ops_branch as OB

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0**-24


def randn(shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(DEV, dtype)


def act64(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    k = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(k * (g + 0.044715 * g**3))
    return g * s, s + g * s * (1 - s) * k * (1 + 3 * 0.044715 * g * g)


def exact(x, w, b, act, dy=None):
    """(y, its error bound, (dx, dw, db), their error bounds) in 64 bits, of the products of the given 16-bit operands.

    A projection is a sum of C products in fp32 in any order: off by at most (C + 2) U of the sum of their magnitudes.  The
    activation and its slope, of size at most |g| and 1.13 and of slope at most 1.13, feel that, and add 2^-19 of their own
    (an exponential and a reciprocal of 1 ulp at an argument rounded in fp32, up to 88, for |g| up to 88: 88 U relative; the
    erf of 4 ulp)."""
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # the least step of fp16 results below its normal range
    xd, wd = x.detach().double(), w.detach().double()
    F = wd.shape[0] // 2
    h, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        h, size = h + b.detach().double(), size + b.detach().double().abs()
    eh = (x.shape[-1] + 2) * U * size
    g, u, eg, eu = h[..., :F], h[..., F:], eh[..., :F], eh[..., F:]
    a, da = act64(g, act)
    own = 2.0**-19
    ea, eda = 1.13 * eg + own * (a.abs() + g.abs() * (g.abs() < 12)), 0.8 * eg + own * (1 + g.abs() * (g.abs() < 12))
    y = a * u
    ey = ea * u.abs() + (a.abs() + ea) * eu + 2 * U * y.abs()
    ey = ey + half * (y.abs() + ey) + tiny
    if dy is None:
        return y, ey
    d = dy.double()
    dg, du = d * u * da, d * a
    # rounded to the operands' type where they enter the products
    edg = d.abs() * ((u.abs() + eu) * eda + da.abs() * eu) + 4 * U * dg.abs()
    edu = d.abs() * ea + 2 * U * du.abs()
    dh, edh = torch.cat([dg, du], -1), torch.cat([edg, edu], -1)
    edh = edh + half * (dh.abs() + edh) + tiny
    dh2, edh2, x2 = dh.reshape(-1, 2 * F), edh.reshape(-1, 2 * F), xd.reshape(-1, xd.shape[-1])
    grads, bounds = [], []
    for lhs, elhs, rhs, n in ((dh, edh, wd, 2 * F), (dh2.t(), edh2.t(), x2, x2.shape[0]), (dh2.t(), edh2.t(), torch.ones_like(x2[:, :1]), x2.shape[0])):
        v = lhs @ rhs
        e = elhs @ rhs.abs() + (n + 66) * U * ((lhs.abs() + elhs) @ rhs.abs())  # parts of rows are added once more
        grads.append(v)
        bounds.append(e + half * (v.abs() + e) + tiny)
    grads[2], bounds[2] = grads[2][:, 0], bounds[2][:, 0]
    return y, ey, grads, bounds


def check(got, want, bound, name):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (name, float((err - bound).max()), float((err / bound).max()))


def operands(M, C, F, dtype, bias=True, seed=0, lead=None):
    x = randn((*(lead or (M,)), C), seed, dtype)
    w = randn((2 * F, C), seed + 1, dtype, C**-0.5)
    b = randn((2 * F,), seed + 2, dtype, 0.2) if bias else None
    return x, w, b


SHAPES = [
    # rows, channels, hidden: single tokens, sizes around the tiles' 64, 128 and 256, channels that fill no stage
    (1, 768, 2048), (1, 8, 1), (2, 16, 3), (5, 64, 64), (16, 72, 65), (17, 128, 127), (33, 136, 129), (64, 192, 130),
    (65, 200, 17), (127, 256, 96), (128, 328, 250), (129, 64, 128), (255, 120, 33), (257, 384, 341), (300, 1024, 682),
    (700, 96, 2730), (1025, 768, 256), (4099, 64, 40), (70, 2048, 64), (512, 8, 512),
]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients_match_64_bits(shape, dtype):
    M, C, F = shape
    act = ("silu", "gelu", "gelu_tanh")[(M + C) % 3]
    bias = F % 2 == 0 or M == 1
    print("case gated_linear", shape, dtype, act, bias, flush=True)
    x, w, b = operands(M, C, F, dtype, bias)
    dy = randn((M, F), 9, dtype)
    y, ey, grads, bounds = exact(x, w, b, act, dy)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    got = OB.gated_linear(x, w, b, act)
    assert got.dtype == dtype
    check(got, y, ey, "y")
    for t, v, e, name in zip(torch.autograd.grad(got, leaves, dy), grads, bounds, ("dx", "dw", "db")):
        assert t.dtype == dtype
        check(t, v, e, name)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_large_tiles(act):
    """Enough rows and columns for the largest tiles, with ragged edges on every side."""
    print("case gated_linear large", act, flush=True)
    M, C, F = 8192 + 77, 136, 1024 + 35
    x, w, b = operands(M, C, F, torch.bfloat16)
    dy = randn((M, F), 9, torch.bfloat16)
    y, ey, grads, bounds = exact(x, w, b, act, dy)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = OB.gated_linear(x, w, b, act)
    check(got, y, ey, "y")
    for t, v, e, name in zip(torch.autograd.grad(got, leaves, dy), grads, bounds, ("dx", "dw", "db")):
        check(t, v, e, name)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_saturated_activations_and_non_finite_rows(act):
    """Gates far out on both sides, and a row of NaN or infinity that stays in its row."""
    print("case gated_linear saturated", act, flush=True)
    M, C, F = 40, 64, 96
    x, w, b = operands(M, C, F, torch.bfloat16)
    x[0] *= 60
    b[: F // 2] -= 30
    y, ey = exact(x, w, b, act)
    check(OB.gated_linear(x, w, b, act), y, ey, "y")
    x[3, 5] = float("nan")
    x[7, 9] = float("inf")
    got = OB.gated_linear(x, w, b, act)
    fine = torch.ones(M, dtype=torch.bool, device=DEV)
    fine[[3, 7]] = False
    check(got[fine], y[fine], ey[fine], "finite rows")
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[7]).any()


def test_layouts_leading_dimensions_and_empty():
    print("case gated_linear layouts", flush=True)
    x, w, b = operands(0, 64, 48, torch.bfloat16, lead=(3, 5, 2))
    y = OB.gated_linear(x, w, b)
    assert y.shape == (3, 5, 2, 48)
    flat = OB.gated_linear(x.reshape(30, 64), w, b)
    assert torch.equal(y.reshape(30, 48), flat)
    assert torch.equal(OB.gated_linear(x[0, 0, 0], w, b), flat[0])  # one vector
    strided = x.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((96, 65), device=DEV, dtype=torch.bfloat16)
    wide[:, 1:] = w  # rows that no vector access fits
    odd = torch.empty(97, device=DEV, dtype=torch.bfloat16)[1:].copy_(b)
    assert torch.equal(OB.gated_linear(strided, wide[:, 1:], odd), y)
    e = torch.empty((0, 64), device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w, b = w.requires_grad_(), b.requires_grad_()
    out = OB.gated_linear(e, w, b)
    assert out.shape == (0, 48)
    gx, gw, gb = torch.autograd.grad(out, (e, w, b), torch.empty_like(out))
    assert gx.shape == e.shape and float(gw.abs().max()) == 0 and float(gb.abs().max()) == 0


def test_partial_gradients_equal_the_full_ones():
    print("case gated_linear partial gradients", flush=True)
    x, w, b = operands(70, 72, 50, torch.bfloat16)
    dy = randn((70, 50), 4, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    full = torch.autograd.grad(OB.gated_linear(*leaves), leaves, dy)
    for need in ((0,), (1,), (2,), (0, 2), (0, 1)):
        for i, t in enumerate(leaves):
            t.requires_grad_(i in need)
        got = torch.autograd.grad(OB.gated_linear(*leaves), [leaves[i] for i in need], dy)
        for i, g in zip(need, got):
            assert torch.equal(g, full[i])
    # an output gradient in another layout
    for t in leaves:
        t.requires_grad_()
    strided = dy.t().contiguous().t()
    for a, c in zip(torch.autograd.grad(OB.gated_linear(*leaves), leaves, strided), full):
        assert torch.equal(a, c)
    (g,) = torch.autograd.grad(OB.gated_linear(*leaves).sum(), x)  # a broadcast one
    (c,) = torch.autograd.grad(OB.gated_linear(*leaves), x, torch.ones_like(dy))
    assert torch.equal(g, c)


def test_gradients_against_differences():
    """A central difference of the 64-bit sum of dy y along a direction, in the operands' own values: the third-order term
    of a step of 2^-6 and the outputs' rounding bound it (about 2^-12 of the sums' size; 5 % of the slope is asked for)."""
    print("case gated_linear differences", flush=True)
    M, C, F = 24, 64, 40
    x, w, b = operands(M, C, F, torch.float16)
    dy = randn((M, F), 5, torch.float16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(OB.gated_linear(*leaves), leaves, dy)
    for i, t in enumerate(leaves):
        step = grads[i].detach() / grads[i].detach().double().norm().half() * 0.25
        moved = []
        for sign in (1, -1):
            args = [u.detach() for u in leaves]
            args[i] = args[i] + sign * step
            moved.append((args[i].double(), float((OB.gated_linear(*args).double() * dy.double()).sum())))
        slope = float((grads[i].double() * (moved[0][0] - moved[1][0])).sum())
        assert abs((moved[0][1] - moved[1][1]) - slope) <= 0.05 * abs(slope), (i, moved[0][1] - moved[1][1], slope)


def test_second_derivative_and_autocast():
    print("case gated_linear double backward, autocast", flush=True)
    x, w, b = operands(12, 32, 20, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    second = []
    for f in (OB.gated_linear, OB.gated_linear_eager):
        first = torch.autograd.grad(f(*leaves).float().square().sum(), leaves, create_graph=True)
        second.append(torch.autograd.grad(sum(g.float().square().sum() for g in first), leaves))
    for a, c in zip(*second):
        # y and the first gradients differ by a rounding each (2^-8 in bf16), and their products feel it
        assert float((a - c).abs().max()) <= 2**-5 * float(c.abs().max())
    master = [t.detach().float().requires_grad_() for t in leaves]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = OB.gated_linear(*master)
    assert y.dtype == torch.bfloat16 and torch.equal(y, OB.gated_linear(*leaves))
    dy = randn(y.shape, 3, torch.bfloat16)
    want = torch.autograd.grad(OB.gated_linear(*leaves), leaves, dy)
    for a, c in zip(torch.autograd.grad(y, master, dy), want):
        assert a.dtype == torch.float32 and torch.equal(a, c.float())


def test_captured_with_its_backward_and_on_a_side_stream():
    print("case gated_linear graph, side stream", flush=True)
    x, w, b = operands(300, 136, 77, torch.bfloat16)
    dy = randn((300, 77), 4, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = OB.gated_linear(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = step()
    side.synchronize()
    for a, c in zip(on_side, step()):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(randn(x.shape, 20 + seed, x.dtype))
            w.copy_(randn(w.shape, 30 + seed, w.dtype, 0.1))
            dy.copy_(randn(dy.shape, 40 + seed, dy.dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, step()):
            assert torch.equal(a, c)


def test_compiled():
    print("case gated_linear compiled", flush=True)
    x, w, b = operands(64, 64, 48, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    f = lambda x, w, b: OB.gated_linear(x, w, b, "gelu_tanh").float().square().mean()  # noqa: E731
    want = torch.autograd.grad(f(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(f)(*leaves), leaves)
    for a, c in zip(got, want):
        # the compiled backward keeps dh in fp32: one rounding (2^-8) less of each term
        assert float((a - c).abs().max()) <= 2**-6 * float(c.abs().max())


def test_refusals():
    print("case gated_linear refusals", flush=True)
    x, w, b = operands(4, 16, 6, torch.bfloat16)
    for args, text in (
        ((x.float(), w.float()), "bf16 or fp16"),
        ((x, w.float()), "dtype"),
        ((x, w, b.float()), "dtype"),
        ((x, w[:11]), "expected"),
        ((x[:, :8], w), "expected"),
        ((x[:, :12], w[:, :12]), "multiple of 8"),
        ((x, w, b[:-1]), "bias"),
        ((x, w.cpu()), "cuda|GPU"),
        ((x, w, b, "relu"), "activation"),
    ):
        with pytest.raises(ValueError, match=text):
            OB.gated_linear(*args)


def test_the_models_feed_forward_with_fused_projections():
    """SwiGLUFFN with the switch on: the eager sequence's function, its roundings of h and silu left out (three of 2^-8)."""
    from flowmatching_lthc_amd.model import SwiGLUFFN

    print("case gated_linear model", flush=True)
    torch.manual_seed(0)
    ffn = SwiGLUFFN(64, 384).to(DEV, torch.bfloat16)
    x = randn((2, 50, 64), 0, torch.bfloat16).requires_grad_()
    dy = randn((2, 50, 64), 1, torch.bfloat16)
    results = []
    for on in (False, True):
        ffn.fused_projections = on
        y = ffn(x)
        results.append([y, *torch.autograd.grad(y, [x, *ffn.parameters()], dy)])
    for a, c in zip(*results):
        assert float((a - c).abs().max()) <= 2**-5 * float(c.abs().max())
    assert not torch.equal(results[0][0], results[1][0])  # the switch does something
    ffn.float()
    x = x.detach().float()
    assert torch.equal(ffn(x), F_ref(ffn, x))  # fp32: the eager sequence


def F_ref(ffn, x):
    g, u = ffn.w12(x).chunk(2, -1)
    return ffn.w3(OB.swiglu(torch.cat([g, u], -1)))


@pytest.mark.parametrize("M", [5, 128, 300])
def test_an_infinite_bias_reaches_only_its_own_sums(M):
    """Rows past the last one add nothing to the bias gradients, whatever the bias makes of them."""
    print("case gated_linear infinite bias", M, flush=True)
    C, Fh = 16, 70
    x, w = randn((M, C), 0, torch.bfloat16).abs(), randn((2 * Fh, C), 1, torch.bfloat16).abs()
    b = torch.zeros(2 * Fh, device=DEV, dtype=torch.bfloat16)
    b[Fh + 3] = math.inf  # an up projection: its gate's gradient is dy inf act'(g), act'(g) > 0
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    dy = randn((M, Fh), 2, torch.bfloat16).abs() + 0.5
    _, dw, db = torch.autograd.grad(OB.gated_linear(x, w, b), [x, w, b], dy)
    assert float(db[3]) == math.inf
    rest = torch.ones(2 * Fh, dtype=torch.bool, device=DEV)
    rest[3] = False
    assert bool(db[rest].isfinite().all()) and bool(dw[rest].isfinite().all())


@pytest.mark.parametrize("M", [3, 700])
def test_the_backward_op_computes_what_is_needed(M):
    print("case gated_linear needs", M, flush=True)
    x, w, b = operands(M, 72, 50, torch.float16)
    dy = randn((M, 50), 4, torch.float16)
    full = OB.gated_linear_backward(dy, x, w, b, "gelu", True, True, True)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        got = OB.gated_linear_backward(dy, x, w, b, "gelu", *need)
        for n, g, c, t in zip(need, got, full, torch.ops.jit_thc.gated_linear_backward(*(t.to("meta") for t in (dy, x, w, b)), "gelu", *need)):
            assert g.shape == t.shape and (torch.equal(g, c) if n else g.numel() == 0)


def test_the_models_feed_forward_calls_a_projection_that_is_more_than_its_weight():
    """With the switch on too: hooks and other modules in w12's place run, and a function mode sees the call."""
    from flowmatching_lthc_amd.model import SwiGLUFFN

    print("case gated_linear model with hooks", flush=True)
    torch.manual_seed(0)
    ffn = SwiGLUFFN(64, 384).to(DEV, torch.bfloat16)
    x = randn((2, 50, 64), 0, torch.bfloat16)
    eager = ffn(x)
    ffn.fused_projections = True
    fused = ffn(x)
    assert not torch.equal(fused, eager)
    seen = []
    handle = ffn.w12.register_forward_hook(lambda m, args, out: seen.append(out.shape))
    assert torch.equal(ffn(x), eager) and len(seen) == 1
    handle.remove()
    assert torch.equal(ffn(x), fused)
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False) as flops:
        assert torch.equal(ffn(x), eager)
    assert flops.get_total_flops() == 2 * 100 * 64 * 512 + 2 * 100 * 256 * 64
    inner = ffn.w12
    ffn.w12 = torch.nn.Sequential(inner, torch.nn.Identity())
    assert torch.equal(ffn(x), eager)


def test_the_models_feed_forward_compiles_to_the_kernels():
    """The compiled forward and backward of SwiGLUFFN with the switch on hold the two operators and the products of w3 alone,
    none of them in fp32, and give the eager call's values."""
    from functorch.compile import make_boxed_func
    from torch._dynamo.backends.common import aot_autograd

    from flowmatching_lthc_amd.model import SwiGLUFFN

    print("case gated_linear compiled model", flush=True)
    torch._dynamo.reset()
    torch.manual_seed(0)
    ffn = SwiGLUFFN(64, 384).to(DEV, torch.bfloat16)
    ffn.fused_projections = True
    x = randn((2, 50, 64), 0, torch.bfloat16).requires_grad_()
    dy = randn((2, 50, 64), 1, torch.bfloat16)
    graphs = []

    def keep(graph, inputs):
        graphs.append([n for n in graph.graph.nodes if n.op == "call_function"])
        return make_boxed_func(graph.forward)

    y = torch.compile(ffn, backend=aot_autograd(fw_compiler=keep, bw_compiler=keep), fullgraph=True)(x)
    got = [y, *torch.autograd.grad(y, [x, *ffn.parameters()], dy)]
    assert len(graphs) == 2
    for nodes, op in zip(graphs, ("gated_linear", "gated_linear_backward")):
        assert f"jit_thc.{op}.default" in {str(n.target) for n in nodes}
        products = [n for n in nodes if any(p in str(n.target) for p in ("aten.mm", "aten.addmm", "aten.bmm"))]
        assert len(products) == (1 if op == "gated_linear" else 2)
        assert all(n.meta["val"].dtype == torch.bfloat16 for n in products)
    want = ffn(x)
    for a, c in zip(got, [want, *torch.autograd.grad(want, [x, *ffn.parameters()], dy)]):
        # w3's own products may be split differently: a rounding of their results
        assert float((a - c).detach().abs().max()) <= 2**-7 * float(c.detach().abs().max())
    torch._dynamo.reset()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(64, 512, (1, 32, 64, 65, 700)), (64, 24, (5, 1365, 1366, 53000)), (1024, 1024, (3, 32, 33))], ids=str)
def test_a_rows_gradient_does_not_depend_on_the_rows_beside_it(shape, dtype):
    """dx of the first rows of a batch is that of the rows by themselves, bit for bit: sums in the same order and the same
    roundings at every number of rows."""
    C, F, rows = shape
    print("case gated_linear rows alone", shape, dtype, flush=True)
    x, w, b = operands(rows[-1], C, F, dtype)
    dy = randn((rows[-1], F), 9, dtype)
    whole, _, _ = OB.gated_linear_backward(dy, x, w, b, "silu", True, False, False)
    for M in rows[:-1]:
        dx, _, _ = OB.gated_linear_backward(dy[:M], x[:M], w, b, "silu", True, False, False)
        assert torch.equal(dx, whole[:M]), M
