"""jit_thc::axial_rope against the rotation in 64 bits (MI355X only)."""

from __future__ import annotations

import pytest
import torch

from flowmatching_lthc_amd import ops_branch as OB

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def inv_freq(sections, theta=10000.0):
    return torch.cat([theta ** (-2.0 * torch.arange(n // 2, dtype=torch.float64) / n) for n in sections]).to(DEV)


def exact(x, positions, freq, sections, interleaved, sign=1):
    """The rotation in 64 bits, pair by pair."""
    x, R = x.detach().double(), sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n // 2)]
    ang = sign * positions.double()[..., axis] * freq
    ang = (ang if ang.dim() == 3 else ang[None]).unsqueeze(2)
    out = x.clone()
    for p in range(R // 2):
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + R // 2)
        c, s = ang[..., p].cos(), ang[..., p].sin()
        out[..., i] = x[..., i] * c - x[..., j] * s
        out[..., j] = x[..., i] * s + x[..., j] * c
    return out


def check(got, x, want, far=0.0):
    """Half a step of the output's type, and of the fp32 arithmetic: a sine or cosine is off by at most 2^-21 (its angle,
    reduced to half a turn and narrowed, by pi 2^-24, and its own evaluation by 2 ulp), two products and a sum by 3 2^-24.
    far: what 64-bit angles of far positions are off by themselves (position * 2^-52)."""
    assert got.dtype == x.dtype and got.shape == x.shape
    half = torch.finfo(x.dtype).eps / 2
    size = x.detach().double().abs().amax(-1, keepdim=True)  # bounds both channels of every pair
    err = (got.double() - want).abs()
    bound = half * want.abs() + 2 * size * (2**-21 + 3 * 2**-24 + far) + torch.finfo(x.dtype).tiny
    assert bool((err <= bound).all()), float((err - bound).max())


def randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def make(B, N, Hq, Hk, D, layout, dtype, seed=0):
    if layout == "qkv":
        qkv = randn((B, N, 3, Hq, D), seed, dtype)
        return qkv[:, :, 0], qkv[:, :, 1]
    if layout == "bhnd":
        return tuple(randn((B, H, N, D), seed + i, dtype).transpose(1, 2) for i, H in enumerate((Hq, Hk)))
    if layout == "dlast":  # the channels of a head not consecutive
        return tuple(randn((B, N, D, H), seed + i, dtype).transpose(2, 3) for i, H in enumerate((Hq, Hk)))
    if layout == "odd":  # rows an odd number of elements apart
        return tuple(randn((B, N, H, D + 1), seed + i, dtype)[..., 1:] for i, H in enumerate((Hq, Hk)))
    return randn((B, N, Hq, D), seed, dtype), randn((B, N, Hk, D), seed + 1, dtype)


CASES = [
    # B, N, Hq, Hk, D, sections, layout, shared positions
    (2, 9, 3, 3, 64, (32, 32), "qkv", True),
    (1, 1, 16, 4, 128, (32, 48, 48), "bnhd", False),
    (3, 17, 5, 1, 84, (20, 26, 18), "bhnd", True),
    (2, 5, 4, 2, 30, (2, 4, 6, 8), "bnhd", False),
    (1, 3, 1, 1, 2, (2,), "bnhd", False),
    (2, 4, 2, 3, 64, (64,), "dlast", False),
    (2, 33, 2, 2, 20, (12, 6), "odd", False),
    (1, 2, 1, 2, 1024, (512, 512), "bnhd", False),
    (1, 700, 7, 3, 256, (96, 80), "qkv", True),
    (65, 1, 12, 12, 64, (16, 24, 24), "qkv", False),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])) + c[6])
def test_forward_and_backward_match_64_bits(case, interleaved, dtype):
    B, N, Hq, Hk, D, sections, layout, shared = case
    print("case axial_rope", case, interleaved, dtype, flush=True)
    if layout == "qkv":
        Hk = Hq
    q, k = make(B, N, Hq, Hk, D, layout, dtype)
    gen = torch.Generator().manual_seed(7)
    shape = (N, len(sections)) if shared else (B, N, len(sections))
    positions = torch.randint(-1000, 1000, shape, generator=gen).to(DEV)
    freq = inv_freq(sections)
    q, k = q.requires_grad_(), k.requires_grad_()
    oq, ok = OB.axial_rope(q, k, positions, freq, sections, interleaved)
    gq, gk = randn(oq.shape, 3, dtype), randn(ok.shape, 4, dtype)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    for got, x, sign in ((oq, q, 1), (ok, k, 1), (dq, gq, -1), (dk, gk, -1)):
        check(got, x, exact(x, positions, freq, sections, interleaved, sign), 1000 * 2**-52)


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_position_types_and_far_positions(ptype):
    print("case axial_rope positions", ptype, flush=True)
    B, N, sections = 2, 6, (16, 8, 8)
    q, k = make(B, N, 2, 1, 32, "bnhd", torch.float32)
    positions = torch.randint(0, 1 << 24, (B, N, 3), generator=torch.Generator().manual_seed(1)).to(DEV, ptype)
    if ptype.is_floating_point:
        positions = positions + 0.25  # fp32: rounded to a step of its own below 2^24, the same number for both sides
    positions = positions.transpose(0, 1).contiguous().transpose(0, 1)  # strided
    freq = inv_freq(sections)
    for got, x in zip(OB.axial_rope(q, k, positions, freq, sections), (q, k)):
        check(got, x, exact(x, positions, freq, sections, True), 2**24 * 2**-51)


def test_channels_past_the_sections_and_empty_sides_are_untouched():
    print("case axial_rope pass-through", flush=True)
    q, k = make(2, 5, 3, 2, 40, "bnhd", torch.bfloat16)
    q[..., 24:] = float("nan")
    q[0, 0, 0, 30] = float("inf")
    pos = torch.arange(5, device=DEV)[:, None].expand(5, 2)
    for interleaved in (True, False):
        oq, ok = OB.axial_rope(q, k, pos, inv_freq((8, 16)), (8, 16), interleaved)
        assert torch.equal(oq[..., 24:].contiguous().view(torch.int16), q[..., 24:].contiguous().view(torch.int16))
        assert torch.equal(ok[..., 24:], k[..., 24:])
        assert torch.isfinite(oq[..., :24]).all()
        assert torch.equal(oq[:, 0, :, :24], q[:, 0, :, :24])  # position 0 turns nothing
    for shape in ((0, 5, 3, 40), (2, 0, 3, 40), (2, 5, 0, 40)):
        e = torch.empty(shape, device=DEV)
        pos = torch.zeros((shape[1], 2), device=DEV, dtype=torch.int64)
        oq, ok = OB.axial_rope(e, e, pos, inv_freq((8, 16)), (8, 16))
        assert oq.shape == shape and ok.shape == shape
    none = q[:, :, :0]
    pos = torch.arange(5, device=DEV)[:, None].expand(5, 2)
    assert torch.equal(OB.axial_rope(none, k, pos, inv_freq((8, 16)), (8, 16))[1], ok_of(k, pos))


def ok_of(k, pos):
    return OB.axial_rope(k, k, pos, inv_freq((8, 16)), (8, 16))[0]


def test_the_grid_tables_of_the_model_are_the_two_axis_case():
    """VisionRotaryEmbeddingFast's rotation: rows on the first half of a head, columns on the second."""
    from flowmatching_lthc_amd.model import VisionRotaryEmbeddingFast

    print("case axial_rope grid", flush=True)
    rope = VisionRotaryEmbeddingFast(32, 7).to(DEV)
    q = randn((2, 49, 3, 64), 0, torch.float32)
    token = torch.arange(49, device=DEV)
    pos = torch.stack([token // 7, token % 7], -1)
    got, _ = OB.axial_rope(q, q, pos, inv_freq((32, 32)), (32, 32))
    want = rope(q.transpose(1, 2)).transpose(1, 2)
    # the table's fp32 angles (up to 6 rad) are off by 6 2^-24, its speeds by as much again
    assert float((got - want).abs().max()) <= 5 * (2 * 6 * 2**-23 + 2**-21)


def test_broadcast_inputs_partial_gradients_and_second_derivative():
    print("case axial_rope broadcast, partial, double backward", flush=True)
    sections, pos = (8, 8), torch.arange(6, device=DEV)[:, None].expand(6, 2)
    freq = inv_freq(sections)
    one = randn((1, 6, 2, 16), 0, torch.float32).requires_grad_()
    k = randn((3, 6, 1, 16), 1, torch.float32)
    g = randn((3, 6, 2, 16), 2, torch.float32)
    oq, ok = OB.axial_rope(one.expand(3, 6, 2, 16), k, pos, freq, sections)
    (d,) = torch.autograd.grad(oq, one, g)  # k asks for none
    check(d, one, exact(g.sum(0, keepdim=True), pos, freq, sections, True, -1), 16 * 2**-22)
    x = randn((3, 6, 2, 16), 3, torch.float32).requires_grad_()
    oq, _ = OB.axial_rope(x, k, pos, freq, sections)
    (first,) = torch.autograd.grad(oq.pow(3).sum(), x, create_graph=True)
    (second,) = torch.autograd.grad(first.sum(), x)
    xd = x.detach().double().requires_grad_()
    (fd,) = torch.autograd.grad(rotated(xd, pos, freq).pow(3).sum(), xd, create_graph=True)
    (sd,) = torch.autograd.grad(fd.sum(), xd)
    assert float((second - sd).abs().max()) <= 1e-4


def rotated(x, pos, freq):
    axis = [0] * 4 + [1] * 4
    ang = (pos.double()[..., axis] * freq)[None, :, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2)


def test_gradient_against_differences():
    """The rotation is linear: a difference of outputs is the rotation of the inputs' difference, and its product with the
    output gradient is the input gradient's with the inputs' difference."""
    print("case axial_rope differences", flush=True)
    sections, freq = (6, 10), inv_freq((6, 10))
    pos = torch.randint(0, 50, (2, 7, 2), generator=torch.Generator().manual_seed(0)).to(DEV)
    q, k = make(2, 7, 2, 2, 20, "bnhd", torch.float32)
    dx, g = randn(q.shape, 5, torch.float32), randn(q.shape, 6, torch.float32)
    q = q.requires_grad_()
    for inter in (True, False):
        out, _ = OB.axial_rope(q, k, pos, freq, sections, inter)
        moved, _ = OB.axial_rope(q.detach() + dx, k, pos, freq, sections, inter)
        (grad,) = torch.autograd.grad(out, q, g)
        left = ((moved.double() - out.detach().double()) * g.double()).sum()
        right = (grad.double() * dx.double()).sum()
        assert abs(float(left - right)) <= 560 * 5 * 5 * 8 * 2**-21


def test_captured_with_its_backward_and_on_a_side_stream():
    print("case axial_rope graph, side stream", flush=True)
    sections, freq = (16, 24, 24), inv_freq((16, 24, 24))
    q, k = make(2, 40, 3, 1, 64, "bnhd", torch.bfloat16)
    pos = torch.randint(0, 500, (2, 40, 3), generator=torch.Generator().manual_seed(0)).to(DEV)
    gq, gk = randn(q.shape, 8, q.dtype), randn(k.shape, 9, k.dtype)
    q, k = q.requires_grad_(), k.requires_grad_()

    def step():
        out = OB.axial_rope(q, k, pos, freq, sections)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), (gq, gk))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = step()
    side.synchronize()
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            q.copy_(randn(q.shape, 20 + seed, q.dtype))
            gk.copy_(randn(k.shape, 30 + seed, k.dtype))
        pos.random_(0, 1000)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_a_second_backward_of_one_graph_and_compiled():
    print("case axial_rope compiled", flush=True)
    sections, freq = (16, 16), inv_freq((16, 16))
    q, k = make(1, 8, 2, 2, 32, "bnhd", torch.float32)
    pos = torch.randint(0, 9, (8, 2), generator=torch.Generator().manual_seed(0)).to(DEV)
    q, k = q.requires_grad_(), k.requires_grad_()

    def f(q, k):
        a, b = OB.axial_rope(q, k, pos, freq, sections, False)
        return (a * b).sum()

    out = f(q, k)
    want = torch.autograd.grad(out, (q, k), retain_graph=True)
    again = torch.autograd.grad(out, (q, k))
    got = torch.autograd.grad(torch.compile(f)(q, k), (q, k))
    for a, b, c in zip(want, again, got):
        assert torch.equal(a, b)
        torch.testing.assert_close(a, c, rtol=1e-6, atol=1e-6)
