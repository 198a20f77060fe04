"""Rows in 8-bit integers, the RMS norm with such an output, linear and gated linear layers on such rows, against 64 bits."""

import math

import pytest
import torch

from flowmatching_lthc_amd import _abi, ops_int8

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24  # a rounding to fp32


def half_step(dt):
    return torch.finfo(dt).eps / 2


def randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=gen, device=DEV).mul_(std).to(dtype)


def check_rows(q, scale, y, slack):
    """(q, scale) as the 8-bit rows of y [..., C] (float64), which they are formed from with an error of up to `slack` [..., 1].

    The scale is the largest magnitude, off by the slack, divided by 127 with one rounding.  q is y (1 / s) with the
    reciprocal's rounding, 2^-24 of at most 127.1, and the rounding to an integer, 1/2: together below 1/2 + 2^-17."""
    c = y.shape[-1]
    assert q.dtype == torch.int8 and scale.dtype == torch.float32
    assert q.shape == (*y.shape[:-1], -(-c // 16) * 16) and scale.shape == y.shape[:-1]
    assert not q[..., c:].any()
    s = scale.double().unsqueeze(-1)
    want = (y.abs().amax(-1, keepdim=True) / 127).clamp(min=2.0**-126)
    assert bool(((s - want).abs() <= slack / 127 + 1.01 * U * want).all())
    assert bool(((q[..., :c].double() * s - y).abs() <= s * (0.5 + 2.0**-17) + slack).all())
    assert int(q.max()) <= 127 and int(q.min()) >= -127


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,c", [(1, 1), (3, 2), (70, 5), (1, 768), (413, 16), (257, 255), (33, 1219), (5, 1537), (9, 2730), (4, 4097), (3, 8192), (2, 8193), (2, 20011)])
def test_quantize_rows(dtype, m, c):
    x = randn(m, c, dtype=dtype) * 3
    q, s = ops_int8.quantize_rows(x)
    check_rows(q, s, x.double(), torch.zeros(m, 1, device=DEV, dtype=torch.float64))
    assert q.stride() == ops_int8.quantize_rows(x.to("meta"))[0].stride()
    # the quotient rounded once: 53 bits hold enough of it for the second rounding, to 24, to be its only one
    assert torch.equal(s, (x.double().abs().amax(-1) / 127).float().clamp(min=ops_int8.TINY))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_of_the_smallest_and_of_the_largest_numbers(dtype):
    info = torch.finfo(dtype)
    small = torch.tensor([0.0, -0.0, info.smallest_normal, -info.smallest_normal / 2], device=DEV, dtype=dtype)
    x = torch.stack([torch.zeros(40, device=DEV, dtype=dtype), small.repeat(10), torch.full((40,), info.max, device=DEV, dtype=dtype), -torch.full((40,), info.max, device=DEV, dtype=dtype)])
    q, s = ops_int8.quantize_rows(x)
    check_rows(q, s, x.double(), torch.zeros(4, 1, device=DEV, dtype=torch.float64))
    assert float(s[0]) == 2.0**-126 and not q[0].any()
    assert bool((q[2, :40] == 127).all()) and bool((q[3, :40] == -127).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [7, 300, 3000, 9001])
def test_rows_that_are_not_finite_have_no_values(dtype, c):
    x = randn(6, c, dtype=dtype)
    x[1, c - 1] = math.nan
    x[3, c // 2] = math.inf
    x[4, 0] = -math.inf
    q, s = ops_int8.quantize_rows(x)
    assert s.isnan().tolist() == [False, True, False, True, True, False]
    assert not q[[1, 3, 4]].any()
    keep = [0, 2, 5]
    check_rows(q[keep], s[keep], x[keep].double(), torch.zeros(3, 1, device=DEV, dtype=torch.float64))
    w = randn(c, dtype=torch.float32)
    _, qn, sn = ops_int8.norm_quantize(x, w, 1e-6)
    assert sn.isnan().tolist() == [False, True, False, True, True, False] and not qn[[1, 3, 4]].any()


def test_rows_of_any_layout():
    base = randn(5, 6, 40, dtype=torch.bfloat16)
    for x in (base[:, :, 1:38], base[::2, 1], base.transpose(0, 1), base[:, 2:3, :].expand(5, 4, 40), base.permute(2, 0, 1), base[1, 1], base[..., 3:4]):
        q, s = ops_int8.quantize_rows(x)
        qc, sc = ops_int8.quantize_rows(x.contiguous())
        assert torch.equal(q, qc) and torch.equal(s, sc) and q.is_contiguous()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [4, 30, 200, 300, 700, 1000, 1500, 2047, 3500, 4096, 8100, 16001, 16400])
def test_rows_at_any_address_of_an_element(dtype, c):
    wide = randn(11, c + 3, dtype=dtype) * 3
    for first in (0, 1, 2, 3):
        x = wide[:, first : first + c]
        q, s = ops_int8.quantize_rows(x)
        want, ws = ops_int8.quantize_rows(x.contiguous())
        check_rows(q, s, x.double(), torch.zeros(11, 1, device=DEV, dtype=torch.float64))
        assert torch.equal(q, want) and torch.equal(s, ws)
        back = ops_int8.dequantize_rows(q, s, c, dtype)
        assert torch.equal(back, ops_int8.dequantize_rows(q.clone(), s, q.shape[1], dtype)[:, :c])
        w = 1 + 0.1 * randn(c, seed=3)
        for keep in ("sum", "update"):
            assert all(torch.equal(a, b) for a, b in zip(ops_int8.norm_quantize(x, w, 1e-6, x, w, keep=keep), ops_int8.norm_quantize(x.contiguous(), w, 1e-6, x.contiguous(), w, keep=keep)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,c,k", [(1, 1, 16), (13, 37, 48), (300, 768, 768), (7, 2730, 2736)])
def test_dequantize_rows(dtype, m, c, k):
    q = torch.randint(-128, 128, (m, k), device=DEV, dtype=torch.int8, generator=torch.Generator(device=DEV).manual_seed(1))
    s = randn(m).abs() * 1e-2
    out = ops_int8.dequantize_rows(q, s, c, dtype)
    want = q[:, :c].double() * s.double().unsqueeze(-1)
    assert out.dtype == dtype and out.shape == (m, c)
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0  # half a step of fp16's subnormal numbers
    assert bool(((out.double() - want).abs() <= (half_step(dtype) + 1.01 * U) * want.abs() + tiny).all())
    wide = torch.zeros(m, k + 32, device=DEV, dtype=torch.int8)
    wide[:, 16 : 16 + k] = q
    assert torch.equal(ops_int8.dequantize_rows(wide[:, 16 : 16 + k], s, c, dtype), out)
    assert torch.equal(ops_int8.dequantize_rows(q[:1].expand(m, k), s[:1].expand(m), c, dtype), out[:1].expand(m, c))


def norm_case(b, n, c, dtype, gate, mod, residual, param=None):
    """Operands of norm_quantize; gate, shift and scale are parts of one row of a sample."""
    x = randn(b, n, c, dtype=dtype, seed=1) * 2
    r = randn(b, n, c, dtype=dtype, seed=2) * 3 if residual else None
    w = 1 + 0.1 * randn(c, seed=3)
    g, sh, sc = randn(b, 3 * c, dtype=param or dtype, seed=4, std=0.5).chunk(3, dim=-1)
    return x, w, r, g if gate else None, sh if mod else None, sc if mod else None


def check_norm(x, w, r, g, sh, sc, keep, eps=1e-6):
    kept, q, s = ops_int8.norm_quantize(x, w, eps, r, g, sh, sc, keep)
    row = lambda t: t.double().unsqueeze(1) if t.dim() == 2 else t.double()  # noqa: E731
    u = x.double() if g is None else x.double() * row(g)
    t = u if r is None else u + r.double()
    y = t / (t.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    shift = torch.zeros_like(y)
    if sc is not None:
        y = y * (1 + row(sc))
        shift = row(sh).expand_as(y)
        y = y + shift
    # t has one rounding; the sum of squares up to 32 in a row of a thread's and those of the additions over threads, half of
    # which pass to the root; the root, its product, w (1 + scale) and the last step one or two each: below 2^-18 of the terms
    slack = (2.0**-18 * (y.abs() + 2 * shift.abs())).amax(-1, keepdim=True)
    check_rows(q, s, y, slack)
    if keep == "none":
        assert kept.numel() == 0 and kept.dtype == x.dtype
        return
    want = t if keep == "sum" else u
    tiny = 2.0**-25 if x.dtype == torch.float16 else 0.0
    assert kept.dtype == x.dtype and kept.shape == x.shape
    step = half_step(x.dtype) + 1.01 * U if x.dtype != torch.float32 else 1.01 * U
    assert bool(((kept.double() - want).abs() <= step * want.abs() + tiny).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep", ["none", "sum", "update"])
@pytest.mark.parametrize("gate,mod,residual", [(False, False, False), (True, True, True), (False, True, True), (True, False, False)])
def test_norm_quantize_forms(dtype, keep, gate, mod, residual):
    check_norm(*norm_case(3, 37, 768, dtype, gate, mod, residual), keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,c", [(1, 1, 1), (1, 1, 768), (2, 3, 9), (64, 1, 48), (5, 77, 255), (3, 5, 1030), (2, 33, 1219), (2, 3, 1540), (1, 3, 2048), (2, 2, 4095), (2, 2, 8192), (1, 3, 8195), (2, 2, 20000)])
def test_norm_quantize_sizes(dtype, b, n, c):
    check_norm(*norm_case(b, n, c, dtype, True, True, True), "sum")


def test_norm_quantize_takes_rows_for_all_samples_other_types_and_two_dimensions():
    x, w, r, g, sh, sc = norm_case(4, 50, 300, torch.bfloat16, True, True, True, param=torch.float32)
    check_norm(x, w, r, g, sh, sc, "update")
    check_norm(x, w.half(), r, g[0], sh[1], sc[1], "sum")
    check_norm(x[0], w.bfloat16(), r[0], g[0], sh[0], sc[0], "sum")
    # strided rows of x and the residual, gate and modulation of unlike strides
    wide = randn(4, 50, 320, dtype=torch.bfloat16, seed=9)
    check_norm(wide[:, :, 5:305], w, wide[:, :, 20:], g.contiguous(), sh, sc.contiguous(), "sum")
    check_norm(x.transpose(0, 1), w, r.transpose(0, 1), None, None, None, "sum")


@pytest.mark.parametrize("keep", ["sum", "update"])
@pytest.mark.parametrize("c", [768, 1100, 9001])  # a row in registers of a wavefront, of a block, and longer ones
def test_what_is_kept_may_take_the_place_of_an_operand(keep, c):
    x, w, r, g, sh, sc = norm_case(2, 21, c, torch.bfloat16, True, True, True)
    want = ops_int8.norm_quantize(x, w, 1e-6, r, g, sh, sc, keep)
    lib, k = _abi.load(), ops_int8.padded(c)
    for place in ("residual", "x"):
        to = {"residual": r.clone(), "x": x.clone()}
        kept, a, b = to[place], to["x"], to["residual"]
        q, s = torch.zeros(42, k, device=DEV, dtype=torch.int8), torch.zeros(42, device=DEV)
        rc = lib.lthc_norm_quantize(
            a.data_ptr(), _abi.BF16, c, b.data_ptr(), c, g.data_ptr(), _abi.BF16, g.stride(0), w.data_ptr(), _abi.F32, sh.data_ptr(),
            sc.data_ptr(), _abi.BF16, sh.stride(0), {"sum": 1, "update": 2}[keep], kept.data_ptr(), q.data_ptr(), k, s.data_ptr(), 2, 21, c,
            1e-6, torch.cuda.current_stream().cuda_stream,
        )  # fmt: skip
        _abi.check(rc, "lthc_norm_quantize")
        for got, w_ in zip((kept, q, s), want):
            assert torch.equal(got.view(-1), w_.reshape(-1))


def test_norm_quantize_of_zeros():
    x = torch.zeros(2, 3, 100, device=DEV, dtype=torch.bfloat16)
    kept, q, s = ops_int8.norm_quantize(x, torch.ones(100, device=DEV), 1e-6, x, keep="sum")
    assert not q.any() and not kept.any() and bool((s == 2.0**-126).all())


def int8_case(m, n, k, seed=0, q_ld=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ints = lambda r, c: torch.randint(-128, 128, (r, c), device=DEV, dtype=torch.int8, generator=gen)  # noqa: E731
    q = ints(m, q_ld or k)[:, :k]
    s = torch.rand(m, device=DEV, generator=gen) * 0.02 + 1e-3
    v = torch.rand(n, device=DEV, generator=gen) * 0.02 / math.sqrt(k) + 1e-4
    return q, s, ints(n, k), v, torch.randn(n, device=DEV, generator=gen)


def product64(q, s, w, v, b):
    """(h, the size of what its fp32 roundings are relative to) in 64 bits."""
    p = torch.matmul(q.double(), w.t().contiguous().double()) * s.double().unsqueeze(-1) * v.double()
    h = p if b is None else p + b.double()
    return h, p.abs() + h.abs()


def check_linear(q, s, w, v, b, dtype):
    y = ops_int8.int8_linear(q, s, w, v, b, dtype)
    h, size = product64(q, s, w, v, b)
    assert y.dtype == dtype and y.shape == h.shape
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    # the sum to fp32, two products and the addition: a rounding each; then the result's own
    store = half_step(dtype) * h.abs() if dtype != torch.float32 else 0.0
    assert bool(((y.double() - h).abs() <= 3.1 * U * size + 1.01 * store + tiny).all())
    return y


SIZES = [(1, 1, 16), (1, 768, 768), (3, 5, 32), (16, 33, 144), (17, 130, 2048), (33, 64, 128), (65, 129, 272), (100, 1, 784), (257, 255, 464), (413, 1219, 160), (700, 130, 4096), (1025, 520, 64), (2048, 2304, 768)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int8_linear(dtype, m, n, k):
    q, s, w, v, b = int8_case(m, n, k)
    y = check_linear(q, s, w, v, b, dtype)
    check_linear(q, s, w, v, None, dtype)
    assert torch.equal(ops_int8.int8_linear(q, s, w, v, b, dtype), y)


def check_gated(q, s, w, v, b, act, dtype):
    y = ops_int8.int8_gated_linear(q, s, w, v, b, act, dtype)
    h, size = product64(q, s, w, v, b)
    g, u = h.chunk(2, -1)
    eg, eu = (3.1 * U * size).chunk(2, -1)
    if act == "silu":
        a = g * torch.sigmoid(g)
    elif act == "gelu":
        a = g * 0.5 * torch.erfc(-g / math.sqrt(2))
    else:
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)))
    # slopes stay below 1.2; the functions themselves are off by (|g| + 6) 2^-24 relative where a power of e is taken of the
    # rounded argument, by 2^-23 |g| / 2 where 1 + erf is formed: both below 2^-19 |g| for |g| up to 25
    assert float(g.abs().max()) < 25
    ea = 1.2 * eg + 2.0**-19 * g.abs()
    want = a * u
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    store = half_step(dtype) if dtype != torch.float32 else U
    bound = ea * u.abs() + (a.abs() + ea) * eu + 1.01 * store * want.abs() + U * want.abs() + tiny
    assert y.dtype == dtype and y.shape == want.shape
    assert bool(((y.double() - want).abs() <= bound).all())
    return y


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,f,k", [(1, 1, 16), (1, 2048, 768), (5, 33, 48), (30, 65, 2736), (40, 64, 128), (100, 7, 64), (413, 1219, 464), (1030, 256, 1024)])
def test_int8_gated_linear(act, m, f, k):
    q, s, w, v, b = int8_case(m, 2 * f, k)
    for dtype in TYPES:
        check_gated(q, s, w, v, b, act, dtype)
    check_gated(q, s, w, v, None, act, torch.bfloat16)


# Sizes that take each of the kernel's tiles: many tiles a block, last tiles that are not whole, stages that are not.
TILED = [
    (16300, 1792, 2048),  # 256 x 256, two tiles a block
    (14500, 1000, 2064),  # 256 x 256, y's rows not whole lines
    (14592, 1002, 1040),  # 256 x 256 for such rows alone
    (14500, 1001, 2096),  # 256 x 256, an odd width
    (16300, 896, 16),  # 256 x 128, one stage
    (15360, 897, 128),  # 256 x 128, an odd width
    (30000, 1200, 784),  # 256 x 128, several tiles a block
    (13307, 1000, 2064),  # 128 x 128, and so are the following
    (13312, 1002, 1040),
    (15300, 896, 16),
    (30000, 1100, 784),
    (16384, 768, 272),
    (4100, 1030, 400),
    (2000, 1100, 784),  # 128 x 64
    (1030, 1450, 2064),
    (700, 2305, 128),
    (1000, 1102, 784),  # 64 x 64
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", TILED)
def test_int8_linear_tiles(dtype, m, n, k):
    q, s, w, v, b = int8_case(m, n, k)
    y = check_linear(q, s, w, v, b, dtype)
    for _ in range(3):
        assert torch.equal(ops_int8.int8_linear(q, s, w, v, b, dtype), y)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", TILED)
def test_int8_gated_linear_tiles(act, m, n, k):
    q, s, w, v, b = int8_case(m, 2 * (n // 2), k)
    dtype = {"silu": torch.bfloat16, "gelu": torch.float32, "gelu_tanh": torch.float16}[act]
    y = check_gated(q, s, w, v, b, act, dtype)
    for _ in range(3):
        assert torch.equal(ops_int8.int8_gated_linear(q, s, w, v, b, act, dtype), y)


@pytest.mark.parametrize("m", [2, 50, 300])
def test_products_of_rows_of_any_layout(m):
    q, s, w, v, b = int8_case(m, 96, 160)
    want = check_linear(q, s, w, v, b, torch.bfloat16)
    wide = torch.randint(-128, 128, (m, 224), device=DEV, dtype=torch.int8)
    wide[:, 32:192] = q
    wide_w = torch.randint(-128, 128, (96, 208), device=DEV, dtype=torch.int8)
    wide_w[:, 16:176] = w
    far = torch.zeros(m, (1 << 22) + 16, device=DEV, dtype=torch.int8)[:, 64:224].copy_(q)  # rows past the kernel's distance
    odd = torch.zeros(m * 160 + 3, device=DEV, dtype=torch.int8)[3:].view(m, 160).copy_(q)
    for a in (wide[:, 32:192], odd, far, q.t().contiguous().t()):
        for c in (w, wide_w[:, 16:176], w.t().contiguous().t()):
            assert torch.equal(ops_int8.int8_linear(a, s, c, v, b, torch.bfloat16), want)
    three = ops_int8.int8_linear(q.view(2, m // 2, 160), s.view(2, m // 2), w, v, b.bfloat16().float(), torch.bfloat16)
    assert three.shape == (2, m // 2, 96)
    same = ops_int8.int8_linear(q[:1].expand(m, 160), s[:1].expand(m), w[:1].expand(96, 160), v, b, torch.float32)
    assert torch.equal(same, ops_int8.int8_linear(q[:1].repeat(m, 1), s[:1].repeat(m), w[:1].repeat(96, 1), v, b, torch.float32))
    assert torch.equal(ops_int8.int8_linear(q, s, w, v, b.bfloat16(), torch.float32), ops_int8.int8_linear(q, s, w, v, b.bfloat16().float(), torch.float32))


@pytest.mark.parametrize("m", [3, 40, 200])
def test_sums_at_the_ends_of_32_bits(m):
    k = 131056
    q = torch.full((m, k), -128, device=DEV, dtype=torch.int8)
    w = torch.full((20, k), -128, device=DEV, dtype=torch.int8)
    w[1::2] = 127
    one = torch.ones(m, device=DEV)
    y = ops_int8.int8_linear(q, one, w, torch.ones(20, device=DEV), None, torch.float32)
    # one rounding of the integer
    want = torch.tensor([128 * 128 * k, -128 * 127 * k] * 10, device=DEV, dtype=torch.float64).float().expand(m, 20)
    assert torch.equal(y, want)
    with pytest.raises(ValueError, match="131056"):
        ops_int8.int8_linear(q.new_zeros(1, k + 16), one[:1], q.new_zeros(4, k + 16), one.new_ones(4), None, torch.float32)


@pytest.mark.parametrize("m", [1, 64, 300])
def test_a_row_that_is_not_finite_gives_nan_in_its_row_alone(m):
    x = randn(m, 256, dtype=torch.bfloat16)
    x[m // 2, 3] = math.inf
    w, v = ops_int8.quantize_rows(randn(80, 256))
    q, s = ops_int8.quantize_rows(x)
    for y in (ops_int8.int8_linear(q, s, w, v, None, torch.bfloat16), ops_int8.int8_gated_linear(q, s, w, v, None, "silu", torch.bfloat16)):
        bad = y.isnan().all(-1)
        assert bad.nonzero().flatten().tolist() == [m // 2] and not y[~bad].isnan().any()


def test_offsets_past_32_bits():
    m, n = 2_100_000, 1040
    q, s, w, v, b = int8_case(m, n, 16)
    y = ops_int8.int8_linear(q, s, w, v, b, torch.bfloat16)
    assert y.numel() > 2**31
    for rows in (slice(0, 64), slice(m // 2, m // 2 + 64), slice(m - 300, m)):
        part = ops_int8.int8_linear(q[rows], s[rows], w, v, b, torch.bfloat16)
        assert torch.equal(y[rows], part)
    q, s = ops_int8.quantize_rows(y)
    assert q.numel() > 2**31
    for rows in (slice(0, 64), slice(m - 64, m)):
        qr, sr = ops_int8.quantize_rows(y[rows])
        assert torch.equal(q[rows], qr) and torch.equal(s[rows], sr)
    back = ops_int8.dequantize_rows(q, s, n, torch.bfloat16)
    assert torch.equal(back[-64:], ops_int8.dequantize_rows(q[-64:], s[-64:], n, torch.bfloat16))
    del back, q, s
    one = torch.ones(n, device=DEV)
    kept, q, s = ops_int8.norm_quantize(y, one, 1e-6, y, keep="sum")
    tail, qt, st = ops_int8.norm_quantize(y[-64:], one, 1e-6, y[-64:], keep="sum")
    assert torch.equal(kept[-64:], tail) and torch.equal(q[-64:], qt) and torch.equal(s[-64:], st)


def test_no_rows():
    w, v = ops_int8.quantize_rows(randn(48, 32))
    for lead in ((0,), (0, 5), (3, 0)):
        x = torch.empty(*lead, 32, device=DEV, dtype=torch.bfloat16)
        kept, q, s = ops_int8.norm_quantize(x, torch.ones(32, device=DEV), 1e-6, x, keep="sum")
        assert kept.shape == x.shape and q.shape == x.shape and s.shape == lead
        q, s = ops_int8.quantize_rows(x)
        assert ops_int8.dequantize_rows(q, s, 32, torch.float32).shape == x.shape
        assert ops_int8.int8_linear(q, s, w, v).shape == (*lead, 48)
        assert ops_int8.int8_gated_linear(q, s, w, v).shape == (*lead, 24)


def test_refusals():
    x = randn(4, 6, 32, dtype=torch.bfloat16)
    ones = torch.ones(32, device=DEV)
    q, s = ops_int8.quantize_rows(x)
    w, v = ops_int8.quantize_rows(randn(24, 32))
    bad = [
        (lambda: ops_int8.quantize_rows(x.double()), "dtype"),
        (lambda: ops_int8.quantize_rows(x[..., :0]), "channel"),
        (lambda: ops_int8.quantize_rows(x.requires_grad_()), "no_grad"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones.clone().requires_grad_(), 1e-6), "no_grad"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones[:31], 1e-6), "weight"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, x.detach()[:3]), "residual"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, x.detach().float()), "residual"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, gate=ones.expand(6, 32)), "gate"),
        (lambda: ops_int8.norm_quantize(x.detach()[0], ones, 1e-6, gate=ones.expand(6, 32)), "gate"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, shift=ones), "together"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, shift=ones, scale=ones.half()), "dtype"),
        (lambda: ops_int8.norm_quantize(x.detach(), ones, 1e-6, keep="all"), "keep"),
        (lambda: ops_int8.dequantize_rows(q, s, 33), "channels"),
        (lambda: ops_int8.dequantize_rows(q, s, 0), "channels"),
        (lambda: ops_int8.dequantize_rows(q, s[0], 32), "scales"),
        (lambda: ops_int8.dequantize_rows(q, s, 32, torch.float64), "dtype"),
        (lambda: ops_int8.int8_linear(q.float(), s, w, v), "int8"),
        (lambda: ops_int8.int8_linear(q[..., :24], s, w[:, :24], v), "multiple of 16"),
        (lambda: ops_int8.int8_linear(q, s.double(), w, v), "scales"),
        (lambda: ops_int8.int8_linear(q, s, w[:, :16], v), "expected"),
        (lambda: ops_int8.int8_linear(q, s, w, v[:5]), "scales"),
        (lambda: ops_int8.int8_linear(q, s, w, v, ones), "bias"),
        (lambda: ops_int8.int8_linear(q, s, w, v, None, torch.int32), "dtype"),
        (lambda: ops_int8.int8_linear(q, s.clone().requires_grad_(), w, v), "no_grad"),
        (lambda: ops_int8.int8_linear(q, s, w.cpu(), v.cpu()), "need GPU tensors"),
        (lambda: ops_int8.int8_gated_linear(q, s, w[:23], v[:23]), "2F"),
        (lambda: ops_int8.int8_gated_linear(q, s, w, v, None, "relu"), "activation"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
