"""The AdamW step over many tensors, its 8-bit states, the norm of all gradients and the optimizer on them, against the
formulas in 64 bits (MI355X only)."""

from __future__ import annotations

import copy
import math

import pytest
import torch

from flowmatching_lthc_amd import optim

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0**-24  # half a step of fp32, relative
HYPER = dict(step=7, lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.05)
RUN = optim.STATE_RUN


def randn(shape, seed, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(DEV, dtype)


def spread(shape, seed, std):
    """Magnitudes over several decades, zeros among them."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * std * 10.0 ** (torch.rand(shape, generator=gen) * 4 - 4)
    return torch.where(torch.rand(shape, generator=gen) < 0.05, 0.0, x).to(DEV)


def codes(m, v, seed):
    """8-bit states: any codes, and scales of the values' sizes."""
    n, gen = m.numel(), torch.Generator().manual_seed(seed)
    runs = -(-n // RUN)
    m8 = torch.randint(-127, 128, (n,), generator=gen, dtype=torch.int8)
    v8 = torch.randint(0, 256, (n,), generator=gen).to(torch.uint8)
    scales = torch.stack([torch.rand(runs, generator=gen) * 1e-3, torch.rand(runs, generator=gen) * 1e-6])
    scales[:, ::5] = 0  # runs that hold nothing yet
    return m8.to(DEV), v8.to(DEV), scales.to(DEV)


def exact_values(m8, v8, scales):
    run = torch.arange(m8.numel(), device=DEV) // RUN
    c, d = m8.double(), v8.double()
    return scales[0].double()[run] * c * c.abs() / 127**2, scales[1].double()[run] * (d / 255) ** 4


class State:
    def __init__(self, shapes, dtype=F32, gdtype=F32, bits=32, master=False, ema=False, seed=0, offset=0):
        def place(t):  # `offset` elements past an allocation's start: addresses that no vector access fits
            flat = torch.empty(t.numel() + offset, device=DEV, dtype=t.dtype)
            return flat[offset:].view(t.shape).copy_(t)

        self.bits = bits
        w = [randn(s, seed + i, std=0.05) for i, s in enumerate(shapes)]
        self.p = [place(t.to(dtype)) for t in w]
        self.g = [place(spread(s, seed + 100 + i, 1e-2).to(gdtype)) for i, s in enumerate(shapes)]
        self.m = [place(spread(s, seed + 200 + i, 1e-3)) for i, s in enumerate(shapes)]
        self.v = [place(spread(s, seed + 300 + i, 1e-3).square()) for i, s in enumerate(shapes)]
        self.scales = []
        if bits == 8:
            got = [codes(m, v, seed + 400 + i) for i, (m, v) in enumerate(zip(self.m, self.v))]
            self.m, self.v, self.scales = [place(t[0]) for t in got], [place(t[1]) for t in got], [t[2] for t in got]
        self.master = [place(t) for t in w] if master else []
        self.ema = [place(t + 0.01) for t in w] if ema else []

    def lists(self):
        return [*self.p, *self.m, *self.v, *self.scales, *self.master, *self.ema]

    def step(self, **kw):
        optim.adamw_step(self.p, self.g, self.m, self.v, scales=self.scales, masters=self.master, emas=self.ema,
                         ema_decay=0.9 if self.ema else 0.0, **{**HYPER, **kw})  # fmt: skip


def check(before: State, after: State, clip=1.0, hyper=HYPER):
    """Each value within its arithmetic's rounding: products and sums are off by U of their terms."""
    (b1, b2), lr, step = hyper["betas"], hyper["lr"], hyper["step"]
    for i in range(len(before.p)):
        if before.p[i].numel() == 0:
            continue
        g = before.g[i].double().flatten() * clip
        old = exact_values(before.m[i], before.v[i], before.scales[i]) if before.bits == 8 else (before.m[i].double(), before.v[i].double())
        m0, v0 = (t.flatten() for t in old)
        m, v = m0 * b1 + g * (1 - b1), v0 * b2 + g * g * (1 - b2)
        # 8-bit values take 5 roundings of their own, clip 3, products and sums the rest
        dm = 12 * U * (m0.abs() * b1 + g.abs() * (1 - b1)) + 1e-44
        dv = 16 * U * v + 1e-44
        if before.bits == 8:
            run = torch.arange(m.numel(), device=DEV) // RUN
            for got, want, slack, code, power, top, least in (
                (exact_values(after.m[i], after.v[i], after.scales[i])[0], m, dm, after.m[i], 2, 127, 0),
                (exact_values(after.m[i], after.v[i], after.scales[i])[1], v, dv, after.v[i], 4, 255, 1),
            ):
                scale = torch.zeros(int(run[-1]) + 1, device=DEV, dtype=torch.float64).scatter_reduce(0, run, want.abs(), "amax")
                assert bool(((after.scales[i][0 if power == 2 else 1] - scale).abs() <= 16 * U * scale + 1e-44).all())
                s = scale[run]
                at = top * (want.abs() / s.clamp(min=1e-300)) ** (1 / power)
                half = 0.5 + 1e-3  # half a code, and what a rounded ratio and root move it by
                low = s * ((at - half).clamp(min=0) / top) ** power
                high = s * ((at + half).clamp(min=float(least) + 1e-3) / top) ** power
                assert bool(((got.abs() >= low * (1 - 1e-6) - slack) & (got.abs() <= high * (1 + 1e-6) + slack)).all())
                assert bool((got * want >= 0).all())
                assert bool((code[want == 0] == 0).all())
                if least:
                    assert bool((code[(want > 1e-40) & (s > 0)] > 0).all())
        else:
            assert bool(((after.m[i].double().flatten() - m).abs() <= dm).all())
            assert bool(((after.v[i].double().flatten() - v).abs() <= dv).all())
        w = (before.master[i] if before.master else before.p[i]).double().flatten()
        root = math.sqrt(1 - b2**step)
        move = lr / (1 - b1**step) * m / (v.sqrt() / root + hyper["eps"])
        p = w * (1 - lr * hyper["weight_decay"]) - move
        # the move: its own 8 roundings, m's error, and v's as half of it under the root
        dp = 3 * U * w.abs() + move.abs() * 16 * U + lr / (1 - b1**step) * dm / (v.sqrt() / root + hyper["eps"])
        if before.master:
            assert bool(((after.master[i].double().flatten() - p).abs() <= dp).all())
            assert torch.equal(after.p[i], after.master[i].to(after.p[i].dtype))
        else:
            fi = torch.finfo(after.p[i].dtype)
            half = fi.eps / 2 if after.p[i].dtype != F32 else 0.0
            err = (after.p[i].double().flatten() - p).abs()
            assert bool((err <= dp * (1 + half) + half * p.abs() + (fi.tiny * fi.eps if half else 0.0)).all())
        if before.ema:
            e = before.ema[i].double().flatten() * 0.9 + p * 0.1
            de = 4 * U * (before.ema[i].double().flatten().abs() + p.abs()) + dp
            assert bool(((after.ema[i].double().flatten() - e).abs() <= de).all())


ODD = [(1,), (3,), (255,), (256,), (257,), (4096,), (4097,), (33, 129), (2, 0, 5), (7, 5, 3), (20000,)]
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16), (F16, BF16)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(d)[6:] for d in t))
@pytest.mark.parametrize("extra", ["plain", "ema", "master_ema"])
@pytest.mark.parametrize("offset", [0, 1])
def test_step_matches_64_bits(bits, types, extra, offset):
    print("case adamw", bits, types, extra, offset, flush=True)
    dtype, gdtype = types
    master = extra == "master_ema" and dtype != F32
    s = State(ODD, dtype, gdtype, bits, master, "ema" in extra, offset=offset)
    before = copy.deepcopy(s)
    s.step()
    check(before, s)


def test_more_tensors_than_a_launch_holds_and_long_ones():
    print("case adamw many", flush=True)
    for bits in (32, 8):
        s = State([(n % 97 + 1, 3) for n in range(150)] + [(1 << 21,)], bits=bits)
        before = copy.deepcopy(s)
        s.step(step=1)
        check(before, s, hyper={**HYPER, "step": 1})


def test_strided_gradients_and_permuted_parameters():
    """A channels-last parameter and its states; a gradient in another layout is brought into it."""
    print("case adamw layouts", flush=True)
    s = State([(6, 4, 3, 5), (16, 8)])
    like = lambda t: t.to(memory_format=torch.channels_last)  # noqa: E731
    plain = copy.deepcopy(s)
    plain.step()
    for name in ("p", "m", "v"):
        getattr(s, name)[0] = like(getattr(s, name)[0])
        getattr(s, name)[1] = getattr(s, name)[1].t().contiguous().t()
    s.g[1] = s.g[1][:1].expand(16, 8)
    plain2 = State([(6, 4, 3, 5), (16, 8)])
    plain2.g[1] = s.g[1].contiguous()
    s.step()
    plain2.step()
    for name in ("p", "m", "v"):
        assert torch.equal(getattr(s, name)[0], getattr(plain, name)[0])
        assert torch.equal(getattr(s, name)[1], getattr(plain2, name)[1])
    with pytest.raises(ValueError, match="exp_avg 0"):
        optim.adamw_step([like(plain.p[0])], [plain.g[0]], [plain.m[0]], [plain.v[0]], step=1)


def test_norm_and_clipping():
    print("case grad norm", flush=True)
    for dtype in (F32, BF16, F16):
        gs = [spread(s, i, 3.0).to(dtype) for i, s in enumerate(ODD * 30)] + [randn((1 << 21,), 5, dtype)[1:]]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        got = optim.grad_norm(gs)
        assert got.shape == () and got.dtype == F32 and abs(float(got) - want) <= 2 * U * want
        assert torch.equal(got, optim.grad_norm(gs))
    big = [torch.full((9,), 3e38, device=DEV)]
    assert abs(float(optim.grad_norm([t * 0.3 for t in big])) / 2.7e38 - 1) < 1e-6  # squares past fp32's range
    assert float(optim.grad_norm([torch.empty(0, device=DEV)])) == 0.0
    strided = randn((40, 30), 1)[:, ::2]
    assert abs(float(optim.grad_norm([strided])) - float(strided.double().norm())) <= 2 * U * float(strided.double().norm())
    s = State(ODD)
    before = copy.deepcopy(s)
    norm = optim.grad_norm(s.g)
    s.step(grad_norm=norm, max_norm=0.25 * float(norm))
    check(before, s, clip=0.25 * float(norm) / (float(norm) + 1e-6))
    wide = copy.deepcopy(before)
    wide.step(grad_norm=norm, max_norm=4 * float(norm))  # within the limit: no clipping
    before.step()
    for a, b in zip(wide.lists(), before.lists()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    """A norm that is not finite leaves every tensor as it is; without one, a NaN stays in its element (32 bits) or its run
    of 256 (8 bits)."""
    print("case adamw non-finite", bits, flush=True)
    for value in (float("nan"), float("inf")):
        s = State([(1000,), (64,)], BF16, bits=bits, master=True, ema=True)
        s.g[0][700] = value
        before = copy.deepcopy(s)
        norm = optim.grad_norm(s.g)
        assert not math.isfinite(float(norm))
        s.step(grad_norm=norm, max_norm=1.0)
        for a, b in zip(s.lists(), before.lists()):
            assert torch.equal(a, b)
        s.step()
        fine = torch.ones(1000, dtype=torch.bool, device=DEV)
        fine[700] = False
        assert torch.equal(torch.isfinite(s.p[0]), fine)
        if bits == 8:
            fine[512:768] = False
            m, v = optim.state_values(s.m, s.v, s.scales)
            assert torch.equal(torch.isfinite(m[0]), fine) and torch.equal(torch.isfinite(v[0]), fine)
        else:
            assert torch.equal(torch.isfinite(s.m[0]), fine)


def test_state_values():
    print("case adamw values", flush=True)
    for n in (1, 255, 256, 1000, 70001):
        m8, v8, scales = codes(torch.empty(n), None, n)
        (m,), (v,) = optim.state_values([m8], [v8], [scales])
        em, ev = exact_values(m8, v8, scales)
        # t = c fl(1/127 or 1/255): 2 U; t^2: 4 U and its own; times A: 6 U in all.  t^4: twice 5 U and its own, times B: 12 U
        assert m.shape == (n,) and bool(((m - em).abs() <= 6 * U * em.abs()).all()) and bool(((v - ev).abs() <= 12 * U * ev).all())
        big = torch.empty(n + 1, device=DEV, dtype=torch.int8)[1:].copy_(m8)  # odd addresses
        (m1,), _ = optim.state_values([big], [v8], [scales])
        assert torch.equal(m, m1)


def test_refusals():
    print("case adamw refusals", flush=True)
    s = State([(300,), (5,)])
    kw = dict(step=1)
    for args, text in (
        (([s.p[0], s.p[0]], [s.g[0], s.g[0]], [s.m[0], s.m[0].clone()], [s.v[0], s.v[0].clone()]), "overlap"),
        (([s.p[0]], [s.g[0]], [s.m[0]], [s.m[0]]), "overlap"),
        (([s.p[0]], [s.g[0]], [s.m[0]], []), "exp_avg_sqs"),
        (([s.p[0]], [s.g[1]], [s.m[0]], [s.v[0]]), "gradient 0"),
        (([s.p[0]], [s.g[0]], [s.m[0].bfloat16()], [s.v[0]]), "exp_avgs"),
        (([s.p[0], s.p[1].bfloat16()], s.g, s.m, s.v), "one dtype"),
        (([s.p[0]], [s.g[0].double()], [s.m[0]], [s.v[0]]), "dtype"),
        (([s.p[0][::2]], [s.g[0][::2]], [s.m[0][::2]], [s.v[0][::2]]), "fill its memory"),
        (([s.p[0]], [s.g[0].cpu()], [s.m[0]], [s.v[0]]), "device|GPU|cuda"),
    ):
        with pytest.raises(ValueError, match=text):
            optim.adamw_step(*args, **kw)
    m8, v8, scales = codes(s.m[0], None, 0)
    with pytest.raises(ValueError, match="scales"):
        optim.adamw_step([s.p[0]], [s.g[0]], [m8], [v8], scales=[scales[:, :1]], **kw)
    with pytest.raises(ValueError, match="exp_avgs"):
        optim.adamw_step([s.p[0]], [s.g[0]], [s.m[0]], [v8], scales=[scales], **kw)
    with pytest.raises(ValueError, match="16-bit"):
        optim.adamw_step([s.p[0]], [s.g[0]], [s.m[0]], [s.v[0]], masters=[s.p[0].clone()], **kw)
    with pytest.raises(ValueError, match="grad_norm"):
        optim.adamw_step([s.p[0]], [s.g[0]], [s.m[0]], [s.v[0]], grad_norm=torch.zeros(2, device=DEV), max_norm=1.0, **kw)
    with pytest.raises(ValueError, match="max_norm"):
        optim.adamw_step([s.p[0]], [s.g[0]], [s.m[0]], [s.v[0]], grad_norm=torch.zeros((), device=DEV), **kw)
    optim.adamw_step([], [], [], [], step=1)


def test_autograd_sees_the_change_of_a_parameter():
    print("case adamw version", flush=True)
    s = State([(8,)])
    p = s.p[0].requires_grad_()
    loss = (p * p).sum()
    s.step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_reads_step_and_rate_anew(bits):
    print("case adamw graph", bits, flush=True)
    shapes = [(300,), (4099,), (64, 32)]
    s, e = (State(shapes, bits=bits) for _ in range(2))
    count, lr = torch.zeros((), device=DEV), torch.full((), 1e-3, device=DEV)

    def step(state, n, rate):
        norm = optim.grad_norm(state.g)
        state.step(step=n, lr=rate, grad_norm=norm, max_norm=0.01)

    scratch = State(shapes, bits=bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(scratch, count + 1, lr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count.add_(1)
        step(s, count, lr)
    for t in range(1, 4):
        lr.fill_(1e-3 * t)
        for i, g in enumerate(s.g):
            g.copy_(spread(g.shape, 1000 * t + i, 1e-2))
            e.g[i].copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        step(e, torch.full((), float(t), device=DEV), lr)
        torch.cuda.synchronize()
        for a, b in zip(s.lists(), e.lists()):
            assert torch.equal(a, b)
    host = State(shapes, bits=bits)  # the host's step and rate give the same scalars
    dev = copy.deepcopy(host)
    host.step(step=3, lr=0.5)
    dev.step(step=torch.full((), 3.0, device=DEV), lr=torch.full((), 0.5, device=DEV))
    for a, b in zip(host.p, dev.p):
        assert float((a - b).abs().max()) <= 1e-6


def test_side_stream():
    print("case adamw side stream", flush=True)
    a, b = State(ODD, bits=8), State(ODD, bits=8)
    a.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step()
    side.synchronize()
    for x, y in zip(a.lists(), b.lists()):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------
# the optimizer
# ---------------------------------------------------------------------------
def model(dtype=F32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 200), torch.nn.GELU(), torch.nn.Linear(200, 8)).to(DEV, dtype)


def backward(m, seed):
    dtype = next(m.parameters()).dtype
    m(randn((64, 40), seed, dtype)).float().square().mean().backward()


def test_optimizer_takes_torch_adamws_steps():
    """Three steps, clipping included: fp32 arithmetic in another order, a few U of |p| and of the move a step."""
    print("case optimizer", flush=True)
    a, b = model(), model()
    ours = optim.AdamW(a.parameters(), lr=1e-3, weight_decay=0.1, max_norm=0.01)
    theirs = torch.optim.AdamW(b.parameters(), lr=1e-3, weight_decay=0.1)
    for t in range(3):
        for m in (a, b):
            m.zero_grad()
        backward(a, t)
        with torch.no_grad():  # the same gradients for both, whatever the products round to
            for p, q in zip(a.parameters(), b.parameters()):
                q.grad = p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(b.parameters(), 0.01)
        ours.step()
        theirs.step()
        assert abs(float(norm) - float(ours.last_grad_norm)) <= 1e-5 * float(norm)
        with torch.no_grad():
            for p, q in zip(a.parameters(), b.parameters()):
                # clip differs by 2^-21 of it; m / sqrt(v) does not feel a common factor but through eps and the roundings
                assert float((p - q).abs().max()) <= (t + 1) * (8 * U * float(q.abs().max()) + 1e-3 * 2**-17)
                q.copy_(p)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_in_bf16_with_master_weights_and_its_checkpoint(bits, tmp_path):
    from flowmatching_lthc_amd import checkpoint

    print("case optimizer bf16", bits, flush=True)
    kw = dict(lr=1e-2, state_bits=bits, master_weights=True, ema_decay=0.9, max_norm=1.0)
    a = model(BF16)
    opt = optim.AdamW(a.parameters(), **kw)
    for t in range(2):
        a.zero_grad()
        backward(a, t)
        opt.step()
    if bits == 8:
        big, small = a[0].weight, a[0].bias
        assert opt.state[big]["exp_avg"].dtype == torch.int8 and "scales" in opt.state[big] and "scales" not in opt.state[small]
    path = tmp_path / "ckpt.pt"
    checkpoint.save_checkpoint(path, a, opt, opt.ema_params(a.parameters()), 2)
    ckpt = checkpoint.load_checkpoint(path, map_location=DEV)
    b = model(BF16)
    checkpoint.load_model_state(b, ckpt, "model")
    opt2 = optim.AdamW(b.parameters(), **kw)
    opt2.load_state_dict(ckpt["optimizer"])
    for m in (a, b):
        m.zero_grad()
    backward(a, 9)
    for p, q in zip(a.parameters(), b.parameters()):
        q.grad = p.grad.clone()
    opt.step()
    opt2.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and torch.equal(p, opt.state[p]["master"].bfloat16())
        for key, value in opt.state[p].items():
            assert torch.equal(torch.as_tensor(value), torch.as_tensor(opt2.state[q][key])), key
    for e, p in zip(opt.ema_params(a.parameters()), a.parameters()):
        assert e.dtype == F32 and e.shape == p.shape


def test_gradients_may_be_there_twice_but_not_in_written_memory():
    print("case adamw gradients shared", flush=True)
    s = State([(300,), (300,)])
    t = State([(300,), (300,)])
    kw = dict(lr=1e-2, step=1)
    optim.adamw_step(s.p, [s.g[0], s.g[0]], s.m, s.v, **kw)
    optim.adamw_step(t.p, [s.g[0], s.g[0].clone()], t.m, t.v, **kw)
    for a, c in zip((*s.p, *s.m, *s.v), (*t.p, *t.m, *t.v)):
        assert torch.equal(a, c)
    whole = torch.zeros(700, device=DEV)
    for g in (s.p[1], s.m[1]):
        with pytest.raises(ValueError, match="overlaps"):
            optim.adamw_step(s.p, [s.g[0], g], s.m, s.v, **kw)
    with pytest.raises(ValueError, match="overlaps"):
        optim.adamw_step([whole[:300]], [whole[299:599]], s.m[:1], s.v[:1], **kw)
    optim.adamw_step([whole[:300]], [whole[300:600]], s.m[:1], s.v[:1], **kw)  # side by side
    with pytest.raises(ValueError, match="overlaps"):
        optim.adamw_step([whole[:300]], s.g[:1], s.m[:1], s.v[:1], lr=1e-2, step=whole[:1])
    with pytest.raises(ValueError, match="overlaps"):
        optim.adamw_step([whole[:300]], s.g[:1], s.m[:1], s.v[:1], lr=1e-2, step=1, grad_norm=whole[299:300], max_norm=1.0)


@pytest.mark.parametrize("decay", [0.9999, 0.4, 0.0])
def test_the_moving_average_keeps_no_bias_over_many_steps(decay):
    """Against the recursion in 64 bits on the same noisy weights, in the mean of 4096 elements.

    A step rounds the difference, its product and the sum: at most U of a value near 1 for the sum, and 1 - d as much of the
    move for the others.  These roundings fall on either side alike; remembered for 1 / (1 - d) steps they leave
    0.6 U sqrt(1 / (2 (1 - d))) an element at most, 2.5e-6 at 0.9999, and a 64th of that in the mean: 4e-8.  2e-6 is asked for (3e-5 of an element);
    weights of d and 1 - d that are rounded by themselves would be off by 1.7e-4 (1 - 0.9999^4000) = 5.5e-5."""
    print("case adamw moving average", decay, flush=True)
    n, steps = 4096, 4000 if decay > 0.9 else 50
    noise = randn((64, n), 1, std=0.05) + 0.8
    p, g, m, v, e = (torch.zeros(n, device=DEV) for _ in range(5))
    e.fill_(0.8)
    want = e.double()
    for t in range(steps):
        p.copy_(noise[t % 64].roll(t))
        optim.adamw_step([p], [g], [m], [v], step=t + 1, lr=0.0, emas=[e], ema_decay=decay)
        want = want + (p.double() - want) * (1 - decay)
    assert abs(float((e.double() - want).mean())) <= 2e-6
    assert float((e.double() - want).abs().max()) <= 3e-5
    if decay == 0.0:
        assert torch.equal(e, p)
