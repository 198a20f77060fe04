"""Refusals, fakes and host logic of the training step's operators: CPU only, no kernel runs."""

from __future__ import annotations

import copy
import ctypes

import pytest
import torch
import torch.testing._internal.two_tensor

from flowmatching_lthc_amd import _abi, optim
from flowmatching_lthc_amd import ops_branch as OB


def err(rc):
    return rc, _abi.load().lthc_last_error().decode()


FAKE = ctypes.c_void_p(4096)  # never dereferenced: the checks fail first


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def rope(sections=(32, 32), D=64, heads=2, N=4, dtype=_abi.BF16, q=FAKE, interleaved=1, strides=None, pos=1, axes=None, B=2):
    s = strides or i64(N * heads * D, heads * D, D, N * heads * D, heads * D, D)
    n = len(sections) if axes is None else axes
    return err(_abi.load().lthc_axial_rope(q, FAKE, s, heads, FAKE, FAKE, s, heads, dtype, FAKE, pos, i64(0, n, 1), FAKE,
                                           i64(*sections), n, interleaved, 0, B, N, D, None))  # fmt: skip


def test_axial_rope_refusals_of_the_c_entry():
    for kw, text in (
        (dict(sections=(31, 32)), "even"),
        (dict(sections=(0, 32)), "even"),
        (dict(sections=(64, 32)), "wider"),
        (dict(sections=(2,) * 5), "axes"),
        (dict(axes=0), "axes"),
        (dict(dtype=5), "dtype"),
        (dict(pos=9), "position"),
        (dict(q=None), "NULL"),
        (dict(q=ctypes.c_void_p(4097)), "misaligned"),
        (dict(q=ctypes.c_void_p(4098)), "even"),
        (dict(strides=i64(8, 65, 64, 8, 64, 64)), "even"),
        (dict(D=65, strides=i64(520, 130, 65, 520, 130, 65)), "even"),
        (dict(sections=(1024, 1024), D=2048), "wide"),
        (dict(B=-1), "negative"),
        (dict(N=1 << 31), "tokens"),
    ):
        rc, msg = rope(**kw)
        assert rc in (_abi.ERR_INVALID, _abi.ERR_UNSUPPORTED) and text in msg, (kw, rc, msg)
    assert rope(B=0)[0] == _abi.OK and rope(N=0)[0] == _abi.OK and rope(heads=0)[0] == _abi.OK


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, device="meta", dtype=dtype)


def test_axial_rope_refuses_cpu_tensors_and_predicts_its_outputs():
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="no CPU fallback"):
        OB.axial_rope(q, q, torch.zeros(4, 1), torch.zeros(2, dtype=torch.float64), (4,))
    x = meta(2, 3, 4, 10, 16, dtype=torch.bfloat16)
    q, k = x.select(2, 0), meta(2, 10, 3, 16).transpose(1, 2)
    a, b = torch.ops.jit_thc.axial_rope(q, k, meta(3, 2), meta(4, dtype=torch.float64), [4, 4], True, False)
    assert a.shape == q.shape and a.is_contiguous() and b.stride() == k.stride()


def test_axial_rope_has_no_gradient_of_positions():
    q = torch.zeros(1, 4, 2, 8, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        OB.axial_rope(q, q, torch.zeros(4, 1, requires_grad=True), torch.zeros(2, dtype=torch.float64), (4,))


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
def adamw(n=1, numel=8, p=4096, dtype=_abi.F32, g=_abi.F32, bits=32, scales=None, masters=None, step=1.0, b1=0.9, norm=None, max_norm=1.0, eps=1e-8, ema=0.5):
    arr = (ctypes.c_void_p * n)(*([4096] * n))
    ps = (ctypes.c_void_p * n)(*([p] * n))
    return err(_abi.load().lthc_adamw_step(ps, dtype, arr, g, arr, arr, bits, scales, masters, None, i64(*([numel] * n)), n, step,
                                           1e-3, b1, 0.99, eps, 0.0, ema, None, None, norm, max_norm, None))  # fmt: skip


def test_adamw_refusals_of_the_c_entries():
    arr = (ctypes.c_void_p * 1)(4096)
    for kw, text in (
        (dict(dtype=4), "dtype"),
        (dict(bits=16), "32 or 8"),
        (dict(bits=8), "scales"),
        (dict(p=0), "NULL"),
        (dict(p=4098), "misaligned"),
        (dict(numel=-1), "numel"),
        (dict(step=0.0), "step"),
        (dict(b1=1.0), "betas"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=float("nan")), "eps"),
        (dict(ema=1.5), "ema"),
        (dict(masters=arr), "16-bit"),
        (dict(norm=4096, max_norm=0.0), "max_norm"),
    ):
        rc, msg = adamw(**kw)
        assert rc in (_abi.ERR_INVALID, _abi.ERR_UNSUPPORTED) and text in msg, (kw, rc, msg)
    assert adamw(n=0)[0] == _abi.OK
    assert adamw(numel=0, p=0)[0] == _abi.OK  # empty tensors need no memory
    lib = _abi.load()
    need = lib.lthc_grad_norm_workspace_bytes(i64(5), 1)
    assert need > 0
    rc, msg = err(lib.lthc_grad_norm(arr, _abi.F32, i64(5), 1, 4096, 4096, need - 1, None))
    assert rc == _abi.ERR_INVALID and "workspace" in msg
    rc, msg = err(lib.lthc_grad_norm(arr, _abi.F32, i64(5), 1, None, 4096, need, None))
    assert rc == _abi.ERR_INVALID and "out" in msg
    # many tensors: a place of its own for every launch's partial sums
    assert lib.lthc_grad_norm_workspace_bytes(i64(*([5] * 1001)), 1001) >= 6 * need
    rc, msg = err(lib.lthc_adamw_state_values(arr, arr, arr, arr, (ctypes.c_void_p * 1)(2), i64(5), 1, None))
    assert rc == _abi.ERR_INVALID and "misaligned" in msg


def test_adamw_refuses_cpu_tensors_and_bad_options():
    t = [torch.zeros(3)]
    with pytest.raises(ValueError, match="no CPU fallback"):
        optim.adamw_step(t, t, t, t, step=1)
    with pytest.raises(ValueError, match="no CPU fallback"):
        optim.grad_norm(t)
    with pytest.raises(ValueError, match="no CPU fallback"):
        optim.state_values(t, t, t)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=4), dict(ema_decay=2.0),
               dict(max_norm=0.0), dict(lr=torch.tensor(1e-3))):  # fmt: skip
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(torch.zeros(2))], **kw)


# ---- the class on stand-in kernels
def plain_step(params, grads, avgs, sqs, scales, masters, emas, step, lr, b1, b2, eps, wd, d, dstep, dlr, norm, max_norm):
    step, lr = (step if dstep is None else float(dstep)), (lr if dlr is None else float(dlr))
    for i, (p, g, m, v) in enumerate(zip(params, grads, avgs, sqs)):
        if scales:
            raise NotImplementedError
        g = g.float() * (1.0 if norm is None else min(1.0, max_norm / (float(norm) + 1e-6)))
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).add_(g * g, alpha=1 - b2)
        w = masters[i] if masters else p.float()
        w = w * (1 - lr * wd) - lr / (1 - b1**step) * m / ((v / (1 - b2**step)).sqrt() + eps)
        if masters:
            masters[i].copy_(w)
        p.copy_(w)
        if emas:
            emas[i].mul_(d).add_(w, alpha=1 - d)


@pytest.fixture
def cpu_kernels():
    lib = torch.library.Library("jit_thc", "IMPL")
    lib.impl("adamw_step", plain_step, "CPU")
    lib.impl("grad_norm", lambda gs: torch.linalg.vector_norm(torch.cat([g.float().flatten() for g in gs])), "CPU")
    yield
    lib._destroy()


def parameters(seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype)) for s in ((4, 3), (7,), (2, 2, 2))]


def run(opt, params, steps, seed=100, skip=()):
    for t in range(steps):
        gen = torch.Generator().manual_seed(seed + t)
        for i, p in enumerate(params):
            g = torch.randn(p.shape, generator=gen).to(p.dtype)
            p.grad = None if (t, i) in skip else g
        opt.step()


def test_adamw_takes_torch_adamws_steps(cpu_kernels):
    """Parameters without a gradient on some steps too: each counts its own steps."""
    ours, theirs = parameters(0), parameters(0)
    a = optim.AdamW(ours, lr=1e-2, betas=(0.8, 0.9), weight_decay=0.1)
    b = torch.optim.AdamW(theirs, lr=1e-2, betas=(0.8, 0.9), weight_decay=0.1)
    for opt, ps in ((a, ours), (b, theirs)):
        run(opt, ps, 5, skip={(0, 1), (3, 2)})
    for p, q in zip(ours, theirs):
        torch.testing.assert_close(p, q, rtol=1e-6, atol=1e-6)
    assert [a.state[p]["step"] for p in ours] == [5, 4, 4]


@pytest.mark.parametrize("source", ["own", "torch"])
@pytest.mark.parametrize("capturable", [False, True])
def test_adamw_state_dicts_load(cpu_kernels, source, capturable):
    first = parameters(0, torch.bfloat16)
    kw = dict(lr=1e-2, weight_decay=0.1)
    a = optim.AdamW(first, **kw, master_weights=True, ema_decay=0.9) if source == "own" else torch.optim.AdamW(first, **kw)
    run(a, first, 3)
    saved = copy.deepcopy(a.state_dict())
    second = [torch.nn.Parameter(p.detach().clone()) for p in first]
    b = optim.AdamW(second, **kw, master_weights=True, ema_decay=0.9, capturable=capturable)
    b.load_state_dict(saved)
    if source == "own":
        assert b.param_groups[0]["capturable"] is False  # a saved group's options are the optimizer's
        for p, q in zip(first, second):
            for key in ("exp_avg", "exp_avg_sq", "master", "ema"):
                assert b.state[q][key].dtype == torch.float32 and torch.equal(a.state[p][key], b.state[q][key])
        run(a, first, 2, seed=7)
        run(b, second, 2, seed=7)
        for p, q in zip(first, second):
            assert torch.equal(p, q) and b.state[q]["step"] == 5
    else:
        run(b, second, 1)
        assert all(b.state[q]["step"] == 4 for q in second)
        assert all(b.state[q]["exp_avg"].dtype == torch.float32 for q in second)


def test_adamw_capturable_counts_on_the_device_and_round_trips(cpu_kernels):
    params = parameters(0)
    a = optim.AdamW(params, lr=torch.tensor(1e-2), capturable=True)
    run(a, params, 3)
    counts = {id(a.state[p]["step"]) for p in params}
    assert len(counts) == 1 and float(a.state[params[0]]["step"]) == 3
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    b = optim.AdamW(other, lr=torch.tensor(1e-2), capturable=True)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    run(a, params, 2, seed=9)
    run(b, other, 2, seed=9)
    for p, q in zip(params, other):
        assert torch.equal(p, q) and float(b.state[q]["step"]) == 5


def test_adamw_ema_and_clipping_norm(cpu_kernels):
    params = parameters(0)
    a = optim.AdamW(params, lr=1e-2, ema_decay=0.5, max_norm=1.0)
    before = [p.detach().clone() for p in params]
    assert all(torch.equal(e, p) for e, p in zip(a.ema_params(), before))
    run(a, params, 1)
    want = torch.linalg.vector_norm(torch.cat([p.grad.flatten() for p in params]))
    torch.testing.assert_close(a.last_grad_norm, want)
    for e, p, q in zip(a.ema_params(params), params, before):
        torch.testing.assert_close(e, 0.5 * q + 0.5 * p)


def test_adamw_refuses_states_it_does_not_have(cpu_kernels):
    params = parameters(0)
    b = torch.optim.AdamW(params, amsgrad=True)
    run(b, params, 1)
    with pytest.raises(ValueError, match="amsgrad"):
        optim.AdamW(params).load_state_dict(b.state_dict())


# ---------------------------------------------------------------------------
# gated linear layer
# ---------------------------------------------------------------------------
def gated(M=4, C=16, F=6, x=4096, w=4096, b=4096, y=4096, dtype=_abi.BF16, act=0):
    return err(_abi.load().lthc_gated_linear_fwd(x, w, b, dtype, act, y, M, C, F, None))


def test_gated_linear_refusals_of_the_c_entries():
    for kw, text in (
        (dict(C=12), "multiple of 8"),
        (dict(C=0), "positive"),
        (dict(F=0), "positive"),
        (dict(M=-1), "positive"),
        (dict(dtype=_abi.F32), "bf16 or fp16"),
        (dict(act=3), "activation"),
        (dict(x=None), "aligned"),
        (dict(w=4104), "aligned"),
        (dict(b=4097), "bias"),
        (dict(y=None), "y is NULL"),
        (dict(C=1 << 16, F=1 << 14), "range"),
    ):
        rc, msg = gated(**kw)
        assert rc in (_abi.ERR_INVALID, _abi.ERR_UNSUPPORTED) and text in msg, (kw, rc, msg)
    assert gated(M=0, x=None, w=None, y=None)[0] == _abi.OK
    lib = _abi.load()
    need = lib.lthc_gated_linear_bwd_workspace_bytes(100, 16, 6)
    assert need >= 100 * 16 * 2 + 16 * 16 * 2 and lib.lthc_gated_linear_bwd_workspace_bytes(0, 16, 6) == 0
    for ws, size, text, db, dw in (
        (4096, need - 1, "workspace", 4096, 4096),
        (4096 + 16, need, "workspace", 4096, 4096),
        (None, need, "workspace", 4096, 4096),
        (4096, need, "dw must", 4096, 4104),
        (4096, need, "db must", 4098, 4096),
    ):
        rc, msg = err(lib.lthc_gated_linear_bwd(4096, 4096, 4096, None, _abi.BF16, 0, 4096, dw, db, 100, 16, 6, ws, size, None))
        assert rc == _abi.ERR_INVALID and text in msg, (msg, text)


def test_gated_linear_refuses_cpu_tensors_and_predicts_its_outputs():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        OB.gated_linear(x, w)
    y = OB.gated_linear(meta(2, 5, 8, dtype=torch.bfloat16), meta(6, 8, dtype=torch.bfloat16))
    assert y.shape == (2, 5, 3) and y.dtype == torch.bfloat16
    gx, gw, gb = OB.gated_linear_backward(y, meta(2, 5, 8), meta(6, 8), None, "silu", True, False, False)
    assert gx.shape == (2, 5, 8) and gw.shape == (0, 8) and gb.shape == (0,)


def test_gated_linear_eager_is_swiglu_of_the_projections():
    x, w, b = torch.randn(4, 8), torch.randn(6, 8), torch.randn(6)
    want = OB.swiglu_eager(torch.nn.functional.linear(x, w, b))
    torch.testing.assert_close(OB.gated_linear_eager(x, w, b), want)


def test_gated_linear_stays_off_in_the_model_by_default():
    from flowmatching_lthc_amd.model import SwiGLUFFN

    ffn = SwiGLUFFN(16, 48)
    assert ffn.fused_projections is False
    x = torch.randn(3, 16)
    ffn.fused_projections = True  # CPU tensors keep the eager sequence
    torch.testing.assert_close(ffn(x), ffn.w3(OB.swiglu_eager(ffn.w12(x))))


class Wrapped(torch.nn.Module):
    """A layer around another, as adapters and loggers are; it has no weight of its own."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x) + 1


def test_the_feed_forward_runs_a_replaced_projection():
    from flowmatching_lthc_amd.model import SwiGLUFFN

    ffn, x = SwiGLUFFN(16, 48), torch.randn(3, 16)
    ffn.w12 = Wrapped(ffn.w12)
    torch.testing.assert_close(ffn(x), ffn.w3(OB.swiglu_eager(ffn.w12.inner(x) + 1)))


def test_a_feed_forward_without_the_switch_in_its_own_state_runs():
    """As a whole module that was saved before the switch existed."""
    from flowmatching_lthc_amd.model import SwiGLUFFN

    ffn, x = SwiGLUFFN(16, 48), torch.randn(3, 16)
    old = SwiGLUFFN.__new__(SwiGLUFFN)
    old.__dict__.update({k: v for k, v in ffn.__dict__.items() if k != "fused_projections"})
    assert torch.equal(old(x), ffn(x))


class Scaled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


def projections():
    from flowmatching_lthc_amd.model import CastLinear

    class Adapted(CastLinear):
        def forward(self, x):
            return super().forward(x) + 1

    def hooked(register):
        layer = CastLinear(8, 8)
        getattr(layer, register)(lambda *args: None)
        return layer

    parametrized, own_forward, subclass = CastLinear(8, 8), CastLinear(8, 8), CastLinear(8, 8)
    torch.nn.utils.parametrize.register_parametrization(parametrized, "weight", Scaled())
    own_forward.forward = lambda x: x
    subclass.weight = torch.nn.Parameter(torch.testing._internal.two_tensor.TwoTensor(torch.ones(8, 8), torch.ones(8, 8)))
    yield from ((n, hooked("register_" + n)) for n in ("forward_hook", "forward_pre_hook", "full_backward_hook", "full_backward_pre_hook"))
    yield from (("another module", Wrapped(CastLinear(8, 8))), ("subclass", Adapted(8, 8)), ("parametrized", parametrized))
    yield from (("forward of its own", own_forward), ("tensor subclass", subclass))


def test_the_fused_feed_forward_passes_by_plain_projections_only():
    from flowmatching_lthc_amd.model import CastLinear, _plain_projection

    assert _plain_projection(CastLinear(8, 8)) and _plain_projection(CastLinear(8, 8, bias=False))
    for name, layer in projections():
        assert not _plain_projection(layer), name
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *args: None)
    try:
        assert not _plain_projection(CastLinear(8, 8))
    finally:
        handle.remove()


def test_adamw_capturable_counts_part_where_steps_part(cpu_kernels):
    """A parameter without a gradient in a step keeps its count, as without capturable."""
    ours, plain = parameters(0), parameters(0)
    a = optim.AdamW(ours, lr=1e-2, capturable=True)
    b = optim.AdamW(plain, lr=1e-2)
    skip = {(1, 0), (2, 0), (3, 2)}
    run(a, ours, 5, skip=skip)
    run(b, plain, 5, skip=skip)
    for p, q in zip(ours, plain):
        assert float(a.state[p]["step"]) == b.state[q]["step"]
        assert torch.equal(p, q)
    assert [b.state[q]["step"] for q in plain] == [3, 5, 4]


def test_adamw_refuses_captures_that_would_not_replay(cpu_kernels, monkeypatch):
    params = parameters(0)
    a = optim.AdamW(params, lr=1e-2, capturable=True)
    b = optim.AdamW(params, lr=1e-2)
    c = optim.AdamW(params, lr=1e-2, capturable=True, ema_decay=0.9)
    run(a, params, 1)
    run(b, params, 1)
    before = [p.detach().clone() for p in params]
    monkeypatch.setattr(optim, "_capturing", lambda t: True)
    run(a, params, 1)  # laid out before: as it should be
    for opt, skip, text in ((b, (), "capturable"), (c, (), "outside the capture"), (a, {(0, 1)}, "same gradients")):
        now = [p.detach().clone() for p in params]
        with pytest.raises(RuntimeError, match=text):
            run(opt, params, 1, skip=skip)
        assert all(torch.equal(p, q) for p, q in zip(params, now))
    assert not all(torch.equal(p, q) for p, q in zip(params, before))


def test_gated_linear_workspace_of_sizes_out_of_range():
    query = _abi.load().lthc_gated_linear_bwd_workspace_bytes
    for sizes in ((0, 8, 8), (8, -8, 8), (1 << 40, 8, 8), (8, 1 << 40, 8), (8, 8, 1 << 40), (8, 1 << 19, 1 << 19), (-1, 1 << 62, 1 << 62)):
        assert query(*sizes) == 0, sizes
    assert query(8, 8, 8) > 0


def test_adamw_copies_and_pickles(cpu_kernels, tmp_path):
    params = parameters(0)
    a = optim.AdamW(params, lr=1e-2, max_norm=0.5, ema_decay=0.9)
    run(a, params, 2)
    held = [a.state[p]["exp_avg"] for p in params]
    torch.save(a, tmp_path / "opt.pt")
    copies = [copy.deepcopy(a), torch.load(tmp_path / "opt.pt", weights_only=False)]
    run(a, params, 1, seed=7)
    for b in copies:
        others = b.param_groups[0]["params"]
        assert b.max_norm == 0.5 and b.last_grad_norm is not None
        run(b, others, 1, seed=7)
        for p, q in zip(params, others):
            assert p is not q and torch.equal(p, q) and torch.equal(a.state[p]["ema"], b.state[q]["ema"])
    assert all(a.state[p]["exp_avg"] is h for p, h in zip(params, held))


def test_a_capture_right_after_capturable_is_set_is_refused(cpu_kernels, monkeypatch):
    """Counts that are still the host's would be captured as constants: every replay would take the same step."""
    first, params = parameters(0), parameters(0)
    a = optim.AdamW(first, lr=1e-2)
    run(a, first, 2)
    b = optim.AdamW(params, lr=1e-2, capturable=True)
    b.load_state_dict(a.state_dict())  # a saved group's options are the optimizer's: not capturable
    b.param_groups[0]["capturable"] = True
    capturing = True
    monkeypatch.setattr(optim, "_capturing", lambda t: capturing)
    with pytest.raises(RuntimeError, match="outside the capture"):
        run(b, params, 1)
    capturing = False
    run(b, params, 1)
    capturing = True
    run(b, params, 1)
    assert all(float(b.state[p]["step"]) == 4 for p in params)


@pytest.mark.parametrize("capturable", [False, True])
def test_adamw_groups_take_their_own_options(cpu_kernels, capturable):
    """Two groups of unlike types and options, one norm over both, against torch's optimizer on clipped gradients; a third
    group added later counts its own steps."""
    small = parameters(0), parameters(1, torch.bfloat16), parameters(2)
    ours, theirs = ([[torch.nn.Parameter(p.detach().clone()) for p in ps] for ps in small] for _ in range(2))
    options = (dict(lr=1e-2, weight_decay=0.1, ema_decay=0.5), dict(lr=3e-2, betas=(0.5, 0.8)), dict(lr=1e-3, eps=1e-4))
    plain = [{k: v for k, v in o.items() if k != "ema_decay"} for o in options]
    a = optim.AdamW([{"params": ps, **o} for ps, o in zip(ours[:2], options)], max_norm=0.5, capturable=capturable)
    b = torch.optim.AdamW([{"params": ps, **o} for ps, o in zip(theirs[:2], plain)])
    for t in range(5):
        if t == 3:
            a.add_param_group({"params": ours[2], **options[2]})
            b.add_param_group({"params": theirs[2], **plain[2]})
        gen = torch.Generator().manual_seed(50 + t)
        grads = [[torch.randn(p.shape, generator=gen).to(p.dtype) for p in ps] for ps in small[: len(a.param_groups)]]
        clip = 0.5 / (torch.linalg.vector_norm(torch.cat([g.flatten().float() for gs in grads for g in gs])) + 1e-6)
        for mine, other, gs in zip(ours, theirs, grads):
            for p, q, g in zip(mine, other, gs):
                p.grad, q.grad = g, (g.float() * clip).to(g.dtype)
        a.step()
        b.step()
    for mine, other in zip(ours, theirs):
        for p, q in zip(mine, other):
            # bf16: five steps' weights are rounded (2^-8 each), and there the states and the clipped gradients too, whose
            # steps of 3e-2 they move by a few 2^-8 more
            rtol, atol = (1e-5, 1e-6) if p.dtype == torch.float32 else (6 * 2.0**-8, 5 * 3e-2 * 8 * 2.0**-8)
            torch.testing.assert_close(p, q, rtol=rtol, atol=atol)
            assert float(a.state[p]["step"]) == float(b.state[q]["step"])
    assert all("ema" in a.state[p] for p in ours[0]) and not any("ema" in a.state[p] for p in (*ours[1], *ours[2]))
