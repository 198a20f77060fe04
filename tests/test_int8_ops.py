"""The 8-bit inference operators' argument checks and shapes (CPU only, no kernel is launched)."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flowmatching_lthc_amd import _abi, ops_int8

FAKE = ctypes.c_void_p(4096)  # never dereferenced: the checks fail first
ODD = ctypes.c_void_p(4097)


def refused(rc, code, text):
    message = _abi.load().lthc_last_error().decode()
    assert rc == code and text in message, (rc, message)


def test_row_entry_points_refuse_bad_arguments():
    lib = _abi.load()
    inv, uns = _abi.ERR_INVALID, _abi.ERR_UNSUPPORTED
    refused(lib.lthc_quantize_rows(FAKE, 7, 8, FAKE, 16, FAKE, 2, 8, None), inv, "dtype")
    refused(lib.lthc_quantize_rows(FAKE, 1, 8, FAKE, 16, FAKE, 2, 0, None), inv, "positive")
    refused(lib.lthc_quantize_rows(FAKE, 1, 8, FAKE, 16, FAKE, -1, 8, None), inv, "positive")
    refused(lib.lthc_quantize_rows(FAKE, 1, -8, FAKE, 16, FAKE, 2, 8, None), inv, "stride")
    refused(lib.lthc_quantize_rows(ODD, 1, 8, FAKE, 16, FAKE, 2, 8, None), inv, "misaligned")
    refused(lib.lthc_quantize_rows(FAKE, 1, 8, ODD, 16, FAKE, 2, 8, None), inv, "16-byte")
    refused(lib.lthc_quantize_rows(FAKE, 1, 8, FAKE, 16, None, 2, 8, None), inv, "scales")
    refused(lib.lthc_quantize_rows(FAKE, 1, 8, FAKE, 16, FAKE, 2, (1 << 28) + 1, None), uns, "channels")
    refused(lib.lthc_quantize_rows(FAKE, 1, 24, FAKE, 16, FAKE, 2, 24, None), inv, "multiple of 16")
    refused(lib.lthc_quantize_rows(FAKE, 1, 24, FAKE, 40, FAKE, 2, 24, None), inv, "multiple of 16")
    refused(lib.lthc_dequantize_rows(FAKE, 24, FAKE, FAKE, 0, 2, 20, None), inv, "multiple of 16")
    refused(lib.lthc_dequantize_rows(FAKE, 16, FAKE, FAKE, 0, 2, 20, None), inv, "multiple of 16")
    norm = lambda **k: lib.lthc_norm_quantize(*({  # noqa: E731
        "x": FAKE, "dt": 1, "ld": 8, "r": FAKE, "rld": 8, "g": FAKE, "gdt": 1, "gld": 8, "w": FAKE, "wdt": 0, "sh": FAKE, "sc": FAKE,
        "mdt": 1, "mld": 8, "keep": 1, "kept": FAKE, "q": FAKE, "qld": 16, "s": FAKE, "b": 2, "n": 3, "c": 8, "eps": 1e-6, "st": None,
    } | k).values())  # fmt: skip
    refused(norm(w=None), inv, "weight")
    refused(norm(sh=None), inv, "together")
    refused(norm(keep=3), inv, "keep")
    refused(norm(kept=None), inv, "kept")
    refused(norm(gdt=5), inv, "dtype")
    refused(norm(r=ODD), inv, "misaligned")
    refused(norm(mld=-1), inv, "stride")
    refused(norm(b=-1), inv, "negative")
    refused(norm(n=1 << 31), uns, "range")
    assert norm(b=0, w=None) == _abi.OK


def test_row_entry_points_refuse_sizes_whose_products_leave_64_bits():
    lib, uns = _abi.load(), _abi.ERR_UNSUPPORTED
    many = 1 << 60
    refused(lib.lthc_quantize_rows(FAKE, 1, 16, FAKE, 16, FAKE, many, 16, None), uns, "rows")
    refused(lib.lthc_dequantize_rows(FAKE, 16, FAKE, FAKE, 1, many, 16, None), uns, "rows")
    for b, n in ((1 << 40, 1 << 30), (1 << 30, 1 << 30), (1 << 20, 1 << 40)):
        refused(lib.lthc_norm_quantize(FAKE, 1, 16, None, 0, None, 0, 0, FAKE, 0, None, None, 0, 0, 0, None, FAKE, 16, FAKE, b, n, 16, 1e-6, None), uns, "")


@pytest.mark.parametrize("gated", [False, True])
def test_product_entry_points_refuse_bad_arguments(gated):
    lib = _abi.load()
    inv, uns = _abi.ERR_INVALID, _abi.ERR_UNSUPPORTED

    def call(**k):
        a = {"q": FAKE, "ql": 32, "s": FAKE, "w": FAKE, "wl": 32, "v": FAKE, "b": FAKE, "act": 0, "y": FAKE, "dt": 1, "m": 4, "n": 6, "k": 32, "st": None} | k
        if not gated:
            a.pop("act")
        return (lib.lthc_int8_gated_linear if gated else lib.lthc_int8_linear)(*a.values())

    refused(call(k=24), uns, "multiple of 16")
    refused(call(k=131072, wl=131072), uns, "131056")
    refused(call(n=0), inv, "positive")
    refused(call(m=-1), inv, "positive")
    refused(call(n=(1 << 20) + 1), uns, "range")
    refused(call(dt=4), inv, "dtype")
    refused(call(ql=40), inv, "strides")
    refused(call(wl=16), inv, "strides")
    refused(call(wl=1 << 23), inv, "strides")
    refused(call(q=ODD), inv, "16-byte")
    refused(call(w=None), inv, "16-byte")
    refused(call(v=None), inv, "scales")
    refused(call(b=ODD), inv, "bias")
    refused(call(y=ODD), inv, "y is")
    assert call(m=0, q=None) == _abi.OK
    if gated:
        refused(call(act=3), inv, "activation")


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 32)
    q, s = ops_int8.quantize_rows_eager(x)
    for call in (
        lambda: ops_int8.quantize_rows(x),
        lambda: ops_int8.dequantize_rows(q, s, 32),
        lambda: ops_int8.norm_quantize(x, torch.ones(32), 1e-6),
        lambda: ops_int8.int8_linear(q, s, q, s),
        lambda: ops_int8.int8_gated_linear(q, s, q, s),
    ):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


def test_shapes_of_fake_tensors():
    with FakeTensorMode():
        x = torch.empty(2, 5, 40, device="cuda", dtype=torch.float16)
        q, s = ops_int8.quantize_rows(x)
        assert q.shape == (2, 5, 48) and q.dtype == torch.int8 and s.shape == (2, 5) and s.dtype == torch.float32
        kept, q, s = ops_int8.norm_quantize(x, x[0, 0].float(), 1e-6, x, keep="sum")
        assert kept.shape == x.shape and kept.dtype == x.dtype and q.shape == (2, 5, 48)
        assert ops_int8.norm_quantize(x, x[0, 0], 1e-6)[0].shape == (0,)
        long, _ = ops_int8.quantize_rows(torch.empty(3, 2, 2730, device="cuda"))
        assert long.shape == (3, 2, 2736) and long.stride() == (5632, 2816, 1)
        w, v = torch.empty(6, 48, device="cuda", dtype=torch.int8), torch.empty(6, device="cuda")
        y = ops_int8.int8_linear(q, s, w, v, None, torch.float32)
        assert y.shape == (2, 5, 6) and y.dtype == torch.float32
        assert ops_int8.int8_gated_linear(q, s, w, v).shape == (2, 5, 3)
        back = ops_int8.dequantize_rows(q, s, 40, torch.float16)
        assert back.shape == x.shape and back.dtype == x.dtype


@pytest.mark.parametrize("op", ["quantize_rows", "norm_quantize"])
def test_a_call_that_autograd_records_is_refused(op):
    x = torch.empty(2, 32, device="meta", requires_grad=True)
    call = lambda: ops_int8.quantize_rows(x) if op == "quantize_rows" else ops_int8.norm_quantize(x, torch.empty(32, device="meta"), 1e-6)  # noqa: E731
    with pytest.raises(ValueError, match="no_grad"):
        call()
    with torch.no_grad():
        call()


def test_the_eager_rows():
    x = torch.tensor([[127.0, -1.0, 0.4, 63.6], [0.0, 0.0, 0.0, 0.0], [float("nan"), 1.0, 2.0, 3.0], [float("inf"), 1.0, 2.0, 3.0]])
    q, s = ops_int8.quantize_rows_eager(x)
    assert q.shape == (4, 16) and not q[:, 4:].any()
    assert q[0, :4].tolist() == [127, -1, 0, 64] and float(s[0]) == 1.0
    assert not q[1:].any() and float(s[1]) == ops_int8.TINY and s[2:].isnan().all()
