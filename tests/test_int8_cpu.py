"""The 8-bit inference ops without a GPU: what they refuse, the shapes and layouts they promise, and the C ABI's status codes."""

import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from dmf_b200 import _lib
from dmf_b200.int8 import MAX_K, Int8Rows, int8_linear, ln_modulate_int8, quantize_int8, rms_norm_int8

FAKE = 0x10000  # never dereferenced by validation


def test_no_cpu_path():
    x = torch.randn(3, 64)
    rows = Int8Rows(torch.zeros(3, 64, dtype=torch.int8), torch.ones(3))
    for f in (lambda: quantize_int8(x), lambda: rms_norm_int8(x, torch.ones(64)), lambda: rows.dequantize(),
              lambda: ln_modulate_int8(x[None], x[:1], x[:1]), lambda: int8_linear(rows, rows)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


@pytest.fixture
def cuda_shapes():
    """CUDA tensors that have a type, a shape and strides, but no data"""
    with FakeTensorMode(allow_non_fake_inputs=False):
        yield lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda:0")


def test_shapes_and_layouts(cuda_shapes):
    t = cuda_shapes
    rows = quantize_int8(t(2, 5, 100), "gelu")
    assert rows.values.shape == (2, 5, 100) and rows.values.stride() == (5 * 112, 112, 1) and rows.values.dtype == torch.int8
    assert rows.scale.shape == (2, 5) and rows.scale.dtype == torch.float32
    rows, z = rms_norm_int8(t(7, 48), t(48), residual=t(7, 48, dtype=torch.float32))
    assert rows.values.stride() == (48, 1) and z.dtype == torch.float32 and z.shape == (7, 48)
    rows, z = ln_modulate_int8(t(2, 7, 33), t(2, 33), t(2, 1, 33), gate=t(2, 33), h=t(2, 7, 33))
    assert rows.values.stride() == (7 * 48, 48, 1) and z.dtype == torch.bfloat16
    w = quantize_int8(t(20, 33))
    assert int8_linear(rows, w, t(20), out_dtype=torch.float16).shape == (2, 7, 20)
    assert rows.dequantize(torch.float32).shape == (2, 7, 33)


def test_refusals(cuda_shapes):
    t = cuda_shapes
    r8 = lambda *s: Int8Rows(t(*s, dtype=torch.int8), t(*s[:-1], dtype=torch.float32))
    for error, f in [
        (ValueError, lambda: quantize_int8(t(3, 64), "relu")),
        (TypeError, lambda: quantize_int8(t(3, 64, dtype=torch.float64))),
        (TypeError, lambda: quantize_int8(t(3, 64, dtype=torch.int8))),
        (ValueError, lambda: quantize_int8(t(3, 0))),
        (ValueError, lambda: quantize_int8(t())),
        (ValueError, lambda: rms_norm_int8(t(3, 64), t(63))),
        (ValueError, lambda: rms_norm_int8(t(3, 64), t(64), residual=t(2, 64))),
        (ValueError, lambda: ln_modulate_int8(t(3, 64), t(1, 64), t(1, 64))),
        (ValueError, lambda: ln_modulate_int8(t(2, 3, 64), t(1, 64), t(2, 64))),
        (ValueError, lambda: ln_modulate_int8(t(2, 3, 64), t(2, 64), t(2, 3, 64))),
        (ValueError, lambda: ln_modulate_int8(t(2, 3, 64), t(2, 64), t(2, 64), gate=t(2, 64))),
        (ValueError, lambda: ln_modulate_int8(t(2, 3, 64), t(2, 64), t(2, 64), gate=t(2, 64), h=t(2, 4, 64))),
        (ValueError, lambda: int8_linear(r8(3, 64), r8(5, 63))),
        (ValueError, lambda: int8_linear(r8(3, 64), r8(2, 5, 64))),
        (ValueError, lambda: int8_linear(r8(3, 64), r8(0, 64))),
        (ValueError, lambda: int8_linear(r8(3, 64), r8(5, 64), t(4))),
        (ValueError, lambda: int8_linear(r8(3, MAX_K + 1), r8(5, MAX_K + 1))),
        (ValueError, lambda: int8_linear(r8(3, 1), r8(2 ** 30 + 1, 1))),
        (ValueError, lambda: quantize_int8(t(2, 2 ** 20 + 1))),
        (ValueError, lambda: quantize_int8(t(2 ** 31, 1))),
        (TypeError, lambda: int8_linear(r8(3, 64), r8(5, 64), out_dtype=torch.int32)),
        (TypeError, lambda: int8_linear(r8(3, 64), r8(5, 64), t(5, dtype=torch.int32))),
        (TypeError, lambda: int8_linear(Int8Rows(t(3, 64), t(3, dtype=torch.float32)), r8(5, 64))),
        (TypeError, lambda: int8_linear(Int8Rows(t(3, 64, dtype=torch.int8), t(3)), r8(5, 64))),
        (ValueError, lambda: int8_linear(Int8Rows(t(3, 64, dtype=torch.int8), t(2, dtype=torch.float32)), r8(5, 64))),
        (TypeError, lambda: r8(3, 64).dequantize(torch.int32)),
    ]:
        with pytest.raises(error):
            f()


def _row_args(a):
    a.batch, a.seqlen, a.channels = 2, 16, 100
    a.x = _lib.Rows(FAKE, 1600, 100)
    a.out = _lib.Int8Matrix(FAKE, 112, FAKE)
    return a


def test_row_entry_points_reject_bad_arguments():
    lib = _lib.load()
    assert lib.dmf_int8_quantize(None) == 1
    for change, status in [(dict(dtype=3), 2), (dict(act=3), 5), (dict(channels=0), 5), (dict(batch=-1), 5), (dict(batch=1 << 30), 5),
                           (dict(x=_lib.Rows(None, 1600, 100)), 1), (dict(x=_lib.Rows(FAKE + 1, 1600, 100)), 7),
                           (dict(x=_lib.Rows(FAKE, -1, 100)), 6), (dict(out=_lib.Int8Matrix(FAKE, 99, FAKE)), 6),
                           (dict(out=_lib.Int8Matrix(None, 112, FAKE)), 1), (dict(out=_lib.Int8Matrix(FAKE, 112, None)), 1),
                           (dict(out=_lib.Int8Matrix(FAKE, 112, FAKE + 2)), 7)]:
        a = _row_args(_lib.Int8QuantizeArgs())
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.dmf_int8_quantize(C.byref(a)) == status, change
    a = _row_args(_lib.Int8RmsNormArgs())
    assert lib.dmf_int8_rmsnorm(C.byref(a)) == 1                       # no weight
    a.weight = FAKE
    a.residual = _lib.Rows(FAKE, 1600, 100)
    assert lib.dmf_int8_rmsnorm(C.byref(a)) == 1                       # a residual without a sum
    a.sum = _lib.Rows(FAKE, 1600, 100)
    a.stream_dtype = 9
    assert lib.dmf_int8_rmsnorm(C.byref(a)) == 2
    b = _row_args(_lib.Int8LnModulateArgs())
    assert lib.dmf_int8_ln_modulate(C.byref(b)) == 1                   # no shift
    b.shift, b.scale = _lib.Mod(FAKE, 600), _lib.Mod(FAKE, 600)
    b.h, b.sum = _lib.Rows(FAKE, 1600, 100), _lib.Rows(FAKE, 1600, 100)
    assert lib.dmf_int8_ln_modulate(C.byref(b)) == 1                   # h without a gate
    b.gate = _lib.Mod(FAKE, -1)
    assert lib.dmf_int8_ln_modulate(C.byref(b)) == 6


def test_linear_rejects_bad_arguments():
    lib = _lib.load()

    def good():
        a = _lib.Int8LinearArgs()
        a.m, a.n, a.k = 3, 5, 64
        a.x, a.w = _lib.Int8Matrix(FAKE, 64, FAKE), _lib.Int8Matrix(FAKE, 64, FAKE)
        a.out, a.out_stride = FAKE, 5
        return a
    for change, status in [(dict(m=-1), 5), (dict(n=0), 5), (dict(k=0), 5), (dict(k=131072), 5), (dict(n=(1 << 30) + 1, out_stride=1 << 31), 5), (dict(out_dtype=3), 2),
                           (dict(bias=FAKE, bias_dtype=7), 2), (dict(bias=FAKE + 1), 7), (dict(out=None), 1), (dict(out=FAKE + 1), 7),
                           (dict(out_stride=4), 6), (dict(x=_lib.Int8Matrix(None, 64, FAKE)), 1), (dict(x=_lib.Int8Matrix(FAKE, -1, FAKE)), 6),
                           (dict(w=_lib.Int8Matrix(FAKE, 64, None)), 1)]:
        a = good()
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.dmf_int8_linear(C.byref(a)) == status, change
    if not torch.cuda.is_available():
        assert lib.dmf_int8_linear(C.byref(good())) == 8               # all checks pass: no device here
        assert lib.dmf_int8_quantize(C.byref(_row_args(_lib.Int8QuantizeArgs()))) == 8
    d = _lib.Int8DequantizeArgs()
    d.rows, d.channels, d.x, d.out, d.out_stride = 3, 64, _lib.Int8Matrix(FAKE, 64, FAKE), FAKE, 63
    assert lib.dmf_int8_dequantize(C.byref(d)) == 6


def test_rows_are_copied_unless_the_tensor_cores_can_read_them():
    from dmf_b200.int8 import _pitched
    buf = torch.arange(0, 2000, dtype=torch.int64).to(torch.int8)
    for v in (buf[:48].expand(9, 48), buf.as_strided((9, 48), (16, 1)), buf[:9 * 50].view(9, 50), buf[1:].as_strided((9, 48), (48, 1))):
        out = _pitched(v)
        assert out.stride(0) == -(-v.shape[1] // 16) * 16 and out.data_ptr() % 16 == 0 and torch.equal(out, v)
    for v in (buf[:9 * 48].view(9, 48), buf.as_strided((9, 40), (64, 1)), buf[:50].view(1, 50), buf.as_strided((1, 50), (0, 1))):
        assert _pitched(v).data_ptr() == v.data_ptr()


def test_dequantize_rejects_rows_that_are_too_wide():
    lib, a = _lib.load(), _lib.Int8DequantizeArgs()
    a.rows, a.x, a.out = 3, _lib.Int8Matrix(FAKE, 1 << 32, FAKE), FAKE
    for channels, status in ((2 ** 20 + 1, 5), (2 ** 31 - 1, 5), (0, 5)):
        a.channels, a.out_stride = channels, 1 << 32
        assert lib.dmf_int8_dequantize(C.byref(a)) == status
