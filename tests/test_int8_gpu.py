"""The 8-bit inference ops against fp64: rows in 8 bits behind activations and norms, and the product of such rows.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32):
* a quantised element is the nearest integer to 127 y / a, where y and a carry the fp32 errors of what stands before: off by at
  most 0.5 + 127 e for a relative error e of the row, with e = 2 u for the quantisation itself (127 / a, times y), and
  - activations: exp and the division within a few u; exp(-t) within (2 + 1.2 |t|) u, and the result's share of a row's maximum is
    below exp(-|t|) |t|, so 16 u covers it;
  - norms: sums of C terms taken as at most C / 32 per thread and a tree of ten: (C / 32 + 10) u, twice (mean and variance), and
    with data of standard deviation about the mean's size a factor of 4: e = 8 (C / 32 + 10) u.
* a scale is within the same e of a / 127, plus one division.
* a product's sum is exact; its conversion, two scales and the bias are four roundings of the terms' magnitudes, and the result is
  rounded once to its type."""

import pytest
import torch

from dmf_b200.int8 import Int8Rows, int8_linear, ln_modulate_int8, quantize_int8, rms_norm_int8
from oracle import int8_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(*shape, dtype=F32, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * sum(shape))
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _check_rows(rows, y, e):
    """rows against the fp64 rows y that were to be quantised, with relative fp32 error e in front of the quantisation"""
    assert rows.values.dtype == torch.int8 and rows.scale.dtype == F32
    assert rows.values.shape == y.shape and rows.scale.shape == y.shape[:-1]
    real, scale = orc.real_rows(y)
    assert int(rows.values.min()) >= -127
    assert float((rows.values.double() - real).abs().max()) <= 0.5 + 127 * (e + 2 * U)
    assert bool(((rows.scale.double() - scale).abs() <= scale * (e + 2 * U)).all())


def _norm_error(C):
    return 8 * (C / 32 + 10) * U


WIDTHS = [1, 7, 8, 64, 100, 257, 384, 1000, 1152, 2040, 4608, 9000]


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
def test_quantize(C, act, dtype):
    for M in (1, 37):
        x = _randn(M, C, dtype=dtype, std=2.0)
        _check_rows(quantize_int8(x, act), orc.act(x, act), 16 * U if act else 0.0)


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (BF16, F32), (FP16, FP16), (F32, BF16), (F32, F32)])
def test_rms_norm(C, dtype, stream):
    w = 1 + _randn(C, std=0.2, seed=3)
    for M in (1, 29):
        x, res = _randn(M, C, dtype=dtype), _randn(M, C, dtype=stream, seed=1)
        _check_rows(rms_norm_int8(x, w), orc.rms_norm(x, w, 1e-6)[0], _norm_error(C))
        rows, z = rms_norm_int8(x, w.to(dtype), 1e-3, residual=res)
        y, z_ref = orc.rms_norm(x, w.to(dtype), 1e-3, res)
        _check_rows(rows, y, _norm_error(C))
        assert z.dtype == stream and torch.equal(z, (res.float() + x.float()).to(stream))


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("stream,dtype,mod", [(BF16, BF16, BF16), (F32, BF16, F32), (FP16, FP16, FP16), (F32, F32, BF16)])
def test_ln_modulate(C, stream, dtype, mod):
    for B, L in ((1, 1), (3, 11)):
        x, h = _randn(B, L, C, dtype=stream) + 0.5, _randn(B, L, C, dtype=dtype, seed=1)
        mods = _randn(B, 1, 6 * C, dtype=mod, seed=2, std=0.4)
        gate, shift, scale = mods.chunk(6, dim=-1)[2:5]          # slices of one projection, as in the block
        if C > 1:
            _check_rows(ln_modulate_int8(x, shift, scale), orc.ln_modulate(x, shift, scale, 1e-6)[0], _norm_error(C))
        rows, z = ln_modulate_int8(x, shift[:, 0], scale[:, 0], 1e-2, gate=gate[:, 0], h=h)
        y, z_ref = orc.ln_modulate(x, shift, scale, 1e-2, gate, h)
        _check_rows(rows, y, _norm_error(C))
        # one rounding to the stream's type, of a sum that fp32 forms with at most two
        half = torch.finfo(stream).eps / 2
        near = half * z_ref.abs() + 2 * U * (x.double().abs() + (gate.double() * h.double()).abs()) + 2.0 ** -25
        assert z.dtype == stream and bool(((z.double() - z_ref).abs() <= near).all())


@pytest.mark.parametrize("C", [511, 513, 777, 1023, 1153, 1535, 1919, 2047, 4001, 4095, 8191, 8193])
def test_odd_widths(C):
    """rows an element at a time: one, two, four and eight warps on a row, and what is wider; 21 rows fill no block"""
    x, h, res = _randn(21, C, dtype=BF16) + 0.25, _randn(21, C, dtype=BF16, seed=1), _randn(21, C, seed=2)
    for act in (None, "gelu", "silu"):
        _check_rows(quantize_int8(x, act), orc.act(x, act), 16 * U if act else 0.0)
    w = 1 + _randn(C, std=0.2, seed=3)
    rows, z = rms_norm_int8(h, w.half(), residual=res)
    _check_rows(rows, orc.rms_norm(h, w.half(), 1e-6, res)[0], _norm_error(C))
    assert torch.equal(z, res + h.float())
    mods = _randn(3, 1, 6 * C, dtype=BF16, seed=4, std=0.4)
    gate, shift, scale = mods.chunk(6, dim=-1)[2:5]
    x3, h3 = x.view(3, 7, C), h.view(3, 7, C)
    rows, z = ln_modulate_int8(x3, shift, scale, gate=gate, h=h3)
    _check_rows(rows, orc.ln_modulate(x3, shift, scale, 1e-6, gate, h3)[0], _norm_error(C))
    assert torch.equal(rows.dequantize(F32), rows.values.float() * rows.scale[..., None])


def test_rows_of_zeros_tiny_values_and_large_ones():
    x = _randn(7, 96, std=1.0)
    x[0] = 0.0
    x[1] *= 2.0 ** -130                      # below the limit: counts as zeros
    x[2] *= 2.0 ** -110
    x[3] *= 2.0 ** 120
    x[4, 5:] = 0.0
    rows = quantize_int8(x)
    assert not rows.values[:2].any() and float(rows.scale[:2].abs().max()) == 0.0
    _check_rows(Int8Rows(rows.values[2:], rows.scale[2:]), x[2:].double(), 0.0)
    assert not rows.dequantize(F32)[:2].any()
    z = torch.zeros(3, 64, device=DEV, dtype=BF16)
    rms = rms_norm_int8(z, torch.ones(64, device=DEV))
    assert not rms.values.any() and not rms.scale.any()
    ln = ln_modulate_int8(torch.full((1, 3, 64), 2.0, device=DEV), z[:1], z[:1])        # no variance: zeros
    assert not ln.values.any()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("C", [96, 1152, 4608])
def test_activations_at_their_ends(act, C):
    """rows whose results are tiny, nothing or as large as the type's largest"""
    x = _randn(12, C, std=0.3)
    x[0] -= 12.0                      # results of 1e-30 and less
    x[1] = -8.0 - x[1].abs()
    x[2] = -100.0
    x[3] = 3e38
    x[3, 1::2] = -3e38
    x[4] = -40.0
    x[4, 7] = 1e-14                   # the row's maximum is far below the activations' own limits
    x[5] = -9.0
    x[5, 0] = 5.0
    y = orc.act(x, act)
    for rows in (quantize_int8(x, act), Int8Rows(*(t.view(12, *t.shape[2:]) for t in quantize_int8(x.view(4, 3, C), act)))):
        real, scale = orc.real_rows(y)
        # exp(v) within (2 + 1.2 |v|) steps, and |v| may reach 88 where a row has nothing larger: 150 u
        some = scale > 0
        assert torch.equal(rows.scale > 0, some)
        assert float((rows.values.double() - real)[some].abs().max()) <= 0.5 + 127 * 150 * U
        assert bool(((rows.scale.double() - scale).abs() <= scale * 150 * U).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("C", [40, 1152, 1153])
def test_a_value_that_is_not_finite_spoils_its_row_and_no_other(bad, C):
    x = _randn(6, C, dtype=BF16)
    clean = x.clone()
    x[2, C // 2] = bad
    w, other = quantize_int8(_randn(24, C)), [0, 1, 3, 4, 5]
    shift = torch.zeros(1, C, device=DEV, dtype=BF16)
    for f in (quantize_int8, lambda t: quantize_int8(t, "gelu"), lambda t: quantize_int8(t, "silu"),
              lambda t: rms_norm_int8(t, torch.ones(C, device=DEV)),
              lambda t: Int8Rows(*(v[0] for v in ln_modulate_int8(t[None], shift, shift)))):
        rows, ref = f(x), f(clean)
        assert torch.isnan(rows.scale[2]) and not rows.values[2].any()
        assert torch.isnan(rows.dequantize()[2]).all() and torch.isnan(int8_linear(rows, w)[2]).all()
        assert torch.equal(rows.values[other], ref.values[other]) and torch.equal(rows.scale[other], ref.scale[other])


def test_strides_and_alignments():
    C = 384
    big = _randn(3, 20, 3, C, dtype=BF16)
    sliced = big[:, :, 1]                                          # strided rows
    assert torch.equal(quantize_int8(sliced).values, quantize_int8(sliced.contiguous()).values)
    odd = _randn(5 * (C + 3) + 1, dtype=BF16)[1:].view(5, C + 3)[:, 1:C + 1]     # odd base and pitch
    assert torch.equal(quantize_int8(odd).values, quantize_int8(odd.contiguous()).values)
    for shift in (1, 4):                                           # fp32 rows at 4 and at 16 bytes
        moved = _randn(9 * C + 8)[shift:shift + 9 * C].view(9, C)
        assert torch.equal(quantize_int8(moved).values, quantize_int8(moved.clone()).values)
        w = torch.ones(C + 8, device=DEV)[shift:shift + C]
        rows, z = rms_norm_int8(moved, w, residual=moved)
        assert torch.equal(z, moved + moved)
        _check_rows(rows, orc.rms_norm(moved, w, 1e-6, moved)[0], _norm_error(C))
    t = _randn(C, 9, dtype=BF16).t()                               # no unit stride
    assert torch.equal(quantize_int8(t).values, quantize_int8(t.contiguous()).values)
    row = _randn(C, dtype=BF16).expand(7, C)                       # one row seven times
    rows = quantize_int8(row)
    assert torch.equal(rows.values, quantize_int8(row.contiguous()).values)
    one = quantize_int8(row[0])                                    # no leading dimension
    assert one.values.shape == (C,) and one.scale.shape == () and torch.equal(one.values, rows.values[0])
    perm = _randn(4, 5, 6, C, dtype=BF16).permute(2, 0, 1, 3)      # leading dimensions that do not collapse
    assert torch.equal(quantize_int8(perm).values, quantize_int8(perm.contiguous()).values)


def _random8(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * sum(shape))
    q = torch.randint(-128, 128, shape, device=DEV, generator=g, dtype=torch.int8)
    scale = torch.rand(shape[:-1], device=DEV, generator=g) * 0.02 + 1e-3
    return Int8Rows(q, scale)


def _pitched(r, pitch=None):
    K = r.values.shape[-1]
    buf = torch.full((*r.values.shape[:-1], -(-K // 16) * 16 if pitch is None else pitch), 99, dtype=torch.int8, device=DEV)
    buf[..., :K] = r.values
    return Int8Rows(buf[..., :K], r.scale)


def _check_linear(x, w, bias, out_dtype):
    out = int8_linear(x, w, bias, out_dtype=out_dtype)
    ref, size = orc.linear(x.values, x.scale, w.values, w.scale, bias)
    assert out.shape == (*x.values.shape[:-1], w.values.shape[0]) and out.dtype == out_dtype and out.is_contiguous()
    half = torch.finfo(out_dtype).eps / 2 if out_dtype != F32 else 0.0
    near = ref.abs() * half + size * 4 * U * (1 + half) + 2.0 ** -25
    assert bool(((out.double() - ref).abs() <= near).all()), float(((out.double() - ref).abs() / near).max())
    return out


LINEAR_SHAPES = [(1, 1, 1), (1, 16, 1), (1, 1152, 6912), (2, 48, 130), (5, 33, 7), (16, 1152, 384), (17, 100, 129), (64, 384, 300),
                 (128, 128, 128), (130, 1001, 258), (256, 4608, 1152), (257, 640, 513), (300, 31, 1000), (1000, 1152, 200),
                 (2049, 144, 776), (4000, 1152, 1152), (8200, 256, 1152), (5000, 128, 3456), (20000, 130, 1100), (19000, 64, 257), (2000, 1001, 300), (1, 100003, 2700)]


@pytest.mark.parametrize("shape", LINEAR_SHAPES)
@pytest.mark.parametrize("out_dtype", [BF16, FP16, F32])
def test_linear(shape, out_dtype):
    M, K, N = shape
    x, w = _random8(M, K), _random8(N, K, seed=1)
    bias = _randn(N, dtype=out_dtype)
    plain = _check_linear(x, w, None, out_dtype)
    _check_linear(_pitched(x), _pitched(w), bias, out_dtype)
    # one result per element whatever the layout of its rows: the sums are exact
    assert torch.equal(int8_linear(_pitched(x), _pitched(w), out_dtype=out_dtype), plain)
    assert torch.equal(int8_linear(_pitched(x, K + 17), w, out_dtype=out_dtype), plain)


def test_linear_is_the_same_for_a_row_alone_and_in_a_batch():
    x, w = _pitched(_random8(700, 1152)), _pitched(_random8(1152, 1152, seed=1))
    bias = _randn(1152)
    whole = int8_linear(x, w, bias)
    for lo, hi in ((0, 1), (3, 5), (100, 133), (200, 456), (0, 699)):
        assert torch.equal(int8_linear(Int8Rows(x.values[lo:hi], x.scale[lo:hi]), w, bias), whole[lo:hi])


def test_linear_largest_sums():
    """every product -128 * -128 over the longest sum there may be"""
    K = 131071
    for M in (1, 200):
        x = Int8Rows(torch.full((M, K), -128, dtype=torch.int8, device=DEV), torch.ones(M, device=DEV))
        w = Int8Rows(torch.full((3, K), -128, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV))
        assert torch.equal(int8_linear(x, w, out_dtype=F32), torch.full((M, 3), float(K * 16384), device=DEV))
        assert torch.equal(int8_linear(_pitched(x), _pitched(w), out_dtype=F32), torch.full((M, 3), float(K * 16384), device=DEV))


def test_linear_shapes_of_x_and_empty_batches():
    w = _pitched(_random8(40, 64, seed=1))
    x = _random8(2, 3, 5, 64)
    out = int8_linear(x, w)
    assert out.shape == (2, 3, 5, 40)
    assert torch.equal(out[1, 2], int8_linear(Int8Rows(x.values[1, 2], x.scale[1, 2]), w))
    one = Int8Rows(x.values[0, 0, 0], x.scale[0, 0, 0])
    assert torch.equal(int8_linear(one, w), out[0, 0, 0])
    none = quantize_int8(torch.empty(0, 64, device=DEV))
    assert int8_linear(none, w).shape == (0, 40) and none.dequantize().shape == (0, 64)
    assert rms_norm_int8(torch.empty(2, 0, 64, device=DEV), torch.ones(64, device=DEV)).values.shape == (2, 0, 64)
    rows, z = ln_modulate_int8(torch.empty(2, 0, 64, device=DEV), *(torch.ones(2, 64, device=DEV),) * 2,
                               gate=torch.ones(2, 64, device=DEV), h=torch.empty(2, 0, 64, device=DEV))
    assert rows.scale.shape == (2, 0) and z.shape == (2, 0, 64)


@pytest.mark.parametrize("C", [5, 64, 1152, 1155])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
def test_dequantize(C, dtype):
    for r in (_random8(33, C), _pitched(_random8(33, C)), _random8(2, 3, C), quantize_int8(_randn(3, 5, C))):
        out = r.dequantize(dtype)
        assert out.is_contiguous() and torch.equal(out, (r.values.float() * r.scale[..., None]).to(dtype))


def test_large_products_of_rows_the_tensor_cores_cannot_read():
    """sliced columns, an odd base, expanded rows and leading dimensions that do not collapse: the result of rows side by side"""
    K, N = 600, 500
    big, w = _random8(1200, K + 40), _random8(N, K, seed=1)
    ref_w = _pitched(w)
    base = torch.empty(N * K + 5, dtype=torch.int8, device=DEV)[5:].view(N, K).copy_(w.values)
    for x in (Int8Rows(big.values[:, 3:K + 3], big.scale), Int8Rows(big.values[:, :K], big.scale),
              Int8Rows(big.values[:1, :K].expand(1200, K), big.scale),
              Int8Rows(big.values.view(4, 300, -1).transpose(0, 1)[..., 1:K + 1], big.scale.view(4, 300).t())):
        ref = int8_linear(_pitched(Int8Rows(x.values.contiguous(), x.scale.contiguous())), ref_w)
        for weight in (w, ref_w, Int8Rows(base, w.scale)):
            assert torch.equal(int8_linear(x, weight), ref)
            flat = Int8Rows(x.values.reshape(-1, K), x.scale.reshape(-1))
            assert torch.equal(torch.ops.dmf_b200.int8_linear(*flat, *weight, None, BF16).view(ref.shape), ref)


def test_rows_behind_the_last_one_stay_as_they_were():
    """the C ABI on buffers that are larger than the call"""
    import ctypes as C

    from dmf_b200 import _lib
    x, w = _pitched(_random8(130, 96)), _pitched(_random8(100, 96, seed=1))
    out = torch.full((200, 128), 7.0, device=DEV, dtype=BF16)
    a = _lib.Int8LinearArgs()
    a.m, a.n, a.k, a.out_dtype = 130, 100, 96, _lib.INT8_BF16
    a.x = _lib.Int8Matrix(x.values.data_ptr(), x.values.stride(0), x.scale.data_ptr())
    a.w = _lib.Int8Matrix(w.values.data_ptr(), w.values.stride(0), w.scale.data_ptr())
    a.out, a.out_stride, a.stream = out.data_ptr(), 128, torch.cuda.current_stream().cuda_stream
    for m in (130, 5):
        out.fill_(7.0)
        a.m = m
        assert _lib.load().dmf_int8_linear(C.byref(a)) == 0
        ref = int8_linear(Int8Rows(x.values[:m], x.scale[:m]), w)
        assert torch.equal(out[:m, :100], ref)
        assert bool((out[m:] == 7.0).all()) and bool((out[:, 100:] == 7.0).all())
    rows = torch.full((50, 112), 55, dtype=torch.int8, device=DEV)
    scale = torch.full((50,), 3.0, device=DEV)
    src = _randn(40, 100)
    b = _lib.Int8QuantizeArgs()
    b.batch, b.seqlen, b.channels, b.dtype = 1, 40, 100, _lib.INT8_F32
    b.x = _lib.Rows(src.data_ptr(), 0, 100)
    b.out = _lib.Int8Matrix(rows.data_ptr(), 112, scale.data_ptr())
    b.stream = a.stream
    assert _lib.load().dmf_int8_quantize(C.byref(b)) == 0
    assert bool((rows[40:] == 55).all()) and bool((rows[:, 100:] == 55).all()) and bool((scale[40:] == 3.0).all())
    assert torch.equal(rows[:40, :100], quantize_int8(src).values)


@pytest.mark.parametrize("C,M", [(1152, 2000), (1152, 5), (100, 9), (99, 9), (4608, 1300)])
def test_the_sum_may_be_written_where_its_term_was(C, M):
    """the C ABI with sum = residual and sum = x, against results in buffers of their own"""
    import ctypes

    from dmf_b200 import _lib
    stream = torch.cuda.current_stream().cuda_stream
    x, res, w = _randn(M, C, dtype=BF16), _randn(M, C, seed=1), 1 + _randn(C, std=0.1, seed=2)
    want, total = rms_norm_int8(x, w, residual=res)
    q, scale = torch.empty(M, -(-C // 16) * 16, dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    a = _lib.Int8RmsNormArgs()
    a.batch, a.seqlen, a.channels, a.dtype, a.stream_dtype, a.weight_dtype, a.eps = 1, M, C, _lib.INT8_BF16, _lib.INT8_F32, _lib.INT8_F32, 1e-6
    a.x, a.residual, a.sum = _lib.Rows(x.data_ptr(), 0, C), _lib.Rows(res.data_ptr(), 0, C), _lib.Rows(res.data_ptr(), 0, C)
    a.weight, a.out, a.stream = w.data_ptr(), _lib.Int8Matrix(q.data_ptr(), q.stride(0), scale.data_ptr()), stream
    assert _lib.load().dmf_int8_rmsnorm(ctypes.byref(a)) == 0
    assert torch.equal(res, total) and torch.equal(q[:, :C], want.values) and torch.equal(scale, want.scale)
    x3, h = x[None].clone(), _randn(1, M, C, dtype=BF16, seed=3)
    gate, shift, sc = (_randn(1, C, dtype=BF16, seed=s, std=0.3) for s in (4, 5, 6))
    want, total = ln_modulate_int8(x3, shift, sc, gate=gate, h=h)
    b = _lib.Int8LnModulateArgs()
    b.batch, b.seqlen, b.channels, b.eps = 1, M, C, 1e-6
    b.x, b.h, b.sum = _lib.Rows(x3.data_ptr(), 0, C), _lib.Rows(h.data_ptr(), 0, C), _lib.Rows(x3.data_ptr(), 0, C)
    b.gate, b.shift, b.scale = (_lib.Mod(t.data_ptr(), 0) for t in (gate, shift, sc))
    b.out, b.stream = _lib.Int8Matrix(q.data_ptr(), q.stride(0), scale.data_ptr()), stream
    assert _lib.load().dmf_int8_ln_modulate(ctypes.byref(b)) == 0
    assert torch.equal(x3, total) and torch.equal(q[:, :C], want.values[0]) and torch.equal(scale, want.scale[0])


def test_more_than_2_to_the_31_elements():
    M, C, tail = 600_000, 4096, 1300                   # 2.46e9 elements; the end alone takes the same kernels
    row = _randn(1000, C, dtype=BF16)
    x = row.repeat(M // 1000, 1)
    x[-tail:] = _randn(tail, C, dtype=BF16, seed=9)
    w, bias = quantize_int8(_randn(24, C, seed=2)), _randn(24)
    for act in (None, "gelu"):
        rows = quantize_int8(x, act)
        end = quantize_int8(x[-tail:], act)
        assert torch.equal(rows.values[-tail:], end.values) and torch.equal(rows.scale[-tail:], end.scale)
    assert torch.equal(rows.dequantize()[-tail:], end.dequantize())
    out = int8_linear(rows, w, bias)
    assert torch.equal(out[-tail:], int8_linear(end, w, bias)) and torch.equal(out[:1000], out[1000:2000])
    ones = torch.ones(C, device=DEV)
    rows, z = rms_norm_int8(x, ones, residual=x)
    end, z_end = rms_norm_int8(x[-tail:], ones, residual=x[-tail:])
    assert torch.equal(rows.values[-tail:], end.values) and torch.equal(z[-tail:], z_end)
    del rows, z, out
    mod = _randn(2, 6 * C, dtype=BF16, std=0.2)
    g, sh, sc = mod.chunk(6, -1)[2:5]
    x3 = x.view(2, M // 2, C)
    rows, z = ln_modulate_int8(x3, sh, sc, gate=g, h=x3)
    end, z_end = ln_modulate_int8(x3[1:, -tail:], sh[1:], sc[1:], gate=g[1:], h=x3[1:, -tail:])
    assert torch.equal(rows.values[1, -tail:], end.values[0]) and torch.equal(z[1, -tail:], z_end[0])


def test_a_block_half_as_it_is_used():
    """adaLN, first product, GELU, second product, gate: the ops one after the other against the same steps in fp64 on their own
    8-bit operands, and against the layer in fp64 with the error that 8 bits have"""
    from dmf_b200 import adaln
    B, L, C = 2, 96, 384
    x, h = _randn(B, L, C, dtype=BF16), _randn(B, L, C, dtype=BF16, seed=1)
    g_a, shift, scale, g_m = (_randn(B, 1, C, dtype=BF16, seed=s, std=0.3) for s in (2, 3, 4, 5))
    w1, w2 = _randn(4 * C, C, seed=6, std=C ** -0.5), _randn(C, 4 * C, seed=7, std=(4 * C) ** -0.5)
    b1, b2 = _randn(4 * C, dtype=BF16, seed=8, std=0.1), _randn(C, dtype=BF16, seed=9, std=0.1)
    q1, q2 = quantize_int8(w1), quantize_int8(w2)
    rows, z = ln_modulate_int8(x, shift, scale, gate=g_a, h=h)
    u = int8_linear(rows, q1, b1)
    rows2 = quantize_int8(u, "gelu")
    out = adaln.gate_residual(z, g_m, int8_linear(rows2, q2, b2))
    y, z64 = orc.ln_modulate(x, shift, scale, 1e-6, g_a, h)
    _check_rows(rows, y, _norm_error(C))
    _check_rows(rows2, orc.act(u, "gelu"), 16 * U)
    full = z64 + g_m.double() * (orc.act(y @ w1.double().t() + b1.double(), "gelu") @ w2.double().t() + b2.double())
    # each of the four quantised operands is off by at most half a scale, about amax / 254 with amax below 6 standard
    # deviations: uniform errors of (6 / 127) / sqrt(12) = 1.4 % of a standard deviation each, GELU's output 2 times that
    assert float((out.double() - full).norm() / full.norm()) < 0.05


def test_another_stream_and_a_graph():
    x, w = _randn(300, 1152, dtype=BF16), quantize_int8(_randn(640, 1152))
    ref = int8_linear(quantize_int8(x), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = int8_linear(quantize_int8(x), w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    static = x.clone()
    graphs = []
    for _ in range(2):                       # two graphs of the same calls, replayed one after the other and together
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = int8_linear(quantize_int8(static), w)
        graphs.append((g, o))
    static.copy_(x * 0.5 + 1)
    want = int8_linear(quantize_int8(static), w)
    streams = [torch.cuda.Stream() for _ in graphs]
    for (g, _), s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, o in graphs)


def test_a_graph_that_forks_and_joins():
    """operands made on two streams, one behind the package's own kernels and one behind torch's, and used behind the join"""
    x, w = _randn(3000, 1152, dtype=BF16), _randn(640, 1152, dtype=BF16, seed=1)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def both(x, w, side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            rows = quantize_int8(quantize_int8(x, "gelu").dequantize() * 2, "silu")
        weight = quantize_int8(rms_norm_int8(w, torch.ones(1152, device=DEV)).dequantize())
        main.wait_stream(side)
        return int8_linear(rows, weight), int8_linear(rows, weight, out_dtype=F32)
    with torch.cuda.graph(graph):
        out = both(x, w, side)
    for i in range(10):
        x.copy_(_randn(3000, 1152, dtype=BF16, seed=10 + i))
        w.copy_(_randn(640, 1152, dtype=BF16, seed=50 + i))
        graph.replay()
        got = [o.clone() for o in out]
        rows = quantize_int8(quantize_int8(x, "gelu").dequantize() * 2, "silu")
        torch.cuda.synchronize()
        weight = quantize_int8(rms_norm_int8(w, torch.ones(1152, device=DEV)).dequantize())
        torch.cuda.synchronize()
        assert torch.equal(got[0], int8_linear(rows, weight)) and torch.equal(got[1], int8_linear(rows, weight, out_dtype=F32))


def test_many_calls_in_a_row_reuse_memory():
    """calls whose buffers the allocator hands on at once: each kernel starts while the one before it ends"""
    x = [_randn(m, 384, dtype=BF16, seed=m) for m in (7, 300, 1500, 5000)]
    w = quantize_int8(_randn(384, 384))
    want = []
    for t in x:
        for _ in range(3):
            t = int8_linear(quantize_int8(t, "gelu"), w)
            torch.cuda.synchronize()
        want.append(t)
    for _ in range(20):
        for t, ref in zip(x, want):
            for _ in range(3):
                t = int8_linear(quantize_int8(t, "gelu"), w)
            assert torch.equal(t, ref)


def test_two_threads_at_once():
    import threading
    w = quantize_int8(_randn(1152, 1152))
    xs = [quantize_int8(_randn(m, 1152, seed=m)) for m in (1, 100, 600, 2000)]
    refs = [int8_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(x, ref):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(int8_linear(x, w), ref):
                    bad.append(x.values.shape)
    threads = [threading.Thread(target=work, args=p) for p in zip(xs, refs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals_of_gradients_and_tangents():
    x = _randn(4, 64).requires_grad_(True)
    w, bias = quantize_int8(_randn(8, 64)), _randn(8).requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradients"):
        quantize_int8(x)
    with pytest.raises(RuntimeError, match="gradients"):
        rms_norm_int8(x, torch.ones(64, device=DEV))
    with pytest.raises(RuntimeError, match="gradients"):
        int8_linear(quantize_int8(x.detach()), w, bias)
    with torch.no_grad():
        assert not int8_linear(quantize_int8(x), w, bias).requires_grad
    with torch.inference_mode():
        int8_linear(quantize_int8(x), w, bias)
    with pytest.raises(RuntimeError, match="tangents"):
        torch.func.jvp(lambda t: quantize_int8(t).scale, (x.detach(),), (x.detach(),))
    # an input of a transform that carries no tangent of its own
    y, _ = torch.func.jvp(lambda t: t * quantize_int8(x.detach()).scale[:, None], (x.detach(),), (x.detach(),))
    assert torch.equal(y, x.detach() * quantize_int8(x.detach()).scale[:, None])


def test_traced_and_under_other_transforms():
    w = quantize_int8(_randn(48, 100))
    x, y = _randn(6, 100, dtype=BF16), _randn(6, 100, dtype=BF16, seed=1)
    f = lambda t: int8_linear(quantize_int8(t), w)
    assert torch.equal(torch.jit.trace(f, (x,))(y), f(y))
    both = torch.stack([x, y])
    assert torch.equal(torch.func.vmap(f)(both), torch.stack([f(x), f(y)]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: quantize_int8(t).scale.sum())(x.float())


def test_compiled():
    w = quantize_int8(_randn(48, 100))
    x = _randn(6, 100, dtype=BF16)
    f = lambda t: int8_linear(quantize_int8(t, "silu"), w) + 1
    assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(x), f(x))


def test_the_registered_ops_give_the_native_paths_bits():
    ops = torch.ops.dmf_b200
    x, res, w = _randn(3, 40, 200, dtype=BF16), _randn(3, 40, 200, seed=1), 1 + _randn(200, std=0.1, seed=2)
    shift, scale, gate = (_randn(3, 1, 200, dtype=BF16, seed=s, std=0.3) for s in (3, 4, 5))
    pairs = [(quantize_int8(x, "gelu"), ops.quantize_int8(x, 1)),
             (rms_norm_int8(x, w), ops.rms_norm_int8(x, w, 1e-6)),
             (ln_modulate_int8(x, shift, scale), ops.ln_modulate_int8(x, shift, scale, 1e-6))]
    rows, z = rms_norm_int8(x, w, residual=res)
    pairs.append(((*rows, z), ops.add_rms_norm_int8(x, res, w, 1e-6)))
    rows, z = ln_modulate_int8(x, shift, scale, gate=gate[:, 0], h=x)
    pairs.append(((*rows, z), ops.gate_ln_modulate_int8(x, gate, x, shift, scale, 1e-6)))
    wq, bias = quantize_int8(_randn(77, 200)), _randn(77)
    pairs.append(((int8_linear(rows, wq, bias, out_dtype=F32),), (ops.int8_linear(*rows, *wq, bias, F32),)))
    pairs.append(((rows.dequantize(FP16),), (ops.dequantize_int8(*rows, FP16),)))
    for native, general in pairs:
        for a, b in zip(native, general):
            assert a.stride() == b.stride() and torch.equal(a, b)


# ---- the model in 8 bits ----------------------------------------------------------------------------------------------

def _model(name="DMFT-S/2", **kw):
    from dmf_b200.harness.model import build_dmft
    torch.manual_seed(0)
    kw = dict(dict(input_size=32, dmf_depth=8, num_classes=1000, attn_func="fa3", use_logvar=False, qk_norm=False), **kw)
    model = build_dmft(name, **kw)
    model.initialize_weights(zero_init=False)      # zero gates would hide the blocks
    return model.to(DEV).requires_grad_(False).eval()


# A layer's two operands are off by (a / rms) / 127 / sqrt(12) each, a the row's largest value: a / rms is about 4 behind a norm, 6
# behind GELU, 1.7 for a weight, so 1.0 % of a product behind a norm or the attention and 1.5 % behind GELU.  qkv, attention and
# proj in one branch, fc1 and fc2 in the other, and the modulation of both: at most 2.5 % of a branch in quadrature; the sum over
# the blocks grows no faster than the branches themselves.  Twice that, and 1 % for the 16-bit model it is compared with.
MODEL_TOL = 0.06


@pytest.mark.parametrize("dtype,kw", [(BF16, {}), (BF16, {"qk_norm": True}), (F32, {})])
def test_model_in_8_bits_is_near_the_model(dtype, kw):
    from dmf_b200.harness.int8_model import int8_model
    model = _model(**kw).to(dtype)
    state = {k: v.clone() for k, v in model.state_dict().items()}
    quantised = int8_model(model)
    assert all(torch.equal(v, state[k]) for k, v in model.state_dict().items()) and len(model.blocks) == 12
    x, y = _randn(4, 4, 32, 32, dtype=dtype), torch.randint(0, 1000, (4,), device=DEV)
    t, r = torch.rand(4, device=DEV, dtype=dtype) * 0.5 + 0.5, torch.rand(4, device=DEV, dtype=dtype) * 0.5
    with torch.no_grad(), torch.autocast("cuda", BF16, enabled=dtype == F32):
        got, ref = quantised(x, t, r, y), model(x, t, r, y)
    assert got.dtype == ref.dtype and got.shape == ref.shape
    assert float((got.double() - ref.double()).norm() / ref.double().norm()) < MODEL_TOL


def test_sampler_in_8_bits_eager_and_graphed():
    from dmf_b200.harness.int8_model import int8_model
    from dmf_b200.harness.sampler import GraphedSampler, euler_sampler
    model = _model().bfloat16()
    quantised = int8_model(model)
    z, y = _randn(2, 4, 32, 32, dtype=BF16), torch.randint(0, 1000, (2,), device=DEV)
    out = euler_sampler(quantised, z, y, num_steps=2, cfg_scale=1.5)
    ref = euler_sampler(model, z, y, num_steps=2, cfg_scale=1.5)
    # two steps, of which guidance weighs the branches with 1.5 and -0.5
    assert float((out - ref).norm() / ref.norm()) < 2 * 1.6 * MODEL_TOL
    graphed = GraphedSampler(quantised, 2, latent_shape=(4, 32, 32), num_steps=2, cfg_scale=1.5)
    assert torch.equal(graphed(z, y), out)
    z2 = _randn(2, 4, 32, 32, dtype=BF16, seed=5)
    assert torch.equal(graphed(z2, y), euler_sampler(quantised, z2, y, num_steps=2, cfg_scale=1.5))


def test_model_in_8_bits_moves_and_casts_without_touching_its_scales():
    from dmf_b200.harness.int8_model import int8_model
    quantised = int8_model(_model().bfloat16())
    layer = quantised.blocks[0].qkv
    values, scale = layer.values.clone(), layer.scale.clone()
    quantised.bfloat16()
    assert layer.scale.dtype == F32 and torch.equal(layer.scale, scale) and torch.equal(layer.values, values)
    quantised.cpu().to(DEV)
    assert torch.equal(layer.scale, scale) and torch.equal(layer.values, values)


def test_model_refusals():
    from dmf_b200.harness.int8_model import int8_model
    with pytest.raises(ValueError, match="fa2"):
        int8_model(_model(attn_func="base"))
    with pytest.raises(ValueError, match="GPU"):
        int8_model(_model().cpu())
    with pytest.raises(ValueError, match="fp32 or bf16"):
        int8_model(_model().half())


# Results far below their row's maximum, of large negative values: real numbers of magnitude x e^-|x|, which round to 0.  The rows: one
# such value among ordinary ones; beside a row maximum near 2^-40 (just below, just above); nothing else (all results are below 2^-120: scale 0).
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("C", [96, 1152, 1153, 4608])
@pytest.mark.parametrize("dtype", [BF16, F32, FP16])
def test_activations_of_large_negative_values(act, C, dtype):
    for M in (12, 1500):                       # a block per row; loops over rows, where there is one
        x = _randn(M, C, std=2.0)
        large = [-1030.0, -1e5, -1e18, -1e20, -3e38] if dtype != FP16 else [-1030.0, -6e4]
        for r in range(M):
            v, kind = large[r % len(large)], r % 12
            if kind < 6:                       # one, two and half a row of them among ordinary values
                x[r, r % C] = v
                x[r, (5 * r + 1) % C] = v
                if kind == 5:
                    x[r, ::2] = v
            elif kind < 9:                     # a row whose maximum, half of 2^-39 or 2^-40.5, is near the limit of the fast form
                x[r] = -200.0
                x[r, (3 * r + 2) % C] = (2.0 ** -39, 2.0 ** -38.5, 2.0 ** -40.5)[kind - 6] if dtype != FP16 else 2.0 ** -20
                x[r, r % C] = v
            else:
                x[r] = v
        x = x.to(dtype)
        _check_rows(quantize_int8(x, act), orc.act(x, act), 16 * U)


@pytest.mark.parametrize("C,gated", [(4080, True), (4096, True), (6120, False), (6144, False)])
def test_ln_modulate_as_a_programs_first_call(C, gated):
    """vectors of just up to 48 KB in shared memory: with the block's own words more than a kernel has unless it was allowed more, which
    an earlier and wider call of the same kernel does too; so in a program of its own"""
    import subprocess
    import sys
    program = f"""
import torch
from dmf_b200.int8 import ln_modulate_int8
x = torch.randn(2, 700, {C}, device="cuda").bfloat16()
gate, shift, scale = torch.randn(2, 1, 3 * {C}, device="cuda").bfloat16().chunk(3, -1)
rows = ln_modulate_int8(x, shift, scale, gate=gate, h=x)[0] if {gated} else ln_modulate_int8(x, shift, scale)
few = ln_modulate_int8(x[:1, :3], shift[:1], scale[:1], gate=gate[:1], h=x[:1, :3])[0] if {gated} else ln_modulate_int8(x[:1, :3], shift[:1], scale[:1])
assert int((rows.values[:1, :3].int() - few.values.int()).abs().max()) <= 1
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_large_products_of_expanded_and_overlapping_rows_copy_them():
    """rows at a pitch of 0, or of 16 bytes and less than a row: a copy goes to the tensor cores (seen as memory that the call takes)"""
    M, K, N = 1200, 640, 500
    w, scale = _pitched(_random8(N, K, seed=1)), torch.rand(M, device=DEV)
    for values in (_random8(1, K).values.expand(M, K), _random8(1, 16 * M + K).values[0].as_strided((M, K), (16, 1))):
        ref = int8_linear(Int8Rows(values.clone(memory_format=torch.contiguous_format), scale), w)
        for f in (lambda: int8_linear(Int8Rows(values, scale), w),
                  lambda: torch.ops.dmf_b200.int8_linear(values, scale, *w, None, BF16)):
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            out = f()
            assert torch.cuda.max_memory_allocated() - before >= M * N * 2 + M * K
            assert torch.equal(out, ref)


def test_rows_wider_than_2_to_the_20_are_refused_on_every_route():
    wide, ok = 2 ** 20 + 1, 2 ** 20
    scale = torch.ones(2, device=DEV)
    values = torch.ones(2, wide, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="at most"):
        Int8Rows(values, scale).dequantize()
    with pytest.raises(RuntimeError):
        torch.ops.dmf_b200.dequantize_int8(values, scale, BF16)
    assert bool((Int8Rows(values[:, :ok], scale).dequantize() == 1).all())
    with pytest.raises(ValueError, match="at most"):
        quantize_int8(torch.ones(2, wide, dtype=BF16, device=DEV))


# ---- the kernels that take many rows: from eight rows per SM on (1184 on a B200), a warp per row up to 1280 channels, a block on wider ones

MANY_WIDTHS = [64, 384, 512, 520, 1152, 1280, 1288, 2040, 4608]


@pytest.mark.parametrize("C", MANY_WIDTHS)
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
def test_quantize_many_rows(C, act, dtype):
    x = _randn(1511, C, dtype=dtype, std=2.0)
    _check_rows(quantize_int8(x, act), orc.act(x, act), 16 * U if act else 0.0)
    x = _randn(7, 3, 211, C, dtype=dtype, seed=1)[:, 1]           # samples that do not lie side by side
    _check_rows(quantize_int8(x, act), orc.act(x, act), 16 * U if act else 0.0)


@pytest.mark.parametrize("C", MANY_WIDTHS)
@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (FP16, FP16), (BF16, F32), (FP16, F32), (F32, BF16), (F32, FP16), (F32, F32)])
def test_rms_norm_many_rows(C, dtype, stream):
    w = 1 + _randn(C, std=0.2, seed=3)
    x, res = _randn(7, 211, C, dtype=dtype), _randn(7, 211, C, dtype=stream, seed=1)
    _check_rows(rms_norm_int8(x, w), orc.rms_norm(x, w, 1e-6)[0], _norm_error(C))
    rows, z = rms_norm_int8(x, w.to(dtype), 1e-3, residual=res)
    _check_rows(rows, orc.rms_norm(x, w.to(dtype), 1e-3, res)[0], _norm_error(C))
    assert torch.equal(z, (res.float() + x.float()).to(stream))


@pytest.mark.parametrize("C", MANY_WIDTHS)
@pytest.mark.parametrize("stream,dtype,mod", [(BF16, BF16, BF16), (FP16, FP16, FP16), (BF16, F32, F32), (FP16, F32, BF16), (F32, BF16, F32),
                                              (F32, FP16, FP16), (F32, F32, BF16)])
def test_ln_modulate_many_rows(C, stream, dtype, mod):
    for B, L in ((5, 307), (1, 1201), (150, 8)):       # samples with vectors of their own; no block's share of rows divides 307 or 1201
        x, h = _randn(B, L, C, dtype=stream) + 0.5, _randn(B, L, C, dtype=dtype, seed=1)
        gate, shift, scale = _randn(B, 1, 6 * C, dtype=mod, seed=2, std=0.4).chunk(6, dim=-1)[2:5]
        _check_rows(ln_modulate_int8(x, shift, scale), orc.ln_modulate(x, shift, scale, 1e-6)[0], _norm_error(C))
        rows, z = ln_modulate_int8(x, shift, scale, 1e-2, gate=gate, h=h)
        y, z_ref = orc.ln_modulate(x, shift, scale, 1e-2, gate, h)
        _check_rows(rows, y, _norm_error(C))
        half = torch.finfo(stream).eps / 2
        near = half * z_ref.abs() + 2 * U * (x.double().abs() + (gate.double() * h.double()).abs()) + 2.0 ** -25
        assert z.dtype == stream and bool(((z.double() - z_ref).abs() <= near).all())


@pytest.mark.parametrize("step", [None, "ln_modulate", "act", "rms_norm", "linear"])
def test_smoke_run_sees_a_wrong_result_of_every_step(step, monkeypatch):
    """with the oracle's step off by 1 % the comparison fails"""
    from __graft_entry__ import _smoke_int8
    g = torch.Generator().manual_seed(1)
    args = [torch.device(DEV)] + [torch.randn(2, n, 384, generator=g) for n in (64, 1, 1)] + [g]
    if step is None:
        assert _smoke_int8(*args) < 3e-3
        return
    true = getattr(orc, step)

    def wrong(*a, **kw):
        out = true(*a, **kw)
        return (out[0] * 1.01, *out[1:]) if isinstance(out, tuple) else out * 1.01
    monkeypatch.setattr(orc, step, wrong)
    with pytest.raises(AssertionError):
        _smoke_int8(*args)
