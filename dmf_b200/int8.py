"""Inference in 8-bit integers: a block's linear layers with int8 weights and activations, a scale per token and per output
channel, and the norms in front of them with their result in that form.

    rows = ln_modulate_int8(x, shift, scale)          # or rms_norm_int8, quantize_int8
    y = int8_linear(rows, weight, bias)               # weight = quantize_int8(linear.weight.detach()), once

The reference samples with 16-bit linear layers (models/layers.py:119-201); on a B200 their products are most of a sampling
step, and the tensor cores multiply 8-bit integers at twice the 16-bit rate.  ``harness.int8_model`` puts the layers of a DMFT
model on these ops.

Rows in 8 bits (``Int8Rows``): of a row y, a = max|y|, scale = a / 127 and q = y * (127 / a) rounded to the nearest integer, so
the error of an element is at most half a scale.  Rows of zeros (below 2^-120) have scale 0; a row with a NaN or an infinity has
scale NaN, and so has everything computed from it.  Norms, activations and scales are fp32, the sums of a product exact.

These are ops for inference: they have no gradients and no tangents, and refuse inputs that ask for either.  There is no CPU
path.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
import torch.autograd.forward_ad as fwAD

from . import _lib, _native
from . import ops as _ops

_DTYPES = {torch.bfloat16: _lib.INT8_BF16, torch.float16: _lib.INT8_FP16, torch.float32: _lib.INT8_F32}
MAX_ROWS, MAX_WIDTH = 2 ** 31 - 1, 2 ** 20
MAX_N = 2 ** 30     # rows of a weight
MAX_K = 131071      # of a product: beyond it a sum of 8-bit products could leave int32


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``values`` (..., C) int8 and ``scale`` (...) fp32; an element stands for value * scale of its row.
    The ops return values whose rows start at multiples of 16 bytes, which the tensor-core product reads directly; a large
    product of other rows copies them first."""

    values: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """What the rows stand for, as a contiguous (..., C) tensor of a floating type."""
        if _native.takes(*self):
            out = _native.dequantize_int8(*self, dtype)
            if out is not None:
                return out
        _check_rows8(self)
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
        _refuse_derivatives(self.scale)
        return torch.ops.dmf_b200.dequantize_int8(self.values, self.scale, dtype)


# ---- checks -----------------------------------------------------------------------------------------------------------

def _refuse_derivatives(*tensors) -> None:
    tensors = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("dmf_b200 int8 ops have no gradients: call them under torch.no_grad()")
    if any(fwAD.unpack_dual(t).tangent is not None for t in tensors if t.is_floating_point()):
        raise RuntimeError("dmf_b200 int8 ops have no tangents")


def _check_floating(*tensors) -> None:
    ref = tensors[0]
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("dmf_b200 int8 ops run on CUDA (sm_100a) only; there is no CPU path")
        if t.dtype not in _DTYPES:
            raise TypeError(f"dmf_b200 int8 ops take bf16, fp16 and fp32, got {t.dtype}")
        if t.device != ref.device:
            raise ValueError("all tensors must be on one device")


def _check_rows8(r: Int8Rows) -> None:
    values, scale = r
    if not values.is_cuda:
        raise RuntimeError("dmf_b200 int8 ops run on CUDA (sm_100a) only; there is no CPU path")
    if values.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"expected int8 values and fp32 scales, got {values.dtype} and {scale.dtype}")
    if values.dim() < 1 or scale.shape != values.shape[:-1] or scale.device != values.device:
        raise ValueError(f"a scale per row: values {tuple(values.shape)} on {values.device}, scale {tuple(scale.shape)} on {scale.device}")
    _check_width(values)


def _check_width(x: torch.Tensor) -> None:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected rows of at least one element, got shape {tuple(x.shape)}")
    if x.shape[-1] > MAX_WIDTH or x.numel() // x.shape[-1] > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows of at most {MAX_WIDTH} elements")


def _mod2(t: torch.Tensor, B: int, Cn: int) -> torch.Tensor:
    """A (B, C) or (B, 1, C) modulation tensor as (B, C) with unit channel stride."""
    if t.dim() == 3 and t.shape[1] == 1:
        t = t[:, 0]
    if t.shape != (B, Cn):
        raise ValueError(f"shift / scale / gate must have shape ({B}, {Cn}) or ({B}, 1, {Cn}), got {tuple(t.shape)}")
    return t if t.stride(-1) == 1 else t.contiguous()


# ---- calls of the C ABI -----------------------------------------------------------------------------------------------

def _rows3(x: torch.Tensor) -> torch.Tensor:
    """(..., C) as (B, L, C) with unit channel stride, without a copy where strides allow."""
    if x.dim() != 3:
        x = x.reshape(1, -1, x.shape[-1])
    return x if x.stride(-1) == 1 else x.contiguous()


def _r(t: Optional[torch.Tensor]) -> _lib.Rows:
    return _lib.Rows(None, 0, 0) if t is None else _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _m(t: Optional[torch.Tensor]) -> _lib.Mod:
    return _lib.Mod(None, 0) if t is None else _lib.Mod(t.data_ptr(), t.stride(0))


def _pitch(columns: int) -> int:
    return -(-columns // 16) * 16


def _empty_rows8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised (values, scale) for rows of x's shape, values at a pitch of whole 16-byte units."""
    strides, step = [1], _pitch(x.shape[-1])
    for n in reversed(x.shape[:-1]):
        strides.append(step)
        step *= n
    return (torch.empty_strided(x.shape, strides[::-1], dtype=torch.int8, device=x.device),
            torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))


def _launch(name: str, a, device: torch.device) -> None:
    a.stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check(getattr(_lib.load(), name)(C.byref(a)))
    _ops._count(1)


def quantize_int8_raw(x, act: int):
    with torch.cuda.device(x.device):
        x3 = _rows3(x)
        q, scale = _empty_rows8(x)
        a = _lib.Int8QuantizeArgs()
        a.batch, a.seqlen, a.channels = x3.shape
        a.dtype, a.act = _DTYPES[x.dtype], act
        a.x = _r(x3)
        a.out = _lib.Int8Matrix(q.data_ptr(), _pitch(x.shape[-1]), scale.data_ptr())
        _launch("dmf_int8_quantize", a, x.device)
    return q, scale


def rms_norm_int8_raw(x, weight, residual, eps: float):
    """q, scale and, with a residual, the sum (like residual)."""
    with torch.cuda.device(x.device):
        x3 = _rows3(x)
        weight = weight.contiguous()
        q, scale = _empty_rows8(x)
        total = None if residual is None else torch.empty(residual.shape, dtype=residual.dtype, device=x.device)
        a = _lib.Int8RmsNormArgs()
        a.batch, a.seqlen, a.channels = x3.shape
        a.dtype, a.weight_dtype, a.eps = _DTYPES[x.dtype], _DTYPES[weight.dtype], float(eps)
        if residual is not None:
            residual = _rows3(residual)
            a.stream_dtype = _DTYPES[residual.dtype]
            a.residual, a.sum = _r(residual), _r(_rows3(total))
        a.x, a.weight = _r(x3), weight.data_ptr()
        a.out = _lib.Int8Matrix(q.data_ptr(), _pitch(x.shape[-1]), scale.data_ptr())
        _launch("dmf_int8_rmsnorm", a, x.device)
    return q, scale, total


def ln_modulate_int8_raw(x, shift, scale, gate, h, eps: float):
    """q, row scale and, with gate and h, the sum (like x)."""
    B, _, Cn = x.shape
    md = shift.dtype
    if any(t is not None and t.dtype != md for t in (scale, gate)):      # the kernel reads the three as one type
        md = torch.float32
    with torch.cuda.device(x.device):
        x3 = _rows3(x)
        shift, scale, gate = (None if t is None else _mod2(t.to(md), B, Cn) for t in (shift, scale, gate))
        q, row_scale = _empty_rows8(x)
        total = None if h is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a = _lib.Int8LnModulateArgs()
        a.batch, a.seqlen, a.channels = x3.shape
        a.stream_dtype, a.mod_dtype, a.eps = _DTYPES[x.dtype], _DTYPES[md], float(eps)
        if h is not None:
            h = _rows3(h)
            a.dtype = _DTYPES[h.dtype]
        a.x, a.h, a.sum = _r(x3), _r(h), _r(total)
        a.gate, a.shift, a.scale = _m(gate), _m(shift), _m(scale)
        a.out = _lib.Int8Matrix(q.data_ptr(), _pitch(Cn), row_scale.data_ptr())
        _launch("dmf_int8_ln_modulate", a, x.device)
    return q, row_scale, total


def _matrix8(values: torch.Tensor) -> torch.Tensor:
    v = values.reshape(-1, values.shape[-1])
    return v if v.stride(1) == 1 or v.shape[1] == 1 else v.contiguous()


# Products of this many terms and more are worth a copy of rows that the tensor cores cannot read: the integer pipe, which reads any
# row, adds up 4e13 terms a second, and a copy takes a few microseconds.
COPY_FROM = 2 ** 28


def _pitched(v: torch.Tensor) -> torch.Tensor:
    """(M, K) int8 with rows that start at multiples of 16 bytes and do not overlap, as the tensor-core kernels read them."""
    if v.data_ptr() % 16 == 0 and (v.shape[0] == 1 or (v.stride(0) % 16 == 0 and v.stride(0) >= v.shape[1])):
        return v
    out = torch.empty_strided(v.shape, (_pitch(v.shape[1]), 1), dtype=torch.int8, device=v.device)
    return out.copy_(v)


def int8_linear_raw(xq, x_scale, wq, w_scale, bias, out_dtype: torch.dtype):
    N, K = wq.shape
    with torch.cuda.device(xq.device):
        x2, w2 = _matrix8(xq), _matrix8(wq)
        if x2.shape[0] * N * K >= COPY_FROM:
            x2, w2 = _pitched(x2), _pitched(w2)
        x_scale, w_scale = x_scale.contiguous(), w_scale.contiguous()
        bias = None if bias is None else bias.contiguous()
        out = torch.empty((*xq.shape[:-1], N), dtype=out_dtype, device=xq.device)
        a = _lib.Int8LinearArgs()
        a.m, a.n, a.k, a.out_dtype = x2.shape[0], N, K, _DTYPES[out_dtype]
        a.x = _lib.Int8Matrix(x2.data_ptr(), x2.stride(0), x_scale.data_ptr())
        a.w = _lib.Int8Matrix(w2.data_ptr(), w2.stride(0), w_scale.data_ptr())
        if bias is not None:
            a.bias, a.bias_dtype = bias.data_ptr(), _DTYPES[bias.dtype]
        a.out, a.out_stride = out.data_ptr(), N
        a.status_word = _ops._status_word(xq.device).data_ptr()
        _launch("dmf_int8_linear", a, xq.device)
        if _ops._CHECK_EVERY_CALL:
            _ops.check_device_status(xq.device)
    return out


def dequantize_int8_raw(q, scale, dtype: torch.dtype):
    with torch.cuda.device(q.device):
        q2, scale = _matrix8(q), scale.contiguous()
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
        a = _lib.Int8DequantizeArgs()
        a.rows, a.channels, a.out_dtype = q2.shape[0], q2.shape[1], _DTYPES[dtype]
        a.x = _lib.Int8Matrix(q2.data_ptr(), q2.stride(0), scale.data_ptr())
        a.out, a.out_stride = out.data_ptr(), q.shape[-1]
        _launch("dmf_int8_dequantize", a, q.device)
    return out


# ---- torch custom ops -------------------------------------------------------------------------------------------------

@torch.library.custom_op("dmf_b200::quantize_int8", mutates_args=(), device_types="cuda")
def _quantize_op(x: torch.Tensor, act: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return quantize_int8_raw(x, act)


@torch.library.register_fake("dmf_b200::quantize_int8")
def _quantize_fake(x, act):
    return _empty_rows8(x)


@torch.library.custom_op("dmf_b200::rms_norm_int8", mutates_args=(), device_types="cuda")
def _rms_op(x: torch.Tensor, weight: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return rms_norm_int8_raw(x, weight, None, eps)[:2]


@torch.library.register_fake("dmf_b200::rms_norm_int8")
def _rms_fake(x, weight, eps):
    return _empty_rows8(x)


@torch.library.custom_op("dmf_b200::add_rms_norm_int8", mutates_args=(), device_types="cuda")
def _add_rms_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return rms_norm_int8_raw(x, weight, residual, eps)


@torch.library.register_fake("dmf_b200::add_rms_norm_int8")
def _add_rms_fake(x, residual, weight, eps):
    return (*_empty_rows8(x), residual.new_empty(residual.shape))


@torch.library.custom_op("dmf_b200::ln_modulate_int8", mutates_args=(), device_types="cuda")
def _ln_op(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return ln_modulate_int8_raw(x, shift, scale, None, None, eps)[:2]


@torch.library.register_fake("dmf_b200::ln_modulate_int8")
def _ln_fake(x, shift, scale, eps):
    return _empty_rows8(x)


@torch.library.custom_op("dmf_b200::gate_ln_modulate_int8", mutates_args=(), device_types="cuda")
def _gate_ln_op(x: torch.Tensor, gate: torch.Tensor, h: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor,
                eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return ln_modulate_int8_raw(x, shift, scale, gate, h, eps)


@torch.library.register_fake("dmf_b200::gate_ln_modulate_int8")
def _gate_ln_fake(x, gate, h, shift, scale, eps):
    return (*_empty_rows8(x), x.new_empty(x.shape))


@torch.library.custom_op("dmf_b200::int8_linear", mutates_args=(), device_types="cuda")
def _linear_op(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    return int8_linear_raw(xq, x_scale, wq, w_scale, bias, out_dtype)


@torch.library.register_fake("dmf_b200::int8_linear")
def _linear_fake(xq, x_scale, wq, w_scale, bias, out_dtype):
    return xq.new_empty((*xq.shape[:-1], wq.shape[0]), dtype=out_dtype)


@torch.library.custom_op("dmf_b200::dequantize_int8", mutates_args=(), device_types="cuda")
def _dequantize_op(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return dequantize_int8_raw(q, scale, dtype)


@torch.library.register_fake("dmf_b200::dequantize_int8")
def _dequantize_fake(q, scale, dtype):
    return q.new_empty(q.shape, dtype=dtype)


# ---- public functions -------------------------------------------------------------------------------------------------

def quantize_int8(x: torch.Tensor, activation: Optional[str] = None) -> Int8Rows:
    """The rows (last dimension) of x, behind ``activation`` - None, "gelu" (tanh form) or "silu" -, in 8 bits.  Of a weight
    (out_features, in_features) this gives a scale per output channel."""
    if activation not in _lib.INT8_ACTS:
        raise ValueError(f"activation must be None, 'gelu' or 'silu', got {activation!r}")
    if _native.takes(x):
        out = _native.quantize_int8(x, _lib.INT8_ACTS[activation])
        if out is not None:
            return Int8Rows(*out)
    _check_floating(x)
    _check_width(x)
    _refuse_derivatives(x)
    return Int8Rows(*torch.ops.dmf_b200.quantize_int8(x, _lib.INT8_ACTS[activation]))


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None):
    """``z * rsqrt(mean(z^2, -1) + eps) * weight`` in 8 bits, z = x or residual + x, for x (..., C) and weight (C).  With a
    residual returns (rows, z in the residual's type); the norm is of z before that rounding."""
    if _native.takes(x, weight, residual):
        out = _native.rms_norm_int8(x, weight, eps, residual)
        if out is not None:
            return Int8Rows(*out[:2]) if residual is None else (Int8Rows(*out[:2]), out[2])
    _check_floating(x, weight, residual)
    _check_width(x)
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError("x and residual must have the same shape")
    _refuse_derivatives(x, weight, residual)
    if residual is None:
        return Int8Rows(*torch.ops.dmf_b200.rms_norm_int8(x, weight, float(eps)))
    q, scale, total = torch.ops.dmf_b200.add_rms_norm_int8(x, residual, weight, float(eps))
    return Int8Rows(q, scale), total


def ln_modulate_int8(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6, *,
                     gate: Optional[torch.Tensor] = None, h: Optional[torch.Tensor] = None):
    """``layer_norm(z) * (1 + scale) + shift`` in 8 bits, z = x or x + gate * h, for x, h (B, L, C) and shift / scale / gate
    (B, C) or (B, 1, C): adaln.gate_residual and adaln.ln_modulate in one pass.  With gate and h returns (rows, z in x's
    type); the norm is of z before that rounding."""
    if (gate is None) != (h is None):
        raise ValueError("gate and h come together")
    if _native.takes(x, shift, scale, gate, h):
        out = _native.ln_modulate_int8(x, shift, scale, eps, gate, h)
        if out is not None:
            return Int8Rows(*out[:2]) if h is None else (Int8Rows(*out[:2]), out[2])
    _check_floating(x, shift, scale, gate, h)
    _check_width(x)
    if x.dim() != 3:
        raise ValueError("expected a (B, L, C) tensor")
    if h is not None and h.shape != x.shape:
        raise ValueError("x and h must have the same shape")
    for t in (shift, scale, gate):
        if t is not None and t.shape not in ((x.shape[0], x.shape[2]), (x.shape[0], 1, x.shape[2])):
            raise ValueError(f"shift / scale / gate must have shape ({x.shape[0]}, {x.shape[2]}) or ({x.shape[0]}, 1, {x.shape[2]}), "
                             f"got {tuple(t.shape)}")
    _refuse_derivatives(x, shift, scale, gate, h)
    if h is None:
        return Int8Rows(*torch.ops.dmf_b200.ln_modulate_int8(x, shift, scale, float(eps)))
    q, row_scale, total = torch.ops.dmf_b200.gate_ln_modulate_int8(x, gate, h, shift, scale, float(eps))
    return Int8Rows(q, row_scale), total


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None, *,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T + bias`` of rows in 8 bits: x (..., K), weight (N, K), bias (N); the result (..., N) in ``out_dtype``.
    The sums are exact; they, their products with the two scales and the bias's addition are rounded to fp32, the result to its type."""
    (xq, x_scale), (wq, w_scale) = x, weight
    if _native.takes(xq, x_scale, wq, w_scale, bias):
        out = _native.int8_linear(xq, x_scale, wq, w_scale, bias, out_dtype)
        if out is not None:
            return out
    x, weight = Int8Rows(xq, x_scale), Int8Rows(wq, w_scale)
    _check_rows8(x)
    _check_rows8(weight)
    if weight.values.dim() != 2 or weight.values.shape[1] != x.values.shape[-1] or weight.values.shape[0] < 1:
        raise ValueError(f"x (..., K) and weight (N, K) do not fit: {tuple(x.values.shape)} and {tuple(weight.values.shape)}")
    if x.values.shape[-1] > MAX_K:
        raise ValueError(f"rows of at most {MAX_K} elements: longer sums could leave int32")
    if weight.values.shape[0] > MAX_N:
        raise ValueError(f"a weight of at most {MAX_N} rows")
    if out_dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    if weight.values.device != x.values.device:
        raise ValueError("x and weight must be on one device")
    if bias is not None:
        _check_floating(bias)
        if bias.shape != weight.values.shape[:1] or bias.device != x.values.device:
            raise ValueError(f"bias must have shape ({weight.values.shape[0]},) on {x.values.device}")
    _refuse_derivatives(x.scale, weight.scale, bias)
    return torch.ops.dmf_b200.int8_linear(x.values, x.scale, weight.values, weight.scale, bias, out_dtype)
