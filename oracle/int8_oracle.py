"""fp64 oracle of the 8-bit inference ops (dmf_b200.int8): what they compute, from their definitions.  Test infrastructure only."""

from __future__ import annotations

import torch

TINY = 2.0 ** -120


def act(x, name):
    x = x.double()
    if name == "gelu":      # 0.5 x (1 + tanh u) as x sigmoid(2 u): 1 + tanh u loses all its digits below u = -18
        return x * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3))
    return x * torch.sigmoid(x) if name == "silu" else x


def rms_norm(x, weight, eps, residual=None):
    """(y, z)"""
    z = x.double() if residual is None else residual.double() + x.double()
    return z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + eps) * weight.double(), z


def ln_modulate(x, shift, scale, eps, gate=None, h=None):
    """(y, z); shift, scale, gate broadcast over L"""
    z = x.double() if h is None else x.double() + gate.double() * h.double()
    c = z - z.mean(-1, keepdim=True)
    return c * torch.rsqrt(c.pow(2).mean(-1, keepdim=True) + eps) * (1 + scale.double()) + shift.double(), z


def real_rows(y):
    """127 y / a before rounding, and the scale a / 127, for rows y."""
    a = y.abs().amax(-1)
    some = a >= TINY
    return torch.where(some[..., None], 127 * y / a.clamp_min(TINY)[..., None], 0.0), torch.where(some, a / 127, 0.0)


def linear(xq, x_scale, wq, w_scale, bias=None):
    """(result, the same with every term's magnitude: what errors of its sum are relative to)"""
    s = (xq.double() @ wq.double().t()) * x_scale.double()[..., None] * w_scale.double()
    b = 0.0 if bias is None else bias.double()
    return s + b, s.abs() + (0.0 if bias is None else b.abs())
