"""A DMFT model whose transformer blocks run in 8-bit integers (dmf_b200.int8), for sampling.

``int8_model(model)`` returns a copy with the blocks' linear layers - modulation, qkv, proj and the MLP - as int8 products with a
scale per token and per output channel, the weights quantised once and the activations where they arise: behind the adaLN norm, by
the norm's own kernel; behind SiLU, GELU and the attention, by a pass over the rows.  Everything else - patch, time and label
embeddings, attention, the final layer - is the model's, and so is the calling convention:

    sampler = GraphedSampler(int8_model(model), batch)          # or euler_sampler(int8_model(model), z, y)

A block's second residual addition happens in the next kernel that reads the stream (the next block's norm, or the final layer), so
between the blocks travels the triple (x, gate, h) that stands for x + gate * h.
"""

from __future__ import annotations

import copy
from typing import NamedTuple

import torch
import torch.nn as nn

from .. import adaln
from ..flash_attn_jvp import flash_attn_qkvpacked_func
from ..int8 import Int8Rows, int8_linear, ln_modulate_int8, quantize_int8
from .model import DMFT, DiTBlock


class Int8Linear(nn.Module):
    """A linear layer's weight in 8 bits, a scale per output channel; applied to ``Int8Rows``."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        with torch.no_grad():
            values, scale = quantize_int8(linear.weight.detach())
            bias = None if linear.bias is None else linear.bias.detach().clone()
        self.register_buffer("values", values)
        self.register_buffer("scale", scale)
        self.register_buffer("bias", bias)

    def forward(self, rows: Int8Rows, out_dtype: torch.dtype) -> torch.Tensor:
        return int8_linear(rows, Int8Rows(self.values, self.scale), self.bias, out_dtype=out_dtype)

    def _apply(self, fn, recurse=True):
        """Moves like any module, but stays what it is: a model's .half() or .bfloat16() must not round the scales."""
        def keep_scales(t):
            moved = fn(t)
            return t.to(moved.device) if t is self.scale else moved
        return super()._apply(keep_scales, recurse)


class PendingResidual(NamedTuple):
    """x + gate * h, not added yet."""
    x: torch.Tensor
    gate: torch.Tensor
    h: torch.Tensor


class Int8DiTBlock(nn.Module):
    """DiTBlock (models/layers.py:170-201) on 8-bit products; takes and gives the stream or a PendingResidual."""

    def __init__(self, block: DiTBlock):
        super().__init__()
        self.eps1, self.eps2 = block.norm1.eps, block.norm2.eps
        self.num_heads, self.head_dim, self.packed, self.attn = (block.attn.num_heads, block.attn.head_dim, block.attn.packed,
                                                                 block.attn.attn)
        self.q_norm, self.k_norm = block.attn.q_norm, block.attn.k_norm
        self.modulation = Int8Linear(block.adaLN_modulation[1])
        self.qkv, self.proj = Int8Linear(block.attn.qkv), Int8Linear(block.attn.proj)
        self.fc1, self.fc2 = Int8Linear(block.mlp.fc1), Int8Linear(block.mlp.fc2)

    def attention(self, rows: Int8Rows, dtype: torch.dtype) -> torch.Tensor:
        qkv = self.qkv(rows, dtype)
        B, L, _ = qkv.shape
        qkv = qkv.reshape(B, L, 3, self.num_heads, self.head_dim)
        if self.packed:
            o = flash_attn_qkvpacked_func(qkv)
        else:
            q, k, v = qkv.unbind(2)
            o = self.attn(self.q_norm(q), self.k_norm(k), v)
        return self.proj(quantize_int8(o.reshape(B, L, -1)), dtype)

    def forward(self, x, c):
        stream = x.x if isinstance(x, PendingResidual) else x
        dtype = torch.bfloat16 if stream.dtype == torch.float32 else stream.dtype      # what the products give
        sh_a, sc_a, g_a, sh_m, sc_m, g_m = self.modulation(quantize_int8(c, "silu"), dtype).chunk(6, dim=-1)
        if isinstance(x, PendingResidual):
            rows, stream = ln_modulate_int8(x.x, sh_a, sc_a, self.eps1, gate=x.gate, h=x.h)
        else:
            rows = ln_modulate_int8(stream, sh_a, sc_a, self.eps1)
        rows, stream = ln_modulate_int8(stream, sh_m, sc_m, self.eps2, gate=g_a, h=self.attention(rows, dtype))
        return PendingResidual(stream, g_m, self.fc2(quantize_int8(self.fc1(rows, dtype), "gelu"), dtype))


class Int8FinalLayer(nn.Module):
    """The model's final layer behind the last block's addition."""

    def __init__(self, layer: nn.Module):
        super().__init__()
        self.layer = layer

    def forward(self, x, c):
        if isinstance(x, PendingResidual):
            x = adaln.gate_residual(x.x, x.gate, x.h)
        return self.layer(x, c)


def int8_model(model: DMFT) -> DMFT:
    """A copy of a DMFT model on the GPU with its blocks in 8 bits, in eval mode and without gradients; the weights that were
    quantised are not kept in 16 or 32 bits.  The model must use this package's attention ('fa2' / 'fa3').  With an fp32 stream the
    products and the attention give bf16, as under autocast."""
    blocks = list(model.blocks)
    if not all(isinstance(b, DiTBlock) and b.fused for b in blocks):
        raise ValueError("int8_model takes a DMFT model with attn_func 'fa2' or 'fa3'")
    if not all(adaln.usable(p.new_empty((1, 1, p.shape[0]))) for p in (b.attn.proj.weight for b in blocks)):
        raise ValueError("int8_model takes a model on the GPU, in fp32 or bf16, of a width that the adaLN ops are compiled for")
    kept, model.blocks = model.blocks, nn.ModuleList()     # the copy leaves the blocks out: they are converted one by one
    try:
        out = copy.deepcopy(model)
    finally:
        model.blocks = kept
    out.blocks = nn.ModuleList(Int8DiTBlock(copy.deepcopy(b)) for b in blocks)
    out.final_layer = Int8FinalLayer(out.final_layer)
    return out.eval().requires_grad_(False)
