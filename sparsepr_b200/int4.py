"""Linear layers with 4-bit weights under group scales, for a few rows.

A diffusion transformer makes every block's modulation from one conditioning
vector per sample: a product that reads its whole weight for one or two rows, so
its time is the weight's bytes.  :func:`quantize_int4` stores a weight in 4 bits,
:func:`int4_linear` multiplies rows by it (its gradient goes to the rows and the
bias; the codes are frozen), :func:`dequantize_int4` gives the weight back.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K

__all__ = ["Int4Weight", "quantize_int4", "dequantize_int4", "int4_linear"]


class Int4Weight(NamedTuple):
    """``packed`` uint8 [N, groups*group/2] (two codes a byte, the even column in the low
    half), ``scales`` [N, groups], ``zeros`` uint8 [N, groups], or None (8).  Zero codes are 0
    to 15; larger ones are not looked for and give meaningless products."""

    packed: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None


def quantize_int4(weight: torch.Tensor, group_size: int = 64, symmetric: bool = False,
                  scale_dtype: torch.dtype | None = None) -> Int4Weight:
    """4-bit codes of a [N, K] weight by round to nearest, on the weight's device.

    Each run of ``group_size`` columns (a multiple of 32; the last may be partly
    used) has a scale in ``scale_dtype`` (default: the weight's type) and, unless
    ``symmetric``, a zero code; the codes are those nearest under the stored scale.  A
    weight that is not finite, or too large for its scales' type, raises."""
    if weight.dim() != 2 or weight.dtype not in K._DT or weight.numel() == 0:
        raise RuntimeError(f"quantize_int4 expects a non-empty fp32/bf16/fp16 [N, K] weight, got "
                           f"{tuple(weight.shape)} {weight.dtype}")
    if group_size < 32 or group_size % 32:
        raise ValueError(f"group_size must be a positive multiple of 32, got {group_size}")
    sdt = weight.dtype if scale_dtype is None else scale_dtype
    if sdt not in K._DT:
        raise ValueError(f"scale_dtype must be fp32/bf16/fp16, got {sdt}")
    n, k = weight.shape
    groups = -(-k // group_size)
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group_size - k)).view(n, groups, group_size)
    lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
    step = torch.maximum(-lo, hi) / 7.0 if symmetric else (hi - lo) / 15.0
    if sdt == torch.float16:  # below 2^-14, multiples of 2^-24: rounded up, so that all codes fit
        step = torch.where(step < 2.0 ** -14, (step * 2.0 ** 24).ceil().clamp(min=1.0) * 2.0 ** -24, step)
    scales = step.clamp(min=torch.finfo(torch.float32).tiny).to(sdt)  # positive, of groups of zeros too
    s = scales.float()
    if not torch.isfinite(s).all():
        raise RuntimeError(f"quantize_int4: the weight is not finite, or too large for scales in {sdt}")
    zeros = None if symmetric else (-lo / s).round().clamp(0, 15).to(torch.uint8)
    codes = ((w / s[..., None]).round() + (8.0 if symmetric else zeros.float()[..., None])).clamp(0, 15)
    codes = codes.to(torch.uint8).view(n, groups * group_size)
    return Int4Weight(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, zeros)


def dequantize_int4(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, in_features: int,
                    dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The [N, in_features] weight that the codes stand for."""
    n, groups = scales.shape
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).view(n, groups, -1).float()
    w = (codes - (8.0 if zeros is None else zeros.float()[..., None])) * scales.float()[..., None]
    return w.view(n, -1)[:, :in_features].to(dtype)


def _backward(ctx, dy):
    K.refuse_tangents("int4_linear gradient", dy)
    packed, scales, zeros = ctx.saved_tensors
    (n, half), groups, scale_dtype = ctx.weight
    index = dy.get_device()
    packed = K.dense_saved(packed, torch.uint8, n * half, index)
    scales = K.dense_saved(scales, scale_dtype, n * groups, index)
    zeros = zeros if zeros is None else K.dense_saved(zeros, torch.uint8, n * groups, index)
    dx = dbias = None
    if dy.stride(1) != 1 or (dy.shape[0] > 1 and dy.stride(0) < dy.shape[1]):
        dy = dy.contiguous()
    if ctx.needs_input_grad[0]:
        dx = K.int4_linear_grad_checked(dy, packed, scales, zeros, ctx.in_features, n, 2 * half // groups)
    if ctx.needs_input_grad[4]:
        dbias = dy.sum(0)  # 16-bit sums are fp32 inside and rounded once
    return dx, None, None, None, dbias


_backward_once = once_differentiable(_backward)


class _Int4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, packed, scales, zeros, bias):
        ctx.save_for_backward(packed, scales, zeros)
        y = K.int4_linear(x, packed, scales, zeros, bias)
        ctx.in_features, ctx.weight = x.shape[1], (packed.shape, scales.shape[1], scales.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        # The wrapper that refuses second derivatives, where a graph of this pass is asked for.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy)


def int4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with the 4-bit weight ``W`` [N, K] of :func:`quantize_int4`.

    ``x`` [..., K] in fp32, bf16 or fp16 and ``bias`` [N] in x's type; ``packed`` begins on 16
    bytes; the result [..., N] is rounded once from fp32 sums.  Up to eight 16-bit rows are
    multiplied as integers of 31 bits relative to each row's largest value (of up to all its
    columns): entries keep bf16's 8 bits down to 2^-22 of that value and are lost below
    2^-31, which shows only where the codes opposite the larger values are zero; cast ``x``
    to fp32 to keep every entry whole.  Any number of rows is computed, but the
    weights are read again for every 8 to 32 rows: the call is for a few rows.  Gradients
    are of first order, in reverse mode (dual tensors are refused).  A backward pass captured
    into a CUDA graph needs what any captured autograd call needs: no graph of an uncaptured
    forward pass over the same leaves still alive.  The weight is frozen: scales that ask for
    a gradient are refused."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"int4_linear: x must be [..., K], got {tuple(x.shape)}")
    K.refuse_tangents("int4_linear", x, scales, bias)
    if scales.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("int4_linear: the weight is frozen, its scales take no gradient; pass scales.detach()")
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        y = _Int4Linear.apply(rows, packed, scales, zeros, bias)
    else:
        y = K.int4_linear(rows, packed, scales, zeros, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], packed.shape[0])
