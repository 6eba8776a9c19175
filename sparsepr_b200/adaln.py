"""Adaptive layer norm of a diffusion transformer's blocks, with gradients.

* :func:`layer_norm` — ``LN(x) * weight + bias``;
* :func:`modulated_layer_norm` — ``LN(x) * (1 + scale) + shift``;
* :func:`gated_residual_layer_norm` — ``z = x + gate * y`` and the modulated norm of
  ``z`` in one pass, returning both.

``x`` and ``y`` are [..., C] CUDA tensors in fp32, bf16 or fp16 (C <= 16384, fewer than
2^31 rows, the channels contiguous, the axes before them in any order of strides that
``Tensor.view`` can merge).  ``weight``, ``bias``, ``shift``, ``scale`` and ``gate`` are of
one type, x's or fp32, and of one shape: [C], or x's shape with some of the
leading axes of extent 1, where the axes kept and the axes broadcast are each
adjacent: one vector, one per sample ([B, 1, C]), one per token ([B, N, C] or
[1, N, C]).  Results are rounded once to x's type; ``z`` is rounded before it is
normalised, so the norm reads what the residual stream holds.  Statistics and
sums are fp32, and the gradients of shared vectors are summed in a fixed order.

The gradients are of first order, in reverse mode (dual tensors are refused).  A backward
pass captured into a CUDA graph needs what any captured autograd call needs: warm-up
passes on a side stream, and no graph of an uncaptured forward pass over the same leaves
still alive.  :func:`operands` with
:func:`sparsepr_b200.kernels.adaln_forward` and ``adaln_backward`` are the same passes
without autograd.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K

__all__ = ["layer_norm", "modulated_layer_norm", "gated_residual_layer_norm"]


def _split(shape, mod_shape, name):
    """(batch, tokens, batch kept, tokens kept): x's leading axes as two runs, each
    wholly kept or wholly broadcast by a vector of ``mod_shape``."""
    lead = tuple(shape[:-1])
    if len(mod_shape) > len(shape) or not mod_shape or mod_shape[-1] != shape[-1]:
        raise RuntimeError(f"{name} {tuple(mod_shape)} does not match x {tuple(shape)}")
    own = (1,) * (len(shape) - len(mod_shape)) + tuple(mod_shape[:-1])
    runs = []  # [extent, kept]
    for d, m in zip(lead, own):
        if m != d and m != 1:
            raise RuntimeError(f"{name} {tuple(mod_shape)} does not match x {tuple(shape)}")
        if d == 1:
            continue
        kept = m != 1
        if runs and runs[-1][1] == kept:
            runs[-1][0] *= d
        else:
            runs.append([d, kept])
    if len(runs) > 2:
        raise RuntimeError(f"{name} {tuple(mod_shape)} against x {tuple(shape)}: the axes it is broadcast along must "
                           "be adjacent")
    if len(runs) < 2:
        runs.insert(0, [1, False])
    if len(runs) < 2:
        runs.append([1, False])
    return runs[0][0], runs[1][0], runs[0][1], runs[1][1]


def _strides(t, b, n, name):
    """Element strides of the [b, n, C] rows that a [..., C] tensor holds (0 for an extent of 1)."""
    if t.is_contiguous():
        c = t.shape[-1]
        return (n * c if b > 1 else 0), (c if n > 1 else 0)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{name}: channels must be contiguous, got strides {t.stride()}")
    try:
        v = t.view(b, n, t.shape[-1])
    except RuntimeError:
        raise RuntimeError(f"{name}: axes of strides {t.stride()} cannot be viewed as [{b}, {n}, {t.shape[-1]}]; "
                           "make it contiguous") from None
    return (v.stride(0) if b > 1 else 0), (v.stride(1) if n > 1 else 0)


_NONE = (0, 0)


def operands(x, y, gate, shift, scale, scale_offset: float = 1.0):
    """``(AdalnOperands, (batch or 1, tokens or 1) of the vectors)`` of checked tensors."""
    if not x.is_cuda:
        raise RuntimeError(f"sparsepr_b200 kernels need CUDA tensors, got a {x.device} tensor")
    dt, shape = x.dtype, x.shape
    if dt not in K._DT or not shape:
        raise RuntimeError(f"x must be [..., C] fp32/bf16/fp16, got {tuple(shape)} {dt}")
    c = shape[-1]
    if not 1 <= c <= 16384:
        raise RuntimeError(f"layer norm over {c} channels: 1 to 16384 are supported")
    index = x.get_device()
    if y is not None and (y.shape != shape or y.dtype != dt or y.get_device() != index):
        raise RuntimeError(f"y must be {tuple(shape)} {dt} on {x.device} as x is, got {tuple(y.shape)} {y.dtype} on "
                           f"{y.device}")
    first = None
    for name, t in (("gate", gate), ("shift", shift), ("scale", scale)):
        if t is None:
            continue
        if t.get_device() != index:
            raise RuntimeError(f"{name} is on {t.device}, x on {x.device}")
        if first is None:
            first, first_name = t, name
            if t.dtype != dt and t.dtype != torch.float32:
                raise RuntimeError(f"{name} must be {dt} or fp32, got {t.dtype}")
        elif t.shape != first.shape or t.dtype != first.dtype:
            raise RuntimeError(f"{name} {tuple(t.shape)} {t.dtype} must be as {first_name}: {tuple(first.shape)} "
                               f"{first.dtype}")
    if first is None or first.shape == (c,):
        b, n, keep_b, keep_n = 1, x.numel() // c, False, False
    else:
        b, n, keep_b, keep_n = _split(shape, first.shape, first_name)
    if b == 1 and len(shape) > 2 and not all(t is None or t.is_contiguous() for t in (x, y, gate, shift, scale)):
        # One vector for all rows, or one for each: any two runs of x's axes will do.
        b, n, keep_b = math.prod(shape[:-2]), shape[-2], keep_n
    mb, mn = (b if keep_b else 1), (n if keep_n else 1)
    op = K.AdalnOperands(x, y, gate, shift, scale, b, n, c, _strides(x, b, n, "x"),
                         _NONE if y is None else _strides(y, b, n, "y"),
                         _NONE if shift is None else _strides(shift, mb, mn, "shift"),
                         _NONE if scale is None else _strides(scale, mb, mn, "scale"),
                         _NONE if gate is None else _strides(gate, mb, mn, "gate"),
                         dt if first is None else first.dtype, scale_offset)
    return op, (mb, mn)


def _saved(s, name, t, dtype, b, n, index):
    """Point operand ``name`` of ``s`` at a saved tensor, which hooks may have given back in another layout."""
    K.check_saved(t, dtype, b * n * s.channels, index)
    if t.is_contiguous():
        sb, st = (n * s.channels if b > 1 else 0), (s.channels if n > 1 else 0)
    else:
        try:
            sb, st = _strides(t, b, n, name)
        except RuntimeError:
            return _saved(s, name, t.contiguous(), dtype, b, n, index)
    setattr(s, name, t.data_ptr())
    setattr(s, name + "_sb", sb)
    setattr(s, name + "_st", st)
    return t


def _backward(ctx, *grads):
    K.refuse_tangents("layer norm gradient", *grads)
    x, y, gate, scale, stats = ctx.saved_tensors
    dz, dh = grads if y is not None else (None, grads[0])
    if dh is None:
        if dz is None:
            return (None,) * 7
        dh = torch.zeros_like(dz, memory_format=torch.contiguous_format)
    elif not dh.is_contiguous():
        dh = dh.contiguous()
    if dz is not None and not dz.is_contiguous():
        dz = dz.contiguous()
    s, mod_shape, vector_shape, mod_dtype = ctx.operands
    s = type(s).from_buffer_copy(s)
    b, n, index = s.batch, s.tokens, dh.get_device()
    x = _saved(s, "x", x, dh.dtype, b, n, index)  # z, where there is a branch
    y = y if y is None else _saved(s, "y", y, dh.dtype, b, n, index)
    gate = gate if gate is None else _saved(s, "gate", gate, mod_dtype, *mod_shape, index)
    scale = scale if scale is None else _saved(s, "scale", scale, mod_dtype, *mod_shape, index)
    stats = K.dense_saved(stats, torch.float32, 2 * b * n, index)
    mean = stats.data_ptr()
    s.mean, s.rstd = mean, mean + 4 * b * n
    grads = K.adaln_backward_struct(s, y is not None, dh, dz, ctx.needs_input_grad[2:5], mod_shape, vector_shape,
                                    mod_dtype)
    return *grads, None, None


_backward_once = once_differentiable(_backward)


class _AdaLN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, shift, scale, eps, scale_offset):
        op, mod_shape = operands(x, y, gate, shift, scale, scale_offset)
        z, h, stats, struct = K.adaln_forward_struct(op, eps, True)
        ctx.save_for_backward(x if z is None else z, y, gate, scale, stats)
        ctx.set_materialize_grads(False)
        vector = gate if gate is not None else shift if shift is not None else scale
        ctx.operands = struct, mod_shape, None if vector is None else vector.shape, op.mod_dtype
        return h if z is None else (z, h)

    @staticmethod
    def backward(ctx, *grads):
        # The wrapper that refuses second derivatives, where a graph of this pass is asked for.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _wants_grad(x, y, gate, shift, scale):
    K.refuse_tangents("layer norm", x, y, gate, shift, scale)
    return torch.is_grad_enabled() and (x.requires_grad or (y is not None and y.requires_grad)
                                        or (gate is not None and gate.requires_grad)
                                        or (shift is not None and shift.requires_grad)
                                        or (scale is not None and scale.requires_grad))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis."""
    if _wants_grad(x, None, None, bias, weight):
        return _AdaLN.apply(x, None, None, bias, weight, float(eps), 0.0)
    return K.adaln_forward(operands(x, None, None, bias, weight, 0.0)[0], eps, False)[1]


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor | None,
                         eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * (1 + scale) + shift`` over the last axis."""
    if _wants_grad(x, None, None, shift, scale):
        return _AdaLN.apply(x, None, None, shift, scale, float(eps), 1.0)
    return K.adaln_forward(operands(x, None, None, shift, scale)[0], eps, False)[1]


def gated_residual_layer_norm(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor | None,
                              shift: torch.Tensor | None, scale: torch.Tensor | None,
                              eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``(z, modulated_layer_norm(z, shift, scale))`` with ``z = x + gate * y`` (``gate`` None:
    ``x + y``), ``y`` of x's shape and type."""
    if _wants_grad(x, y, gate, shift, scale):
        return _AdaLN.apply(x, y, gate, shift, scale, float(eps), 1.0)
    return K.adaln_forward(operands(x, y, gate, shift, scale)[0], eps, False)[:2]
