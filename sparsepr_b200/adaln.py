"""Adaptive layer norm of a diffusion transformer's blocks, with gradients.

* :func:`layer_norm` — ``LN(x) * weight + bias``;
* :func:`modulated_layer_norm` — ``LN(x) * (1 + scale) + shift``;
* :func:`gated_residual_layer_norm` — ``z = x + gate * y`` and the modulated norm of
  ``z`` in one pass, returning both.

``x`` and ``y`` are [..., C] CUDA tensors in fp32, bf16 or fp16 (C <= 16384, the
channels contiguous, the axes before them in any order of strides that
``Tensor.view`` can merge).  ``weight``, ``bias``, ``shift``, ``scale`` and ``gate`` are of
one type, x's or fp32, and of one shape: [C], or x's shape with some of the
leading axes of extent 1, where the axes kept and the axes broadcast are each
adjacent: one vector, one per sample ([B, 1, C]), one per token ([B, N, C] or
[1, N, C]).  Results are rounded once to x's type; ``z`` is rounded before it is
normalised, so the norm reads what the residual stream holds.  Statistics and
sums are fp32, and the gradients of shared vectors are summed in a fixed order.

The gradients are of first order.  A call captured into a CUDA graph needs what
any captured autograd call needs; :func:`sparsepr_b200.kernels.adaln_forward` and
``adaln_backward`` are the same passes without autograd.
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


def _rows(t, b, n, name):
    """[b, n, C] view of a [..., C] tensor."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{name}: channels must be contiguous, got strides {t.stride()}")
    try:
        return t.view(b, n, t.shape[-1])
    except RuntimeError:
        raise RuntimeError(f"{name}: axes of strides {t.stride()} cannot be viewed as [{b}, {n}, {t.shape[-1]}]; "
                           "make it contiguous") from None


def _prepare(x, y, gate, shift, scale):
    """Checked [B,N,C] views of all operands and the kept extents of the vectors."""
    for name, t in (("x", x), ("y", y), ("gate", gate), ("shift", shift), ("scale", scale)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} is on {t.device}, x on {x.device}")
    if not x.is_cuda:
        raise RuntimeError(f"sparsepr_b200 kernels need CUDA tensors, got a {x.device} tensor")
    if x.dtype not in K._DT or x.dim() < 1:
        raise RuntimeError(f"x must be [..., C] fp32/bf16/fp16, got {tuple(x.shape)} {x.dtype}")
    c = x.shape[-1]
    if not 1 <= c <= 16384:
        raise RuntimeError(f"layer norm over {c} channels: 1 to 16384 are supported")
    if y is not None and (y.shape != x.shape or y.dtype != x.dtype):
        raise RuntimeError(f"y must be {tuple(x.shape)} {x.dtype} as x is, got {tuple(y.shape)} {y.dtype}")
    mods = [(n, t) for n, t in (("gate", gate), ("shift", shift), ("scale", scale)) if t is not None]
    if mods:
        name, first = mods[0]
        if first.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{name} must be {x.dtype} or fp32, got {first.dtype}")
        for other, t in mods[1:]:
            if t.shape != first.shape or t.dtype != first.dtype:
                raise RuntimeError(f"{other} {tuple(t.shape)} {t.dtype} must be as {name}: {tuple(first.shape)} "
                                   f"{first.dtype}")
        b, n, keep_b, keep_n = _split(x.shape, first.shape, name)
    else:
        b, n, keep_b, keep_n = 1, x.numel() // c, False, False
    if b == 1 and not keep_n and x.dim() > 2 and not all(t is None or t.is_contiguous() for t in (x, y)):
        # One vector for all rows: any two runs of x's axes will do.
        b, n = math.prod(x.shape[:-2]), x.shape[-2]
    xv = _rows(x, b, n, "x")
    yv = None if y is None else _rows(y, b, n, "y")
    mb, mn = (b if keep_b else 1), (n if keep_n else 1)
    return xv, yv, *(None if t is None else _rows(t, mb, mn, k) for k, t in
                     (("gate", gate), ("shift", shift), ("scale", scale))), (mb, mn)


def _grad_rows(t, b, n):
    """[b, n, C] view of an incoming gradient of any strides."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t.view(b, n, t.shape[-1])


class _AdaLN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, shift, scale, eps, scale_offset):
        xv, yv, gv, shv, scv, mod_shape = _prepare(x, y, gate, shift, scale)
        z, h, mean, rstd = K.adaln_forward(xv, yv, gv, shv, scv, eps, scale_offset, True)
        h = h.view(x.shape)
        if z is not None:
            z = z.view(x.shape)
        ctx.save_for_backward(x if z is None else z, y, gate, scale, mean, rstd)
        ctx.set_materialize_grads(False)
        ctx.layout = (xv.shape[0], xv.shape[1], mod_shape, scale_offset)
        ctx.mod = next(((t.shape, t.dtype) for t in (gate, shift, scale) if t is not None), (None, None))
        return (h,) if z is None else (z, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, y, gate, scale, mean, rstd = ctx.saved_tensors
        b, n, mod_shape, offset = ctx.layout
        dz, dh = grads if y is not None else (None, grads[0])
        if dh is None and dz is None:
            return (None,) * 7
        dh = torch.zeros_like(x, memory_format=torch.contiguous_format) if dh is None else dh
        mshape, mdtype = ctx.mod
        view = lambda t, nb, nn: None if t is None else t.view(nb, nn, t.shape[-1])  # noqa: E731
        dx, dy, dgate, dshift, dscale = K.adaln_backward(
            view(x, b, n), view(y, b, n), view(gate, *mod_shape), view(scale, *mod_shape), mean, rstd,
            _grad_rows(dh, b, n), _grad_rows(dz, b, n), offset, ctx.needs_input_grad[2:5], mod_shape, mdtype)
        shaped = lambda t, s: None if t is None else t.view(s)  # noqa: E731
        return (dx.view(x.shape), shaped(dy, x.shape), shaped(dgate, mshape), shaped(dshift, mshape),
                shaped(dscale, mshape), None, None)


def _apply(x, y, gate, shift, scale, eps, scale_offset):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, gate, shift, scale)):
        return _AdaLN.apply(x, y, gate, shift, scale, float(eps), scale_offset)
    xv, yv, gv, shv, scv, _ = _prepare(x, y, gate, shift, scale)
    z, h, _, _ = K.adaln_forward(xv, yv, gv, shv, scv, float(eps), scale_offset, False)
    return (h.view(x.shape),) if z is None else (z.view(x.shape), h.view(x.shape))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis."""
    return _apply(x, None, None, bias, weight, eps, 0.0)[0]


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor | None,
                         eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * (1 + scale) + shift`` over the last axis."""
    return _apply(x, None, None, shift, scale, eps, 1.0)[0]


def gated_residual_layer_norm(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor | None,
                              shift: torch.Tensor | None, scale: torch.Tensor | None,
                              eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``(z, modulated_layer_norm(z, shift, scale))`` with ``z = x + gate * y`` (``gate`` None:
    ``x + y``), ``y`` of x's shape and type."""
    return _apply(x, y, gate, shift, scale, eps, 1.0)
