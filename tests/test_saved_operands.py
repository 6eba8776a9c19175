"""Saved-tensor hooks (offloading, compression, checkpoints) under the adaLN passes and
the 4-bit linear: gradients are the same whatever layout the hooks give back, and another
shape, type or device is refused before a kernel reads it."""

import pytest
import torch

import sparsepr_b200 as spr
from sparsepr_b200 import kernels as K

BF, FP = torch.bfloat16, torch.float32


def _turned(t):
    """The same values with the axes' memory order reversed."""
    axes = tuple(reversed(range(t.dim())))
    return t.permute(axes).contiguous().permute(axes)


def _norm(dev, gated):
    g = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn(3, 40, 2 * 96, device=dev, generator=g)
    x, y = wide[..., :96].requires_grad_(), wide[..., 96:].requires_grad_()
    gate, shift, scale = (t.requires_grad_() for t in torch.randn(3, 1, 3 * 96, device=dev, generator=g).chunk(3, -1))
    dh = torch.randn(3, 40, 96, device=dev, generator=g)

    def grads():
        if gated:
            z, h = spr.gated_residual_layer_norm(x, y, gate, shift, scale)
            return torch.autograd.grad((z, h), (x, y, gate, shift, scale), (dh, dh))
        return torch.autograd.grad(spr.modulated_layer_norm(x, shift, scale), (x, shift, scale), dh)

    return grads


def _int4(dev):
    g = torch.Generator(device=dev).manual_seed(6)
    w = spr.quantize_int4(torch.randn(200, 300, device=dev, generator=g).to(BF), 32)
    x = torch.randn(5, 300, device=dev, generator=g).to(BF).requires_grad_()
    dy = torch.randn(5, 200, device=dev, generator=g).to(BF)
    return lambda: torch.autograd.grad(spr.int4_linear(x, *w), x, dy)


def test_checks_of_a_saved_operand():
    t = torch.arange(12.0).view(3, 4)
    assert K.check_saved(_turned(t), FP, 12, -1) is not None
    assert K.dense_saved(t, FP, 12, -1) is t
    back = K.dense_saved(_turned(t), FP, 12, -1)
    assert back.is_contiguous() and torch.equal(back, t)
    for other, index in ((t.double(), -1), (t[:2], -1), (t.view(torch.int32), -1), (t, 0)):
        for f in (K.check_saved, K.dense_saved):
            with pytest.raises(RuntimeError, match="came back as"):
                f(other, FP, 12, index)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["norm", "gated", "int4"])
def test_any_layout_may_come_back(cuda, what):
    grads = _int4(cuda) if what == "int4" else _norm(cuda, what == "gated")
    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _turned):
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["norm", "gated", "int4"])
@pytest.mark.parametrize("change", [lambda t: t.half(), lambda t: t[:1], lambda t: t.cpu()])
def test_other_shapes_types_and_devices_are_refused(cuda, what, change):
    grads = _int4(cuda) if what == "int4" else _norm(cuda, what == "gated")
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        with pytest.raises(RuntimeError, match="came back as"):
            grads()
