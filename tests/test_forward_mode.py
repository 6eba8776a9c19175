"""Forward-mode derivatives through the adaLN passes and the 4-bit linear: not formed, so a
dual tensor in any differentiable place raises instead of losing its tangent."""

import pytest
import torch
from torch.autograd import forward_ad

import sparsepr_b200 as spr

CALLS = {
    "norm": (lambda x, w, b: spr.layer_norm(x, w, b), ((4, 64), (64,), (64,))),
    "modulated": (lambda x, s, c: spr.modulated_layer_norm(x, s, c), ((4, 64), (64,), (64,))),
    "gated": (spr.gated_residual_layer_norm, ((4, 64), (4, 64), (64,), (64,), (64,))),
    "int4": (lambda x, s, b: spr.int4_linear(x, torch.zeros(8, 32, dtype=torch.uint8, device=x.device), s, None, b),
             ((4, 64), (8, 2), (8,))),
}


@pytest.mark.parametrize("name,which", [(n, i) for n, (_f, shapes) in CALLS.items() for i in range(len(shapes))])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_dual_operands_are_refused(name, which, mode):
    f, shapes = CALLS[name]
    args = [torch.ones(s) for s in shapes]
    with mode(), forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones(shapes[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(*args)
        args[which] = forward_ad.unpack_dual(args[which]).primal
        with pytest.raises(RuntimeError, match="need CUDA tensors"):  # without a tangent: as ever
            f(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CALLS))
def test_dual_gradients_are_refused(cuda, name):
    f, shapes = CALLS[name]
    args = [torch.ones(s, device=cuda) for s in shapes]
    args[0].requires_grad_()
    y = f(*args)
    y = y[1] if name == "gated" else y
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, args[0], dy, retain_graph=True)
        torch.autograd.grad(y, args[0], torch.ones_like(y))
