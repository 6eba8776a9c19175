"""The plain and affine norms at the widths where the rows change hands between kernels,
against 64 bits: one rounding to the result's type (half a step), and 32 roundings of
2^-24 on what enters it before."""

import pytest
import torch

import sparsepr_b200 as spr

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("n", [300, 1000])
@pytest.mark.parametrize("c", [2048, 4096, 4352, 5120, 5632, 6144, 7168, 8184, 8192, 8200])
def test_norm_of_wide_rows(cuda, c, n, dtype):
    g = torch.Generator(device=cuda).manual_seed(c)
    x = (torch.randn(2, n, c, device=cuda, generator=g) * 2 + 0.5).to(dtype)
    shift, scale = (torch.randn(s, device=cuda, generator=g) for s in ((c,), (c,)))
    x64 = x.double()
    mean = x64.mean(-1, keepdim=True)
    rstd = ((x64 - mean).square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    norm, spread = (x64 - mean) * rstd, (x64.abs() + mean.abs() + x64.abs().mean(-1, keepdim=True)) * rstd
    for got, w in ((spr.modulated_layer_norm(x, shift, scale), 1 + scale.double()),
                   (spr.layer_norm(x, scale, shift), scale.double())):
        ref = norm * w + shift.double()
        amp = (spread + norm.abs()) * w.abs() + shift.double().abs()
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 32 * 2.0 ** -24 * amp + torch.finfo(dtype).tiny
        assert not ((got.double() - ref).abs() > tol).any()


@pytest.mark.gpu
def test_passes_without_autograd_and_without_a_branch(cuda):
    """The kernels' own backward call with its defaults: no gate, no gradient of one."""
    from sparsepr_b200 import kernels as K
    from sparsepr_b200.adaln import operands

    g = torch.Generator(device=cuda).manual_seed(2)
    x, dh = (torch.randn(2, 30, 256, device=cuda, generator=g) for _ in range(2))
    shift, scale = (torch.randn(256, device=cuda, generator=g).requires_grad_() for _ in range(2))
    op, mod_shape = operands(x, None, None, shift.detach(), scale.detach())
    _z, h, stats = K.adaln_forward(op, 1e-6, True)
    dx, dy, dgate, dshift, dscale = K.adaln_backward(op, stats, dh, mod_shape=mod_shape)
    assert dy is None and dgate is None
    leaf = x.clone().requires_grad_()
    want = spr.modulated_layer_norm(leaf, shift, scale)
    assert torch.equal(want, h)
    for a, b in zip((dx, dshift, dscale), torch.autograd.grad(want, (leaf, shift, scale), dh)):
        assert torch.equal(a.reshape(b.shape), b)
