"""Sums over many rows in the gradients of the adaLN vectors, against 64 bits closely enough
that one run of rows left out, or taken twice, is an error.

The data add up instead of cancelling: every column has a mean of its own in z, and dh, dz
and y have one, so a gradient grows with the rows and its fp32 error stays relative to it.
A column's sum is a chain of a run's rows, then every 32nd run and five joins: fewer than
2,048 roundings of 2^-24 for the sizes here; the terms carry some 64 more.  A run is at
least one 2,368th of the rows (16 runs an SM of 148), so leaving one out moves the sum by
4.2e-4, 3.3 times the bound.  That is asserted on the reference."""

import pytest
import torch

import sparsepr_b200 as spr

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
BOUND = (2048 + 64) * 2.0 ** -24
RUNS = 2368


def _data(dev, b, n, c, dtype):
    g = torch.Generator(device=dev).manual_seed(n + c)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g)

    sign = torch.where(randn(c) < 0, -1.0, 1.0)
    x = (3 * sign + 0.25 * randn(b, n, c)).to(dtype)
    y, dh, dz = ((1 + 0.25 * randn(b, n, c)).to(dtype) for _ in range(3))
    return x, y, dh, dz


def _vectors(dev, b, c, sample, dtype):
    g = torch.Generator(device=dev).manual_seed(c)
    shape = (b, 1, c) if sample else (c,)
    return [(0.1 * torch.randn(shape, device=dev, generator=g)).to(dtype).requires_grad_() for _ in range(3)]


def _reference(z, y, dh, dz, gate, scale, gated):
    """Per-row terms of (dgate, dshift, dscale) in 64 bits."""
    z = z.double()
    mean = z.mean(-1, keepdim=True)
    rstd = ((z - mean).square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    norm = (z - mean) * rstd
    d = dh.double()
    terms = [d, d * norm]
    if gated:
        u = d * (1 + scale.double())
        g = dz.double() + rstd * (u - u.mean(-1, keepdim=True) - norm * (u * norm).mean(-1, keepdim=True))
        terms.insert(0, g * y.double())
    return terms


def _close(got, ref):
    """In norm, beside the one rounding to the gradient's type."""
    return (got.double() - ref).norm() <= (BOUND + torch.finfo(got.dtype).eps / 2) * ref.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("b,n,c,dtype,sample", [
    (1, 70001, 64, BF, False),     # several teams to a CTA
    (7, 10001, 24, FP, True),
    (1, 40000, 264, HF, False),
    (1, 20000, 1280, BF, False),   # the streaming kernels, several runs an SM
    (2, 9001, 2048, FP, True),
    (1, 12000, 5120, BF, False),
    (3, 4001, 5128, HF, True),
    (1, 30000, 1537, BF, False),   # rows that no vectors fit
    (2, 9000, 1003, FP, True),
    (1, 50001, 131, HF, False),
    (1, 3001, 12288, BF, False),   # the widest rows
    (1, 2500, 8193, FP, False),
])
def test_no_run_of_rows_is_lost(cuda, gated, b, n, c, dtype, sample):
    x, y, dh, dz = _data(cuda, b, n, c, dtype)
    gate, shift, scale = _vectors(cuda, b, c, sample, FP)
    if gated:
        z, h = spr.gated_residual_layer_norm(x, y, gate, shift, scale)
        grads = torch.autograd.grad((z, h), (gate, shift, scale), (dz, dh))
    else:
        z, h = x, spr.modulated_layer_norm(x, shift, scale)
        grads = torch.autograd.grad(h, (shift, scale), dh)
    for got, terms in zip(grads, _reference(z.detach(), y, dh, dz, gate.detach(), scale.detach(), gated)):
        terms = terms if sample else terms.flatten(0, 1)[None]
        ref = terms.sum(1)
        got = got.detach().reshape(ref.shape)
        lost = -(-terms.shape[1] // RUNS)
        for i in range(ref.shape[0]):  # each sample's vector by itself
            assert _close(got[i], ref[i])
            assert not _close((ref[i] - terms[i, :lost].sum(0)).float(), ref[i])


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("b,n,c,dtype,sample", [
    (1, 70001, 64, BF, False), (2, 20000, 1536, HF, False), (1, 30000, 1537, BF, False), (3, 7001, 5120, FP, True),
    (1, 3001, 12288, BF, False),
])
def test_sums_of_integers_are_exact(cuda, gated, b, n, c, dtype, sample):
    """dshift is the sum of dh, which small integers make exact in fp32 in any order."""
    x, y, _dh, dz = _data(cuda, b, n, c, dtype)
    g = torch.Generator(device=cuda).manual_seed(1)
    dh = torch.randint(-8, 9, (b, n, c), device=cuda, generator=g).to(dtype)
    gate, shift, scale = _vectors(cuda, b, c, sample, FP)
    if gated:
        z, h = spr.gated_residual_layer_norm(x, y, gate, shift, scale)
    else:
        h = spr.modulated_layer_norm(x, shift, scale)
    got, = torch.autograd.grad(h, shift, dh)
    want = dh.double().sum(1, keepdim=True) if sample else dh.double().sum((0, 1))
    assert torch.equal(got.double(), want)
