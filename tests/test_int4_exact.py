"""The 4-bit product where its sums are exact: rows of small integers and scales that are
powers of two give sums that fp32 holds without a rounding, so that results are
compared bit for bit and one wrong scale, zero code or column is an error.  On the
CPU, the plans that spread the product over a GPU are enumerated and walked."""

import os
import subprocess

import pytest
import torch

import sparsepr_b200 as spr
from sparsepr_b200 import Int4Weight

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
HERE = os.path.dirname(os.path.abspath(__file__))


def test_plans_give_out_all_work_and_keep_scales_until_read(tmp_path):
    walk = str(tmp_path / "walk")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(HERE, "..", "sparsepr_b200", "csrc"),
                    os.path.join(HERE, "int4_plan_walk.cpp"), "-o", walk], check=True)
    out = subprocess.run([walk], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.endswith(" 0 wrong\n"), out.stdout


def _integers(dev, rows, n, k, group, dtype, sdt, zeros, seed):
    """Rows and gradients in -1, 0, 1 (and rows of 2), scales 1/2 and 1: the sums' absolute
    values, in units of 1/2, stay below 2^24 for the sizes here (asserted)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-k // group)
    packed = torch.randint(0, 256, (n, groups * group // 2), device=dev, generator=g).to(torch.uint8)
    scales = (0.5 * torch.randint(1, 3, (n, groups), device=dev, generator=g)).to(sdt)
    z = torch.randint(0, 16, (n, groups), device=dev, generator=g).to(torch.uint8) if zeros else None
    x = torch.randint(-2, 3, (rows, k), device=dev, generator=g).to(dtype)
    dy = torch.randint(-1, 2, (rows, n), device=dev, generator=g).to(dtype)
    return Int4Weight(packed, scales, z), x, dy


def _dense(w, k):
    n, groups = w.scales.shape
    codes = torch.stack((w.packed & 15, w.packed >> 4), -1).view(n, groups, -1).double()
    codes -= 8.0 if w.zeros is None else w.zeros.double()[..., None]
    return codes.mul_(w.scales.double()[..., None]).view(n, -1)[:, :k]


def _check_exact(dev, rows, n, k, group, dtype, sdt, zeros):
    w, x, dy = _integers(dev, rows, n, k, group, dtype, sdt, zeros, seed=n + k)
    dense = _dense(w, k)
    x64, d64 = x.double(), dy.double()
    assert 2 * max((x64.abs() @ dense.abs().t()).max().item(), (d64.abs() @ dense.abs()).max().item()) < 2 ** 24
    x.requires_grad_()
    y = spr.int4_linear(x, *w)
    dx, = torch.autograd.grad(y, x, dy)
    same = torch.equal(y, (x64 @ dense.t()).to(dtype)), torch.equal(dx, (d64 @ dense).to(dtype))
    assert same == (True, True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,dtype,sdt,zeros", [
    (1, 30720, 3328, BF, FP, True),    # thirteen chunks of 256 columns: a last slice of one
    (4, 19968, 4352, BF, BF, True),
    (3, 19968, 7424, BF, BF, False),
    (23, 32636, 3328, BF, BF, True),
    (2, 30720, 4352, HF, FP, True),
    (8, 61440, 7424, BF, BF, True),
    (1, 15360, 13824, FP, FP, True),   # fifty-four: a rest of two
    (5, 15360, 3584, HF, HF, True),
    (2, 15360, 3840, FP, BF, False),   # fifteen: a rest of three
])
def test_groups_of_32_in_several_slices(cuda, rows, n, k, dtype, sdt, zeros):
    _check_exact(cuda, rows, n, k, 32, dtype, sdt, zeros)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [100, -100])
@pytest.mark.parametrize("rows,dtype", [(1, BF), (8, BF), (9, BF), (2, FP)])
def test_large_scales_and_small_rows_and_the_other_way_round(cuda, rows, dtype, power):
    """Scales 2^100 larger and rows (or gradients) 2^100 smaller leave the results as they are."""
    w, x, dy = _integers(cuda, rows, 500, 640, 64, dtype, FP, True, seed=rows)
    dense = _dense(w, 640)
    scaled = Int4Weight(w.packed, w.scales * 2.0 ** power, w.zeros)
    x = (x * 2.0 ** -power).requires_grad_()
    y = spr.int4_linear(x, *scaled)
    dx, = torch.autograd.grad(y, x, dy * 2.0 ** -power)
    same = (torch.equal(y, ((x.detach().double() * 2.0 ** power) @ dense.t()).to(dtype)),
            torch.equal(dx, (dy.double() @ dense).to(dtype)))
    assert same == (True, True)


@pytest.mark.gpu
@pytest.mark.parametrize("k,group,dtype", [(72, 64, BF), (64, 32, FP)])
def test_more_rows_than_a_launch_takes(cuda, k, group, dtype):
    _check_exact(cuda, 65535 + 65535 + 41, 40, k, group, dtype, FP, True)


def test_scales_that_ask_for_a_gradient_are_refused():
    w = spr.quantize_int4(torch.randn(8, 64), 32)
    scales = w.scales.requires_grad_()
    for x in (torch.zeros(1, 64), torch.zeros(1, 64, requires_grad=True)):
        with pytest.raises(RuntimeError, match="frozen"):
            spr.int4_linear(x, w.packed, scales, w.zeros)
        with torch.no_grad(), pytest.raises(RuntimeError, match="need CUDA tensors"):
            spr.int4_linear(x, w.packed, scales, w.zeros)
    with pytest.raises(RuntimeError, match="need CUDA tensors"):
        spr.int4_linear(x, w.packed, scales.detach(), w.zeros)


@pytest.mark.parametrize("std", [1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("dtype", [HF, FP])
@pytest.mark.parametrize("symmetric", [False, True])
def test_small_weights_keep_their_codes_under_fp16_scales(std, dtype, symmetric):
    """Steps below fp16's normal numbers are rounded up to the next multiple of 2^-24: codes are off by half a
    step, or a whole one where a zero code was rounded too."""
    w = (torch.randn(16, 256, generator=torch.Generator().manual_seed(4)) * std).to(dtype)
    q = spr.quantize_int4(w, 64, symmetric=symmetric, scale_dtype=HF)
    groups = w.double().view(16, 4, 64)
    if symmetric:
        step = groups.abs().amax(-1) / 7
    else:
        step = (groups.amax(-1).clamp(min=0) - groups.amin(-1).clamp(max=0)) / 15
    assert (step < 2.0 ** -14).all()
    assert (q.scales.double() >= step * (1 - 2.0 ** -22)).all() and (q.scales.double() <= step + 2.0 ** -24).all()
    err = (spr.dequantize_int4(*q, 256).double() - w.double()).abs().view(16, 4, 64)
    assert (err <= (0.5 if symmetric else 1.0) * (1 + 2.0 ** -20) * q.scales.double()[..., None]).all()


def test_weights_without_a_scale_are_refused():
    for bad in (float("inf"), float("nan")):
        w = torch.ones(2, 64)
        w[1, 5] = bad
        with pytest.raises(RuntimeError, match="not finite"):
            spr.quantize_int4(w, 32)
    with pytest.raises(RuntimeError, match="too large"):
        spr.quantize_int4(torch.full((2, 64), 1e6), 32, scale_dtype=HF)
    spr.quantize_int4(torch.full((2, 64), 1e6), 32, scale_dtype=BF)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,group,dtype,sdt,zeros", [
    (1, 5120, 256, 32, BF, BF, False),
    (2, 17, 130, 64, BF, FP, True),
    (3, 7777, 4999, 64, FP, FP, False),
    (1, 20000, 5120, 64, BF, BF, True),
    (2, 40000, 5120, 128, BF, BF, True),
    (4, 30720, 5120, 64, HF, HF, True),
    (7, 250, 2049, 96, HF, FP, True),
    (8, 3333, 4800, 160, BF, HF, True),
    (2, 3, 16000, 128, FP, FP, True),
    (6, 12001, 96, 96, BF, BF, False),
    (1, 64, 30000, 16384, BF, FP, True),
    (9, 3000, 2560, 256, FP, BF, True),
    (16, 5000, 4096, 64, HF, HF, False),
    (17, 2600, 10000, 512, BF, BF, True),
    (33, 960, 3200, 64, FP, FP, True),
])
def test_exact_sums(cuda, rows, n, k, group, dtype, sdt, zeros):
    _check_exact(cuda, rows, n, k, group, dtype, sdt, zeros)
