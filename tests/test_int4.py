"""4-bit weights: quantisation and argument checks on the CPU, the product and its
gradient on the GPU against the formula in 64 bits.

Tolerances: u = finfo(T).eps / 2 for the one rounding to the result's type, and
the fp32 sums before it bounded by S rounding steps of 2^-23 (a tensor-core sum
may cut off instead of rounding) on the sum of the absolute values of the terms,
S = 64 + the longest chain of additions."""

import pytest
import torch

import sparsepr_b200 as spr
from sparsepr_b200 import Int4Weight, dequantize_int4, quantize_int4

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("n,k,group,symmetric", [(5, 64, 32, False), (3, 100, 64, True), (7, 129, 128, False)])
def test_quantised_weight_is_the_nearest_code(dtype, n, k, group, symmetric):
    g = torch.Generator().manual_seed(k)
    w = (torch.randn(n, k, generator=g) * 0.1 + 0.03).to(dtype)
    q = quantize_int4(w, group, symmetric=symmetric)
    groups = -(-k // group)
    assert q.packed.shape == (n, groups * group // 2) and q.packed.dtype == torch.uint8
    assert q.scales.shape == (n, groups) and q.scales.dtype == dtype and (q.zeros is None) == symmetric
    back = dequantize_int4(*q, k)
    step = q.scales.float().repeat_interleave(group, dim=1)[:, :k]
    # Half a step by rounding; the end codes may lie past the range by what the stored scale was
    # rounded (8 codes from zero at most 15 steps) and the zero code by half a step.
    slack = 0.5 + 15 * torch.finfo(dtype).eps + (0.0 if symmetric else 0.5)
    assert ((back - w.float()).abs() <= slack * step + 1e-7).all()


def test_quantise_constant_and_zero_groups():
    w = torch.zeros(2, 64)
    w[1] = 0.75
    for symmetric in (False, True):
        back = dequantize_int4(*quantize_int4(w, 32, symmetric=symmetric), 64)
        torch.testing.assert_close(back, w, rtol=1e-6, atol=0.0)


def test_code_order():
    """Column k sits in byte k // 2, the even column in the low half."""
    w = torch.zeros(1, 32)
    w[0, :4] = torch.tensor([-7.0, 7.0, 1.0, -1.0])
    q = quantize_int4(w, 32, symmetric=True)
    assert q.packed[0, :3].tolist() == [1 | (15 << 4), 9 | (7 << 4), 8 | (8 << 4)]


def test_cpu_refusals():
    w = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="group_size"):
        quantize_int4(w, 48)
    with pytest.raises(ValueError, match="scale_dtype"):
        quantize_int4(w, 32, scale_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="non-empty"):
        quantize_int4(w[:0], 32)
    with pytest.raises(RuntimeError, match="need CUDA tensors"):
        spr.int4_linear(torch.zeros(1, 64), *quantize_int4(w, 32))


def test_c_entries_refuse_before_any_launch():
    from sparsepr_b200 import _lib, build

    build.build()

    def call(rows=1, n=8, k=64, group=32, dtype=1, sdt=1, packed=256, x=256, stride=64):
        _lib.call("spr_int4_linear", x, stride, dtype, rows, n, k, group, packed, 256, sdt, None, None, 256, None, 0,
                  None)

    def grad(rows=1, n=8, k=64, group=32, dtype=1, sdt=1, packed=256, dx=256, stride=8):
        _lib.call("spr_int4_linear_grad", 256, stride, dtype, rows, n, k, group, packed, 256, sdt, None, dx, None, 0,
                  None)

    for f in (call, grad):
        for kw, msg in ((dict(k=0), "SHAPE"), (dict(rows=-1), "SHAPE"), (dict(group=48), "SHAPE"),
                        (dict(group=0), "SHAPE"), (dict(dtype=5), "DTYPE"), (dict(sdt=-1), "DTYPE"),
                        (dict(packed=264), "ALIGN"), (dict(packed=None), "ARG"), (dict(rows=2, stride=1), "SHAPE")):
            with pytest.raises(RuntimeError, match="SPR_ERR_" + msg):
                f(**kw)
        f(rows=0)  # nothing to do, nothing launched
    call(n=0)


def _weights(dev, n, k, group, sdt, zeros, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, groups * group), device=dev, generator=g).to(torch.uint8)
    scales = (torch.rand(n, groups, device=dev, generator=g) * 0.05 - 0.01).to(sdt)
    z = torch.randint(0, 16, (n, groups), device=dev, generator=g).to(torch.uint8) if zeros else None
    return Int4Weight(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, z)


def _dense64(w, k):
    n, groups = w.scales.shape
    codes = torch.stack((w.packed & 15, w.packed >> 4), -1).view(n, groups, -1).double()
    z = 8.0 if w.zeros is None else w.zeros.double()[..., None]
    return ((codes - z) * w.scales.double()[..., None]).view(n, -1)[:, :k]


def _close(got, ref, terms, chain, what=""):
    u = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    tol = u * ref.abs() + (64 + chain) * 2.0 ** -23 * terms + tiny
    err = (got.detach().double() - ref).abs()
    assert got.shape == ref.shape and not (err > tol).any(), (what, err.max().item(), tol.max().item())


def _check(x, w, bias, dy):
    x = x.detach().requires_grad_()
    bias = None if bias is None else bias.detach().requires_grad_()
    k = x.shape[-1]
    dense = _dense64(w, k)
    y = spr.int4_linear(x, *w, bias)
    with torch.no_grad():
        assert torch.equal(y, spr.int4_linear(x, *w, bias))
    ref = x.detach().double() @ dense.t()
    terms = x.detach().double().abs() @ dense.abs().t()
    if bias is not None:
        ref, terms = ref + bias.detach().double(), terms + bias.detach().double().abs()
    _close(y, ref, terms, k, "y")
    grads = torch.autograd.grad(y, [x] + ([] if bias is None else [bias]), dy)
    d = dy.double()
    _close(grads[0], d @ dense, d.abs() @ dense.abs(), dense.shape[0], "dx")
    if bias is not None:
        lead = list(range(d.dim() - 1))
        _close(grads[1], d.sum(lead), d.abs().sum(lead), d.numel() // d.shape[-1], "dbias")
    return y, grads


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,group,dtype,sdt,zeros,bias", [
    (1, 1, 1, 32, FP, FP, True, True),
    (1, 16, 32, 32, BF, BF, False, False),
    (1, 5120, 256, 32, BF, BF, False, True),
    (2, 17, 130, 64, BF, FP, True, True),
    (3, 777, 999, 64, FP, FP, False, False),
    (4, 1000, 5120, 128, BF, BF, True, True),
    (5, 100, 5120, 256, HF, HF, True, False),
    (7, 250, 2049, 96, HF, FP, True, True),
    (8, 33, 640, 160, BF, HF, True, True),
    (9, 3000, 384, 32, FP, BF, True, True),
    (16, 129, 4096, 64, HF, HF, False, True),
    (17, 260, 1000, 512, BF, BF, True, False),
    (33, 96, 320, 64, FP, FP, True, True),
    (70, 40, 72, 64, BF, BF, True, True),
    (2, 3, 16000, 128, FP, FP, True, False),
    (6, 12001, 96, 96, BF, BF, False, False),
    (1, 64, 30000, 16384, BF, FP, True, True),
])
def test_product_and_gradient(cuda, rows, n, k, group, dtype, sdt, zeros, bias):
    g = torch.Generator(device=cuda).manual_seed(n)
    w = _weights(cuda, n, k, group, sdt, zeros, seed=rows)
    x = torch.randn(rows, k, device=cuda, generator=g).to(dtype)
    b = torch.randn(n, device=cuda, generator=g).to(dtype) if bias else None
    _check(x, w, b, torch.randn(rows, n, device=cuda, generator=g).to(dtype))


@pytest.mark.gpu
def test_leading_axes_strides_and_weight_slices(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    w = _weights(cuda, 100, 200, 64, BF, True)
    wide = torch.randn(2, 3, 417, device=cuda, generator=g).to(BF)
    x, dy = wide[..., 11:211], torch.randn(2, 3, 100, device=cuda, generator=g).to(BF)
    y, _ = _check(x, w, None, dy)
    assert y.shape == (2, 3, 100)
    _check(wide[0, 0, 1:201], w, None, dy[0, 0])                         # one vector, odd offset
    _check(x[0, :1].expand(3, 200), w, None, dy[0])                      # rows of stride 0
    _check(x, w, None, dy[:1, :1].expand(2, 3, 100))                     # an expanded gradient
    _check(x[0].t().contiguous().t(), w, None, dy[0])                    # columns contiguous: copied
    part = Int4Weight(w.packed[13:57], w.scales[13:57], w.zeros[13:57])  # rows of a larger weight
    y13, _ = _check(x, part, None, dy[..., 13:57])
    assert torch.equal(y13, y[..., 13:57])


@pytest.mark.gpu
def test_unused_codes_are_ignored_and_bad_values_stay_in_their_row(cuda):
    w = _weights(cuda, 70, 100, 64, FP, True)
    x = torch.randn(3, 100, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    y = spr.int4_linear(x, *w)
    other = w.packed.clone()
    other[:, 50:] ^= 0xA5  # columns 100..127
    assert torch.equal(spr.int4_linear(x, other, w.scales, w.zeros), y)
    bad = x.clone()
    bad[0, 3], bad[2, 50] = float("inf"), float("nan")
    got = spr.int4_linear(bad, *w)
    ref = bad.double() @ _dense64(w, 100).t()
    assert torch.equal(got[1], y[1]) and got[2].isnan().all()
    assert torch.equal(got[0].isnan(), ref[0].isnan()) and torch.equal(got[0].isinf(), ref[0].isinf())
    big = torch.full((1, 100), 3.4e38, device=cuda)  # near fp32's largest value: no part of it overflows
    one = Int4Weight(torch.full_like(w.packed, 0x99), torch.full_like(w.scales, 2.0 ** -10), None)
    torch.testing.assert_close(spr.int4_linear(big, *one).double(), torch.full((1, 70), 3.4e38 * 100 / 1024,
                               device=cuda, dtype=torch.float64), rtol=1e-5, atol=0.0)
    sub = torch.full((1, 100), 2.0 ** -24, device=cuda, dtype=HF)  # fp16's least subnormal value
    one = Int4Weight(one.packed, torch.ones_like(w.scales), None)
    assert torch.equal(spr.int4_linear(sub, *one), torch.full((1, 70), 100 * 2.0 ** -24, device=cuda, dtype=HF))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows", [1, 8])
def test_values_far_below_the_largest_of_their_row(cuda, dtype, rows):
    """Where the codes opposite a row's largest value are zero, the small values keep their bits."""
    n, k = 100, 640
    w = _weights(cuda, n, k, 64, FP, False)
    w.packed[:, 50] = w.packed[:, 50] & 0xF0 | 8  # column 100
    x = torch.randn(rows, k, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)) * 2.0 ** -6
    x = x.to(dtype)
    x[:, 100] = 2.0 ** 12
    dense = _dense64(w, k)
    ref = x.double() @ dense.t()
    terms = x.double().abs() @ dense.abs().t()  # the largest value's are 0
    err = (spr.int4_linear(x, *w).double() - ref).abs()
    # One rounding, the fp32 sums, and each small value within half of 2^(12 - 29).
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + (64 + k) * 2.0 ** -23 * terms + 2.0 ** -18 * dense.abs().sum(1)
    assert not (err > tol).any(), (err / tol).max().item()


@pytest.mark.gpu
def test_empty_rows_and_outputs(cuda):
    w = _weights(cuda, 8, 64, 32, FP, False)
    x = torch.zeros(0, 64, device=cuda, requires_grad=True)
    b = torch.zeros(8, device=cuda, requires_grad=True)
    y = spr.int4_linear(x, *w, b)
    assert y.shape == (0, 8)
    dx, db = torch.autograd.grad(y, (x, b), torch.zeros_like(y))
    assert dx.shape == (0, 64) and torch.equal(db, torch.zeros_like(b))
    none = Int4Weight(w.packed[:0], w.scales[:0], None)
    x = torch.ones(2, 64, device=cuda, requires_grad=True)
    y = spr.int4_linear(x, *none)
    assert y.shape == (2, 0)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.zeros_like(x))


@pytest.mark.gpu
def test_weight_offsets_past_32_bits(cuda):
    """A weight of more than 2^32 codes: the last rows equal the same rows as a weight of their own."""
    n, k, group = 270_000, 16384, 128
    g = torch.Generator(device=cuda).manual_seed(7)
    packed = torch.randint(0, 256, (n, k // 2), device=cuda, generator=g, dtype=torch.uint8)
    scales = torch.rand(n, k // group, device=cuda, generator=g).to(BF)
    x = torch.randn(2, k, device=cuda, generator=g).to(BF)
    y = spr.int4_linear(x, packed, scales)
    tail = slice(n - 300, n)
    w = Int4Weight(packed[tail].clone(), scales[tail].clone(), None)
    dense = _dense64(w, k)
    _close(y[:, tail], x.double() @ dense.t(), x.double().abs() @ dense.abs().t(), k)
    dy = torch.zeros(1, n, device=cuda, dtype=BF)
    dy[:, tail] = 1.0
    from sparsepr_b200 import kernels as K

    dx = K.int4_linear_grad(dy, packed, scales, None, k)
    d = dy[:, tail].double()
    _close(dx, d @ dense, d.abs() @ dense.abs(), 300)


@pytest.mark.gpu
def test_refusals(cuda):
    w = _weights(cuda, 8, 64, 32, FP, True)
    x = torch.zeros(2, 64, device=cuda)
    for args, msg in (
            ((x.double(), *w), "fp32/bf16/fp16"),
            ((x, w.packed.int(), w.scales, w.zeros), "uint8"),
            ((x, w.packed, w.scales[:4], w.zeros), "uint8 \\[N, K/2\\]"),
            ((x[:, :32], *w), "input features"),
            ((torch.zeros(2, 65, device=cuda), *w), "input features"),
            ((x, w.packed[:, :24].contiguous(), w.scales, w.zeros), "multiple of 32"),
            ((x, w.packed, w.scales, w.zeros.int()), "zeros must be uint8"),
            ((x, w.packed, w.scales, w.zeros[:, :1]), "zeros must be uint8"),
            ((x, w.packed, w.scales.t().contiguous().t(), w.zeros), "contiguous"),
            ((x, *w, torch.zeros(8, device=cuda, dtype=BF)), "bias must be"),
            ((x, *w, torch.zeros(9, device=cuda)), "bias must be"),
            ((x, w.packed.cpu(), w.scales, w.zeros), "CUDA tensors")):
        with pytest.raises(RuntimeError, match=msg):
            spr.int4_linear(*args)


@pytest.mark.gpu
def test_repeatable_and_on_other_streams(cuda):
    w = _weights(cuda, 4000, 2560, 64, BF, True)
    g = torch.Generator(device=cuda).manual_seed(3)
    x, dy = torch.randn(3, 2560, device=cuda, generator=g).to(BF), torch.randn(3, 4000, device=cuda, generator=g).to(BF)
    first = _check(x, w, None, dy)
    runs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            runs.append(_check(x, w, None, dy))
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for y, grads in runs:
        assert torch.equal(y, first[0]) and torch.equal(grads[0], first[1][0])


@pytest.mark.gpu
def test_captured_graph(cuda):
    from sparsepr_b200 import kernels as K

    w = _weights(cuda, 1000, 2560, 64, BF, True)
    g = torch.Generator(device=cuda).manual_seed(3)
    x, dy = torch.randn(2, 2560, device=cuda, generator=g).to(BF), torch.randn(2, 1000, device=cuda, generator=g).to(BF)
    want = K.int4_linear(x, *w), K.int4_linear_grad(dy, *w, 2560)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.int4_linear(x, *w), K.int4_linear_grad(dy, *w, 2560)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
