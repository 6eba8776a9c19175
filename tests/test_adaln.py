"""The adaptive layer norms: argument checks on the CPU, values and gradients on
the GPU against the formulas in 64 bits.

Tolerances: u = finfo(T).eps / 2 is the relative error of the one rounding to the
result's type; the fp32 arithmetic before it is bounded by K rounding steps of
2^-24 on the sum of the absolute values that enter the result (an input's
offset from zero enters with |x| + |mean|); a sum over R rows adds at most one
step per term."""

import pytest
import torch

import sparsepr_b200 as spr
from sparsepr_b200.adaln import _split, operands

EPS32 = 2.0 ** -24
K_STEPS = 32


# ---------------------------------------------------------------- CPU: checks


def test_split_of_the_leading_axes():
    assert _split((2, 5, 8), (8,), "scale") == (1, 10, False, False)
    assert _split((2, 5, 8), (2, 1, 8), "scale") == (2, 5, True, False)
    assert _split((2, 5, 8), (1, 5, 8), "scale") == (2, 5, False, True)
    assert _split((2, 5, 8), (2, 5, 8), "scale") == (1, 10, False, True)
    assert _split((2, 3, 5, 8), (2, 3, 1, 8), "scale") == (6, 5, True, False)
    assert _split((2, 3, 5, 8), (2, 1, 1, 8), "scale") == (2, 15, True, False)
    assert _split((1, 5, 8), (1, 1, 8), "scale") == (1, 5, False, False)
    assert _split((8,), (8,), "scale") == (1, 1, False, False)
    with pytest.raises(RuntimeError, match="adjacent"):
        _split((2, 3, 5, 8), (2, 1, 5, 8), "scale")
    for bad in ((7,), (3, 1, 8), (1, 1, 2, 5, 8), ()):
        with pytest.raises(RuntimeError, match="does not match"):
            _split((2, 5, 8), bad, "scale")


def test_cpu_tensors_are_refused():
    x, v = torch.zeros(2, 8), torch.zeros(8)
    for call in (lambda: spr.layer_norm(x, v, v), lambda: spr.modulated_layer_norm(x, v, v),
                 lambda: spr.gated_residual_layer_norm(x, x, v, v, v)):
        with pytest.raises(RuntimeError, match="need CUDA tensors"):
            call()


def test_c_entries_refuse_before_any_launch():
    import ctypes

    from sparsepr_b200 import _lib, build

    build.build()

    def op(**kw):
        o = _lib.SprAdaln(dtype=1, mod_dtype=1, batch=1, tokens=4, channels=8, eps=1e-6, scale_offset=1.0, x=256, h=256)
        for k, v in kw.items():
            setattr(o, k, v)
        return o

    def fwd(o):
        _lib.call("spr_adaln_forward", ctypes.addressof(o), None)

    for kw, msg in ((dict(channels=0), "SPR_ERR_SHAPE"), (dict(channels=16385), "SPR_ERR_SHAPE"),
                    (dict(batch=1 << 20, tokens=1 << 20), "SPR_ERR_SHAPE"), (dict(dtype=7), "SPR_ERR_DTYPE"),
                    (dict(mod_dtype=2), "SPR_ERR_DTYPE"), (dict(gate=256), "SPR_ERR_ARG"), (dict(x=None), "SPR_ERR_ARG"),
                    (dict(y=256), "SPR_ERR_ARG")):
        with pytest.raises(RuntimeError, match=msg):
            fwd(op(**kw))
    with pytest.raises(RuntimeError, match="SPR_ERR_ARG"):
        _lib.call("spr_adaln_forward", None, None)
    fwd(op(tokens=0))  # nothing to do, nothing launched
    gr = _lib.SprAdalnGrad(dh=256, dx=256, dshift=256)
    o = op(tokens=4096, mean=256, rstd=256)
    with pytest.raises(RuntimeError, match="SPR_ERR_WORKSPACE"):
        _lib.call("spr_adaln_backward", ctypes.addressof(o), ctypes.addressof(gr), None, 0, None)
    with pytest.raises(RuntimeError, match="SPR_ERR_ARG"):
        o = op()  # no statistics
        _lib.call("spr_adaln_backward", ctypes.addressof(o), ctypes.addressof(gr), 256, 1 << 20, None)
    for kw in (dict(scale=256, scale_st=8), dict(y=256, gate=256, gate_st=8), dict(batch=2, scale=256, scale_sb=8)):
        gr = _lib.SprAdalnGrad(dh=256, dx=256, dy=256, dscale=256)  # the strides say that the vectors differ
        o = op(mean=256, rstd=256, **kw)
        with pytest.raises(RuntimeError, match="summed over"):
            _lib.call("spr_adaln_backward", ctypes.addressof(o), ctypes.addressof(gr), 256, 1 << 30, None)


# ---------------------------------------------------------------- 64-bit reference


def _half_step(t):
    return torch.finfo(t.dtype).eps / 2


def _close(got, ref, amp, steps=K_STEPS, what=""):
    """|got - ref| <= u|ref| + steps * 2^-24 * amp (+ half the least subnormal of the type)."""
    got64 = got.detach().double()
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    tol = _half_step(got) * ref.abs() + steps * EPS32 * amp + tiny
    bad = (got64 - ref).abs() > tol
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert not bad.any(), (what, int(bad.sum()), (got64 - ref).abs().max().item(), (tol.max()).item())


def _to_vec(t, shape):
    """Sum t [B,N,C] down to a vector's shape."""
    full = (1,) * (t.dim() - len(shape)) + tuple(shape)
    axes = [i for i in range(t.dim() - 1) if full[i] == 1 and t.shape[i] != 1]
    return (t.sum(axes, keepdim=True) if axes else t).reshape(shape)


def _reference(x, shift, scale, offset, eps, y=None, gate=None, dh=None, dz=None):
    out, amp = {}, {}
    one = torch.ones((), dtype=torch.float64, device=x.device)
    if y is not None:
        # The product and the sum rounded to fp32 in turn, then to the stored type.
        out["z"] = ((x.float() + (y.float() if gate is None else gate.float() * y.float())).to(x.dtype)).double()
        z = out["z"]
    else:
        z = x.double()
    w = one if scale is None else scale.double() + offset
    b = 0.0 * one if shift is None else shift.double()
    mean = z.mean(-1, keepdim=True)
    rstd = ((z - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    n = (z - mean) * rstd
    spread = (z.abs() + mean.abs() + z.abs().mean(-1, keepdim=True)) * rstd + n.abs()
    out["h"], amp["h"] = n * w + b, spread * w.abs() + b.abs()
    if dh is None:
        return out, amp
    d = dh.double()
    u = d * w
    m0, m1 = u.mean(-1, keepdim=True), (u * n).mean(-1, keepdim=True)
    g = rstd * (u - m0 - n * m1)
    ua = u.abs()
    ga = rstd * (ua + ua.mean(-1, keepdim=True) + spread * (ua * spread).mean(-1, keepdim=True))
    if dz is not None:
        g = g + dz.double()
        ga = ga + dz.double().abs()
    out["dx"], amp["dx"] = g, ga
    if y is not None:
        gt = one if gate is None else gate.double()
        out["dy"], amp["dy"] = g * gt, ga * gt.abs()
        if gate is not None:
            out["dgate"], amp["dgate"] = _to_vec(g * y.double(), gate.shape), _to_vec(ga * y.double().abs(), gate.shape)
    if shift is not None:
        out["dshift"], amp["dshift"] = _to_vec(d, shift.shape), _to_vec(d.abs(), shift.shape)
    if scale is not None:
        out["dscale"], amp["dscale"] = _to_vec(d * n, scale.shape), _to_vec(d.abs() * spread, scale.shape)
    return out, amp


def _inputs(dev, b, n, c, dtype, mod_dtype, mods, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = {"vector": (c,), "sample": (b, 1, c), "token": (b, n, c), "shared": (1, n, c)}[mods]

    def randn(*s, t=dtype, std=1.0, mean=0.0):
        return (torch.randn(*s, device=dev, generator=g) * std + mean).to(t)

    x = (torch.randn(b, n, c, device=dev, generator=g) * torch.randn(c, device=dev, generator=g).exp() + 0.7).to(dtype)
    return dict(x=x, y=randn(b, n, c), gate=randn(*shape, t=mod_dtype, std=0.4),
                shift=randn(*shape, t=mod_dtype, std=0.3), scale=randn(*shape, t=mod_dtype, std=0.3),
                dh=randn(b, n, c, std=0.1), dz=randn(b, n, c, std=0.1))


def _check(v, gated, offset=1.0, eps=1e-6):
    """Forward, backward and the inference form of one call against the reference."""
    leaves = {k: v[k].detach().requires_grad_() for k in ("x", "y", "gate", "shift", "scale")}
    x, y, gate, shift, scale = (leaves[k] for k in ("x", "y", "gate", "shift", "scale"))
    rows = x.numel() // x.shape[-1]
    if gated:
        z, h = spr.gated_residual_layer_norm(x, y, gate, shift, scale, eps=eps)
        names = ("x", "y", "gate", "shift", "scale")
        grads = torch.autograd.grad((z, h), [leaves[k] for k in names], (v["dz"], v["dh"]))
        with torch.no_grad():
            z2, h2 = spr.gated_residual_layer_norm(x, y, gate, shift, scale, eps=eps)
        ref, amp = _reference(x, shift, scale, 1.0, eps, y, gate, v["dh"], v["dz"])
        assert torch.equal(z.double(), ref["z"]) and torch.equal(z, z2)
    else:
        def call():
            return (spr.modulated_layer_norm(x, shift, scale, eps=eps) if offset else
                    spr.layer_norm(x, scale, shift, eps=eps))
        h = call()
        names = ("x", "shift", "scale")
        grads = torch.autograd.grad(h, [leaves[k] for k in names], v["dh"])
        with torch.no_grad():
            h2 = call()
        ref, amp = _reference(x, shift, scale, offset, eps, dh=v["dh"])
    assert torch.equal(h, h2)
    assert h.dtype == x.dtype
    _close(h, ref["h"], amp["h"], what="h")
    for name, got in zip(names, grads):
        assert got.dtype == leaves[name].dtype and got.shape == leaves[name].shape
        steps = K_STEPS + (rows if name in ("gate", "shift", "scale") else 0)
        _close(got, ref["d" + name], amp["d" + name], steps, "d" + name)
    return grads


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("b,n,c,dtype,mod_dtype,mods", [
    (1, 1, 1, FP, FP, "vector"),            # one value: n = 0
    (1, 1, 5120, BF, BF, "vector"),
    (2, 3, 8, BF, FP, "sample"),
    (1, 7, 130, HF, HF, "token"),
    (2, 5, 33, FP, FP, "shared"),
    (3, 37, 129, HF, FP, "sample"),
    (1, 300, 512, BF, BF, "vector"),
    (2, 67, 1000, BF, FP, "vector"),
    (1, 130, 1003, FP, FP, "vector"),
    (2, 19, 1536, BF, BF, "token"),
    (2, 200, 2048, HF, HF, "sample"),
    (1, 700, 5120, BF, FP, "vector"),
    (3, 11, 4097, BF, BF, "sample"),
    (1, 9, 8192, FP, FP, "vector"),
    (1, 50, 256, FP, FP, "vector"),
    (2, 40, 132, FP, FP, "sample"),
    (1, 90, 508, FP, FP, "vector"),
    (1, 40, 384, FP, FP, "vector"),
    (1, 60, 272, BF, FP, "vector"),
    (2, 33, 6144, BF, BF, "sample"),
    (1, 20, 5128, FP, FP, "vector"),
    (1, 77, 8192, HF, FP, "vector"),
    (3, 41, 8200, BF, BF, "vector"),
    (1, 70, 1536, BF, BF, "token"),
    (2, 60, 1536, BF, FP, "token"),
    (3, 50, 328, HF, HF, "token"),
    (1, 90, 256, FP, FP, "token"),
    (2, 37, 5120, BF, FP, "token"),
    (1, 40, 4104, HF, HF, "token"),
    (3, 33, 640, BF, FP, "shared"),
    (2, 30, 5120, FP, FP, "token"),
    (1, 25, 5200, BF, BF, "token"),
    (1, 5, 16384, BF, BF, "vector"),
    (1, 3, 16383, FP, FP, "sample"),
    (2, 4, 16384, FP, FP, "shared"),
])
def test_values_and_gradients(cuda, gated, b, n, c, dtype, mod_dtype, mods):
    _check(_inputs(cuda, b, n, c, dtype, mod_dtype, mods, seed=c + n), gated)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("b,n,c,dtype,mod_dtype,mods,pad", [
    (1, 70, 1537, BF, BF, "vector", 0),
    (1, 2000, 1537, BF, FP, "vector", 0),  # several runs of rows
    (2, 40, 1003, FP, FP, "sample", 0),
    (1, 33, 65, HF, HF, "token", 0),
    (2, 20, 4099, BF, FP, "token", 0),     # three slots of gated rows; the gradient's do not fit
    (1, 30, 8191, HF, HF, "vector", 0),
    (3, 17, 2049, FP, FP, "token", 0),
    (1, 24, 5001, FP, FP, "vector", 0),
    (3, 21, 777, BF, BF, "shared", 0),
    (2, 45, 512, BF, BF, "vector", 1),     # rows of whole vectors at odd addresses and strides
    (3, 19, 1024, FP, FP, "sample", 3),
    (2, 23, 640, HF, FP, "token", 5),
])
def test_rows_that_no_vectors_fit(cuda, gated, b, n, c, dtype, mod_dtype, mods, pad):
    v = _inputs(cuda, b, n, c, dtype, mod_dtype, mods, seed=c + n)
    for name in ("x", "y") if pad else ():
        wide = v[name].new_full((b, n, c + pad), float("nan"))
        wide[..., pad:] = v[name]
        v[name] = wide[..., pad:]
    _check(v, gated)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_affine_layer_norm(cuda, dtype):
    v = _inputs(cuda, 1, 77, 1003, dtype, FP, "vector", seed=5)
    _check(v, False, offset=0.0, eps=1e-5)


@pytest.mark.gpu
def test_many_rows_of_few_channels_and_long_sums(cuda):
    """70,001 rows: more than the grid of any persistent launch, sums of many terms."""
    _check(_inputs(cuda, 1, 70001, 64, BF, FP, "vector", seed=3), True)
    _check(_inputs(cuda, 7, 10001, 24, FP, FP, "sample", seed=4), False)


@pytest.mark.gpu
def test_optional_operands(cuda):
    v = _inputs(cuda, 2, 31, 96, BF, FP, "sample", seed=9)
    x, y = v["x"].detach().requires_grad_(), v["y"].detach().requires_grad_()
    h = spr.layer_norm(x)
    ref, amp = _reference(x, None, None, 0.0, 1e-6, dh=v["dh"])
    _close(h, ref["h"], amp["h"])
    _close(torch.autograd.grad(h, x, v["dh"])[0], ref["dx"], amp["dx"])
    h = spr.modulated_layer_norm(x, v["shift"], None)
    _close(h, *(d["h"] for d in _reference(x, v["shift"], None, 1.0, 1e-6)))
    h = spr.modulated_layer_norm(x, None, v["scale"])
    _close(h, *(d["h"] for d in _reference(x, None, v["scale"], 1.0, 1e-6)))
    # No gate, no modulation; one of the two results used alone.
    z, h = spr.gated_residual_layer_norm(x, y, None, None, None)
    ref, amp = _reference(x, None, None, 1.0, 1e-6, y, None, v["dh"], None)
    assert torch.equal(z.double(), ref["z"])
    dx, dy = torch.autograd.grad(h, (x, y), v["dh"], retain_graph=True)
    _close(dx, ref["dx"], amp["dx"])
    _close(dy, ref["dy"], amp["dy"])
    dx, dy = torch.autograd.grad(z, (x, y), v["dz"])
    assert torch.equal(dx, v["dz"]) and torch.equal(dy, v["dz"])
    # Only a vector asks for a gradient.
    scale = v["scale"].detach().requires_grad_()
    ref, amp = _reference(x.detach(), v["shift"], scale, 1.0, 1e-6, dh=v["dh"])
    g, = torch.autograd.grad(spr.modulated_layer_norm(x.detach(), v["shift"], scale), scale, v["dh"])
    _close(g, ref["dscale"], amp["dscale"], K_STEPS + 62)


@pytest.mark.gpu
def test_strides_offsets_and_expanded_gradients(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    b, n, c = 2, 21, 256
    wide = torch.randn(b, n + 5, 3 * c + 8, device=cuda, generator=g).to(BF)
    mods = torch.randn(b, 6 * c, device=cuda, generator=g).to(BF) * 0.3
    shift, scale, gate = (t.unsqueeze(1) for t in mods.chunk(6, dim=1)[:3])  # rows of stride 6c
    for lo in (0, 8, 1):  # 1: no 16-byte alignment
        x, y = wide[:, 2:2 + n, lo:lo + c], wide[:, :n, lo + c:lo + 2 * c]
        v = dict(x=x, y=y, gate=gate, shift=shift, scale=scale,
                 dh=torch.randn(b, n, c, device=cuda, generator=g).to(BF),
                 dz=torch.randn(1, n, 1, device=cuda, generator=g).to(BF).expand(b, n, c))
        _check(v, True)
        v.update(shift=shift[0, 0], scale=scale[0, 0], gate=gate[0, 0])  # one vector, strided rows
        _check(v, False)
    # A vector for every token, each kind a part of one wider tensor, rows with gaps.
    wide_mods = torch.randn(b, n, 3 * c, device=cuda, generator=g).to(BF) * 0.3
    for batch in (slice(0, b), slice(0, 1)):
        v = dict(x=wide[batch, 2:2 + n, 8:8 + c], y=wide[batch, :n, 8 + c:8 + 2 * c],
                 dh=torch.randn(b, n, c, device=cuda, generator=g).to(BF)[batch],
                 dz=torch.randn(b, n, c, device=cuda, generator=g).to(BF)[batch])
        v.update(zip(("gate", "shift", "scale"), wide_mods[batch].chunk(3, dim=-1)))
        _check(v, True)
        _check(v, False)
    # A transposed leading order: [n, b, c] seen as [b, n, c], each sample with its vector.
    x = torch.randn(n, b, c, device=cuda, generator=g).to(BF).transpose(0, 1)
    _check(dict(x=x, y=x * 0.5, gate=gate, shift=shift, scale=scale, dh=x.contiguous(), dz=x), True)


@pytest.mark.gpu
def test_row_offsets_past_32_bits(cuda):
    """Rows of one [3, 2, 64] view lie more than 2^31 elements apart."""
    base = torch.zeros(2 ** 32 + 4096, dtype=BF, device=cuda)
    x = base.as_strided((3, 2, 64), (2 ** 31 + 16, 128, 1))
    v = _inputs(cuda, 3, 2, 64, BF, BF, "sample", seed=1)
    x.copy_(v["x"])
    v["x"] = x
    _check(v, True)
    _check(v, False)


@pytest.mark.gpu
def test_constant_rows_large_offsets_and_bad_values(cuda):
    v = _inputs(cuda, 1, 6, 320, FP, FP, "vector", seed=8)
    x = v["x"].clone()
    x[0, 0] = 3.0                       # variance 0: n = 0
    x[0, 1] = x[0, 1] * 1e-3 + 1000.0   # offset far above the spread: the variance is taken about the mean
    x[0, 2] = x[0, 2] * 1e15
    v["x"] = x
    _check(v, False)
    h = spr.modulated_layer_norm(x, v["shift"], v["scale"])
    assert torch.equal(h[0, 0], v["shift"])
    bad = x.clone()
    bad[0, 3, 7] = float("inf")
    bad[0, 4, 9] = float("nan")
    got = spr.modulated_layer_norm(bad, v["shift"], v["scale"])
    assert got[0, 3:5].isnan().all()
    assert torch.equal(got[0, :3], h[0, :3]) and torch.equal(got[0, 5], h[0, 5])


@pytest.mark.gpu
def test_empty_rows(cuda):
    x = torch.zeros(2, 0, 16, device=cuda, requires_grad=True)
    w = torch.ones(16, device=cuda, requires_grad=True)
    h = spr.layer_norm(x, w, w)
    assert h.shape == x.shape
    dx, dw = torch.autograd.grad(h, (x, w), torch.zeros_like(h))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
    z, h = spr.gated_residual_layer_norm(x, x * 2, w, w, w)
    dx, dw = torch.autograd.grad((z, h), (x, w), (torch.zeros_like(h),) * 2)
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """The directional derivative against a central difference in fp32 (step 2^-6: its
    curvature error is of order step^2 and its rounding error 2^-24 |L| / step)."""
    v = _inputs(cuda, 2, 3, 40, FP, FP, "sample", seed=12)
    leaves = {k: v[k].detach().requires_grad_() for k in ("x", "y", "gate", "shift", "scale")}

    def loss(p):
        z, h = spr.gated_residual_layer_norm(p["x"], p["y"], p["gate"], p["shift"], p["scale"])
        return (z.double() * v["dz"].double()).sum() + (h.double() * v["dh"].double()).sum()

    grads = torch.autograd.grad(loss(leaves), list(leaves.values()))
    g = torch.Generator(device=cuda).manual_seed(1)
    step = 2.0 ** -6
    for (name, t), grad in zip(leaves.items(), grads):
        d = torch.randn(t.shape, device=cuda, generator=g) / t.numel() ** 0.5
        with torch.no_grad():
            hi, lo = ({**leaves, name: t + s * step * d} for s in (1, -1))
            diff = ((loss(hi) - loss(lo)) / (2 * step)).item()
        want = (grad.double() * d.double()).sum().item()
        assert abs(diff - want) <= 2e-3 * (grad.double().norm() * d.double().norm()).item(), (name, diff, want)


@pytest.mark.gpu
def test_second_derivatives_are_refused_and_graphs_kept(cuda):
    x = torch.randn(3, 40, device=cuda, requires_grad=True)
    h = spr.layer_norm(x)
    first, = torch.autograd.grad(h, x, torch.ones_like(h), retain_graph=True)
    again, = torch.autograd.grad(h, x, torch.ones_like(h), retain_graph=True)  # the saved operands stay
    assert torch.equal(first, again)
    g, = torch.autograd.grad(h.square().sum(), x, create_graph=True)  # asking for a graph is no error by itself
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.gpu
def test_saved_operands_may_be_moved(cuda):
    """Hooks that keep saved tensors elsewhere give back other memory."""
    v = _inputs(cuda, 1, 50, 256, BF, FP, "vector", seed=4)
    leaves = [v[k].detach().requires_grad_() for k in ("x", "y", "gate", "shift", "scale")]

    def grads():
        z, h = spr.gated_residual_layer_norm(*leaves)
        return torch.autograd.grad((z, h), leaves, (v["dz"], v["dh"]))

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    z, h = spr.gated_residual_layer_norm(*leaves)
    with torch.no_grad():
        z += 1.0  # the saved stream is the result itself
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, leaves[0], v["dh"])


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_saved_operands_may_come_back_in_another_layout(cuda, gated):
    """Such hooks give back dense copies of strided operands."""
    g = torch.Generator(device=cuda).manual_seed(12)
    wide = torch.randn(3, 40, 2 * 64, device=cuda, generator=g)
    x, y = wide[..., :64].requires_grad_(), wide.transpose(0, 1).contiguous().transpose(0, 1)[..., 64:].requires_grad_()
    gate, shift, scale = (t.requires_grad_() for t in torch.randn(3, 1, 3 * 64, device=cuda, generator=g).chunk(3, -1))
    dh = torch.randn(3, 40, 64, device=cuda, generator=g)

    def grads():
        if gated:
            z, h = spr.gated_residual_layer_norm(x, y, gate, shift, scale)
            return torch.autograd.grad((z, h), (x, y, gate, shift, scale), (dh, dh))
        return torch.autograd.grad(spr.modulated_layer_norm(x, shift, scale), (x, shift, scale), dh)

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals(cuda):
    x, v = torch.zeros(2, 4, 16, device=cuda), torch.zeros(16, device=cuda)
    with pytest.raises(RuntimeError, match="fp32/bf16/fp16"):
        spr.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="must be torch.bfloat16 or fp32"):
        spr.layer_norm(x.bfloat16(), v.half())
    with pytest.raises(RuntimeError, match="must be as"):
        spr.modulated_layer_norm(x, v, v.view(1, 1, 16))
    with pytest.raises(RuntimeError, match="does not match"):
        spr.modulated_layer_norm(x, v[:8], v[:8])
    with pytest.raises(RuntimeError, match="y must be"):
        spr.gated_residual_layer_norm(x, x[:1], v, v, v)
    with pytest.raises(RuntimeError, match="channels must be contiguous"):
        spr.layer_norm(x.transpose(1, 2))
    with pytest.raises(RuntimeError, match="1 to 16384"):
        spr.layer_norm(torch.zeros(1, 16385, device=cuda))
    with pytest.raises(RuntimeError, match="is on cpu"):
        spr.layer_norm(x, v.cpu())
    with pytest.raises(RuntimeError, match="contiguous"):
        spr.layer_norm(torch.zeros(4, 3, 2, 16, device=cuda).permute(2, 0, 1, 3)[:, ::2], v.expand(2, 2, 3, 16))


@pytest.mark.gpu
def test_repeatable_and_on_other_streams(cuda):
    v = _inputs(cuda, 1, 5000, 1280, BF, FP, "vector", seed=6)
    first = _check(v, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = _check(v, True)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_captured_graphs_replayed_together(cuda):
    """Each captured backward pass has its own scratch: two graphs replayed on two streams give what each gives alone."""
    from sparsepr_b200 import kernels as K

    runs = []
    for seed in (1, 2):
        v = _inputs(cuda, 1, 3000, 1280, BF, FP, "vector", seed=seed)
        op, vectors = operands(v["x"], v["y"], v["gate"], v["shift"], v["scale"])

        def step(op=op, v=v):
            z, h, stats = K.adaln_forward(op, 1e-6, True)
            return (z, h, *K.adaln_backward(op._replace(x=z), stats, v["dh"], v["dz"], mod_shape=vectors))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        runs.append((g, got, want, torch.cuda.Stream(), v))  # a graph reads its inputs where they were
    for _ in range(5):
        for g, got, _w, s, _in in runs:
            with torch.cuda.stream(s):
                for t in got:
                    t.zero_()
                g.replay()
    torch.cuda.synchronize()
    for _g, got, want, _s, _in in runs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_autograd_step(cuda):
    """Forward and backward pass captured as a training step captures them: warmed up on a side
    stream, no eager graph of the leaves left alive."""
    v = _inputs(cuda, 1, 1000, 640, BF, FP, "vector", seed=9)
    leaves = [v[k].detach().requires_grad_() for k in ("x", "y", "gate", "shift", "scale")]

    def step():
        z, h = spr.gated_residual_layer_norm(*leaves)
        return torch.autograd.grad((z, h), leaves, (v["dz"], v["dh"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_results_do_not_depend_on_the_calls_before(cuda):
    """The order of a vector gradient's sum is that of a fresh process, whatever other passes over CTAs
    of the same size ran first."""
    import subprocess
    import sys

    script = """
import sys, torch, sparsepr_b200 as spr
g = torch.Generator(device="cuda").manual_seed(3)
def run(c, gated, n, dtype):
    x, y, dh = torch.randn(3, 1, n, c, device="cuda", generator=g).to(dtype)
    v = [torch.randn(c, device="cuda", generator=g).to(dtype).requires_grad_() for _ in range(3)]
    if gated:
        z, h = spr.gated_residual_layer_norm(x, y, *v)
        return torch.autograd.grad((z, h), v, (dh, dh))
    return torch.autograd.grad(spr.modulated_layer_norm(x, *v[:2]), v[:2], dh)
state = g.get_state()
if len(sys.argv) > 1:
    for dtype in (torch.float32, torch.float16):
        for c in (640, 1280, 2560):
            run(c, True, 4096, dtype), run(c, False, 4096, dtype), run(c + 8, True, 4096, dtype)
g.set_state(state)
for c in (1280, 2560):
    for gated in (False, True):
        for t in run(c, gated, 20000, torch.bfloat16):
            print(t.double().sum().item(), t.double().square().sum().item())
"""
    out = [subprocess.run([sys.executable, "-c", script, *args], capture_output=True, text=True, timeout=300)
           for args in ((), ("first",))]
    assert out[0].returncode == 0, out[0].stderr
    assert out[0].stdout and out[0].stdout == out[1].stdout
