"""Cases of the adaLN operators of a diffusion transformer: the modulated layer
norm and the gated residual in front of it, forward and backward, and the
product of a few conditioning vectors with 4-bit weights that makes the
modulation.  Hidden widths are heads x head_dim of 128-wide heads (40 and 12
heads) and odd ones; token counts are those of the 480p and 720p video layers,
text prompts and single vectors."""

import math

import torch

own = False  # False: the plain forms in elementary torch operations; True: the framework's operators

EPS = 1e-6
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # The first norm of a block over all video tokens of a 720p clip (21 x 45 x 80), one modulation vector.
        dict(name="norm_video", kind="norm", batch=1, tokens=75600, channels=5120, dtype="bf16", mods="vector", mod_dtype="bf16"),
        # One conditioning token: latency.
        dict(name="norm_one_token", kind="norm", batch=1, tokens=1, channels=5120, dtype="bf16", mods="vector", mod_dtype="bf16"),
        # A plain affine norm of a short prompt at an odd width, in fp32.
        dict(name="norm_prompt_affine", kind="norm", batch=1, tokens=77, channels=1003, dtype="fp32", mods="affine", mod_dtype="fp32"),
        # Fine-tuning on two 480p clips (21 x 30 x 52), modulation per clip kept in fp32.
        dict(name="norm_train_clips", kind="norm_train", batch=2, tokens=32760, channels=5120, dtype="bf16", mods="sample", mod_dtype="fp32"),
        # Training on short odd sequences at an odd width.
        dict(name="norm_train_odd", kind="norm_train", batch=3, tokens=333, channels=1537, dtype="fp16", mods="sample", mod_dtype="fp16"),
        # The end of an attention branch and the norm before the MLP over a 720p clip, fp32 modulation.
        dict(name="gated_video", kind="gated", batch=1, tokens=75600, channels=5120, dtype="bf16", mods="vector", mod_dtype="fp32"),
        # Image-to-video: every token has a timestep of its own, so a modulation of its own.
        dict(name="gated_per_token", kind="gated", batch=1, tokens=4095, channels=1536, dtype="bf16", mods="token", mod_dtype="bf16"),
        # Fine-tuning on one 480p clip.
        dict(name="gated_train_clip", kind="gated_train", batch=1, tokens=32760, channels=5120, dtype="bf16", mods="vector", mod_dtype="bf16"),
        # The timestep embedding's first layer: the smallest product, latency.
        dict(name="int4_timestep", kind="int4", rows=1, outs=5120, ins=256, group=32, dtype="bf16", scale_dtype="bf16", zeros=False, bias=True),
        # The modulations of eight blocks (six vectors each) for the two guidance branches, in one product.
        dict(name="int4_blocks", kind="int4", rows=2, outs=8 * 6 * 5120, ins=5120, group=128, dtype="bf16", scale_dtype="bf16", zeros=True, bias=True),
        # Ragged sizes in fp32: the last group of each row is only partly used.
        dict(name="int4_ragged_fp32", kind="int4", rows=3, outs=7777, ins=4999, group=64, dtype="fp32", scale_dtype="fp32", zeros=False, bias=False),
        # Fine-tuning through frozen 4-bit modulation weights of one block.
        dict(name="int4_train_block", kind="int4_train", rows=4, outs=6 * 5120, ins=5120, group=64, dtype="bf16", scale_dtype="bf16", zeros=True, bias=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "gated", "gated_train", "int4", "int4_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    limit = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
    if kind.startswith("int4"):
        group = rng.choice([32, 64, 128, 256])
        ins = _log_uniform(rng, 64, 16384)
        if rng.random() < 0.5:
            ins = max(group, ins // group * group)
        case = dict(kind=kind, rows=_log_uniform(rng, 1, 32), outs=_log_uniform(rng, 32, 250000), ins=ins, group=group,
                    dtype=dtype, scale_dtype=rng.choice([dtype, "fp32"]), zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
        size = "outs"
    else:
        channels = _log_uniform(rng, 64, 8192)
        if rng.random() < 0.7:
            channels = channels // 64 * 64
        batch = rng.choice([1, 1, 2, 3])
        mods = rng.choice(["vector", "sample", "token"] + ([] if kind.startswith("gated") else ["affine"]))
        case = dict(kind=kind, batch=batch, tokens=_log_uniform(rng, 1, 75600 // batch), channels=channels, dtype=dtype,
                    mods=mods, mod_dtype=rng.choice([dtype, "fp32"]))
        size = "tokens"
    while work(case)["bytes"] > limit:
        case[size] = case[size] * 2 // 3
    return case


# ---------------------------------------------------------------- inputs


def _mod_shape(case):
    b, n, c = case["batch"], case["tokens"], case["channels"]
    return {"vector": (c,), "affine": (c,), "sample": (b, 1, c), "token": (b, n, c)}[case["mods"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, dtype=dt, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).add_(mean).to(dtype)

    if case["kind"].startswith("int4"):
        m, n, k, gs = case["rows"], case["outs"], case["ins"], case["group"]
        groups = -(-k // gs)
        # Codes of a normally distributed weight row; two to a byte, the even column in the low half.
        codes = torch.randn(n, groups * gs, device="cuda", generator=g).mul_(2.5).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
        packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
        del codes
        sdt = _DTYPES[case["scale_dtype"]]
        scales = (torch.rand(n, groups, device="cuda", generator=g).mul_(0.4).add_(0.8) / (2.5 * math.sqrt(k))).to(sdt)
        zeros = torch.randint(6, 10, (n, groups), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
        x = torch.nn.functional.silu(randn(m, k, dtype=torch.float32)).to(dt)
        s = dict(case=case, x=x, packed=packed, scales=scales, zeros=zeros, bias=randn(n, std=0.1) if case["bias"] else None)
        if case["kind"] == "int4_train":
            s["dout"] = randn(m, n, std=0.02)
            x.requires_grad_()
            if s["bias"] is not None:
                s["bias"].requires_grad_()
        return s
    b, n, c = case["batch"], case["tokens"], case["channels"]
    mdt, ms = _DTYPES[case["mod_dtype"]], _mod_shape(case)
    # A residual stream: channels of different spread, offsets, and a few that stand out.
    spread = torch.randn(c, device="cuda", generator=g).mul_(0.5).exp_()
    spread[torch.randint(0, c, (max(1, c // 256),), device="cuda", generator=g)] *= 20.0
    x = torch.randn(b, n, c, device="cuda", generator=g)
    x = x.mul_(spread).add_(torch.randn(c, device="cuda", generator=g).mul_(0.3)).to(dt)
    s = dict(case=case, x=x, shift=randn(*ms, std=0.3, dtype=mdt),
             scale=randn(*ms, std=0.3, dtype=mdt, mean=1.0 if case["mods"] == "affine" else 0.0))
    grads = [s["x"], s["shift"], s["scale"]]
    if case["kind"].startswith("gated"):
        s["y"], s["gate"] = randn(b, n, c), randn(*ms, std=0.4, dtype=mdt)
        grads += [s["y"], s["gate"]]
    if case["kind"].endswith("train"):
        s["dh"] = randn(b, n, c, std=0.05)
        if case["kind"].startswith("gated"):
            s["dz"] = randn(b, n, c, std=0.05)
        for t in grads:
            t.requires_grad_()
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    with torch.no_grad():
        return _int4_plain(s) if kind.startswith("int4") else _norm_plain(s)


def _run_own(s, kind):
    import sparsepr_b200 as spr

    if kind.startswith("int4"):
        y = spr.int4_linear(s["x"], s["packed"], s["scales"], s["zeros"], s["bias"])
        if kind == "int4":
            return y
        leaves = [s["x"]] + ([s["bias"]] if s["bias"] is not None else [])
        grads = torch.autograd.grad(y, leaves, s["dout"])
        return dict(zip(("y", "dx", "dbias"), (y, *grads)))
    if kind.startswith("gated"):
        z, h = spr.gated_residual_layer_norm(s["x"], s["y"], s["gate"], s["shift"], s["scale"], eps=EPS)
        if kind == "gated":
            return dict(z=z, h=h)
        grads = torch.autograd.grad((z, h), (s["x"], s["y"], s["gate"], s["shift"], s["scale"]), (s["dz"], s["dh"]))
        return dict(zip(("z", "h", "dx", "dy", "dgate", "dshift", "dscale"), (z, h, *grads)))
    if s["case"]["mods"] == "affine":
        h = spr.layer_norm(s["x"], s["scale"], s["shift"], eps=EPS)
    else:
        h = spr.modulated_layer_norm(s["x"], s["shift"], s["scale"], eps=EPS)
    if kind == "norm":
        return h
    grads = torch.autograd.grad(h, (s["x"], s["shift"], s["scale"]), s["dh"])
    return dict(zip(("h", "dx", "dshift", "dscale"), (h, *grads)))


def _to_mod(t, mod):
    """Sum a per-element gradient over the axes that the modulation was broadcast along."""
    lead = tuple(range(t.dim() - mod.dim())) + tuple(i + t.dim() - mod.dim() for i, e in enumerate(mod.shape) if e == 1)
    return (t.sum(lead) if lead else t).reshape(mod.shape).to(mod.dtype)


def _norm_plain(s):
    case, dt = s["case"], s["x"].dtype
    x, shift, scale = s["x"].float(), s["shift"].float(), s["scale"].float()
    factor = scale if case["mods"] == "affine" else 1.0 + scale
    gated = case["kind"].startswith("gated")
    out = {}
    if gated:
        y, gate = s["y"].float(), s["gate"].float()
        out["z"] = (x + gate * y).to(dt)  # the residual stream as it is stored; the norm reads that
        x = out["z"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + EPS)
    normed = centred * rstd
    out["h"] = (normed * factor + shift).to(dt)
    if case["kind"] == "norm":
        return out["h"]
    if case["kind"] == "gated":
        return out
    dh = s["dh"].float()
    u = dh * factor
    dx = (u - u.mean(-1, keepdim=True) - normed * (u * normed).mean(-1, keepdim=True)) * rstd
    if gated:
        dx = dx + s["dz"].float()
        out["dy"], out["dgate"] = (dx * gate).to(dt), _to_mod(dx * y, s["gate"])
    out["dx"], out["dshift"], out["dscale"] = dx.to(dt), _to_mod(dh, s["shift"]), _to_mod(dh * normed, s["scale"])
    return out


def _int4_plain(s):
    case, x = s["case"], s["x"].float()
    n, groups = s["scales"].shape
    codes = torch.stack((s["packed"] & 15, s["packed"] >> 4), dim=-1).view(n, groups, case["group"])
    w = codes.float()
    del codes
    w.sub_(8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]).mul_(s["scales"].float()[:, :, None])
    w = w.view(n, -1)[:, :case["ins"]]
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = y.to(s["x"].dtype)
    if case["kind"] == "int4":
        return y
    dout = s["dout"].float()
    out = dict(y=y, dx=(dout @ w).to(s["x"].dtype))
    if s["bias"] is not None:
        out["dbias"] = dout.sum(0).to(s["bias"].dtype)
    return out


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = _BYTES[case["dtype"]]
    train = case["kind"].endswith("train")
    if case["kind"].startswith("int4"):
        m, n, k, groups = case["rows"], case["outs"], case["ins"], -(-case["ins"] // case["group"])
        nbytes = n * k // 2 + n * groups * (_BYTES[case["scale_dtype"]] + (1 if case["zeros"] else 0)) + e * (m * k + m * n)
        nbytes += e * n if case["bias"] else 0
        if train:  # dout in, dx and dbias out
            nbytes += e * (m * n + m * k) + (e * n if case["bias"] else 0)
        return dict(bytes=nbytes, flops=2 * m * n * k * (2 if train else 1))
    size, mod = case["batch"] * case["tokens"] * case["channels"], _BYTES[case["mod_dtype"]] * math.prod(_mod_shape(case))
    gated = case["kind"].startswith("gated")
    tensors = 4 if gated else 2  # x (y) in, (z) h out
    vectors = 3 if gated else 2
    flops = 10 if gated else 8
    if train:  # dh (dz) in, dx (dy) out, a gradient for each vector
        tensors, vectors, flops = 2 * tensors, 2 * vectors, 2 * flops + 6
    return dict(bytes=e * tensors * size + vectors * mod, flops=flops * size)


# ---------------------------------------------------------------- the same from the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return (_int4_exact if case["kind"].startswith("int4") else _norm_exact)(s)


def _norm_exact(s):
    case = s["case"]
    stream = s["x"].double()
    if case["kind"].startswith("gated"):
        z = torch.addcmul(stream, s["gate"].double(), s["y"].double())
        stream = z.to(s["x"].dtype).double()
    var, mean = torch.var_mean(stream, dim=-1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + EPS)
    normed = (stream - mean) / sigma
    w = s["scale"].double() + (0 if case["mods"] == "affine" else 1)
    h = torch.addcmul(s["shift"].double(), normed, w)
    if case["kind"] == "norm":
        return h
    if case["kind"] == "gated":
        return dict(z=z, h=h)
    dh, c = s["dh"].double(), case["channels"]
    p = dh * w
    # Jacobian of the norm: (I - 1/c 11^T - 1/c normed normed^T) / sigma.
    dx = (c * p - p.sum(-1, keepdim=True) - normed * torch.linalg.vecdot(p, normed)[..., None]) / (c * sigma)
    del p

    def reduced(t):
        shape = _mod_shape(case)
        return t.flatten(0, 1).sum(0) if len(shape) == 1 else t.sum(1, keepdim=True) if shape[1] == 1 and t.shape[1] != 1 else t

    out = dict(h=h, dshift=reduced(dh), dscale=reduced(dh * normed))
    if case["kind"] == "gated_train":
        dx += s["dz"].double()
        out.update(z=z, dy=dx * s["gate"].double(), dgate=reduced(dx * s["y"].double()))
    return dict(out, dx=dx)


def _int4_exact(s):
    case = s["case"]
    n, groups = s["scales"].shape
    x = torch.nn.functional.pad(s["x"].double(), (0, groups * case["group"] - case["ins"]))
    xe, xo = x[:, 0::2], x[:, 1::2]
    y = torch.empty(x.shape[0], n, device=x.device, dtype=torch.float64)
    dx = torch.zeros_like(x)
    rows = max(1, (1 << 27) // max(1, x.shape[1]))
    for a in range(0, n, rows):
        p, sc = s["packed"][a:a + rows], s["scales"][a:a + rows].double().repeat_interleave(case["group"] // 2, dim=1)
        zp = 8 if s["zeros"] is None else s["zeros"][a:a + rows].repeat_interleave(case["group"] // 2, dim=1).double()
        we, wo = (p.remainder(16).double() - zp) * sc, (p.div(16, rounding_mode="floor").double() - zp) * sc
        y[:, a:a + rows] = xe @ we.t() + xo @ wo.t()
        if case["kind"] == "int4_train":
            d = s["dout"][:, a:a + rows].double()
            dx[:, 0::2] += d @ we
            dx[:, 1::2] += d @ wo
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["kind"] == "int4":
        return y
    out = dict(y=y, dx=dx[:, :case["ins"]])
    if s["bias"] is not None:
        out["dbias"] = s["dout"].double().sum(0)
    return out
