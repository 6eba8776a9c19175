"""The DiT with one kind of block alone."""

import torch

from sparsepr_b200.hunyuan_dit import HunyuanDiT, HunyuanDiTConfig, JointAttention


def _run(model, cfg):
    g = torch.Generator().manual_seed(11)
    latent, text, pooled = (torch.randn(s, generator=g) for s in ((16, 2, 4, 8), (6, cfg.text_dim), (cfg.vec_dim,)))

    def inner(_i, q, k, v, _n):
        return torch.softmax(q @ k.transpose(-1, -2) / q.shape[-1] ** 0.5, dim=-1) @ v

    return model.forward(latent, text, torch.tensor(500.0), pooled, torch.tensor(6.0), JointAttention(inner))


def _config(double, single):
    return HunyuanDiTConfig(hidden=64, heads=4, head_dim=16, double_blocks=double, single_blocks=single, text_dim=32,
                            vec_dim=24, rope_axes=(4, 6, 6))


def test_without_single_blocks_the_last_text_branch_is_not_computed():
    """The output layer takes the video tokens: the text stream ends with the last attention."""
    cfg = _config(2, 0)
    model = HunyuanDiT(cfg, "cpu", dtype=torch.float32, seed=1)
    out = _run(model, cfg)
    assert out.shape == (2 * 2 * 4, 64) and torch.isfinite(out).all()
    for key in ("proj", "fc1", "fc2"):
        model.double[1]["txt"][key] = None
    assert torch.equal(_run(model, cfg), out)
    assert not torch.equal(_run(HunyuanDiT(cfg, "cpu", dtype=torch.float32, seed=2), cfg), out)


def test_without_double_blocks():
    cfg = _config(0, 2)
    out = _run(HunyuanDiT(cfg, "cpu", dtype=torch.float32, seed=1), cfg)
    assert out.shape == (2 * 2 * 4, 64) and torch.isfinite(out).all()


def test_streams_and_norms_are_released_when_used(monkeypatch):
    """At an attention call no layer's input or output from before the block's Q/K/V is alive but the streams."""
    import gc
    import weakref

    cfg = _config(2, 1)
    model = HunyuanDiT(cfg, "cpu", dtype=torch.float32, seed=1)
    embedded, normed, alive = [], [], []
    lin = HunyuanDiT._lin

    def record(x, layer):
        out = lin(x, layer)
        if layer is model.patch_in or layer is model.txt_in:
            embedded.append(weakref.ref(out))
        if any(layer is blk[s]["qkv"] for blk in model.double for s in ("img", "txt")):
            normed.append(weakref.ref(x))
        return out

    monkeypatch.setattr(HunyuanDiT, "_lin", staticmethod(record))
    dense = JointAttention(lambda _i, q, k, v, _n: v)

    def attention(i, *qkv):
        gc.collect()
        alive.append((sum(r() is not None for r in embedded), sum(r() is not None for r in normed)))
        return dense(i, *qkv)

    g = torch.Generator().manual_seed(11)
    latent, text, pooled = (torch.randn(s, generator=g) for s in ((16, 2, 4, 8), (6, cfg.text_dim), (cfg.vec_dim,)))
    with torch.no_grad():
        model.forward(latent, text, torch.tensor(500.0), pooled, torch.tensor(6.0), attention)
    assert alive == [(2, 0), (0, 0), (0, 0)]
