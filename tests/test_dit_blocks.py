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
