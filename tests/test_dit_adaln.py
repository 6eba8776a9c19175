"""The DiT with its norms, modulations and gated residuals as fused passes and its
modulation weights in 4 bits, against the same model from separate operations.

Tolerances in fp32: a norm or residual differs by some eight rounding steps of 2^-24;
the dozen of them in the model pass through layers and a softmax whose gain is of
order one, which leaves 1e-4 of the largest output a wide margin; gradients pass
twice as many, and are compared at 1e-3 of their norm."""

import dataclasses

import pytest
import torch

from sparsepr_b200 import dequantize_int4
from sparsepr_b200.hunyuan_dit import HunyuanDiT, HunyuanDiTConfig, JointAttention

HEADS, PROMPT, TEXT = 2, 5, 7


def _config(**kw):
    return HunyuanDiTConfig(hidden=HEADS * 128, heads=HEADS, head_dim=128, double_blocks=2, single_blocks=2, text_dim=32,
                            vec_dim=24, modulation_group=64, **kw)


def _inputs(dev):
    g = torch.Generator().manual_seed(3)
    latent = torch.randn(16, 2, 6, 10, generator=g).to(dev)
    text = torch.randn(TEXT, 32, generator=g).to(dev)
    pooled = torch.randn(24, generator=g).to(dev)
    return latent, text, torch.tensor(700.0, device=dev), pooled, torch.tensor(6.0, device=dev)


def _attention():
    def inner(_i, q, k, v, _n):
        p = torch.softmax(q.float() @ k.float().transpose(-1, -2) / q.shape[-1] ** 0.5, dim=-1)
        return (p @ v.float()).to(q.dtype)

    return JointAttention(inner)


def _loss_and_gradients(model, dev):
    latent, text, t, pooled, guidance = _inputs(dev)
    latent.requires_grad_()
    pooled.requires_grad_()
    weights = [model.double[0]["img"]["qkv"][0], model.double[1]["txt"]["fc2"][1], model.single[0]["lin1"][0],
               model.final[0]]
    for w in weights:
        w.requires_grad_()
    out = model.forward(latent, text, t, pooled, guidance, _attention())
    r = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    return out.detach(), torch.autograd.grad((out * r).sum(), [latent, pooled, *weights])


def _dequantised(model):
    """The same model from separate operations, with the weights that the 4-bit codes stand for."""
    plain = HunyuanDiT(dataclasses.replace(model.cfg, fused_adaln=False, modulation_bits=16), model.device, model.dtype,
                       seed=0)
    weight, bias = model.mod4
    dense = dequantize_int4(*weight, model.cfg.hidden, dtype=model.dtype)
    at = 0
    for owner, key in plain._modulation_layers():
        n = owner[key][0].shape[0]
        owner[key] = (dense[at:at + n], bias[at:at + n])
        at += n
    assert at == dense.shape[0]
    return plain


def test_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        HunyuanDiT(_config(fused_adaln=True), "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        HunyuanDiT(_config(modulation_bits=4), "cpu")
    with pytest.raises(ValueError, match="modulation_bits"):
        _config(modulation_bits=8).validate()


@pytest.mark.gpu
@pytest.mark.parametrize("fused,bits", [(True, 16), (False, 4), (True, 4)])
def test_matches_separate_operations_with_gradients(cuda, fused, bits):
    model = HunyuanDiT(_config(fused_adaln=fused, modulation_bits=bits), cuda, torch.float32, seed=0)
    plain = _dequantised(model) if bits == 4 else HunyuanDiT(_config(), cuda, torch.float32, seed=0)
    out, grads = _loss_and_gradients(model, cuda)
    want, want_grads = _loss_and_gradients(plain, cuda)
    assert (out - want).abs().max() <= 1e-4 * want.abs().max()
    for got, ref in zip(grads, want_grads):
        assert (got - ref).norm() <= 1e-3 * ref.norm()


@pytest.mark.gpu
def test_16_bit_step_stays_as_close_to_fp32(cuda):
    """One rounding a pass instead of one an operation: no further from fp32 than the separate
    operations in bf16 (1.5 times, for the luck of a few hundred values)."""
    exact = HunyuanDiT(_config(), cuda, torch.bfloat16, seed=0)
    ref = HunyuanDiT(_config(), cuda, torch.float32, seed=0)
    for mine, theirs in zip(_tensors(ref), _tensors(exact)):
        mine.copy_(theirs)  # the bf16 weights
    fused = HunyuanDiT(_config(fused_adaln=True), cuda, torch.bfloat16, seed=0)
    with torch.no_grad():
        want, a, b = (m.forward(*_inputs(cuda), _attention()).double() for m in (ref, exact, fused))
    assert (b - want).norm() <= 1.5 * (a - want).norm()


def _tensors(model):
    def walk(v):
        if isinstance(v, torch.Tensor):
            yield v
        elif isinstance(v, (list, tuple)):
            for e in v:
                yield from walk(e)
        elif isinstance(v, dict):
            for e in v.values():
                yield from walk(e)

    for name in ("patch_in", "txt_in", "time_in", "guid_in", "vec_in", "double", "single", "final_mod", "final"):
        yield from walk(getattr(model, name))


@pytest.mark.gpu
def test_sparse_attention_step_with_4_bit_modulation(cuda):
    """The whole step: SparsePR in every block, fused passes, 4-bit modulation."""
    from sparsepr_b200 import N8V6Config
    from sparsepr_b200.hunyuan_dit import SparsePRBlocks

    cfg = _config(fused_adaln=True, modulation_bits=4)
    model = HunyuanDiT(cfg, cuda, seed=2)
    assert all(blk["mod"] is None for blk in model.single) and model.final_mod is None
    sp = N8V6Config(num_q_centroids=16, num_k_centroids=24, kmeans_iter_init=4, probe_rows=16, repair_rank=16,
                    selector_policy="svg_ear_value", role_kv_matmul_precision="highest", kmeans_tol=0.0)
    g = torch.Generator().manual_seed(11)
    latent = torch.randn(16, 4, 16, 32, generator=g).to(cuda)
    text = torch.randn(40, 32, generator=g).to(cuda)
    pooled = torch.randn(24, generator=g).to(cuda)
    blocks = SparsePRBlocks(sp, cfg.double_blocks + cfg.single_blocks, prompt_length=30)
    with torch.no_grad():
        out = model.forward(latent, text, torch.tensor(500.0, device=cuda), pooled, torch.tensor(6.0, device=cuda),
                            JointAttention(blocks))
    assert out.shape == (4 * 8 * 16, 64) and torch.isfinite(out.float()).all()
