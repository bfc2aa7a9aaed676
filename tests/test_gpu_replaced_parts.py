"""Blocks whose attentions or feed-forwards a program has replaced by modules of its own (GPU): they are called
with the arguments that the reference's blocks pass."""

import pytest
import torch

pytestmark = pytest.mark.gpu


class _Around(torch.nn.Module):
    """A part of a block behind the reference's own signature."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.calls = inner, 0


class _Attention(_Around):
    def forward(self, x, context=None, mask=None, pe=None, k_pe=None, perturbation_mask=None, all_perturbed=False):
        self.calls += 1
        return self.inner(x, context=context, mask=mask, pe=pe, k_pe=k_pe, perturbation_mask=perturbation_mask,
                          all_perturbed=all_perturbed)


class _FeedForward(_Around):
    def forward(self, x):
        assert type(x) is torch.Tensor
        self.calls += 1
        return self.inner(x)


def _wrap(model):
    for block in model.blocks:
        for name in ("attn1", "attn2", "audio_attn1", "audio_attn2"):
            setattr(block, name, _Attention(getattr(block, name)))
        block.ff, block.audio_ff = _FeedForward(block.ff), _FeedForward(block.audio_ff)
    return [m for m in model.modules() if isinstance(m, _Around)]


@pytest.mark.parametrize("flags", [{}, {"cross_attention_adaln": False}])
def test_replaced_attentions_and_feed_forwards(flags):
    from test_gpu_fp8_model import _modalities, _small

    cfg, model = _small(**flags)
    v, a = _modalities(cfg, 1, 7)
    with torch.no_grad():
        want = model(v, a, None)
        parts = _wrap(model)
        got = model(v, a, None)
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and all(p.calls == 1 for p in parts)


def test_replaced_parts_around_8_bit_layers():
    """A replaced feed-forward is given the normed tensor, whatever it holds."""
    from test_gpu_fp8_model import _modalities, _small

    import ltx_nn

    cfg, model = _small()
    v, a = _modalities(cfg, 1, 7)
    with torch.no_grad():
        ltx_nn.quantize_fp8(model)
        parts = _wrap(model)
        got = model(v, a, None)
    assert all(torch.isfinite(g).all() for g in got) and all(p.calls == 1 for p in parts)
