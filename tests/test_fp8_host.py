"""What 8-bit layers and kept tokens do before any launch (CPU): derivatives and tracers refused."""

from types import SimpleNamespace

import pytest
import torch

BF16 = torch.bfloat16


def _ff(dim=128):
    import ltx_nn

    ff = ltx_nn.FeedForward(dim).to(BF16).requires_grad_(False)
    ff.proj_in, ff.proj_out = ltx_nn.Fp8Linear(dim, 4 * dim), ltx_nn.Fp8Linear(4 * dim, dim)
    return ff


def _block_ffn(ff, x, pending=None):
    """Block._ffn over a 9-row table."""
    import ltx_dit

    d = x.shape[-1]
    table, emb = torch.zeros(9, d, dtype=BF16), torch.zeros(x.shape[0], 1, 9 * d, dtype=BF16)
    return ltx_dit.Block._ffn(SimpleNamespace(norm_eps=1e-6), x, pending, table, (emb, None), ff, True)


def test_derivatives_are_refused():
    """A gradient to record and a forward-mode tangent, at the layers and in a block, where the norm takes the input;
    without either the calls go on (to the device check: this is the CPU)."""
    import ltx_nn
    from torch.autograd import forward_ad

    ff, x = _ff(), torch.randn(1, 3, 128).to(BF16)
    attn = ltx_nn.Attention(128, 128, 2, 64)
    attn.to_q = attn.to_k = attn.to_v = ltx_nn.Fp8Linear(128, 128)
    calls = [ff, ff.proj_in, ff.proj_in.gelu, lambda t: ltx_nn.project(t, attn.to_q, attn.to_k), lambda t: _block_ffn(ff, t),
             lambda t: _block_ffn(ff, x, (t, None, None)), lambda t: _block_ffn(ff, t, (x, None, None))]
    for call in calls:
        with pytest.raises(RuntimeError, match="inference"):
            call(x.clone().requires_grad_())
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="inference"):
                call(forward_ad.make_dual(x, x))
            with pytest.raises(RuntimeError, match="ROCm device"):  # no tangent on this one
                call(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm device"):
            call(x.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="ROCm device"):
            call(x)


def test_transforms_and_tracers_are_refused():
    """They would see constants, or nothing, in place of the layer."""
    ff, x = _ff(), torch.randn(2, 3, 128).to(BF16)
    for call in (ff, ff.proj_in, lambda t: ff.proj_in.gelu(t), lambda t: _block_ffn(ff, t)):
        with pytest.raises(RuntimeError, match="inference"):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError, match="inference"):
            torch.func.grad(lambda t: call(t).float().sum())(x)
        with pytest.raises(RuntimeError, match="inference"):
            torch.func.vmap(call)(x[:, None])
        with pytest.raises(RuntimeError, match="inference"):
            torch.jit.trace(call, x, check_trace=False)
