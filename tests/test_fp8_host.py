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


@pytest.mark.parametrize("width", [128, 136])  # of 128 columns a bf16 weight has the bytes' shape
@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("strict", [False, True])
def test_a_bf16_state_is_refused(width, assign, strict):
    """A bf16 layer's state (or one cast to another type) is not loaded into an 8-bit layer as if its values were
    bytes; an 8-bit layer's own is, whichever way."""
    import ltx_nn

    layer, plain = ltx_nn.Fp8Linear(width, 40), torch.nn.Linear(width, 40).to(BF16)
    layer.weight.random_(0, 127), layer.weight_scale.fill_(120)
    held = {name: t.clone() for name, t in layer.state_dict().items()}
    half = {name: t.half() for name, t in held.items()}
    values = {**held, "weight": held["weight"].view(torch.float8_e4m3fn)}
    for state in (plain.state_dict(), half, {**held, "weight": plain.weight.detach()}, values):
        with pytest.raises(RuntimeError, match="8-bit|size mismatch"):
            layer.load_state_dict(state, strict=strict, assign=assign)
        assert all(torch.equal(t, held[name]) and t.dtype == held[name].dtype for name, t in layer.state_dict().items())
    other = torch.nn.Sequential(ltx_nn.Fp8Linear(width, 40))
    other.load_state_dict({f"0.{name}": t for name, t in held.items()}, strict=strict, assign=assign)
    assert all(torch.equal(t, held[name]) for name, t in other[0].state_dict().items())


def test_fx_tracing_is_refused():
    """The kernels bypass the dispatcher: a traced graph would hold their results as constants."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    ff, x = _ff(), torch.randn(2, 3, 128).to(BF16)
    for call in (lambda t: ff(t), lambda t: ff.proj_in(t), lambda t: ff.proj_in.gelu(t), lambda t: _block_ffn(ff, t)):
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="inference"):
                make_fx(call, tracing_mode=mode)(x)
        with FlopCounterMode(display=False), pytest.raises(RuntimeError, match="ROCm device"):
            call(x)  # counts what torch runs: these go on
