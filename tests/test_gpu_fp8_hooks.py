"""8-bit layers that hooks or patched calls watch (GPU): they see the modules' own calls, on tensors."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


def _ff(dim=256):
    import ltx_nn

    torch.manual_seed(3)
    return ltx_nn.quantize_fp8(ltx_nn.FeedForward(dim).to(DEV, BF16).requires_grad_(False))


def _seen(module, **kw):
    """The types of what a module's forward hook is given."""
    seen = []
    handle = module.register_forward_hook(lambda m, args, out: seen.append((type(args[0]), type(out))), **kw)
    return seen, handle


TENSORS = [(torch.Tensor, torch.Tensor)]


@pytest.mark.parametrize("name", ["proj_in", "proj_out"])
def test_hooks_on_a_feed_forwards_layers(name):
    """A hook on either layer fires once with tensors, may replace the result, and leaves no trace once removed."""
    import ltxk

    ff, x = _ff(), torch.randn(2, 70, 256, device=DEV).to(BF16)
    plain = ff(x)
    seen, handle = _seen(getattr(ff, name))
    got = ff(x)
    assert seen == TENSORS and not ff.takes_blocks
    hidden = ltxk.linear_fp8(x, ff.proj_in.blocks(), ff.proj_in.bias)
    want = ltxk.linear_fp8(ltxk.gelu_tanh(hidden), ff.proj_out.blocks(), ff.proj_out.bias)
    assert torch.equal(got, want)
    handle.remove()
    assert ff.takes_blocks and torch.equal(ff(x), plain)
    handle = getattr(ff, name).register_forward_pre_hook(lambda m, args: (torch.zeros_like(args[0]),))
    zero = torch.zeros_like(x) if name == "proj_in" else torch.zeros(2, 70, 1024, device=DEV, dtype=BF16)
    got = ff(x)
    handle.remove()
    if name == "proj_out":
        assert torch.equal(got, ff.proj_out(zero))
    else:
        assert torch.equal(got, ff.proj_out(ltxk.gelu_tanh(ff.proj_in(zero))))
    layer = getattr(ff, name)
    layer.forward = lambda t: torch.ones(*t.shape[:-1], layer.out_features, device=DEV, dtype=BF16)
    assert not ff.takes_blocks and ff(x).shape == x.shape


def test_hooks_of_every_module():
    """A global hook sees every module's tensors."""
    from torch.nn.modules.module import register_module_forward_hook

    ff, x, seen = _ff(), torch.randn(1, 9, 256, device=DEV).to(BF16), []
    handle = register_module_forward_hook(lambda m, args, out: seen.append((type(m).__name__, type(args[0]), type(out))))
    try:
        ff(x)
    finally:
        handle.remove()
    assert seen == [("Fp8Linear", *TENSORS[0]), ("Fp8Linear", *TENSORS[0]), ("FeedForward", *TENSORS[0])]


def test_hooks_on_projections_of_one_input():
    """A hooked projection takes the tensor, the others the blocks made once for them: the same results."""
    import ltx_nn

    torch.manual_seed(4)
    attn = ltx_nn.quantize_fp8(ltx_nn.Attention(256, 256, 4, 64).to(DEV, BF16).requires_grad_(False))
    x = torch.randn(2, 40, 256, device=DEV).to(BF16)
    want = ltx_nn.project(x, attn.to_q, attn.to_k, attn.to_v)
    for names in (("to_k",), ("to_q", "to_v"), ("to_q", "to_k", "to_v")):
        hooks = [_seen(getattr(attn, n)) for n in names]
        got = ltx_nn.project(x, attn.to_q, attn.to_k, attn.to_v)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for seen, handle in hooks:
            assert seen == TENSORS
            handle.remove()


def test_hooks_on_a_blocks_feed_forward():
    """A hook on a block's feed-forward is given the normed tensor, as in the bf16 model."""
    from test_gpu_fp8_model import _modalities, _small

    import ltx_nn

    cfg, model = _small()
    v, a = _modalities(cfg, 1, 7)
    ltx_nn.quantize_fp8(model)
    hooks = [_seen(ff) for block in model.blocks for ff in (block.ff, block.audio_ff)]
    with torch.no_grad():
        model(v, a, None)
    assert all(seen == TENSORS for seen, _ in hooks)


def test_layers_that_hooks_watch_stay_bf16():
    """A layer with hooks, a patched forward or a replaced operand is not converted, and Fp8Linear.of refuses it: what
    hangs on it would be lost."""
    import ltx_nn

    def patched(ff):
        ff.proj_in.forward = lambda x: x

    def hooked(ff):
        ff.proj_in.register_forward_hook(lambda *_: None)

    def before(ff):
        ff.proj_in.register_forward_pre_hook(lambda *_: None)

    def parametrized(ff):
        torch.nn.utils.parametrizations.weight_norm(ff.proj_in)

    def broadcast(ff):
        ff.proj_in.bias = torch.nn.Parameter(torch.zeros(1, device=DEV, dtype=BF16))

    for change in (patched, hooked, before, parametrized, broadcast):
        ff = ltx_nn.FeedForward(128).to(DEV, BF16).requires_grad_(False)
        change(ff)
        kept = ff.proj_in
        ltx_nn.quantize_fp8(ff)
        assert ff.proj_in is kept and type(ff.proj_out) is ltx_nn.Fp8Linear and not ff.takes_blocks, change.__name__
        with pytest.raises(ValueError, match="bare"):
            ltx_nn.Fp8Linear.of(kept)
