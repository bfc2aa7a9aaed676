"""8-bit layers and prompts of different lengths through the modules (GPU): Fp8Linear,
feed-forwards and attentions against their bf16 selves over the values held, and whole
models with padded contexts against the same contexts without their padding."""

import importlib.util

import pytest
import torch

from conftest import GOLDEN

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


def _near(got, want, share, what=""):
    """Relative L2 distance: `share`."""
    rel = ((got.double() - want.double()).norm() / want.double().norm()).item()
    assert rel <= share, f"{what}: {rel}"


def _layer(k, n, bias=True):
    layer = torch.nn.Linear(k, n, bias=bias).to(DEV, BF16).requires_grad_(False)
    torch.nn.init.normal_(layer.weight, std=k**-0.5)
    return layer


def test_layer_and_its_refusals():
    import ltx_nn
    import ltxk

    layer = _layer(264, 40)
    made = ltx_nn.Fp8Linear.of(layer)
    x = torch.randn(2, 5, 264, device=DEV).to(BF16)
    want = ltxk.linear_fp8(x, ltxk.quantize_fp8(layer.weight), layer.bias)
    assert torch.equal(made(x), want) and torch.equal(made(ltxk.quantize_fp8(x)), want)
    wide = torch.randn(2, 5, 300, device=DEV).to(BF16)
    assert torch.equal(made(wide[..., :264]), made(wide[..., :264].contiguous()))
    again = ltx_nn.Fp8Linear(264, 40, device=DEV)
    again.load_state_dict(made.state_dict())
    assert torch.equal(again.to(BF16)(x), want)
    with pytest.raises(RuntimeError, match="no gradient"):
        made(x.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(made(x.clone().requires_grad_()), want)
    with pytest.raises(ValueError, match="multiples of 8"):
        ltx_nn.Fp8Linear(264, 12)
    with pytest.raises(ValueError, match="columns"):
        made(x[..., :256].contiguous())
    q, k = ltx_nn.project(x, made, None, again, layer)[::2]
    assert torch.equal(q, want) and torch.equal(k, want)


def test_feed_forward_is_its_own_layers():
    """Both layers 8-bit: the hidden values go between them in blocks, whichever way the input comes."""
    import ltx_nn
    import ltxk

    ff = ltx_nn.FeedForward(256).to(DEV, BF16).requires_grad_(False)
    x = torch.randn(3, 70, 256, device=DEV).to(BF16)
    plain = ff(x)
    assert ltx_nn.quantize_fp8(ff).takes_blocks
    y = ff(x)
    hidden = ltxk.linear_gelu_fp8(x, ff.proj_in.blocks(), ff.proj_in.bias)
    assert torch.equal(y, ltxk.linear_fp8(hidden, ff.proj_out.blocks(), ff.proj_out.bias))
    assert torch.equal(y, ff(ltxk.quantize_fp8(x)))
    # three roundings to e4m3 (input, hidden, weights twice): half a step of 2^-4 each at most, 0.026
    # rms of a value's each where steps are uniform within a binade, so below 0.06 together
    _near(y, plain, 0.06)


@pytest.mark.parametrize("quantized", [False, True])
def test_attention_over_kept_tokens(quantized):
    """A padded batch of contexts gives what each gives alone without its padding."""
    import ltx_nn

    attn = ltx_nn.Attention(256, 128, 4, 64, apply_gated_attention=True).to(DEV, BF16).requires_grad_(False)
    for norm in (attn.q_norm, attn.k_norm):
        torch.nn.init.ones_(norm.weight)
    if quantized:
        ltx_nn.quantize_fp8(attn)
        assert type(attn.to_q) is type(attn.to_out) is ltx_nn.Fp8Linear and type(attn.to_gate_logits) is torch.nn.Linear
    lengths = [1, 37, 200, 64]
    x, context = torch.randn(4, 90, 256, device=DEV).to(BF16), torch.randn(4, 200, 128, device=DEV).to(BF16)
    keep = torch.arange(200, device=DEV)[None, :] < torch.tensor(lengths, device=DEV)[:, None]
    got = attn(x, context=context, keep=keep)
    for i, n in enumerate(lengths):
        want = attn(x[i:i + 1], context=context[i:i + 1, :n].contiguous())
        # bf16 results of two kernels, one of them rounded again by the gate: d = 2^-7 of a value apart at
        # most.  An 8-bit output layer rounds them to steps of at most s = 2^-3 of the value: values d apart fall
        # on both sides of a border in d / s of the cases and are then s apart, rms sqrt(d / s) s = sqrt(d s) = 2^-5,
        # which the product, linear in them, keeps.
        _near(got[i:i + 1], want, 2.0**-5 if quantized else 0.01, f"item {i}")
    assert torch.equal(attn(x, context=context, keep=keep.to(torch.uint8)), got)
    empty = keep.clone()
    empty[2] = False
    none = attn(x, context=context, keep=empty)
    assert torch.equal(none[2], attn.to_out(torch.zeros(90, 256, device=DEV, dtype=BF16)))
    with pytest.raises(ValueError, match="keep"):
        attn(x, context=context, keep=keep[:, :100])
    with pytest.raises(ValueError, match="takes the place"):
        attn(x, context=context, keep=keep, mask=torch.zeros(1, 1, 1, 200, device=DEV, dtype=BF16))


def test_gradient_through_kept_tokens_is_torchs():
    """With a gradient to record the attention is torch's, with keep as its mask."""
    import ltx_nn

    attn = ltx_nn.Attention(128, 128, 2, 64).to(DEV, BF16)
    q, k, v = (torch.randn(2, t, 128, device=DEV).to(BF16).requires_grad_() for t in (9, 20, 20))
    keep = torch.rand(2, 20, device=DEV) < 0.6
    keep[:, 0] = True
    attn.attend(q, k, v, None, keep=keep).float().sum().backward()
    assert all(torch.isfinite(t.grad).all() and t.grad.abs().sum() > 0 for t in (q, k, v))
    assert not k.grad[~keep].any() and not v.grad[~keep].any()


def _golden_module():
    spec = importlib.util.spec_from_file_location("make_block_golden", GOLDEN / "make_block_golden.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _small(**flags):
    import ltx_dit

    mk = _golden_module()
    cfg = ltx_dit.DiTConfig(**{**mk.SMALL, **flags})
    model = ltx_dit.LTXModel(cfg)
    mk.init_weights(model)
    return cfg, model.to(DEV, BF16).eval().requires_grad_(False)


def _modalities(cfg, batch, text, seed=0, keep=None):
    import ltx_dit

    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(BF16)

    sigma = torch.full((batch,), 0.6, device=DEV)
    v = ltx_dit.Modality(latent=normal(batch, 12, cfg.video_in), sigma=sigma, timesteps=sigma.view(-1, 1, 1),
                         positions=ltx_dit.video_positions(batch, 1, 3, 4, 24.0, DEV),
                         context=normal(batch, text, cfg.video_cross_dim), context_keep=keep)
    a = ltx_dit.Modality(latent=normal(batch, 5, cfg.audio_in), sigma=sigma, timesteps=sigma.view(-1, 1, 1),
                         positions=ltx_dit.audio_positions(batch, 5, DEV),
                         context=normal(batch, text, cfg.audio_cross_dim), context_keep=keep)
    return v, a


@pytest.mark.parametrize("quantized", [False, True])
def test_model_with_padded_prompts(quantized):
    """Two prompts of 9 and 23 tokens padded to 23 in one call, and each alone without its padding."""
    import ltx_nn
    from dataclasses import replace

    cfg, model = _small()
    if quantized:
        ltx_nn.quantize_fp8(model)
    lengths = (9, 23)
    keep = torch.arange(23, device=DEV)[None, :] < torch.tensor(lengths, device=DEV)[:, None]
    v, a = _modalities(cfg, 2, 23, keep=keep)
    with torch.no_grad():
        vx, ax = model(v, a, None)
        for i, n in enumerate(lengths):
            one = [replace(m, latent=m.latent[i:i + 1], sigma=m.sigma[i:i + 1], timesteps=m.timesteps[i:i + 1],
                           positions=m.positions[i:i + 1], context=m.context[i:i + 1, :n].contiguous(), context_keep=None)
                   for m in (v, a)]
            wv, wa = model(*one, None)
            # two blocks of bf16 activations, whose roundings the kernels' orders of sums decide
            # (e4m3 roundings, a step of 2^-3 apart, where the layers are 8-bit)
            share = 0.08 if quantized else 0.02
            _near(vx[i:i + 1], wv, share, f"video {i}")
            _near(ax[i:i + 1], wa, share, f"audio {i}")


def test_quantized_model_is_near_its_bf16_self():
    import ltx_nn

    cfg, model = _small()
    v, a = _modalities(cfg, 1, 7)
    with torch.no_grad():
        want = model(v, a, None)
        ltx_nn.quantize_fp8(model)
        assert model.blocks[0].ff.takes_blocks and model.blocks[1].audio_ff.takes_blocks
        got = model(v, a, None)
    for g, w in zip(got, want):
        assert torch.isfinite(g).all()
        # each layer's result is off by 0.026 * sqrt(2) of its size (both operands' roundings); the residual
        # stream carries most of every output past two blocks of them
        _near(g, w, 0.2)
