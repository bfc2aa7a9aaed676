"""Kept context tokens and 8-bit layers through whole models and run_dit's passes (GPU), under weights of which every
branch of the blocks matters: each test also shows that its tolerance would not hold with the branch left out, the
tokens exchanged or the streams' masks swapped."""

from dataclasses import replace

import pytest
import torch

from test_gpu_fp8_model import _golden_module

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16

# Relative distances over two blocks of these weights, from the eager restatement (oracle/model_eager.py) on the CPU: in
# bf16 from fp32 0.008-0.009, and two bf16 models are as far apart at most twice; with the layers' operands rounded to
# their blocks 0.053-0.065.  Two 8-bit models whose activations are bf16 roundings apart (2^-8 of a value) differ by
# steps of 2^-3 in 2^-5 of the values, 2^-5.5 a layer (rms), the same size as that.  Left out, exchanged or
# zeroed branches move the outputs by the shares that the tests state.
NEAR = {False: 0.02, True: 0.08}


def _distance(got, want):
    return [((g.double() - w.double()).norm() / w.double().norm()).item() for g, w in zip(got, want)]


def _model(quantized, audio_head_dim=32, layers=2):
    """Linear weights of variance 1 / K, AdaLN tables of order 1, text attention's gates 3."""
    import ltx_dit
    import ltx_nn

    wide = dict(audio_head_dim=64, audio_cross_dim=128) if audio_head_dim == 64 else {}
    cfg = ltx_dit.DiTConfig(**{**_golden_module().SMALL, **wide, "num_layers": layers})
    model = ltx_dit.LTXModel(cfg)
    g = torch.Generator().manual_seed(11)
    with torch.no_grad():
        for name, p in sorted(model.named_parameters()):
            r = torch.randn(p.shape, generator=g)
            if name.endswith("norm.weight"):
                r = 1 + 0.1 * r
            elif "table" in name:
                r = r * 0.5
            elif p.ndim == 2 and "keyframes" not in name:
                r = r * p.shape[1]**-0.5 * (0.3 if "adaln" in name else 1.0)
            else:
                r = r * 0.1
            p.copy_(r)
        for block in model.blocks:
            for table in (block.scale_shift_table, block.audio_scale_shift_table):
                for row, size in ((2, 1.0), (5, 1.0), (8, 3.0)):
                    table[row] = torch.sign(table[row]) * size
    model = model.to(DEV, BF16).eval().requires_grad_(False)
    return cfg, ltx_nn.quantize_fp8(model) if quantized else model


def _modalities(cfg, batch, v_text, a_text):
    import ltx_dit

    g = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(DEV, BF16)

    sigma = torch.full((batch,), 0.6, device=DEV)
    v = ltx_dit.Modality(latent=normal(batch, 12, cfg.video_in), sigma=sigma, timesteps=sigma.view(-1, 1, 1),
                         positions=ltx_dit.video_positions(batch, 1, 3, 4, 24.0, DEV),
                         context=normal(batch, v_text, cfg.video_cross_dim))
    a = ltx_dit.Modality(latent=normal(batch, 5, cfg.audio_in), sigma=sigma, timesteps=sigma.view(-1, 1, 1),
                         positions=ltx_dit.audio_positions(batch, 5, DEV),
                         context=normal(batch, a_text, cfg.audio_cross_dim))
    return v, a


def _item(m, i, kept=None):
    """Batch item i of a modality, its context cut to the kept tokens."""
    context = m.context[i:i + 1]
    return replace(m, latent=m.latent[i:i + 1], sigma=m.sigma[i:i + 1], timesteps=m.timesteps[i:i + 1],
                   positions=m.positions[i:i + 1], context=context if kept is None else context[:, kept].contiguous(),
                   context_keep=None)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("audio_head_dim", [32, 64])  # torch's attention over the audio's prompt, and the kernel
def test_padded_prompts(quantized, audio_head_dim):
    """Prompts of different lengths and patterns, another mask for each stream and NaN in what is left out, against each
    item alone over its kept tokens."""
    cfg, model = _model(quantized, audio_head_dim)
    v, a = _modalities(cfg, 3, 23, 23)
    at = torch.arange(23, device=DEV)
    v_keep = torch.stack([at < 9, at >= 0, at % 3 == 1])
    a_keep = torch.stack([at >= 17, at < 4, at % 2 == 0])
    masked = [replace(m, context=m.context.masked_fill(~k.unsqueeze(-1), float("nan")), context_keep=k)
              for m, k in ((v, v_keep), (a, a_keep))]
    with torch.no_grad():
        want = [model(_item(v, i, v_keep[i]), _item(a, i, a_keep[i]), None) for i in range(3)]

        def distances(video, audio):
            got = model(video, audio, None)
            return [_distance([g[i:i + 1] for g in got], want[i]) for i in range(3)]

        for i, d in enumerate(distances(*masked)):
            assert max(d) <= NEAR[quantized], (i, d)
        # nothing left out, the others kept instead, the streams' masks swapped: 0.3 and more of the first item
        for wrong in ((v, a), [replace(m, context_keep=~m.context_keep | (at == 0)) for m in (replace(v, context_keep=v_keep),
                      replace(a, context_keep=a_keep))], (replace(v, context_keep=a_keep), replace(a, context_keep=v_keep))):
            d = distances(*wrong)[0]
            assert min(d) >= 3 * NEAR[quantized], d
        one = distances(replace(v, context_keep=v_keep[:1]), replace(a, context_keep=a_keep[:1]))[0]
        assert max(one) <= NEAR[quantized], one  # one mask for every item


@pytest.mark.parametrize("audio_head_dim", [32, 64])
def test_quantized_model(audio_head_dim):
    """All layers 8-bit against the bf16 model, and what a branch of zeros would do."""
    with torch.no_grad():
        cfg, model = _model(False, audio_head_dim)
        v, a = _modalities(cfg, 1, 23, 23)
        want = model(v, a, None)
        del model
        cfg, model = _model(True, audio_head_dim)
        near = 0.1  # the blocks' rounding and two models' in bf16
        assert max(_distance(model(v, a, None), want)) <= near

        def without(*names):
            zeroed = _model(True, audio_head_dim)[1]
            for name in names:
                layer = zeroed.get_submodule(name)
                layer.weight.zero_(), layer.bias.zero_() if layer.bias is not None else None
            return _distance(zeroed(v, a, None), want)

        assert min(without(*(f"blocks.{i}.{s}ff.proj_out" for i in (0, 1) for s in ("", "audio_")))) >= 2.5 * near
        assert min(without(*(f"blocks.{i}.{s}attn{n}.to_out" for i in (0, 1) for s in ("", "audio_") for n in (1, 2)))) >= 5 * near
        for name, stream in (("blocks.0.ff.proj_out", 0), ("blocks.1.audio_ff.proj_out", 1), ("blocks.0.attn2.to_out", 0),
                             ("blocks.0.video_to_audio_attn.to_out", 1)):
            assert without(name)[stream] >= 1.5 * near, name


def _states(cfg):
    import ltx_dit

    g = torch.Generator().manual_seed(5)
    v, a = (torch.randn(1, t, n, generator=g).to(DEV, BF16) for t, n in ((12, cfg.video_in), (5, cfg.audio_in)))
    ones = [torch.ones(1, t.shape[1], 1, device=DEV) for t in (v, a)]
    return (ltx_dit.LatentState(v, ones[0], ltx_dit.video_positions(1, 1, 3, 4, 24.0, DEV), torch.zeros_like(v)),
            ltx_dit.LatentState(a, ones[1], ltx_dit.audio_positions(1, 5, DEV), torch.zeros_like(a)))


@pytest.mark.parametrize("given", [("pos", "neg"), ("pos",), ("neg",)])
def test_run_dit_keeps_each_passes_tokens(given):
    """Every pass of a guided step, its prompt's kept tokens, against the same step over those tokens alone; a prompt
    without a mask is whole."""
    import ltx_dit

    cfg, model = _model(False, 64)
    p = ltx_dit.GuiderParams(3.0, 1.0, 0.7, 2.0, (1,))
    g = torch.Generator().manual_seed(9)
    at = torch.arange(20, device=DEV)
    keeps = {"v_pos": at < 5, "v_neg": at >= 16, "a_pos": at % 4 == 2, "a_neg": at < 2}
    contexts = {n: torch.randn(1, 20, 128, generator=g).to(DEV, BF16) for n in keeps}
    for n in keeps:
        if n[2:] not in given:
            keeps[n] = torch.ones_like(keeps[n])
    sigmas, seen = torch.tensor([0.9, 0.5], device=DEV), []

    def passes(contexts):
        return ltx_dit.guided_denoise_step(model, *_states(cfg), contexts, sigmas[0], 0, p, p, cfg)[2]

    masked = {**{n: c.masked_fill(~keeps[n][None, :, None], float("nan")) for n, c in contexts.items()},
              **{f"{n}_keep": k[None] for n, k in keeps.items() if n[2:] in given}}
    ltx_dit.run_dit(model, cfg, masked, *_states(cfg), sigmas, p, p, on_step=lambda *args: seen.append(args[4]))
    got = seen[0]
    with torch.no_grad():
        for prompt, names in (("pos", ("cond", "ptb", "mod")), ("neg", ("uncond",))):
            cut = {f"{s}_{n}": contexts[f"{s}_{prompt}"][:, keeps[f"{s}_{prompt}"]].contiguous()
                   for s in ("v", "a") for n in ("pos", "neg")}
            want = passes(cut)
            for name in names:
                d = _distance(got[name], want[name])
                assert max(d) <= NEAR[False], (name, d)
            whole = passes({f"{s}_{n}": contexts[f"{s}_{prompt}"] for s in ("v", "a") for n in ("pos", "neg")})
            if prompt in given:
                assert min(_distance(whole[names[0]], want[names[0]])) >= 3 * NEAR[False]
        other = passes({f"{s}_{n}": contexts[f"{s}_{q}"][:, keeps[f"{s}_{q}"]].contiguous()
                        for s in ("v", "a") for n, q in (("pos", "neg"), ("neg", "neg"))})
        assert min(_distance(got["cond"], other["cond"])) >= 3 * NEAR[False]  # the other prompt's tokens


@pytest.mark.parametrize("registers", [0, 32])  # attention masked (torch's), or unmasked once registers fill the padding
def test_quantized_connector(registers):
    """The text path's connectors take 8-bit layers like the blocks."""
    import ltx_nn
    import ltx_te

    torch.manual_seed(2)
    connector = ltx_te.Embeddings1DConnector(4, 64, 2, [128], registers, True, True).to(DEV, BF16).requires_grad_(False)
    for name, p in connector.named_parameters():
        if name.endswith("norm.weight"):
            torch.nn.init.ones_(p)
        else:
            torch.nn.init.normal_(p, std=p.shape[-1]**-0.5 if p.ndim == 2 and "registers" not in name else 1.0 if p.ndim == 2 else 0.1)
    x = torch.randn(2, 64, 256, device=DEV).to(BF16)
    mask = torch.zeros(2, 1, 1, 64, device=DEV, dtype=BF16)
    mask[1, ..., 40:] = torch.finfo(BF16).min
    want = connector(x, mask)[0]
    layers = ltx_nn.quantize_fp8(connector).blocks
    assert all(b.ff.takes_blocks and type(b.attn1.to_q) is type(b.attn1.to_out) is ltx_nn.Fp8Linear for b in layers)
    near = 0.1  # the operands' rounding, 0.037 a layer, over four branches as large as the stream they are added to
    assert _distance([connector(x, mask)[0]], [want])[0] <= near
    for part in ("attn1.to_out", "ff.proj_out"):
        held = [b.get_submodule(part).weight.clone() for b in layers]
        for b in layers:
            b.get_submodule(part).weight.zero_()
        assert _distance([connector(x, mask)[0]], [want])[0] >= 2.5 * near, part
        for b, w in zip(layers, held):
            b.get_submodule(part).weight.copy_(w)
