"""Attention(keep=) where it is torch's (CPU): left-out tokens may hold anything there, too, and items without a
kept token give zeros."""

import math

import pytest
import torch


def _attention(heads, dim_head, gated=False):
    import ltx_nn

    torch.manual_seed(1)
    attn = ltx_nn.Attention(64, 64, heads, dim_head, apply_gated_attention=gated)
    attn.to_out = torch.nn.Identity()
    return attn


def _plain(q, k, v, h, keep):
    """Softmax attention over the kept keys in fp64, item by item; zeros where nothing is kept."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    dh = q.shape[-1] // h
    for i in range(q.shape[0]):
        kept = keep[i if keep.shape[0] > 1 else 0]
        if not kept.any():
            continue
        for j in range(h):
            c = slice(j * dh, (j + 1) * dh)
            w = torch.softmax(q[i, :, c].double() @ k[i, kept][:, c].double().t() / math.sqrt(dh), -1)
            out[i, :, c] = w @ v[i, kept][:, c].double()
    return out


@pytest.mark.parametrize("heads,dh", [(2, 32), (1, 64), (3, 24)])
@pytest.mark.parametrize("tk", [1, 17, 64])
def test_left_out_tokens_may_hold_anything(heads, dh, tk):
    attn = _attention(heads, dh)
    g = torch.Generator().manual_seed(tk)
    q, k, v = (torch.randn(4, t, heads * dh, generator=g) for t in (5, tk, tk))
    keep = torch.rand(4, tk, generator=g) < 0.6
    keep[0], keep[1], keep[2, 0] = True, False, True
    want = _plain(q, k, v, heads, keep)
    k[~keep], v[~keep] = float("nan"), float("inf")
    held = k.clone(), v.clone()
    for mask in (keep, keep.to(torch.uint8) * 7):
        got = attn.attend(q, k, v, None, keep=mask).double()
        # fp32 sums of tk weights and dh products, an exponential of 2 ulp
        assert (got - want).abs().max() <= 2.0**-23 * (tk + dh + 8) * 4 and not got[1].any()
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(held, (k, v)))  # left as they were
    one = keep[:1]
    k, v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    assert torch.equal(attn.attend(q, k, v, None, keep=one), attn.attend(q, k, v, None, keep=one.expand(4, tk)))


def test_gradients_of_left_out_tokens_are_zero():
    """They stay finite where the tokens do not, and beside an item without a kept token."""
    attn = _attention(2, 32)
    q, k, v = (torch.randn(3, t, 64) for t in (5, 9, 9))
    keep = torch.rand(3, 9) < 0.5
    keep[0], keep[1, 0] = False, True
    k[~keep], v[~keep] = float("inf"), float("nan")
    for t in (q, k, v):
        t.requires_grad_()
    attn.attend(q, k, v, None, keep=keep).square().sum().backward()
    assert all(torch.isfinite(t.grad).all() for t in (q, k, v))
    assert not k.grad[~keep].any() and not v.grad[~keep].any() and not q.grad[0].any() and v.grad[1:][keep[1:]].any()


def test_no_tokens_at_all():
    attn = _attention(2, 32)
    q, none = torch.randn(2, 5, 64), torch.zeros(2, 0, 64)
    got = attn.attend(q, none, none, None, keep=torch.zeros(2, 0, dtype=torch.bool))
    assert got.shape == q.shape and not got.any()


def test_keep_goes_with_no_perturbation():
    """A perturbed attention passes the values through: there is nothing to leave out."""
    attn = _attention(2, 32)
    x, keep = torch.randn(2, 5, 64), torch.ones(2, 5, dtype=torch.bool)
    with pytest.raises(ValueError, match="no perturbation"):
        attn(x, keep=keep, all_perturbed=True)
    with pytest.raises(ValueError, match="no perturbation"):
        attn.attend(x, x, x, None, keep=keep, perturbation_mask=torch.ones(2, 1, 1))
    assert torch.equal(attn(x, all_perturbed=True), attn.to_v(x))


def test_passes_take_their_prompts_masks():
    """run_dit's masks by pass: the positive prompt's for all but the unconditional one; a prompt without a mask is whole."""
    import ltx_dit

    assert ltx_dit.PASSES == ("cond", "uncond", "ptb", "mod")
    contexts = {f"{s}_{p}": torch.zeros(1, n, 8) for s, n in (("v", 5), ("a", 3)) for p in ("pos", "neg")}
    assert ltx_dit._passes_keep(contexts, "v") is None and ltx_dit._passes_keep(contexts, "a") is None
    pos, neg, audio = (torch.tensor([row]) for row in ([1, 1, 0, 0, 0], [0, 0, 0, 1, 1], [0, 1, 0]))
    contexts.update(v_pos_keep=pos.bool(), v_neg_keep=neg, a_neg_keep=audio.to(torch.uint8))
    v, a = (ltx_dit._passes_keep(contexts, s) for s in ("v", "a"))
    assert v.dtype == a.dtype == torch.bool
    assert torch.equal(v.int(), torch.cat([pos, neg, pos, pos]).int())
    assert torch.equal(a.int(), torch.cat([torch.ones_like(audio), audio, torch.ones_like(audio), torch.ones_like(audio)]).int())
    del contexts["v_neg_keep"]
    assert torch.equal(ltx_dit._passes_keep(contexts, "v")[1], torch.ones(5, dtype=torch.bool))
    contexts["v_pos_keep"] = torch.ones(1, 4, dtype=torch.bool)
    with pytest.raises(RuntimeError):
        ltx_dit._passes_keep(contexts, "v")


def test_additive_masks_are_refused():
    """Their zeros are what to attend to: read as a keep they would attend to the padding."""
    import ltx_dit

    attn = _attention(2, 32)
    x, mask = torch.randn(2, 5, 64), torch.zeros(2, 5)
    mask[:, 3:] = -math.inf
    for dtype in (torch.float32, torch.bfloat16):
        with pytest.raises(ValueError, match="keep is"):
            attn.attend(x, x, x, None, keep=mask.to(dtype))
        with pytest.raises(ValueError, match="keep is"):
            ltx_dit._passes_keep({"v_pos": torch.zeros(1, 5, 8), "v_neg_keep": mask[:1].to(dtype)}, "v")
    assert torch.equal(attn.attend(x, x, x, None, keep=(mask == 0).long()), attn.attend(x, x, x, None, keep=mask == 0))
