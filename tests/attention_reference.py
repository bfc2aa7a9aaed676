"""Attention of single sequences in fp64, and how far a kernel may be from it."""

import math

import torch


def seen_keys(queries: int, keys: int, prefix: int, causal: bool, window=None):
    """(first, end) of the own keys that each query sees, and whether it sees the prefix."""
    pos = torch.arange(keys - queries, keys)
    end = (pos + 1).clamp(min=0) if causal else torch.full_like(pos, keys)
    first = (end - window).clamp(min=0) if window else torch.zeros_like(pos)
    return first, end, (pos >= 0) if causal else torch.ones_like(pos, dtype=torch.bool)


def one_sequence(q, k, v, heads, kv_heads, scale=None, prefix=0, causal=True, window=None):
    """q (n, H*Dh) over k, v (prefix + m, KVH*Dh), whose first `prefix` keys are shared ones: the result, and its weights'
    sum over |v|, both (n, H*Dh) in fp64.  Masked values take no part, whatever they hold."""
    (n, w), dh = q.shape, q.shape[1] // heads
    scale = 1 / math.sqrt(dh) if scale is None else scale
    first, end, all_prefix = (x.to(q.device) for x in seen_keys(n, k.shape[0] - prefix, prefix, causal, window))
    j = torch.arange(k.shape[0], device=q.device) - prefix
    seen = torch.where(j < 0, all_prefix[:, None], (j >= first[:, None]) & (j < end[:, None]))
    want, spread = torch.zeros(n, w, dtype=torch.float64, device=q.device), torch.zeros(n, w, dtype=torch.float64, device=q.device)
    if not n or not k.shape[0]:
        return want, spread
    for h in range(heads):
        a, b = slice(h * dh, (h + 1) * dh), slice(h // (heads // kv_heads) * dh, (h // (heads // kv_heads) + 1) * dh)
        s = (q[:, a].double() @ k[:, b].double().t().contiguous()) * scale
        s = torch.where(seen, s, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(0.0, neginf=0.0, posinf=math.inf))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        p = torch.where(seen, p, 0.0)
        x = v[:, b].double()
        if not bool(torch.isfinite(x).all()):  # a value that is not finite counts where it is seen
            bad = ~torch.isfinite(x)
            clean = torch.where(bad, 0.0, x)
            hit = seen.double() @ bad.double() > 0
            want[:, a] = torch.where(hit, math.nan, p @ clean)
            spread[:, a] = p @ clean.abs()
        else:
            want[:, a], spread[:, a] = p @ x, p @ x.abs()
    return want, spread


def assert_near(got, want, spread, what="", score=0.0):
    """A weight rounded to bf16 is off by at most 2^-8 of it, which moves the result by at most 2^-8 sum_j w_j |v_j|; the
    result's own rounding by 2^-8 of it.  The fp32 products, exponentials and sums are far below that (2 %).  Rows of
    zeros are zeros, and what is not finite is not.  `score`: the largest magnitude of a score where that is thousands: it
    rounds before the maximum is taken off, by at most 2^-24 of it, and so does the maximum, which moves a weight by that
    share of it.  A weight below 2^-126, the least normal number of fp32, may be zero: 2^20 of them and values up to 2^5 move a
    result by no more than 2^-101, which is below 1e-30."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: {int((torch.isfinite(got) != fine).sum())} values finite or not"
    err = torch.where(fine, got - want, 0.0).abs()
    bound = torch.where(fine, (spread + want.abs()) * 2.0**-8 * 1.02 + (1e-6 + 2 * score * 2.0**-24) * spread + 1e-30, 0.0)
    ratio = err / bound.clamp(min=1e-30)
    assert bool((err <= bound).all()), f"{what}: {ratio.max().item():.3f} of the bound at {int(ratio.argmax())} of {tuple(got.shape)}"
