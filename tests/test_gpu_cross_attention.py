"""ltxk_cross_attention (csrc/flash.hip) against softmax attention over the kept keys in
fp64 (GPU): any pattern of kept keys, none of them, keys cut over units, views of
wider rows, and keys left out that hold anything."""

import pytest
import torch

from test_gpu_flash import _check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _keep(kind, b, tk, g):
    at = torch.arange(tk, device=DEV).expand(b, tk)
    n = torch.randint(1, tk + 1, (b, 1), device=DEV, generator=g)
    if kind == "front":
        return (at < n).contiguous()
    if kind == "back":
        return (at >= tk - n).contiguous()
    if kind == "one":
        return (at == n - 1).contiguous()
    keep = torch.rand(b, tk, device=DEV, generator=g) < 0.6
    if kind == "empty":
        keep[-1] = False
    return keep


def _against_kept(q, k, v, h, keep, logits, got):
    for i in range(q.shape[0]):
        kept = keep[i if keep.shape[0] > 1 else 0].bool()
        if not kept.any():
            assert not got[i].any(), f"item {i}: nothing is kept"
            continue
        _check(q[i:i + 1], k[i:i + 1, kept].contiguous(), v[i:i + 1, kept].contiguous(), h,
               None if logits is None else logits[i:i + 1], got[i:i + 1])


@pytest.mark.parametrize("kind", ["front", "back", "one", "holes", "empty"])
@pytest.mark.parametrize("b,tq,tk,h,dh,gated", [
    (1, 1, 1, 2, 64, True), (2, 128, 64, 1, 128, False), (3, 129, 65, 3, 64, True), (2, 127, 333, 2, 128, True),
    (4, 126, 1024, 4, 64, True), (3, 5, 4099, 3, 128, True), (2, 70, 8192, 2, 64, True), (2, 3, 8193, 1, 128, False),
    (3, 40, 9001, 2, 64, True), (2, 257, 2050, 2, 64, False), (2, 4100, 700, 8, 128, True)])
def test_matches_fp64_over_the_kept_keys(kind, b, tq, tk, h, dh, gated):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(tq * 7 + tk)
    q, k, v = ((torch.randn(b, t, h * dh, device=DEV, generator=g) * s).to(torch.bfloat16)
               for t, s in ((tq, 1.5), (tk, 1.0), (tk, 1.0)))
    keep = _keep(kind, b, tk, g)
    logits = torch.randn(b, tq, h, device=DEV, generator=g).to(torch.bfloat16) if gated else None
    # what is left out may hold anything
    k[~keep], v[~keep] = float("nan"), float("inf")
    _against_kept(q, k, v, h, keep, logits, ltxk.cross_attention(q, k, v, h, keep, logits))


@pytest.mark.parametrize("tk", [320, 1000, 2500])
def test_all_kept_equals_no_mask(tk):
    """A mask that keeps everything, and no mask, give the same bits (`attention`'s, where neither cuts the
    keys); uint8 masks count every non-zero byte; one row of a mask serves every batch item."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(2, t, 256, device=DEV, generator=g).to(torch.bfloat16) for t in (200, tk, tk))
    logits = torch.randn(2, 200, 4, device=DEV, generator=g).to(torch.bfloat16)
    every = torch.ones(2, tk, device=DEV, dtype=torch.bool)
    assert torch.equal(ltxk.cross_attention(q, k, v, 4, None, logits), ltxk.cross_attention(q, k, v, 4, every, logits))
    want = ltxk.cross_attention(q, k, v, 4)
    if tk == 320:
        assert torch.equal(want, ltxk.attention(q, k, v, 4))
    assert torch.equal(ltxk.cross_attention(q, k, v, 4, torch.full((2, tk), 200, device=DEV, dtype=torch.uint8)), want)
    row = torch.rand(1, tk, device=DEV, generator=g) < 0.5
    one = ltxk.cross_attention(q, k, v, 4, row)
    assert torch.equal(one, ltxk.cross_attention(q, k, v, 4, row.expand(2, tk).contiguous()))
    out = torch.full_like(q, 3.0)
    assert ltxk.cross_attention(q, k, v, 4, row, out=out) is out and torch.equal(out, one)


def test_no_keys_and_views():
    """No keys at all give zeros; q, k and v as columns of wider rows, and keys shared by the
    batch (stride 0), equal the contiguous call bit for bit."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(2)
    q = torch.randn(3, 70, 128, device=DEV, generator=g).to(torch.bfloat16)
    none = q[:, :0]
    assert not ltxk.cross_attention(q, none, none, 2, torch.empty(3, 0, dtype=torch.bool, device=DEV)).any()
    assert not ltxk.cross_attention(q, none, none, 2).any()
    assert ltxk.cross_attention(none, q, q, 2).shape == (3, 0, 128)
    wide = torch.randn(1, 300, 392, device=DEV, generator=g).to(torch.bfloat16)
    k, v = wide[..., 8:136].expand(3, 300, 128), wide[..., 264:].expand(3, 300, 128)
    keep = torch.rand(3, 300, device=DEV, generator=g) < 0.4
    got = ltxk.cross_attention(q, k, v, 2, keep)
    assert torch.equal(got, ltxk.cross_attention(q, k.contiguous(), v.contiguous(), 2, keep))
    _against_kept(q, k.contiguous(), v.contiguous(), 2, keep, None, got)


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (torch.randn(2, t, 256, device=DEV, generator=g).to(torch.bfloat16) for t in (60, 3000, 3000))
    keeps = [torch.rand(2, 3000, device=DEV, generator=g) < s for s in (0.2, 0.9)]
    want = [ltxk.cross_attention(q, k, v, 4, m) for m in keeps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in keeps]
    got = [[], []]
    for _ in range(8):
        for s, m, o in zip(streams, keeps, got):
            with torch.cuda.stream(s):
                o.append(ltxk.cross_attention(q, k, v, 4, m))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(w, x) for x in o)


@pytest.mark.parametrize("b,tq,tk,h,dh", [(4, 40, 23, 4, 32), (3, 1, 300, 2, 32), (65, 16, 16, 32, 64), (3, 70, 2048, 4, 32)])
def test_kept_tokens_where_attention_is_torchs(b, tq, tk, h, dh):
    """Heads that the kernel does not take, and many short sequences: left-out tokens may hold anything there, too,
    and an item without a kept token gives zeros."""
    import ltx_nn

    attn = ltx_nn.Attention(h * dh, h * dh, h, dh, apply_gated_attention=True)
    attn.to_out = torch.nn.Identity()
    g = torch.Generator(device=DEV).manual_seed(tk)
    q, k, v = (torch.randn(b, t, h * dh, device=DEV, generator=g).to(torch.bfloat16) for t in (tq, tk, tk))
    gates = torch.randn(b, tq, h, device=DEV, generator=g).to(torch.bfloat16)
    keep = torch.rand(b, tk, device=DEV, generator=g) < 0.6
    keep[0], keep[1] = True, False
    k[~keep], v[~keep] = float("nan"), float("inf")
    assert not ltx_nn.fused_attention_applies(q, k, v, h, dh)
    got = attn.attend(q, k, v, gates, keep=keep)
    assert not got[1].any()
    q4, k4, v4 = (t.double().view(b, -1, h, dh).transpose(1, 2).contiguous() for t in (q, k, v))
    k4, v4 = (t.masked_fill(~keep[:, None, :, None], 0.0) for t in (k4, v4))
    score = (q4 @ k4.transpose(-1, -2).contiguous()) * dh**-0.5
    p = torch.exp(score).masked_fill(~keep[:, None, None, :], 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    gate = (2 * torch.sigmoid(gates.double())).transpose(1, 2).unsqueeze(-1)
    want, size = (((p @ t) * gate).transpose(1, 2).reshape(b, tq, h * dh) for t in (v4, v4.abs()))
    # weights in bf16, the output's rounding and the gated one's: half a step each; a quarter more for the exponentials
    assert ((got.double() - want).abs() <= size * 2.0**-8 * 3.25 + 1e-30).all()


def test_captured_calls_past_the_listed_keys():
    """Two graphs, keys listed by a launch of its own and cut over units: replays in turn equal the eager calls."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(6)
    calls = []
    for tk in (8193, 9001):
        q, k, v = (torch.randn(2, t, 128, device=DEV, generator=g).to(torch.bfloat16) for t in (40, tk, tk))
        keep = torch.rand(2, tk, device=DEV, generator=g) < 0.3
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            ltxk.cross_attention(q, k, v, 2, keep)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = ltxk.cross_attention(q, k, v, 2, keep)
        calls.append((graph, out, q, k, v, keep))
    for i in range(4):
        for _, _, q, _, _, keep in calls:
            q.copy_(torch.randn(q.shape, device=DEV, generator=g))
            keep.copy_(torch.rand(keep.shape, device=DEV, generator=g) < 0.2 * (i + 1))
            keep[i % 2] &= i > 1  # an item without any
        for graph, *_ in calls:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, q, k, v, keep in calls:
            assert torch.equal(out, ltxk.cross_attention(q, k, v, 2, keep)), f"replay {i}"
