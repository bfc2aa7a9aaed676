"""Packed and prefix attention with scores past 2^20, in every kind of tile and joined ones (GPU).

Queries are whole multiples of a power of two, keys and values small whole numbers, so that every product is exact in fp32.
In units of the softmax's exponents, scores of a large row are multiples of 2^17: those that equal the row's largest
weigh exactly as much as it, all others nothing.  Every other row has ordinary scores, whose tiles large ones share.
So nothing is allowed for the rounding of large scores."""

import math

import pytest
import torch

from attention_reference import assert_near, one_sequence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
SCALE = 0.125


def _offsets(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)


def _whole(g, *shape):
    return torch.randint(-3, 4, shape, device=DEV, generator=g).to(torch.bfloat16)


def _queries(g, rows, width, heads, size):
    q = _whole(g, rows, heads, width // heads)
    large = torch.arange(rows * heads, device=DEV).view(rows, heads, 1) % 2 == 0
    return torch.where(large, q * size, q).view(rows, width)


def _past(q, k, heads, kv_heads):
    """Whether a score is past 2^20 in the softmax's exponents."""
    dh = q.shape[1] // heads
    first = (q[:, :dh].double() @ k[:, :dh].double().t().contiguous()).abs().max().item()
    return first * SCALE * math.log2(math.e) > 2**20


@pytest.mark.parametrize("size", [2.0**20, 2.0**36, 2.0**100])
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("queries,keys,heads,kv_heads", [
    ([150, 50], None, 2, 2),        # tiles of 128 rows
    ([700], None, 4, 2),            # two groups of waves
    ([100], [4000], 4, 2),          # their keys cut
    ([3, 1, 2], [300, 40, 9], 4, 2),  # few rows
    ([1, 5], [6000, 3000], 4, 2),   # their keys cut
    ([1] * 20 + [300] * 30, None, 8, 8)])
def test_packed(queries, keys, heads, kv_heads, dh, size):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(len(queries))
    qo, ko = _offsets(queries), _offsets(keys or queries)
    q, k, v = _queries(g, sum(queries), heads * dh, heads, size), _whole(g, int(ko[-1]), kv_heads * dh), _whole(g, int(ko[-1]), kv_heads * dh)
    assert _past(q, k, heads, kv_heads)
    for mask in (dict(causal=True), dict(causal=False), dict(causal=True, window=90)):
        got = ltxk.packed_attention(q, k, v, heads, qo, kv_heads, ko, scale=SCALE, **mask)
        for s in {0, 1 % len(queries), len(queries) - 1}:
            rows, at = slice(int(qo[s]), int(qo[s + 1])), slice(int(ko[s]), int(ko[s + 1]))
            assert_near(got[rows], *one_sequence(q[rows], k[at], v[at], heads, kv_heads, SCALE, **mask), f"sequence {s}, {mask}")


@pytest.mark.parametrize("size", [2.0**20, 2.0**36, 2.0**100])
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("b,tq,prefix,room", [(64, 1, 9000, 300), (30, 5, 12000, 700), (3, 2, 60000, 40), (2, 1, 900, 2000), (5, 90, 500, 90)])
def test_prefix(b, tq, prefix, room, dh, size):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(b)
    heads, kv_heads = 4, 2
    q = _queries(g, b * tq, heads * dh, heads, size).view(b, tq, -1)
    k, v, pk, pv = (_whole(g, *x, kv_heads * dh) for x in ((b, room), (b, room), (prefix,), (prefix,)))
    assert _past(q[0], pk, heads, kv_heads)
    lengths = [room - i % 9 for i in range(b)]
    got = ltxk.prefix_attention(q, k, v, pk, pv, heads, kv_heads, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=SCALE)
    for i in {0, 1, b - 1}:
        n = lengths[i]
        want = one_sequence(q[i], torch.cat([pk, k[i, :n]]), torch.cat([pv, v[i, :n]]), heads, kv_heads, SCALE, prefix=prefix)
        assert_near(got[i], *want, f"item {i}")


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("queries,keys", [([300], [300]), ([100], [3000]), ([2], [4000]), ([1], [200])])
def test_scores_next_to_each_other(queries, keys, dh):
    """Scores of 2^21 and whole quarters beside it: each rounds by at most 2^-24 of itself before its weight is taken."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dh)
    qo, ko = _offsets(queries), _offsets(keys)
    q, k, v = _whole(g, sum(queries), 2 * dh), _whole(g, sum(keys), 2 * dh), _whole(g, sum(keys), 2 * dh)
    for x in (q, k):  # 2^22 in each of two places
        x.view(-1, 2, dh)[:, :, :2] = 2.0**11
    got = ltxk.packed_attention(q, k, v, 2, qo, 2, ko, scale=0.25)
    assert_near(got, *one_sequence(q, k, v, 2, 2, 0.25), score=(2.0**23 + 9 * dh) * 0.25)
