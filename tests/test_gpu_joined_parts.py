"""Packed and prefix attention whose keys are cut into parts: what a part that weighs nothing still brings (GPU)."""

import pytest
import torch

from attention_reference import assert_near, one_sequence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _offsets(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)


def _draw(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g).to(torch.bfloat16)


def _positive(g, *shape):
    """Queries whose products with negative keys are all negative, and never of zero with an infinity."""
    return (torch.randn(*shape, device=DEV, generator=g).abs() * 1.5).clamp(min=0.01).to(torch.bfloat16)


def _sink(k, low):
    """Keys whose scores are hundreds below the others' (at least sqrt(64) * 1.5 * 40 * 2 / pi = 305 on average, in heads of
    64), or minus infinity."""
    k.copy_(-(k.abs() * 40).clamp(min=0.1) if low == "low" else torch.full_like(k, float("-inf")))


def _spoil(v, dh):
    """A NaN in the first key head, an infinity in the second, in different parts and tiles."""
    v[min(5, len(v) - 1), 3] = float("nan")
    v[len(v) * 2 // 3, dh + 5] = float("-inf")


@pytest.mark.parametrize("low", ["low", "minus infinity"])
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("queries,keys", [([1], [5000]), ([3, 2], [3000, 4000]), ([1] * 64, [900] * 63 + [6000]),
                                          ([100], [2000]), ([300], [4000])])
def test_packed_values_of_low_scored_keys(queries, keys, dh, low):
    """Values that are not finite make the rows that see them so, however little their keys weigh."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dh + len(queries))
    qo, ko = _offsets(queries), _offsets(keys)
    q, k, v = _positive(g, sum(queries), 4 * dh), _draw(g, sum(keys), 2 * dh), _draw(g, sum(keys), 2 * dh)
    first, end = int(ko[-2]), int(ko[-2]) + keys[-1] // 2  # of the last sequence: its queries see later keys, too
    _sink(k[first:end], low)
    for spoilt in (False, True):
        if spoilt:
            _spoil(v[first:end], dh)
        got = ltxk.packed_attention(q, k, v, 4, qo, 2, ko)
        for s in {0, len(queries) - 1}:
            rows, at = slice(int(qo[s]), int(qo[s + 1])), slice(int(ko[s]), int(ko[s + 1]))
            assert_near(got[rows], *one_sequence(q[rows], k[at], v[at], 4, 2), f"sequence {s}")
        assert bool(got.isfinite().all()) != spoilt
        last = got[int(qo[-2]):].view(queries[-1], 4, dh)
        assert bool(last[:, :2, 3].isfinite().any()) != spoilt and bool(last[:, 2:, 5].isfinite().any()) != spoilt


@pytest.mark.parametrize("low", ["low", "minus infinity"])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("b,tq,prefix,room", [(64, 1, 9000, 300), (30, 5, 12000, 700), (3, 2, 60000, 40), (2, 1, 900, 2000)])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_prefix_values_of_low_scored_keys(b, tq, prefix, room, dh, where, low):
    """The same of a shared prefix, and of one item's own keys behind it, whose other items stay finite."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dh + b)
    q, k, v = _positive(g, b, tq, 4 * dh), _draw(g, b, room, 2 * dh), _draw(g, b, room, 2 * dh)
    pk, pv = _draw(g, prefix, 2 * dh), _draw(g, prefix, 2 * dh)
    lengths = [room] * b
    if where == "own":
        _sink(k[1, :room - tq], low)  # (each query sees its own key, which is not one of these)
        _spoil(v[1, :room - tq], dh)
    else:
        _sink(pk[:prefix // 2], low)
        _spoil(pv[:prefix // 2], dh)
    got = ltxk.prefix_attention(q, k, v, pk, pv, 4, 2, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    for i in (0, 1, b - 1):
        want = one_sequence(q[i], torch.cat([pk, k[i]]), torch.cat([pv, v[i]]), 4, 2, prefix=prefix)
        assert_near(got[i], *want, f"item {i}")
    bad = ~got.view(b, tq, 4, dh)[:, :, 0, 3].isfinite()
    assert bool(bad[1].all()) and bool(bad.all()) == (where == "prefix")
