"""ltxk_packed_attention against attention of each sequence in fp64 (GPU)."""

import pytest
import torch

from attention_reference import assert_near, one_sequence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _offsets(counts, start=0):
    at = [start]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _draw(g, rows, width, scale=1.0):
    return (torch.randn(rows, width, device=DEV, generator=g) * scale).to(torch.bfloat16)


def _check(got, q, k, v, qo, ko, heads, kv_heads, **kw):
    qo, ko = qo.tolist(), ko.tolist()
    for s in range(len(qo) - 1):
        want, spread = one_sequence(q[qo[s]:qo[s + 1]], k[ko[s]:ko[s + 1]], v[ko[s]:ko[s + 1]], heads, kv_heads, **kw)
        assert_near(got[qo[s]:qo[s + 1]], want, spread, f"sequence {s}")


# queries and keys of each sequence (None: as many), query heads, key heads, head dimension
SHAPES = [
    ([1], None, 1, 1, 64), ([5, 126], None, 16, 8, 256), ([0, 1, 0, 64, 65, 0], None, 4, 4, 128),
    ([127, 128, 129], None, 3, 3, 64), ([33, 31, 32, 500], None, 8, 1, 128), ([700, 3], None, 6, 2, 256),
    ([17, 300, 257, 1, 1, 1, 90], None, 14, 2, 128), ([1] * 70, None, 5, 5, 64), ([1100], None, 4, 2, 128),
    # queries behind earlier keys, keys alone, and queries without (all of their) keys
    ([1] * 9, [1, 63, 64, 65, 0, 1000, 2, 128, 4100], 8, 2, 128), ([5, 1, 40], [700, 64, 41], 6, 1, 64),
    ([3, 0, 7], [5000, 20, 7], 32, 4, 256), ([1], [20000], 4, 1, 64), ([70, 70], [10, 0], 2, 1, 128),
    ([2] * 40, [333] * 40, 7, 1, 256), ([1, 1], [9000, 1], 40, 5, 64), ([600, 1, 1], [600, 3000, 40], 8, 8, 64),
    ([40] * 3, [40, 2000, 90], 4, 1, 128),
]
MASKS = [dict(causal=True), dict(causal=False), dict(causal=True, window=1), dict(causal=True, window=100)]


@pytest.mark.parametrize("mask", MASKS, ids=["causal", "open", "window1", "window100"])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,dh", SHAPES)
def test_matches_fp64(queries, keys, heads, kv_heads, dh, mask):
    """Rows before the first and behind the last sequence hold NaN, and out's are left as they were."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(sum(queries) * 7 + dh)
    qo, ko = _offsets(queries, 3), _offsets(keys or queries, 3)
    tq, tk = int(qo[-1]) + 5, int(ko[-1]) + 5
    q, k, v = _draw(g, tq, heads * dh, 1.5), _draw(g, tk, kv_heads * dh), _draw(g, tk, kv_heads * dh)
    for x, o in ((q, qo), (k, ko), (v, ko)):
        x[:3], x[int(o[-1]):] = float("nan"), float("nan")
    out = torch.full_like(q, 7.0)
    got = ltxk.packed_attention(q, k, v, heads, qo, kv_heads, None if keys is None else ko, out=out, **mask)
    assert got is out
    _check(got, q, k, v, qo, ko, heads, kv_heads, **mask)
    assert bool((got[:3] == 7).all()) and bool((got[int(qo[-1]):] == 7).all())


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("mask", [dict(causal=True), dict(causal=True, window=50)], ids=["causal", "window"])
def test_masked_values_may_hold_anything(dh, mask):
    """NaN and infinities among keys and values reach the queries that see them and no others."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dh)
    for queries, keys in (([300, 90], [300, 90]), ([3, 40], [3000, 200]), ([100], [2000])):
        qo, ko = _offsets(queries), _offsets(keys)
        q, k, v = _draw(g, sum(queries), 4 * dh, 1.5), _draw(g, sum(keys), 2 * dh), _draw(g, sum(keys), 2 * dh)
        late = int(ko[1]) - 2  # the first sequence's last query but one sees it, and the last one
        v[late, 3], v[late, dh + 5] = float("nan"), float("inf")
        v[int(ko[-1]) - 60, 7] = float("-inf")
        got = ltxk.packed_attention(q, k, v, 4, qo, 2, ko, **mask)
        _check(got, q, k, v, qo, ko, 4, 2, **mask)
        assert bool(got[0].isfinite().all()) and not bool(got[queries[0] - 1].isfinite().all())
        k[late] = float("nan")  # the score of a masked key counts as little
        got = ltxk.packed_attention(q, k, v, 4, qo, 2, ko, **mask)
        _check(got, q, k, v, qo, ko, 4, 2, **mask)
        assert bool(got[queries[0] - 2:queries[0]].isnan().all())


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("queries,heads", [([1, 1], 2), ([9, 40], 4), ([300], 2), ([1] * 30, 8)])
def test_every_cut_of_the_keys(queries, heads, dh):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(heads)
    q = _draw(g, sum(queries), heads * dh, 1.5)
    for most in list(range(1, 2400, 157)) + list(range(2400, 9000, 601)):
        keys = [most * (i + 1) // len(queries) for i in range(len(queries))]
        k, v = _draw(g, sum(keys), 2 * dh), _draw(g, sum(keys), 2 * dh)
        qo, ko = _offsets(queries), _offsets(keys)
        got = ltxk.packed_attention(q, k, v, heads, qo, 2, ko)
        for s in {0, len(queries) - 1}:
            rows, at = slice(int(qo[s]), int(qo[s + 1])), slice(int(ko[s]), int(ko[s + 1]))
            assert_near(got[rows], *one_sequence(q[rows], k[at], v[at], heads, 2), f"{most} keys, sequence {s}")


@pytest.mark.parametrize("queries,keys,heads,kv_heads,dh", [
    ([1, 0, 2] * 1700, None, 4, 2, 64), ([0] * 4100 + [5] + [0] * 4100 + [3], None, 2, 1, 128),
    ([1] * 100 + [2000], [700] * 100 + [2000], 8, 2, 128), ([900] + [1] * 60, [900] + [50, 6000] * 30, 4, 4, 64),
    ([1], [150_000], 2, 1, 64), ([2], [40_000], 3, 1, 256), ([1] * 3, [100_000, 3, 40_000], 8, 8, 128)])
def test_many_and_unequal_sequences(queries, keys, heads, kv_heads, dh):
    """Thousands of sequences, most of them empty; one prompt among single tokens; keys in hundreds of parts."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(len(queries))
    qo, ko = _offsets(queries), _offsets(keys or queries)
    q, k, v = _draw(g, sum(queries), heads * dh, 1.5), _draw(g, int(ko[-1]), kv_heads * dh), _draw(g, int(ko[-1]), kv_heads * dh)
    out = torch.full_like(q, float("nan"))
    got = ltxk.packed_attention(q, k, v, heads, qo, kv_heads, None if keys is None else ko, out=out)
    assert bool(got.isfinite().all())
    at, kt = qo.tolist(), ko.tolist()
    some = [s for s, n in enumerate(queries) if n]
    for s in {*some[:6], *some[-6:], *some[:: max(1, len(some) // 20)]}:
        rows, cols = slice(at[s], at[s + 1]), slice(kt[s], kt[s + 1])
        assert_near(got[rows], *one_sequence(q[rows], k[cols], v[cols], heads, kv_heads), f"sequence {s}")


@pytest.mark.parametrize("seed", range(30))
def test_any_sizes(seed):
    """Sizes of all magnitudes, with more keys than queries, fewer, and none, in every mask."""
    import random

    import ltxk

    r, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    dh, kv_heads, group = r.choice((64, 128, 256)), r.choice((1, 2, 3, 4, 8, 16)), r.choice((1, 1, 2, 3, 4, 8))
    seqs, causal = int(2 ** r.uniform(0, 7)), r.random() < 0.7
    most_q, most_k = r.choice((1, 3, 40, 700)), int(2 ** r.uniform(1, 12))
    queries = [r.randint(0, most_q) for _ in range(seqs)]
    keys = [r.randint(0, most_k) + (n if r.random() < 0.8 else 0) for n in queries]
    heads, qo, ko = kv_heads * group, _offsets(queries), _offsets(keys)
    kw = dict(causal=causal, window=r.choice((None, None, 1, 37, 500)) if causal else None)
    q, k, v = _draw(g, sum(queries), heads * dh, 1.5), _draw(g, sum(keys), kv_heads * dh), _draw(g, sum(keys), kv_heads * dh)
    got = ltxk.packed_attention(q, k, v, heads, qo, kv_heads, ko, out=torch.full_like(q, float("nan")), **kw)
    assert bool(got.isfinite().all())
    at, kt = qo.tolist(), ko.tolist()
    for s in {0, seqs - 1, *range(0, seqs, max(1, seqs // 8))}:
        rows, cols = slice(at[s], at[s + 1]), slice(kt[s], kt[s + 1])
        assert_near(got[rows], *one_sequence(q[rows], k[cols], v[cols], heads, kv_heads, **kw), f"sequence {s}")


def test_views_scale_and_equal_offsets():
    """Columns of one projection's rows, and lengths shared by queries and keys, give the same bits; a scale of its own."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(3)
    wide = _draw(g, 333, 8 * 64 + 2 * 2 * 64 + 24)
    q, k, v = wide[:, 8:520], wide[:, 520:648], wide[:, 656:784]
    offsets = _offsets([200, 0, 133])
    got = ltxk.packed_attention(q, k, v, 8, offsets, 2)
    assert torch.equal(got, ltxk.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), 8, offsets, 2, offsets.clone()))
    _check(got, q, k, v, offsets, offsets, 8, 2)
    _check(ltxk.packed_attention(q, k, v, 8, offsets, 2, scale=1.0), q, k, v, offsets, offsets, 8, 2, scale=1.0)


@pytest.mark.parametrize("scale", [300.0, 3e4])
def test_large_scores(scale):
    """Scores of thousands and more: the largest weight is one."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = ((torch.randint(-3, 4, (200, 128), device=DEV, generator=g) * s).to(torch.bfloat16) for s in (scale, 1, 1))
    offsets = _offsets([150, 50])
    got = ltxk.packed_attention(q, k, v, 2, offsets, scale=0.125)
    score = max((q[:, h].double() @ k[:, h].double().t()).abs().max().item() * 0.125 for h in (slice(0, 64), slice(64, 128)))
    assert score > 4096
    for rows in (slice(0, 150), slice(150, 200)):
        assert_near(got[rows], *one_sequence(q[rows], k[rows], v[rows], 2, 2, scale=0.125), score=score)


def test_offsets_are_cut_to_the_tensors():
    """Entries outside the tensors name their ends; no sequences, no queries and no keys are no work."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = _draw(g, 90, 256), _draw(g, 200, 128), _draw(g, 200, 128)

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    want = ltxk.packed_attention(q, k, v, 4, ints(0, 40, 90), 2, ints(0, 100, 200))
    assert torch.equal(want, ltxk.packed_attention(q, k, v, 4, ints(-9, 40, 2**31 - 1), 2, ints(-2**31, 100, 2**30)))
    out = torch.full_like(q, 7.0)
    assert bool((ltxk.packed_attention(q, k, v, 4, ints(0), 2, ints(0), out=out) == 7).all())
    assert bool((ltxk.packed_attention(q, k, v, 4, ints(0, 0, 0), 2, ints(0, 100, 200), out=out) == 7).all())
    assert bool((ltxk.packed_attention(q, k, v, 4, ints(60, 20), 2, ints(0, 100), out=out) == 7).all())  # not ascending
    assert not bool(ltxk.packed_attention(q, k[:0], v[:0], 4, ints(0, 90), 2, ints(0, 0)).any())
    assert ltxk.packed_attention(q[:0], k, v, 4, ints(0, 0), 2, ints(0, 200)).shape == (0, 256)


def test_keys_past_32_bit_offsets():
    """Keys and values in rows of 48 KB: those of the last sequences, and the end of a long one, lie past 2^32 bytes."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(6)
    rows, width = 100_000, 24_576  # 4.9 GB
    wide = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    k, v = wide[:, :128], wide[:, -128:]
    for x in (k, v):
        x.copy_(_draw(g, rows, 128))
    for queries, keys in (([3, 40, 1], [90_000, 5000, 5000]), ([200], [100_000])):
        q = _draw(g, sum(queries), 4 * 64, 1.5)
        qo, ko = _offsets(queries), _offsets(keys)
        _check(ltxk.packed_attention(q, k, v, 4, qo, 2, ko), q, k, v, qo, ko, 4, 2)


def test_two_streams_and_two_graphs():
    """Calls on two streams, and graphs replayed in turn with new lengths, equal the eager calls."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(7)
    calls = []
    for lengths, keys in (([1] * 6, [900, 10, 5000, 64, 1, 25]), ([100, 28, 0, 72], [200, 2700, 1, 99])):
        q, k, v = _draw(g, sum(lengths), 512, 1.5), _draw(g, sum(keys), 256), _draw(g, sum(keys), 256)
        calls.append((q, k, v, 4, _offsets(lengths), 2, _offsets(keys)))
    want = [ltxk.packed_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for _ in range(8):
        for s, c, o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(ltxk.packed_attention(*c))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(w, x) for x in o)
    graphs = []
    for s, c in zip(streams, calls):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            graphs.append((graph, ltxk.packed_attention(*c)))
    for i in range(4):
        for q, _, _, _, _, _, ko in calls:
            q.copy_(torch.randn(q.shape, device=DEV, generator=g))
            ko[1:-1] = torch.sort(torch.randint(0, int(ko[-1]), (len(ko) - 2,), device=DEV, generator=g)).values.int()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), c in zip(graphs, calls):
            assert torch.equal(out, ltxk.packed_attention(*c)), f"replay {i}"
