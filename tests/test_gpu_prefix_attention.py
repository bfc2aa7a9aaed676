"""ltxk_prefix_attention against attention of each item in fp64, and with ltxk_packed_attention as they are used (GPU)."""

import pytest
import torch

from attention_reference import assert_near, one_sequence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _draw(g, *shape, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(torch.bfloat16)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check(got, q, k, v, pk, pv, lengths, heads, kv_heads, **kw):
    for b, n in enumerate(lengths):
        want, spread = one_sequence(q[b], torch.cat([pk, k[b, :n]]), torch.cat([pv, v[b, :n]]), heads, kv_heads,
                                    prefix=pk.shape[0], **kw)
        assert_near(got[b], want, spread, f"item {b}")


# queries an item, prefix, room for own keys, lengths, query heads, key heads, head dimension
SHAPES = [
    (1, 1, 1, [1], 1, 1, 64), (1, 333, 128, [1, 126, 40, 128], 16, 8, 256), (1, 64, 5, [0, 5], 4, 4, 128),
    (1, 0, 70, [70, 0, 1], 8, 2, 128), (1, 5000, 300, [300, 1, 64, 65, 200, 8, 9], 32, 4, 64),
    (1, 8200, 40, [33] * 70, 8, 8, 128), (5, 700, 90, [90, 5, 3, 0], 16, 8, 256), (3, 1000, 64, [64] * 40, 7, 1, 128),
    (2, 65, 4000, [4000, 2], 5, 5, 64), (40, 300, 64, [40, 64, 13, 1], 6, 2, 128), (126, 1024, 126, [126, 90, 33], 4, 1, 64),
    (300, 77, 300, [300, 10, 299], 4, 2, 256), (1, 20000, 1, [1], 4, 1, 128), (9, 4290, 30, [30] * 17, 28, 4, 64),
    (17, 0, 200, [200, 3], 3, 3, 256), (1, 3000, 200, [200, 100, 7] * 30, 40, 5, 64), (130, 2000, 130, [130], 8, 2, 128),
]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "open"])
@pytest.mark.parametrize("tq,prefix,room,lengths,heads,kv_heads,dh", SHAPES)
def test_matches_fp64(tq, prefix, room, lengths, heads, kv_heads, dh, causal):
    """What lies past an item's length holds NaN."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(tq * 7 + prefix)
    b = len(lengths)
    q, k, v = _draw(g, b, tq, heads * dh, scale=1.5), _draw(g, b, room, kv_heads * dh), _draw(g, b, room, kv_heads * dh)
    pk, pv = _draw(g, prefix, kv_heads * dh), _draw(g, prefix, kv_heads * dh)
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = float("nan"), float("nan")
    out = torch.full_like(q, 7.0)
    got = ltxk.prefix_attention(q, k, v, pk, pv, heads, kv_heads, _ints(lengths), causal=causal, out=out)
    assert got is out
    _check(got, q, k, v, pk, pv, lengths, heads, kv_heads, causal=causal)


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("b,tq", [(2, 1), (40, 1), (12, 5), (3, 70)])
def test_every_cut_of_a_prefix(b, tq, dh):
    """Prefixes of every number of key tiles, last tiles of every length, cut into parts of every size."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(b)
    pk, pv = _draw(g, 9000, 2 * dh), _draw(g, 9000, 2 * dh)
    q, k, v = _draw(g, b, tq, 4 * dh, scale=1.5), _draw(g, b, 80, 2 * dh), _draw(g, b, 80, 2 * dh)
    lengths = [80, 79] + [70 + i % 9 for i in range(b - 2)]
    for prefix in list(range(1, 2400, 157)) + list(range(2400, 9000, 601)):
        got = ltxk.prefix_attention(q, k, v, pk[:prefix], pv[:prefix], 4, 2, _ints(lengths))
        _check(got[-2:], q[-2:], k[-2:], v[-2:], pk[:prefix], pv[:prefix], lengths[-2:], 4, 2)


@pytest.mark.parametrize("b,tq,prefix,room,heads,kv_heads,dh", [
    (1500, 1, 2000, 20, 4, 2, 128), (300, 3, 3000, 400, 4, 1, 64), (2, 1, 120_000, 9000, 8, 1, 128), (90, 9, 900, 64, 6, 2, 256),
    (1, 700, 5000, 700, 4, 2, 128)])
def test_many_items_and_long_prefixes(b, tq, prefix, room, heads, kv_heads, dh):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(b)
    q, k, v = _draw(g, b, tq, heads * dh, scale=1.5), _draw(g, b, room, kv_heads * dh), _draw(g, b, room, kv_heads * dh)
    pk, pv = _draw(g, prefix, kv_heads * dh), _draw(g, prefix, kv_heads * dh)
    lengths = [(37 * i) % (room + 1) for i in range(b)]
    got = ltxk.prefix_attention(q, k, v, pk, pv, heads, kv_heads, _ints(lengths), out=torch.full_like(q, float("nan")))
    assert bool(got.isfinite().all())
    for i in {0, 1 % b, b - 1, *range(0, b, max(1, b // 12))}:
        _check(got[i:i + 1], q[i:i + 1], k[i:i + 1], v[i:i + 1], pk, pv, lengths[i:i + 1], heads, kv_heads)


@pytest.mark.parametrize("seed", range(30))
def test_any_sizes(seed):
    """Sizes of all magnitudes: each way to share a prefix, to cut it and own keys, and to lay out few and many rows."""
    import random

    import ltxk

    r, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    dh, kv_heads, group = r.choice((64, 128, 256)), r.choice((1, 2, 3, 4, 8, 16)), r.choice((1, 1, 2, 3, 4, 8))
    b, tq = int(2 ** r.uniform(0, 7)), r.choice((1, 1, 1, 2, 5, 9, 30, 70))
    prefix, room = int(2 ** r.uniform(0, 15)) - 1, int(2 ** r.uniform(0, 11)) - 1
    while b * room * kv_heads * dh > 1 << 27:
        room //= 2
    heads, lengths, causal = kv_heads * group, [r.randint(0, room) for _ in range(b)], r.random() < 0.7
    q, k, v = _draw(g, b, tq, heads * dh, scale=1.5), _draw(g, b, room, kv_heads * dh), _draw(g, b, room, kv_heads * dh)
    pk, pv = _draw(g, prefix, kv_heads * dh), _draw(g, prefix, kv_heads * dh)
    got = ltxk.prefix_attention(q, k, v, pk, pv, heads, kv_heads, _ints(lengths), causal, out=torch.full_like(q, float("nan")))
    assert bool(got.isfinite().all())
    for i in {0, b - 1, *range(0, b, max(1, b // 6))}:
        _check(got[i:i + 1], q[i:i + 1], k[i:i + 1], v[i:i + 1], pk, pv, lengths[i:i + 1], heads, kv_heads, causal=causal)


@pytest.mark.parametrize("tq,prefix", [(4, 200), (4, 9000), (150, 200)])
def test_masked_values_may_hold_anything(tq, prefix):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(tq)
    b, room = 5, 200
    q, k, v = _draw(g, b, tq, 512, scale=1.5), _draw(g, b, room, 256), _draw(g, b, room, 256)
    pk, pv = _draw(g, prefix, 256), _draw(g, prefix, 256)
    lengths = [200, 160, 151, 190, 170]
    for i, n in enumerate(lengths):
        v[i, n - 2, 3], v[i, n - 1, 130] = float("nan"), float("inf")  # the last two queries, and the last one, see them
    got = ltxk.prefix_attention(q, k, v, pk, pv, 4, 2, _ints(lengths))
    _check(got, q, k, v, pk, pv, lengths, 4, 2)
    assert bool(got[:, 0].isfinite().all()) and not bool(got[:, -1].isfinite().all())


def test_lengths_and_views():
    """Lengths are cut to the cache; None is all of it; views of wider rows, of a larger cache, and one item's keys for all
    (stride 0) give the same bits."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(2)
    for tq in (1, 40):
        q = _draw(g, 3, tq, 512, scale=1.5)
        cache = _draw(g, 3, 2, 300, 392)
        k, v = cache[:, 1, :150, 8:136], cache[:, 1, :150, 264:]
        wide = _draw(g, 500, 264)
        pk, pv = wide[:, 8:136], wide[:, 136:]
        want = ltxk.prefix_attention(q, k, v, pk, pv, 8, 2)
        assert torch.equal(want, ltxk.prefix_attention(q, k.contiguous(), v.contiguous(), pk.contiguous(), pv.contiguous(), 8, 2,
                                                       _ints([150, 2**31 - 1, 151])))
        _check(want, q, k, v, pk, pv, [150] * 3, 8, 2)
        none = ltxk.prefix_attention(q, k, v, pk, pv, 8, 2, _ints([-5, 0, -2**31]), causal=False)
        _check(none, q, k, v, pk, pv, [0] * 3, 8, 2, causal=False)
        none = ltxk.prefix_attention(q, k[:, :0], v[:, :0], pk, pv, 8, 2, causal=False)  # (a call may be cut by its room)
        _check(none, q, k, v, pk, pv, [0] * 3, 8, 2, causal=False)
        one = ltxk.prefix_attention(q, k[:1].expand(3, 150, 128), v[:1].expand(3, 150, 128), pk, pv, 8, 2, scale=0.25)
        _check(one, q, k[:1].expand(3, 150, 128), v[:1].expand(3, 150, 128), pk, pv, [150] * 3, 8, 2, scale=0.25)
    empty = ltxk.prefix_attention(q, k[:, :0], v[:, :0], pk[:0], pv[:0], 8, 2, causal=False)
    assert empty.shape == q.shape and not bool(empty.any())
    assert ltxk.prefix_attention(q[:0], k[:0], v[:0], pk, pv, 8, 2).shape == (0, 40, 512)


def test_long_prefix_past_32_bit_offsets():
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(3)
    rows, width = 100_000, 24_576  # 4.9 GB
    wide = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    pk, pv = wide[:, :128], wide[:, -128:]
    for x in (pk, pv):
        x.copy_(_draw(g, rows, 128))
    for b, tq in ((2, 1), (70, 1), (2, 130)):
        q, k, v = _draw(g, b, tq, 256, scale=1.5), _draw(g, b, 140, 128), _draw(g, b, 140, 128)
        _check(ltxk.prefix_attention(q, k, v, pk, pv, 4, 2)[:2], q, k, v, pk, pv, [140] * 2, 4, 2)


def test_two_streams_and_two_graphs():
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(4)
    calls = []
    for b, tq, prefix in ((9, 1, 6000), (20, 4, 900)):
        calls.append((_draw(g, b, tq, 512, scale=1.5), _draw(g, b, 80, 256), _draw(g, b, 80, 256), _draw(g, prefix, 256),
                      _draw(g, prefix, 256), 4, 2, torch.randint(0, 80, (b,), device=DEV, generator=g).int()))
    want = [ltxk.prefix_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for _ in range(8):
        for s, c, o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(ltxk.prefix_attention(*c))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(w, x) for x in o)
    graphs = []
    for s, c in zip(streams, calls):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            graphs.append((graph, ltxk.prefix_attention(*c)))
    for i in range(4):
        for c in calls:
            c[0].copy_(torch.randn(c[0].shape, device=DEV, generator=g))
            c[-1].copy_(torch.randint(0, 81, c[-1].shape, device=DEV, generator=g))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), c in zip(graphs, calls):
            assert torch.equal(out, ltxk.prefix_attention(*c)), f"replay {i}"


@pytest.mark.parametrize("heads,kv_heads,dh", [(16, 8, 256), (32, 4, 64), (8, 8, 128)])
def test_prefix_prompts_and_tokens_together(heads, kv_heads, dh):
    """Common instructions once, prompts behind them left-padded, then tokens one at a time, by a cache of each item's own
    and by packed keys: each equals packed attention over the whole sequences."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dh)
    prefix, lengths, more = 200, [31, 64, 7], 3
    room = max(lengths) + more
    rows = [_draw(g, prefix + n + more, (heads + 2 * kv_heads) * dh) for n in lengths]
    for r in rows:
        r[:prefix] = rows[0][:prefix]
    cut = (heads * dh, kv_heads * dh, kv_heads * dh)
    split = [r.split(cut, 1) for r in rows]
    offsets = _ints([0, *torch.tensor([len(r) for r in rows]).cumsum(0).tolist()])
    q, k, v = (torch.cat([s[i] for s in split]) for i in range(3))
    whole = ltxk.packed_attention(q, k, v, heads, offsets, kv_heads)
    ends = [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]
    exact = [one_sequence(*s, heads, kv_heads) for s in split]
    for (a, b), e in zip(ends, exact):
        assert_near(whole[a:b], *e)

    def near(x, i, first, n):  # x stands for rows first .. first + n - 1 of sequence i
        assert_near(x, *(e[first:first + n] for e in exact[i]))

    pq, pk, pv = (x[:prefix] for x in split[0])
    near(ltxk.packed_attention(pq, pk, pv, heads, _ints([0, prefix]), kv_heads), 0, 0, prefix)

    keys, values = (torch.zeros(len(rows), room, kv_heads * dh, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    prompts = torch.zeros(len(rows), max(lengths), heads * dh, dtype=torch.bfloat16, device=DEV)
    for i, (n, s) in enumerate(zip(lengths, split)):
        prompts[i, max(lengths) - n:] = s[0][prefix:prefix + n]
        keys[i, :n], values[i, :n] = s[1][prefix:prefix + n], s[2][prefix:prefix + n]
    got = ltxk.prefix_attention(prompts, keys, values, pk, pv, heads, kv_heads, _ints(lengths))
    for i, n in enumerate(lengths):
        near(got[i, max(lengths) - n:], i, prefix, n)
        assert not bool(got[i, :max(lengths) - n].any())
    for step in range(more):
        now = [n + step for n in lengths]
        token = torch.stack([s[0][prefix + n] for s, n in zip(split, now)])
        for i, (n, s) in enumerate(zip(now, split)):
            keys[i, n], values[i, n] = s[1][prefix + n], s[2][prefix + n]
        got = ltxk.prefix_attention(token[:, None], keys, values, pk, pv, heads, kv_heads, _ints([n + 1 for n in now]))
        upto = [prefix + n + 1 for n in now]
        also = ltxk.packed_attention(token, torch.cat([s[1][:e] for s, e in zip(split, upto)]),
                                     torch.cat([s[2][:e] for s, e in zip(split, upto)]), heads,
                                     _ints(range(len(rows) + 1)), kv_heads,
                                     _ints([0, *torch.tensor(upto).cumsum(0).tolist()]))
        for i, n in enumerate(now):
            near(got[i], i, prefix + n, 1)
            near(also[i:i + 1], i, prefix + n, 1)
