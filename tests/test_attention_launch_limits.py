"""Sizes of packed and prefix attention that come near what a launch holds."""

import pytest
import torch

from attention_reference import assert_near, one_sequence
from test_packed_refusals import _lib, _packed, _prefix


@pytest.mark.parametrize("sizes", [(32768, 64, 64, 4096, 32, 32, 64), (1 << 20, 1, 40, 4096, 64, 8, 64),
                                   (1 << 20, 2, 0, 600, 64, 4, 128), (1 << 20, 1, 7, 8192, 64, 8, 256),
                                   (1 << 20, 1, 4, 4096, 64, 1, 64)])
def test_large_batches_do_not_share_a_prefix(sizes):
    """(batch, tokens_q, tokens_k, prefix, heads, kv_heads, head_dim) whose rows are too many to join need no workspace;
    a hundredth of the items share it."""
    _, lib = _lib()
    assert lib.ltxk_prefix_attention_workspace_bytes(*sizes) == 0
    assert lib.ltxk_prefix_attention_workspace_bytes(sizes[0] // 100, *sizes[1:]) > 0


# 2^24 workgroups and more, where the header's bound ends
PACKED = [(1 << 20, 1 << 20, 16, 16, 64), (1 << 20, 1 << 20, 64, 64, 128), (1 << 25, 1 << 20, 16, 16, 64),
          (1, 1 << 20, 1 << 16, 1 << 16, 64)]
PREFIX = [(1 << 20, 1, 16, 16, 64), (1 << 20, 16, 32, 32, 256), (1 << 20, 2, 256, 16, 128)]


@pytest.mark.parametrize("tq,seqs,heads,kv_heads,dh", PACKED)
def test_packed_launches_past_2_to_32_threads_are_refused(tq, seqs, heads, kv_heads, dh):
    """By the call, whatever workspace it is given, and by the workspace's size, which is 0 then."""
    ltxk, lib = _lib()
    assert tq * heads // 32 + (seqs + 7) * kv_heads >= 1 << 24
    assert lib.ltxk_packed_attention_workspace_bytes(tq, tq, seqs, heads, kv_heads, dh) == 0
    strides = dict(qt=heads * dh, kt=kv_heads * dh, vt=kv_heads * dh)
    assert _packed(lib, seqs=seqs, tq=tq, tk=tq, heads=heads, kv_heads=kv_heads, dh=dh, **strides) == ltxk.E_ARG
    assert "too many row tiles" in ltxk.last_error()


@pytest.mark.parametrize("b,tq,heads,kv_heads,dh", PREFIX)
def test_prefix_launches_past_2_to_32_threads_are_refused(b, tq, heads, kv_heads, dh):
    ltxk, lib = _lib()
    assert b * tq * heads // 32 + (b + 7) * kv_heads >= 1 << 24
    for prefix in (0, 30, 9000):
        assert lib.ltxk_prefix_attention_workspace_bytes(b, tq, 20, prefix, heads, kv_heads, dh) == 0
        wide, narrow = heads * dh, kv_heads * dh
        assert _prefix(lib, b=b, tq=tq, tk=20, prefix=prefix, heads=heads, kv_heads=kv_heads, dh=dh, qt=wide, kt=narrow,
                       vt=narrow, pkt=narrow, pvt=narrow) == ltxk.E_ARG
        assert "too many row tiles" in ltxk.last_error()


@pytest.mark.gpu
def test_a_million_items_behind_a_prefix():
    """2^26 rows, which are too many to join: the prefix is not shared, and the call is taken."""
    import ltxk

    dev, (b, heads, dh, prefix, room) = torch.device("cuda"), (1 << 20, 64, 64, 700, 3)
    g = torch.Generator(device=dev).manual_seed(1)

    def draw(*shape):
        return torch.randn(*shape, device=dev, generator=g).to(torch.bfloat16)

    pk, pv, lengths = draw(prefix, dh), draw(prefix, dh), torch.randint(1, room + 1, (b,), device=dev, generator=g).int()
    q = torch.empty(b, 1, heads * dh, dtype=torch.bfloat16, device=dev)
    for part in q.split(1 << 16):
        part.copy_(draw(*part.shape))
    k, v = draw(b, room, dh), draw(b, room, dh)
    got = ltxk.prefix_attention(q, k, v, pk, pv, heads, 1, lengths)
    for i in (0, 1, 77777, b // 2, b - 2, b - 1):
        n = int(lengths[i])
        want = one_sequence(q[i], torch.cat([pk, k[i, :n]]), torch.cat([pv, v[i, :n]]), heads, 1, prefix=prefix)
        assert_near(got[i], *want, f"item {i}")
