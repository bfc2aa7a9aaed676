"""What packed and prefix attention refuse, before any launch (CPU)."""

import ctypes

import pytest
import torch

P, ODD, BYTE = ctypes.c_void_p(256), ctypes.c_void_p(264), ctypes.c_void_p(257)
BIG = 1 << 40


def _lib():
    import ltxk

    return ltxk, ltxk.load()


def _packed(lib, out=P, q=P, qt=512, k=P, kt=128, v=P, vt=128, offsets=P, k_offsets=P, seqs=2, tq=10, tk=20, heads=8,
            kv_heads=2, dh=64, causal=1, window=0, scale=0.125, ws=P, size=BIG):
    as_ints = [ctypes.cast(x, ctypes.c_void_p) if x is not None else None for x in (offsets, k_offsets)]
    return lib.ltxk_packed_attention(out, q, qt, k, kt, v, vt, *as_ints, seqs, tq, tk, heads, kv_heads, dh, causal, window,
                                     scale, ws, size, None)


def _prefix(lib, out=P, q=P, qb=5120, qt=512, k=P, kb=2560, kt=128, v=P, vb=2560, vt=128, pk=P, pkt=128, pv=P, pvt=128,
            lengths=None, b=2, tq=10, tk=20, prefix=30, heads=8, kv_heads=2, dh=64, causal=1, scale=0.125, ws=P, size=BIG):
    return lib.ltxk_prefix_attention(out, q, qb, qt, k, kb, kt, v, vb, vt, pk, pkt, pv, pvt, lengths, b, tq, tk, prefix,
                                     heads, kv_heads, dh, causal, scale, ws, size, None)


SHARED_ARG = [dict(tq=-1), dict(tk=-1), dict(heads=0), dict(kv_heads=0), dict(heads=-8), dict(kv_heads=-2), dict(kv_heads=3),
              dict(heads=1 << 17, kv_heads=1 << 17), dict(dh=32), dict(dh=0), dict(dh=192), dict(dh=-64), dict(scale=0.0),
              dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(out=None),
              dict(q=None), dict(k=None), dict(v=None), dict(qt=504), dict(kt=120), dict(vt=0), dict(kt=-128),
              dict(vt=(1 << 23) + 8), dict(qt=1 << 62), dict(tq=1 << 28), dict(tk=(1 << 31) - 1), dict(tq=1 << 62),
              dict(tk=1 << 62)]
SHARED_ALIGN = [dict(out=ODD), dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(qt=516), dict(kt=130), dict(vt=131)]


@pytest.mark.parametrize("kw", SHARED_ARG + [dict(seqs=-1), dict(seqs=(1 << 20) + 1), dict(window=-1),
                                             dict(window=5, causal=0), dict(offsets=None), dict(k_offsets=None)])
def test_packed_refuses_arguments(kw):
    ltxk, lib = _lib()
    assert _packed(lib, **kw) == ltxk.E_ARG and ltxk.last_error().startswith("packed_attention")


@pytest.mark.parametrize("kw", SHARED_ALIGN + [dict(offsets=BYTE), dict(k_offsets=BYTE)])
def test_packed_refuses_alignments(kw):
    ltxk, lib = _lib()
    assert _packed(lib, **kw) == ltxk.E_ALIGN


@pytest.mark.parametrize("kw", SHARED_ARG + [dict(b=-1), dict(b=(1 << 20) + 1), dict(prefix=-1), dict(prefix=1 << 31),
                                             dict(prefix=1 << 62), dict(pk=None), dict(pv=None), dict(pkt=120),
                                             dict(pvt=1 << 24), dict(b=1 << 20, tq=1 << 10)])
def test_prefix_refuses_arguments(kw):
    ltxk, lib = _lib()
    assert _prefix(lib, **kw) == ltxk.E_ARG and ltxk.last_error().startswith("prefix_attention")


@pytest.mark.parametrize("kw", SHARED_ALIGN + [dict(pk=ODD), dict(pv=ODD), dict(pkt=132), dict(qb=5124), dict(kb=-8),
                                               dict(vb=4), dict(lengths=BYTE)])
def test_prefix_refuses_alignments(kw):
    ltxk, lib = _lib()
    assert _prefix(lib, **kw) == ltxk.E_ALIGN


def test_no_work_is_no_error():
    _, lib = _lib()
    assert _packed(lib, seqs=0, out=None, q=None) == 0 and _packed(lib, tq=0, out=None, q=None) == 0
    assert _prefix(lib, b=0, out=None, q=None) == 0 and _prefix(lib, tq=0, out=None, q=None) == 0


def test_binding_refuses_what_is_not_on_the_device():
    ltxk, _ = _lib()
    q, k = torch.zeros(4, 512, dtype=torch.bfloat16), torch.zeros(4, 128, dtype=torch.bfloat16)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ltxk.packed_attention(q, k, k, 8, offsets, 2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ltxk.prefix_attention(q[None], k[None], k[None], k, k, 8, 2)
    with pytest.raises(ValueError, match="not a multiple"):
        ltxk.packed_attention(q, k, k, 8, offsets, 3)
    with pytest.raises(ValueError, match="not a multiple"):
        ltxk.prefix_attention(q[None], k[None], k[None], k, k, 8, 0)
    with pytest.raises(ValueError, match="heads of 64, 128 or 256"):
        ltxk.packed_attention(q, k, k, 16, offsets, 2)
    with pytest.raises(ValueError, match="tensor"):
        ltxk.packed_attention(q[None], k, k, 8, offsets, 2)
    with pytest.raises(ValueError, match="tensors"):
        ltxk.prefix_attention(q, k, k, k, k, 8, 2)


def _gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


@pytest.mark.gpu
def test_binding_refuses_tensors():
    ltxk, _ = _lib()
    q, k, o = _gpu(6, 512), _gpu(6, 128), _gpu(3, dtype=torch.int32)

    def packed(err, match, q=q, k=k, v=k, heads=8, offsets=o, kv_heads=2, **kw):
        with pytest.raises(err, match=match):
            ltxk.packed_attention(q, k, v, heads, offsets, kv_heads, **kw)

    packed(ValueError, "dtype", q=q.float())
    packed(ValueError, "dtype", k=k.half())
    packed(ValueError, "expected", k=_gpu(6, 64))
    packed(ValueError, "5 values", v=k[:5])
    packed(ValueError, "need k_offsets", k=_gpu(7, 128), v=_gpu(7, 128))
    packed(ValueError, "contiguous", q=_gpu(512, 6).t())
    packed(ValueError, "multiple of 8", k=_gpu(6, 132)[:, :128])
    packed(ValueError, "cover", v=_gpu(128)[None].expand(6, 128))
    packed(ValueError, "dtype", offsets=o.long())
    packed(ValueError, "sequences", offsets=o[:0])
    packed(ValueError, "sequences", offsets=o[None])
    packed(ValueError, "must be", k_offsets=_gpu(4, dtype=torch.int32))
    packed(RuntimeError, "ROCm device", offsets=o.cpu())
    packed(ValueError, "window", window=0)
    packed(ValueError, "window", window=4, causal=False)
    packed(RuntimeError, "positive and finite", scale=float("nan"))
    packed(ValueError, "out", out=_gpu(5, 512))
    packed(ValueError, "dtype", out=_gpu(6, 512).float())
    packed(RuntimeError, "misaligned", q=_gpu(6 * 512 + 4)[4:].view(6, 512))

    b = dict(q=_gpu(2, 3, 512), k=_gpu(2, 6, 128), v=_gpu(2, 6, 128), prefix_k=_gpu(9, 128), prefix_v=_gpu(9, 128))

    def prefix(err, match, heads=8, kv_heads=2, lengths=None, out=None, **kw):
        with pytest.raises(err, match=match):
            ltxk.prefix_attention(**{**b, **kw}, heads=heads, kv_heads=kv_heads, lengths=lengths, out=out)

    prefix(ValueError, "expected", k=_gpu(3, 6, 128))
    prefix(ValueError, "expected", v=_gpu(2, 5, 128))
    prefix(ValueError, "expected", prefix_k=_gpu(2, 9, 128))
    prefix(ValueError, "8 values", prefix_v=_gpu(8, 128))
    prefix(ValueError, "dtype", prefix_v=_gpu(9, 128).float())
    prefix(ValueError, "dtype", lengths=_gpu(2, dtype=torch.int64))
    prefix(ValueError, "must be", lengths=_gpu(3, dtype=torch.int32))
    prefix(ValueError, "out", out=_gpu(2, 2, 512))
    prefix(TypeError, "Tensor", prefix_k=None)


@pytest.mark.parametrize("kw", [dict(tq=1 << 62), dict(tk=1 << 62), dict(items=1 << 62), dict(heads=1 << 62), dict(kv_heads=3),
                                dict(head_dim=96), dict(tq=0), dict(tq=-1), dict(items=0), dict(prefix=1 << 62), dict(kv_heads=0)])
def test_workspaces_of_refused_sizes(kw):
    """A size that a call refuses needs none, however large: no sum or quotient of it is taken."""
    _, lib = _lib()
    a = {**dict(items=4, tq=8, tk=4096, prefix=1 << 16, heads=8, kv_heads=2, head_dim=128), **kw}
    assert lib.ltxk_prefix_attention_workspace_bytes(a["items"], a["tq"], a["tk"], a["prefix"], a["heads"], a["kv_heads"],
                                                     a["head_dim"]) == 0
    if "prefix" not in kw:
        assert lib.ltxk_packed_attention_workspace_bytes(a["tq"], a["tk"], a["items"], a["heads"], a["kv_heads"],
                                                         a["head_dim"]) == 0
    assert lib.ltxk_prefix_attention_workspace_bytes(4, 8, 4096, 1 << 16, 8, 2, 128) > 0
