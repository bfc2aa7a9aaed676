"""What the 8-bit layers and cross attention refuse, before any launch (CPU)."""

import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _lib():
    import ltxk

    return ltxk, ltxk.load()


def test_quantize_refusals():
    ltxk, lib = _lib()
    for rows, k in ((-1, 64), (4, 0), (4, -8), (4, 12)):
        assert lib.ltxk_quantize_fp8(P, P, P, rows, k, None) == ltxk.E_ARG
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert lib.ltxk_quantize_fp8(*args, 4, 64, None) == ltxk.E_ARG and "null" in ltxk.last_error()
    for args in ((ODD, P, P), (P, ODD, P), (P, P, ODD)):
        assert lib.ltxk_quantize_fp8(*args, 4, 64, None) == ltxk.E_ALIGN
    for rows, k in ((1 << 24, 8), (1, 1 << 31), (1 << 20, 2048), (1 << 62, 8), (1, 1 << 62)):
        assert lib.ltxk_quantize_fp8(P, P, P, rows, k, None) == ltxk.E_ARG and "2^31" in ltxk.last_error()
    assert lib.ltxk_quantize_fp8(None, None, None, 0, 64, None) == 0


def test_norm_refusals():
    ltxk, lib = _lib()

    def call(x_out=P, q=P, qs=P, x=P, f=P, gate=None, mask=None, rows=4, tokens=4, dim=64, shift=None):
        return lib.ltxk_add_norm_modulate_fp8(x_out, q, qs, x, f, gate, mask, rows, tokens, dim, 1e-6, shift, None, None)

    for kw in (dict(rows=-1), dict(tokens=0), dict(dim=0), dict(dim=12), dict(dim=16392), dict(rows=5), dict(q=None),
               dict(qs=None), dict(x=None), dict(f=None), dict(x_out=None), dict(x_out=None, f=None, mask=P),
               dict(rows=1 << 24, tokens=1)):
        assert call(**kw) == ltxk.E_ARG, kw
    for kw in (dict(x=ODD), dict(q=ODD), dict(x_out=ODD), dict(f=ODD), dict(mask=ctypes.c_void_p(257)),
               dict(shift=ctypes.byref(ltxk.Ada(264, None, 0, 0, None, 0)))):
        assert call(**kw) == ltxk.E_ALIGN, kw
    assert call(shift=ctypes.byref(ltxk.Ada(None, 256, 0, 64, 256, 0))) == ltxk.E_ARG and "emb_rows" in ltxk.last_error()
    assert call(rows=0) == 0


@pytest.mark.parametrize("gelu", [False, True])
def test_linear_refusals(gelu):
    ltxk, lib = _lib()

    def call(y=P, ys=P, ops=(P, P, P, P), bias=None, m=4, n=16, k=64, ws=P, size=1 << 40):
        if gelu:
            return lib.ltxk_linear_gelu_fp8(y, ys, *ops, bias, m, n, k, ws, size, None)
        return lib.ltxk_linear_fp8(y, *ops, bias, m, n, k, ws, size, None)

    for kw in (dict(m=-1), dict(n=0), dict(k=0), dict(n=12), dict(k=20), dict(y=None)):
        assert call(**kw) == ltxk.E_ARG, kw
    for i in range(4):
        ops = [P] * 4
        ops[i] = None
        if i != 1:  # without scales x is bf16
            assert call(ops=ops) == ltxk.E_ARG and "null" in ltxk.last_error()
        ops[i] = ODD
        assert call(ops=ops) == ltxk.E_ALIGN
    assert call(bias=ODD) == ltxk.E_ALIGN and call(y=ODD) == ltxk.E_ALIGN
    for m, n, k in ((1 << 24, 16, 64), (1, 1 << 24, 64), (1 << 16, 1 << 15, 64), (1, 8, 1 << 31), (1, 1 << 31, 8),
                    (1 << 62, 8, 8)):
        assert call(m=m, n=n, k=k) == ltxk.E_ARG and "2^3" in ltxk.last_error(), (m, n, k)
    assert call(m=0) == 0
    for m, n, k in ((4, 16, 64), (126, 2048, 2048), (1024, 4096, 4096)):
        for quantize in (0, 1):
            need = lib.ltxk_linear_fp8_workspace_bytes(m, n, k, int(gelu), quantize)
            assert need >= 0
            if need:
                for kw in (dict(ws=None), dict(size=need - 1), dict(ws=ODD)):
                    kw["ops"] = (P, None if quantize else P, P, P)
                    assert call(m=m, n=n, k=k, **kw) == ltxk.E_ARG and "workspace" in ltxk.last_error()
    assert lib.ltxk_linear_fp8_workspace_bytes(0, 16, 64, 1, 1) == 0
    assert lib.ltxk_linear_fp8_workspace_bytes(1 << 40, 16, 1 << 40, 1, 1) == 0


def test_cross_attention_refusals():
    ltxk, lib = _lib()

    def call(keep=P, kb=100, out=P, q=P, row=128, b=2, tq=4, tk=100, h=2, dh=64, scale=0.125, ws=P, size=1 << 40):
        return lib.ltxk_cross_attention(out, q, tq * row, row, P, tk * row, row, P, tk * row, row, keep, kb, None, b, tq,
                                        tk, h, dh, scale, ws, size, None)

    for kw in (dict(kb=-1), dict(dh=96), dict(h=0), dict(b=-1), dict(tk=0), dict(scale=0.0),
               dict(scale=float("nan")), dict(out=None), dict(row=64), dict(tk=1 << 24)):
        assert call(**kw) == ltxk.E_ARG, kw
    assert call(q=ODD) == ltxk.E_ALIGN and call(row=132) == ltxk.E_ALIGN
    for tk in (4096, 9000):
        need = lib.ltxk_cross_attention_workspace_bytes(2, 4, tk, 2, 64)
        assert need >= lib.ltxk_attention_workspace_bytes(2, 4, tk, 2, 64) > 0
        for kw in (dict(ws=None), dict(size=need - 1), dict(ws=ODD), dict(keep=None, ws=None)):
            assert call(tk=tk, **kw) == ltxk.E_ARG and "workspace" in ltxk.last_error()
    assert call(tq=0) == 0 and call(b=0) == 0


def test_binding_refuses_before_the_device():
    import ltxk

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: ltxk.quantize_fp8(x), lambda: ltxk.norm_modulate_fp8(x),
                 lambda: ltxk.add_norm_modulate_fp8(x, x), lambda: ltxk.cross_attention(x[None], x[None], x[None], 1)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="needs f"):
        ltxk.add_norm_modulate_fp8(x, None)
    with pytest.raises(TypeError, match="Fp8Blocks"):
        ltxk.linear_fp8(x, x)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ltxk.Fp8Blocks(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 4, 4, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="tensors"):
        ltxk.cross_attention(x, x, x, 1)


def test_blocks_refuse_negative_sizes():
    """Two of them multiply to a count of rows that fits."""
    import ltxk

    blocks = ltxk.Fp8Blocks._made((6, 64), "cpu")
    assert blocks.view(2, 3, 64).shape == (2, 3, 64) and blocks.view(1, 6, 64).rows == 6
    for shape in ((-2, -3, 64), (-1, -6, 64), (-1, 64), (5, 64), (6, 128), ()):
        with pytest.raises(ValueError, match="no view"):
            blocks.view(*shape)
