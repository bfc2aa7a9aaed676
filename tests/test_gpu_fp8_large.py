"""8-bit operands and results just below 2^31 values (GPU): rows that repeat give results that repeat, all of them, and
the first ones against fp64."""

import pytest
import torch

from test_gpu_fp8 import _exact_blocks, _gelu64, _near_blocks

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16
PERIOD = 1021  # of the rows: no tile's


def _repeated(base, rows):
    import ltxk

    index = torch.arange(rows, device=DEV) % base.rows
    data = base.data.view(torch.uint8).index_select(0, index).view(torch.float8_e4m3fn)
    return ltxk.Fp8Blocks(data, base.scale.index_select(1, index), (rows, base.shape[-1]))


def _repeats(big, small, dim=0):
    """big is `small` over and over along `dim`."""
    period, n = small.shape[dim], big.shape[dim]
    whole = n // period * period
    first = big.narrow(dim, 0, whole).unflatten(dim, (whole // period, period))
    for i in range(first.shape[dim]):  # a piece at a time: no second tensor of this size
        if not torch.equal(first.select(dim, i), small):
            return False
    return torch.equal(big.narrow(dim, whole, n - whole), small.narrow(dim, 0, n - whole))


@pytest.mark.parametrize("m,n,k", [(524287, 8, 4096), (524287, 256, 4096), (100, 524280, 4096), (4, 524280, 4096),
                                   (65535, 32768, 128), (65535, 32760, 264)])
def test_products_of_nearly_2_31_values(m, n, k):
    """Many rows of x, many columns, a large result; with GELU, too."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + n)
    xs, ws = (_exact_blocks(min(rows, PERIOD), k, g) for rows in (m, n))
    x, w = _repeated(xs, m), _repeated(ws, n)
    assert (1 << 31) - (1 << 18) < max(x.data.numel(), w.data.numel(), m * -(-n // 128) * 128) < 1 << 31
    sums = xs.float().double() @ ws.float().double().t().contiguous()
    y = ltxk.linear_fp8(x, w)
    assert _repeats(y, y[:xs.rows]) and _repeats(y[:xs.rows], sums.to(BF16), 1)
    del y
    got = ltxk.linear_gelu_fp8(x, w)
    first = ltxk.Fp8Blocks(got.data[:xs.rows].contiguous(), got.scale[:, :xs.rows].contiguous(), (xs.rows, n))
    assert _repeats(got.data.view(torch.uint8), first.data.view(torch.uint8)) and _repeats(got.scale, first.scale, 1)
    want = _gelu64(sums)
    want = want[:, torch.arange(n, device=DEV) % ws.rows]
    _near_blocks(first, want, want.abs() * 2.0**-20 + 2.0**-24)  # sums that fp32 holds: GELU's own evaluation


def test_rows_of_nearly_2_31_values():
    """Quantising and the norms that write blocks."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(1)
    m, k = 524287, 4096
    small, f = (torch.randn(1, PERIOD, k, device=DEV, generator=g).to(BF16) for _ in range(2))
    index = torch.arange(m, device=DEV) % PERIOD
    x = small.index_select(1, index)
    got, want = ltxk.quantize_fp8(x), ltxk.quantize_fp8(small)
    assert _repeats(got.data.view(torch.uint8), want.data.view(torch.uint8)) and _repeats(got.scale, want.scale, 1)
    del got
    scale = ltxk.AdaRef(torch.randn(1, k, device=DEV, generator=g).to(BF16), 0)
    fs = f.index_select(1, index)
    out, got = ltxk.add_norm_modulate_fp8(x, fs, scale=scale)
    want_out, want = ltxk.add_norm_modulate_fp8(small, f, scale=scale)
    assert _repeats(out[0], want_out[0])
    assert _repeats(got.data.view(torch.uint8), want.data.view(torch.uint8)) and _repeats(got.scale, want.scale, 1)
