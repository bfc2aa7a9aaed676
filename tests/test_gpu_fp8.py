"""Blocks of 128 e4m3 values (csrc/fp8_rows.hip) and the 8-bit linear layers
(csrc/gemm_fp8.hip) against the format and the products in fp64 (GPU)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F64 = torch.float64


def _grid():
    """The non-negative finite e4m3 values in order (the byte's own), in fp64."""
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).to(F64)


def _exponent(top):
    """The least e with top <= 448 * 2^e, at least -127, for a tensor of magnitudes in fp64."""
    e = torch.full_like(top, -127)
    for i in range(-127, 128):
        e = torch.where(top > 448 * 2.0**i, i + 1, e)
    return e


def _blocks_ref(x):
    """(values, exponents) of x (rows, k) fp64 on the CPU: the nearest grid value, halves to the even byte."""
    rows, k = x.shape
    grid = _grid()
    b = torch.nn.functional.pad(x, (0, -k % 128)).view(rows, -1, 128)
    e = _exponent(b.abs().amax(-1, keepdim=True))
    y = b.abs() / torch.exp2(e)
    hi = torch.searchsorted(grid, y).clamp(max=126)     # grid[hi] >= y
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y, y - grid[lo]
    i = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    i = torch.where(grid[hi] == y, hi, i)
    return (grid[i] * torch.sign(b) * torch.exp2(e)).view(rows, -1), e.squeeze(-1)


def _held(w):
    """(values fp64 on the GPU, Fp8Blocks) of a weight: the values as held."""
    import ltxk

    blocks = ltxk.quantize_fp8(w)
    return blocks.float().to(F64), blocks


def _same_blocks(blocks, x):
    """Values and scales equal to the reference's bit for bit, the padding zero."""
    want, e = _blocks_ref(x.reshape(-1, x.shape[-1]).double().cpu())
    rows, k, nb = want.shape[0], x.shape[-1], e.shape[1]
    scale = blocks.scale.cpu().transpose(0, 1).reshape(rows, -1)
    assert torch.equal(scale[:, :nb].double(), e + 127) and not scale[:, nb:].any()
    got = torch.ldexp(blocks.data.float().cpu().double().view(rows, nb, 128), e[..., None].int()).view(rows, -1)
    assert torch.equal(got, want) and not got[:, k:].any()
    assert torch.equal(blocks.float().double().cpu().reshape(rows, k), want[:, :k])


@pytest.mark.parametrize("rows,k", [(1, 8), (3, 128), (5, 136), (2, 512), (7, 520), (130, 4096), (33, 1544)])
def test_quantize_is_the_formats_rounding(rows, k):
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(rows * 1000 + k)
    x = torch.randn(rows, k, device=DEV, generator=g) * torch.exp2(torch.randint(-20, 20, (1, k), device=DEV, generator=g))
    x = x.to(torch.bfloat16)
    _same_blocks(ltxk.quantize_fp8(x), x)


def test_quantize_borders():
    """Maxima on and next to 448 * 2^e, every bf16 magnitude's exponent, zeros, subnormals,
    halves between two steps, and blocks with an infinity or NaN."""
    import ltxk

    x = torch.zeros(260, 256, dtype=torch.bfloat16, device=DEV)
    for i in range(254):
        top = torch.tensor([(i << 7) | 0x60], dtype=torch.int16).view(torch.bfloat16).to(DEV)  # 1.75 * 2^(i - 127)
        x[i, :128] = top * torch.linspace(-1, 1, 128, device=DEV).to(torch.bfloat16)
        x[i, 3] = top
        x[i, 128] = torch.tensor([(i << 7) | 0x61], dtype=torch.int16).view(torch.bfloat16).to(DEV)  # the next value
    x[254, :128] = torch.arange(128, device=DEV) + 320.0   # halves of steps of 32
    x[254, 128:] = (torch.arange(128, device=DEV) * 2.0**-11)  # below the smallest step of a block with maximum 448
    x[254, 255] = 448.0
    _same_blocks(ltxk.quantize_fp8(x), x)
    bad = torch.ones(3, 256, dtype=torch.bfloat16, device=DEV)
    bad[0, 5], bad[1, 200], bad[2, 0] = float("nan"), float("inf"), -float("inf")
    got = ltxk.quantize_fp8(bad)
    nan = torch.isnan(got.float())
    assert nan[0, :128].all() and nan[1, 128:].all() and nan[2, :128].all() and int(nan.sum()) == 3 * 128
    assert torch.isnan(got.data.float())[nan].all()
    w = ltxk.quantize_fp8(torch.ones(8, 256, dtype=torch.bfloat16, device=DEV))
    assert torch.isnan(ltxk.linear_fp8(got, w)).all()


def _product_bound(x, w, want):
    """The scaled matrix instruction cuts the products of 8 neighbouring values of k off at 2^-13 of
    their largest (which keeps its own bits), so a group's sum is off by less than 7 * 2^-13 of it; from there on
    fp32: 16 groups of an instruction in a tree and the sums of K / 128 of them run on, plus the parts of a cut K,
    each step off by at most 2^-23 of the sum of magnitudes."""
    steps = -(-x.shape[1] // 128) + 8 + 16
    x, w = (torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)) for t in (x, w))
    top = [t.view(t.shape[0], -1, 8).amax(-1) for t in (x, w)]
    return (x @ w.t().contiguous()) * 2.0**-23 * steps + (top[0] @ top[1].t().contiguous()) * (7 * 2.0**-13) \
        + want.abs() * 2.0**-24


def _exact_blocks(rows, k, g):
    """Blocks whose products and sums take at most 24 bits: values +-(1 + i/8) of 2^-1 and 1 (and zeros), scales 1 and 2.
    A product is a multiple of 2^-8 and below 4, so none is cut off beside another of its group (2^-13 of at least
    2^-2), and at 1.2 * 2.25 a product on average, sums of 16384 of them stay below 2^16."""
    import ltxk

    kp = -(-k // 128) * 128
    v = (1 + torch.randint(0, 8, (rows, kp), device=DEV, generator=g) / 8) * 2.0 ** -torch.randint(0, 2, (rows, kp), device=DEV, generator=g)
    v = v * torch.randint(-4, 5, (rows, kp), device=DEV, generator=g).sign()
    v[:, k:] = 0
    groups = -(-kp // 512)
    scale = torch.randint(127, 129, (groups, rows, 4), device=DEV, generator=g, dtype=torch.uint8)
    return ltxk.Fp8Blocks(v.to(torch.float8_e4m3fn), scale, (rows, k))


SHAPES = [(1, 8, 8), (1, 4096, 4096), (3, 24, 136), (16, 40, 520), (17, 128, 384), (33, 72, 2048), (65, 200, 640),
          (126, 2048, 2048), (129, 264, 128), (250, 512, 1152), (300, 520, 776), (1000, 776, 4096), (257, 1000, 8192),
          (2100, 2064, 512), (4100, 1032, 256), (100, 16384, 256), (64, 48, 16384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_exact(m, n, k):
    """Sums that fp32 holds exactly, in whatever order: the result is their one rounding, bit for bit."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x, w = _exact_blocks(m, k, g), _exact_blocks(n, k, g)
    want = x.float().to(F64) @ w.float().to(F64).t().contiguous()
    assert float((x.float().abs().to(F64) @ w.float().abs().to(F64).t().contiguous()).max()) < 2.0**16
    got = ltxk.linear_fp8(x, w)
    assert torch.equal(got, want.to(torch.bfloat16)), (got.to(F64) - want).abs().max().item()
    bias = torch.randint(-64, 64, (n,), device=DEV, generator=g).to(torch.bfloat16)
    assert torch.equal(ltxk.linear_fp8(x, w, bias), (want + bias.to(F64)).to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_matches_fp64(m, n, k, bias):
    """Products of the held values: 2^-8 of the value for the one rounding to bf16."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + 3 * n + 7 * k)
    x = (torch.randn(m, k, device=DEV, generator=g) * (1 + 20 * (torch.rand(k, device=DEV, generator=g) < 0.02))).to(torch.bfloat16)
    w, held = _held((torch.randn(n, k, device=DEV, generator=g) * k**-0.5).to(torch.bfloat16))
    b = torch.randn(n, device=DEV, generator=g).to(torch.bfloat16) if bias else None
    xb = ltxk.quantize_fp8(x)
    xv = xb.float().to(F64)
    want = xv @ w.t().contiguous()
    bound = _product_bound(xv, w, want)
    if bias:
        want = want + b.to(F64)
    got = ltxk.linear_fp8(x, held, b)
    assert got.dtype == torch.bfloat16 and got.shape == (m, n)
    err = (got.to(F64) - want).abs()
    assert bool((err <= bound * 1.01 + want.abs() * 2.0**-8 + 1e-30).all()), (err / (bound + want.abs() * 2.0**-8 + 1e-30)).max().item()
    assert torch.equal(got, ltxk.linear_fp8(xb, held, b))  # the same call over blocks, and again: the same bits


def _gelu64(u):
    return u * torch.special.expit(2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u**3))


def _near_blocks(blocks, want, slack):
    """Blocks of values known to within `slack`: each is held to half a step of its own (2^-4 of
    the value, or half of the block's smallest step 2^(e - 9)), under a scale that a maximum within the slack gives."""
    rows, k = want.shape
    nb = -(-k // 128)

    def tops(v):
        return torch.nn.functional.pad(v, (0, -k % 128)).view(rows, nb, 128).amax(-1)

    e = blocks.scale.transpose(0, 1).reshape(rows, -1).to(F64) - 127
    assert not blocks.scale.transpose(0, 1).reshape(rows, -1)[:, nb:].any()
    e = e[:, :nb]
    assert bool((e >= _exponent((tops(want.abs() - slack)).clamp(min=0))).all())
    assert bool((e <= _exponent(tops(want.abs() + slack))).all())
    got = blocks.float().to(F64).view(rows, k)
    half = torch.exp2(e - 10).repeat_interleave(128, 1)[:, :k]
    err = (got - want).abs()
    bound = slack + torch.maximum((want.abs() + slack) * 2.0**-4, half)
    assert bool((err <= bound).all()), (err / bound).max().item()
    pad = blocks.data.view(torch.uint8)[:, k:]
    assert not (pad & 0x7f).any()


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_gelu_matches_fp64(m, n, k, bias):
    """GELU's slope is below 1.13, and its own evaluation is within 2^-20 of the value and 2^-24."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + 5 * n + 11 * k)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    w, held = _held((torch.randn(n, k, device=DEV, generator=g) * 1.5 * k**-0.5).to(torch.bfloat16))
    b = torch.randn(n, device=DEV, generator=g).to(torch.bfloat16) if bias else None
    xb = ltxk.quantize_fp8(x)
    xv = xb.float().to(F64)
    u = xv @ w.t().contiguous()
    slack = _product_bound(xv, w, u)
    if bias:
        u = u + b.to(F64)
    want = _gelu64(u)
    slack = slack * 1.13 + (u.abs() * 2.0**-23) * 1.13 + want.abs() * 2.0**-20 + 2.0**-24
    got = ltxk.linear_gelu_fp8(xb, held, b)
    assert got.shape == (m, n)
    _near_blocks(got, want, slack)
    again = ltxk.linear_gelu_fp8(x, held, b)
    assert torch.equal(got.data.view(torch.uint8), again.data.view(torch.uint8)) and torch.equal(got.scale, again.scale)


# Every way that a product is cut: 32 rows that are quantised in the call, a tile of several and over a cut K; K one
# value past what is; 64 x 32 and 64 x 64 tiles over a cut K; GELU in tiles of 32 x 128, of one block and at both its
# borders; 256 x 128 tiles of odd sizes, and of one block; large tiles of two steps, of an odd rest whole and in parts; 128 x 128 tiles in parts.
VARIANTS = [(100, 256, 128), (64, 512, 376), (126, 2040, 512), (1, 1024, 17152), (1, 1024, 17160), (31, 520, 16384),
            (126, 1024, 16384), (250, 1160, 16392), (1, 8, 24),
            (70, 1000, 512), (252, 4104, 2056), (252, 4096, 4096), (97, 12280, 1000), (520, 712, 648), (2100, 4200, 2568), (2305, 2056, 1000), (3001, 4104, 120), (3001, 4104, 136), (8200, 2056, 520), (4136, 4112, 2056),
            (900, 1544, 8200), (4100, 4104, 4104)]


@pytest.mark.parametrize("m,n,k", VARIANTS)
def test_linear_variants_exact(m, n, k):
    """As above, and equal for x in bf16, of which the blocks' rounding leaves nothing away."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x, w = _exact_blocks(m, k, g), _exact_blocks(n, k, g)
    want = x.float().to(F64) @ w.float().to(F64).t().contiguous()
    assert float((x.float().abs().to(F64) @ w.float().abs().to(F64).t().contiguous()).max()) < 2.0**16
    bias = torch.randint(-64, 64, (n,), device=DEV, generator=g).to(torch.bfloat16)
    for b, value in ((None, want), (bias, want + bias.to(F64))):
        assert torch.equal(ltxk.linear_fp8(x, w, b), value.to(torch.bfloat16))
        assert torch.equal(ltxk.linear_fp8(x.float().to(torch.bfloat16), w, b), value.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", VARIANTS)
def test_linear_gelu_variants_match_fp64(m, n, k):
    test_linear_gelu_matches_fp64(m, n, k, True)


@pytest.mark.parametrize("m,n,k", [(20, 256, 512), (100, 2048, 256), (500, 1024, 512), (1000, 1032, 384), (3001, 4104, 264)])
def test_not_finite_stays_in_its_row(m, n, k):
    """A NaN or an infinity in a row of x makes that row of the result NaN, one in a row of w that column; nothing else."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    w = torch.randn(n, k, device=DEV, generator=g).to(torch.bfloat16)
    clean, clean_gelu = ltxk.linear_fp8(x, ltxk.quantize_fp8(w)), ltxk.linear_gelu_fp8(x, ltxk.quantize_fp8(w)).float()
    x[3, 5], x[m - 1, k - 1], w[9, 0] = float("nan"), float("inf"), float("-inf")
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[3], bad[m - 1], bad[:, 9] = True, True, True
    w = ltxk.quantize_fp8(w)
    for v in (x, ltxk.quantize_fp8(x)):
        got = ltxk.linear_fp8(v, w)
        assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], clean[~bad])
        got = ltxk.linear_gelu_fp8(v, w).float()
        assert got[bad].isnan().all()
        # a block that holds a NaN may be NaN as a whole; the others are what they were
        bad_blocks = bad.clone()
        bad_blocks[:, :128] = True
        assert torch.equal(got[~bad_blocks], clean_gelu[~bad_blocks])


@pytest.mark.parametrize("m,n,k", [(20, 256, 512), (30, 4096, 16384), (126, 4104, 512), (500, 1024, 512), (1000, 1032, 384),
                                   (2305, 2056, 1000), (3001, 4104, 264), (4136, 4112, 2056)])
def test_not_finite_takes_its_block(m, n, k):
    """A NaN, or an infinity, of the hidden values makes its block of 128 NaN, as in quantize_fp8, whichever kernel
    writes it; every other block is what it was."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(m + 1)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    w = ltxk.quantize_fp8((torch.randn(n, k, device=DEV, generator=g) * k**-0.5).to(torch.bfloat16))
    bias = torch.randn(n, device=DEV, generator=g).to(torch.bfloat16)
    clean = ltxk.linear_gelu_fp8(x, w, bias)
    bias[7], bias[n - 5] = float("nan"), float("inf")
    got = ltxk.linear_gelu_fp8(x, w, bias)
    last = (n - 1) // 128 * 128
    v, want = got.float(), clean.float()
    assert v[:, :128].isnan().all() and v[:, last:].isnan().all()
    assert torch.equal(v[:, 128:last], want[:, 128:last])
    # the bytes themselves: NaN values under scale 255
    assert ((got.data.view(torch.uint8)[:, :128] & 0x7F) == 0x7F).all()
    groups = got.scale.transpose(0, 1).reshape(m, -1)
    assert (groups[:, 0] == 255).all() and (groups[:, last // 128] == 255).all() and not groups[:, last // 128 + 1:].any()


@pytest.mark.parametrize("batch,tokens,dim", [(1, 1, 8), (2, 3, 128), (1, 7, 200), (2, 65, 2048), (1, 130, 4096), (3, 5, 4104),
                                              (1, 4, 8192), (1, 3, 16384), (2, 9, 640), (2, 1601, 264),
                                              (1, 900, 2056), (3, 800, 4096)])
@pytest.mark.parametrize("form", ["plain", "residual", "gated", "masked", "indexed", "tokens"])
def test_add_norm_modulate_fp8(batch, tokens, dim, form):
    """x' equals add_norm_modulate's bit for bit; the blocks hold the fp64 norm of it to within
    fp32's rounding (the sum of squares: 2^-24 a step, at most dim / 256 + 16 of them; six more operations)."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dim + tokens)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(torch.bfloat16)

    x, f = normal(batch, tokens, dim, scale=3.0), normal(batch, tokens, dim)
    table = normal(4, dim, scale=0.5)
    index = None
    if form == "indexed":
        index = ltxk.TimestepIndex(torch.randint(0, 3, (batch * tokens,), device=DEV, generator=g).to(torch.int32), 3)
        emb = normal(1, 3, 4 * dim, scale=0.5)
    else:
        emb = normal(batch, tokens if form == "tokens" else 1, 4 * dim, scale=0.5)
    gate, shift, scale = (ltxk.AdaRef(table, i, emb, index=index) for i in range(3))
    mask = torch.arange(batch, device=DEV).to(torch.bfloat16) if form == "masked" else None

    def value(i):
        e = emb[..., i * dim:(i + 1) * dim].float()
        if index is not None:
            e = e[0][index.index.long()].view(batch, tokens, dim)
        return (table[i].float() + e).to(torch.bfloat16).to(F64)

    if form == "plain":
        res, got = x, ltxk.norm_modulate_fp8(x, shift=shift, scale=scale)
    else:
        kw = dict(gate=None if form == "residual" else gate, mask=mask, shift=shift, scale=scale)
        res, got = ltxk.add_norm_modulate_fp8(x, f, **kw)
        want_x, _ = ltxk.add_norm_modulate(x, f, **kw)
        assert torch.equal(res, want_x)
        mine = x.clone()
        again = ltxk.add_norm_modulate_fp8(mine, f, **kw, x_out=mine)[1]
        assert torch.equal(mine, want_x) and torch.equal(again.scale, got.scale)
        assert torch.equal(again.data.view(torch.uint8), got.data.view(torch.uint8))
    r = res.to(F64)
    n = r / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-6)
    want = n * (1 + value(2)) + value(1)
    slack = ((n * (1 + value(2))).abs() + value(1).abs()) * 2.0**-24 * (dim / 256 + 22)
    assert got.shape == x.shape
    _near_blocks(got, want.view(-1, dim), slack.view(-1, dim))


def test_outputs_behind_the_rows_stay():
    """Nothing is written behind the last row of values, scales or results."""
    import ltxk

    lib, st = ltxk.load(), ltxk._stream(torch.empty(1, device=DEV))
    for m, n, k in ((5, 40, 136), (70, 264, 640), (300, 520, 1152)):
        x = torch.randn(m, k, device=DEV).to(torch.bfloat16)
        w = ltxk.quantize_fp8(torch.randn(n, k, device=DEV).to(torch.bfloat16))
        xb = ltxk.quantize_fp8(x)
        rows, kp, np_ = m, -(-k // 128) * 128, -(-n // 128) * 128
        q = torch.full((rows * kp + 256,), 77, device=DEV, dtype=torch.uint8)
        s = torch.full((xb.scale.numel() + 256,), 77, device=DEV, dtype=torch.uint8)
        assert lib.ltxk_quantize_fp8(q.data_ptr(), s.data_ptr(), x.data_ptr(), m, k, st) == 0
        assert (q[rows * kp:] == 77).all() and (s[xb.scale.numel():] == 77).all()
        y = torch.full((m * n + 256,), 7.0, device=DEV, dtype=torch.bfloat16)
        ws = torch.empty(max(16, *(lib.ltxk_linear_fp8_workspace_bytes(m, n, k, g, 0) for g in (0, 1))), dtype=torch.uint8,
                         device=DEV)
        ops = [t.data_ptr() for t in (xb.data, xb.scale, w.data, w.scale)]
        assert lib.ltxk_linear_fp8(y.data_ptr(), *ops, None, m, n, k, ws.data_ptr(), ws.numel(), st) == 0
        assert (y[m * n:] == 7).all() and torch.equal(y[:m * n].view(m, n), ltxk.linear_fp8(xb, w))
        q = torch.full((m * np_ + 256,), 77, device=DEV, dtype=torch.uint8)
        size = -(-np_ // 512) * m * 4
        s = torch.full((size + 256,), 77, device=DEV, dtype=torch.uint8)
        assert lib.ltxk_linear_gelu_fp8(q.data_ptr(), s.data_ptr(), *ops, None, m, n, k, ws.data_ptr(), ws.numel(), st) == 0
        assert (q[m * np_:] == 77).all() and (s[size:] == 77).all()


def test_empty_and_views():
    import ltxk

    w = ltxk.quantize_fp8(torch.randn(16, 64, device=DEV).to(torch.bfloat16))
    empty = torch.empty(2, 0, 64, device=DEV, dtype=torch.bfloat16)
    assert ltxk.linear_fp8(empty, w).shape == (2, 0, 16) and ltxk.linear_gelu_fp8(empty, w).shape == (2, 0, 16)
    x = torch.randn(2, 3, 64, device=DEV).to(torch.bfloat16)
    b = ltxk.quantize_fp8(x)
    assert b.shape == (2, 3, 64) and torch.equal(ltxk.linear_fp8(b.view(6, 64), w), ltxk.linear_fp8(x, w).view(6, 16))
    one = ltxk.linear_fp8(x[0, 0], w)  # a single row without a leading dimension
    assert one.shape == (16,) and torch.equal(one, ltxk.linear_fp8(x, w)[0, 0])


def test_captured_run_replays_equal():
    """Residual + norm, both layers of a feed-forward and masked attention in one captured graph: every
    replay with other inputs and eager work between equals the eager calls bit for bit."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(3)

    def fresh(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(torch.bfloat16)

    x, f = fresh(2, 70, 512), fresh(2, 70, 512)
    w1, w2 = (ltxk.quantize_fp8(fresh(*s, scale=0.05)) for s in ((2048, 512), (512, 2048)))
    kv = fresh(2, 1500, 1024)
    keep = torch.rand(2, 1500, device=DEV, generator=g) < 0.5
    scale = ltxk.AdaRef(fresh(1, 512), 0)

    def call():
        r, h = ltxk.add_norm_modulate_fp8(x, f, scale=scale)
        y = ltxk.linear_fp8(ltxk.linear_gelu_fp8(h, w1), w2)
        return r, y, ltxk.cross_attention(y, kv[..., :512], kv[..., 512:], 4, keep)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    for i in range(4):
        x.copy_(fresh(2, 70, 512))
        kv.copy_(fresh(2, 1500, 1024))
        keep.copy_(torch.rand(2, 1500, device=DEV, generator=g) < 0.1 * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        for a, b in zip(got, call()):
            assert torch.equal(a, b), f"replay {i}"


def test_two_streams_at_once():
    """Calls on two streams have results and workspaces of their own: cut K, quantised x, blocks of the GELU."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(8)
    shapes = [(300, 520, 4096), (126, 1024, 16384), (64, 2048, 512)]
    ops = [(torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16),
            ltxk.quantize_fp8(torch.randn(n, k, device=DEV, generator=g).to(torch.bfloat16))) for m, n, k in shapes]

    def run():
        out = [ltxk.linear_fp8(x, w) for x, w in ops]
        return out + [t for x, w in ops for b in (ltxk.linear_gelu_fp8(x, w),) for t in (b.data.view(torch.uint8), b.scale)]

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for s, o in zip(streams, got):
            with torch.cuda.stream(s):
                o.append(run())
    torch.cuda.synchronize()
    for runs in got:
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(want, r))


def test_binding_refusals():
    """What the binding refuses of tensors on the GPU, before any launch."""
    import ltxk

    x = torch.zeros(6, 256, device=DEV, dtype=torch.bfloat16)
    w = ltxk.quantize_fp8(torch.zeros(16, 256, device=DEV, dtype=torch.bfloat16))
    bias = torch.zeros(16, device=DEV, dtype=torch.bfloat16)
    flat = torch.zeros(6 * 256 + 8, device=DEV, dtype=torch.bfloat16)
    bad = [
        (ValueError, lambda: ltxk.quantize_fp8(x.float())), (ValueError, lambda: ltxk.quantize_fp8(x[:, :12].contiguous())),
        (ValueError, lambda: ltxk.quantize_fp8(x[:, :128])), (RuntimeError, lambda: ltxk.quantize_fp8(flat[1:1537].view(6, 256))),
        (ValueError, lambda: ltxk.linear_fp8(x[:, :128].contiguous(), w)), (ValueError, lambda: ltxk.linear_fp8(x.half(), w)),
        (ValueError, lambda: ltxk.linear_fp8(x.t(), w)), (ValueError, lambda: ltxk.linear_fp8(x, w, bias[:8])),
        (ValueError, lambda: ltxk.linear_fp8(x, w, bias.float())), (RuntimeError, lambda: ltxk.linear_fp8(x, w, bias.cpu())),
        (RuntimeError, lambda: ltxk.linear_fp8(flat[1:1537].view(6, 256), w)), (TypeError, lambda: ltxk.linear_fp8(x, x)),
        (TypeError, lambda: ltxk.linear_gelu_fp8([1.0], w)),
        (ValueError, lambda: ltxk.linear_fp8(x, ltxk.quantize_fp8(torch.zeros(12, 256, device=DEV, dtype=torch.bfloat16)))),
        (ValueError, lambda: ltxk.Fp8Blocks(w.data, w.scale, (16, 128))), (ValueError, lambda: ltxk.Fp8Blocks(w.data, w.scale, (8, 256))),
        (ValueError, lambda: ltxk.Fp8Blocks(w.data, w.scale[..., :2], (16, 256))),
        (ValueError, lambda: ltxk.Fp8Blocks(w.data.view(torch.uint8), w.scale, (16, 256))),
        (ValueError, lambda: w.view(16, 128)), (ValueError, lambda: w.view(4, 8, 256)),
        (ValueError, lambda: ltxk.add_norm_modulate_fp8(x, x[:3])), (ValueError, lambda: ltxk.add_norm_modulate_fp8(x, None)),
        (ValueError, lambda: ltxk.add_norm_modulate_fp8(x, x, x_out=x[:3])),
        (ValueError, lambda: ltxk.norm_modulate_fp8(x, shift=ltxk.AdaRef(bias.view(1, 16), 0))),
        (TypeError, lambda: ltxk.cross_attention(x[None], x[None], x[None], 4, [True] * 6)),
        (ValueError, lambda: ltxk.cross_attention(x[None], x[None], x[None], 4, torch.ones(1, 5, device=DEV, dtype=torch.bool))),
        (ValueError, lambda: ltxk.cross_attention(x[None], x[None], x[None], 4, torch.ones(1, 6, device=DEV))),
        (ValueError, lambda: ltxk.cross_attention(x[None], x[None], x[None], 3)),
        (RuntimeError, lambda: ltxk.cross_attention(x[None], x[None], x[None], 4, torch.ones(1, 6, dtype=torch.bool))),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was not refused")
    assert not ltxk.linear_fp8(x, w, bias).any()  # the good call still runs


def test_blocks_as_tensors():
    """Blocks that a kernel made give their tensors when asked, also without rows and past the object's life; a quantised
    weight's two tensors share no memory, so that they can be saved apart; views hold the same bytes."""
    import ltxk

    x = torch.randn(6, 264, device=DEV).to(torch.bfloat16)
    w = ltxk.quantize_fp8(torch.randn(520, 264, device=DEV).to(torch.bfloat16))
    assert w.data.untyped_storage().data_ptr() != w.scale.untyped_storage().data_ptr()
    made = ltxk.linear_gelu_fp8(x, w)
    assert made.data.shape == (6, 640) and made.scale.shape == (2, 6, 4) and made.device == x.device
    other = ltxk.Fp8Blocks(made.data.clone(), made.scale.clone(), made.shape)
    w2 = ltxk.quantize_fp8(torch.randn(16, 520, device=DEV).to(torch.bfloat16))
    want = ltxk.linear_fp8(other, w2)
    assert torch.equal(ltxk.linear_fp8(made, w2), want)
    assert torch.equal(ltxk.linear_fp8(made.view(2, 3, 520), w2), want.view(2, 3, 16))
    data, scale = made.data, made.scale
    del made
    assert torch.equal(data.view(torch.uint8), other.data.view(torch.uint8)) and torch.equal(scale, other.scale)
    empty = ltxk.linear_gelu_fp8(x[:0], w)
    assert empty.data.shape == (0, 640) and empty.scale.shape == (2, 0, 4) and empty.float().shape == (0, 520)
    assert ltxk.linear_fp8(empty, w2).shape == (0, 16)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dim", [8, 136, 520, 1032, 2056, 4040])
def test_norm_padding_beside_values_not_finite(dim, residual):
    """Rows with a NaN or an infinity, and an infinite modulation of the first column: the columns past the last are
    zeros in every row all the same (7f in a block that is NaN as a whole), so the last block is NaN for values of
    its own only, the scale bytes past it are zero, and many rows (which workgroups walk) hold the bytes that
    few rows (a workgroup each) do."""
    import ltxk

    g = torch.Generator(device=DEV).manual_seed(dim)
    tokens, blocks = 1100, -(-dim // 128)
    x, f = (torch.randn(1, tokens, dim, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    x[0, 3, 1], x[0, 900, dim - 1], x[0, 1099, 0] = float("nan"), float("inf"), float("-inf")
    f[0, 5, 2], f[0, 6, 0] = float("nan"), 0.0

    def call(lo, hi, gate, shift, scale):
        part = [t[:, lo:hi].contiguous() for t in (x, f)]
        mods = dict(shift=ltxk.AdaRef(shift, 0), scale=ltxk.AdaRef(scale, 0))
        if residual:
            return ltxk.add_norm_modulate_fp8(*part, gate=ltxk.AdaRef(gate, 0), **mods)[1]
        return ltxk.norm_modulate_fp8(part[0], **mods)

    for which in ("none", "gate", "shift", "scale"):
        mods = {name: torch.full((1, dim), 0.5, dtype=torch.bfloat16, device=DEV) for name in ("gate", "shift", "scale")}
        if which != "none":
            mods[which][0, 0] = float("inf")
        many = call(0, tokens, **mods)
        scale = many.scale.transpose(0, 1).reshape(tokens, -1)
        assert not scale[:, blocks:].any(), which
        tail, bad = many.data.view(torch.uint8)[:, dim:], scale[:, blocks - 1] == 255
        assert not tail[~bad].any(), which
        for lo in (0, 400, 898, 1092):
            few = call(lo, lo + 8, **mods)
            assert torch.equal(few.scale, many.scale[:, lo:lo + 8]), (which, lo)
            assert torch.equal(few.data.view(torch.uint8), many.data.view(torch.uint8)[lo:lo + 8]), (which, lo)
