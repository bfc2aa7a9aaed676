"""Cases of the 8-bit linear layers, the feed-forward made of them, and cross attention to padded prompts.

A case is one call (or the short run of calls that a block makes) at the widths of the 48-block configuration: video
stream 4096 wide (32 heads of 128), audio stream 2048 wide (32 heads of 64), feed-forward 4x, 1024 text tokens, 6144 or
4290 video and 126 audio tokens, a guidance batch of four.

  linear     bf16 rows through a layer whose weight is held in blocks of 128 e4m3 values with a power-of-two scale each
  ffn        residual + gate + norm + modulation, both layers of the feed-forward, hidden values in the same blocks
  attention  queries over the kept ones of an encoder's states, another number in each batch item
"""
import math
import pathlib
import sys

import torch

own = False

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "ltx-nv_amd"))

DEV = "cuda"
EPS = 1e-6
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
BLOCK, GROUP = 128, 4  # values of a scale; scales of a row that lie together


def listed():
    return [
        # One timestep through the timestep embedder's second layer: the smallest call, latency counts.
        dict(name="linear_timestep", kind="linear", rows=1, k=4096, n=4096, bias=True),
        # Four passes' timesteps through the AdaLN layer (9 rows of 4096): the weight's bytes count.
        dict(name="linear_adaln", kind="linear", rows=4, k=4096, n=36864, bias=True),
        # An audio stream's query projection.
        dict(name="linear_audio", kind="linear", rows=126, k=2048, n=2048, bias=True),
        # Keys of one prompt's text context.
        dict(name="linear_text", kind="linear", rows=1024, k=4096, n=4096, bias=True),
        # A video projection at a ragged length.
        dict(name="linear_ragged", kind="linear", rows=4290, k=4096, n=4096, bias=False),
        # A video projection of the guidance batch.
        dict(name="linear_video_b4", kind="linear", rows=24576, k=4096, n=4096, bias=True),
        # The audio stream's feed-forward.
        dict(name="ffn_audio", kind="ffn", batch=1, tokens=126, dim=2048, bias=True),
        # The video stream's feed-forward, the largest part of a block.
        dict(name="ffn_video", kind="ffn", batch=1, tokens=6144, dim=4096, bias=False),
        # The same in the guidance batch at a ragged length: the largest call.
        dict(name="ffn_video_b4", kind="ffn", batch=4, tokens=4290, dim=4096, bias=False),
        # One query over a short prompt.
        dict(name="attention_one", kind="attention", batch=1, tq=1, tk=333, heads=32, dim_head=64, keep="front", gated=True),
        # Audio tokens over the guidance batch's prompts (some of them left-padded).
        dict(name="attention_audio", kind="attention", batch=4, tq=126, tk=1024, heads=32, dim_head=64, keep="back", gated=True),
        # Video tokens over the guidance batch's prompts.
        dict(name="attention_video", kind="attention", batch=4, tq=6144, tk=1024, heads=32, dim_head=128, keep="front", gated=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "ffn", "attention", "attention"])
    if kind == "linear":
        # K and N in steps of 8; the work stays below the largest listed layer's
        k, n = 8 * _log_int(rng, 8, 2048), 8 * _log_int(rng, 1, 4608)
        most = max(1, min(24576, (1 << 38) // (k * n)))
        return dict(kind=kind, rows=_log_int(rng, 1, most), k=k, n=n, bias=rng.random() < 0.7)
    if kind == "ffn":
        dim = 64 * rng.randint(4, 64)
        most = max(1, min(17160, (1 << 38) // (dim * dim)))
        rows = _log_int(rng, 1, most)
        batch = rng.choice([1, 1, 2, 4])
        return dict(kind=kind, batch=batch, tokens=max(1, rows // batch), dim=dim, bias=rng.random() < 0.5)
    batch, heads, dim_head = rng.randint(1, 4), rng.choice([1, 2, 5, 16, 32]), rng.choice([64, 128])
    tk = _log_int(rng, 1, 6144)
    most = max(1, min(6144, (1 << 29) // (batch * heads * tk)))
    return dict(kind=kind, batch=batch, tq=_log_int(rng, 1, most), tk=tk, heads=heads, dim_head=dim_head,
                keep=rng.choice(["none", "front", "back", "holes", "empty"]), gated=rng.random() < 0.6)


# ------------------------------------------------------------------ blocks of 128 e4m3 values --


def _blocks(x, dtype):
    """x (rows, k) in whole blocks: (rows, blocks, 128), zeros past k."""
    rows, k = x.shape
    return torch.nn.functional.pad(x.to(dtype), (0, -k % BLOCK)).view(rows, -1, BLOCK)


def _exponents(blocks):
    """The least e with max |x| <= 448 * 2^e for each block, at least -127 (448 = 0.875 * 2^9)."""
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    e = exponent - 9 + (mantissa > 0.875)
    return torch.where(mantissa == 0, -127, e).clamp(min=-127)


def _rounded(x):
    """x (rows, k) as its blocks' values e4m3(x 2^-e) 2^e, in x's type (fp32 or fp64)."""
    b = _blocks(x, x.dtype)
    e = _exponents(b)
    q = torch.ldexp(b, -e).to(torch.float8_e4m3fn).to(x.dtype)
    return torch.ldexp(q, e).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _held(w):
    """A weight (n, k) as a program keeps it: e4m3 values (n, whole blocks) and one byte per block, e + 127, four of a
    row side by side: (ceil(blocks / 4), n, 4)."""
    b = _blocks(w, F32)
    e = _exponents(b)
    data = torch.ldexp(b, -e).to(torch.float8_e4m3fn).reshape(w.shape[0], -1)
    bytes_ = torch.nn.functional.pad((e.squeeze(-1) + 127).to(torch.uint8), (0, -e.shape[1] % GROUP))
    return data, bytes_.view(w.shape[0], -1, GROUP).transpose(0, 1).contiguous(), (w.shape[0], w.shape[1])


def _values(held, dtype):
    """What a held weight stands for."""
    data, scale, (n, k) = held
    e = scale.transpose(0, 1).reshape(n, -1)[:, :data.shape[1] // BLOCK].to(torch.int32) - 127
    return torch.ldexp(data.to(dtype).view(n, -1, BLOCK), e.unsqueeze(-1)).reshape(n, -1)[:, :k]


# ------------------------------------------------------------------------------- inputs --


def _lengths(case, g):
    b, tk = case["batch"], case["tk"]
    at = torch.arange(tk, device=DEV).expand(b, tk)
    n = (torch.rand(b, 1, device=DEV, generator=g) * 0.9 + 0.1) * tk
    if case["keep"] == "none":
        return None
    if case["keep"] == "front":  # padded behind the prompt
        return at < n.ceil()
    if case["keep"] == "back":   # padded in front of it
        return at >= tk - n.ceil()
    holes = torch.rand(b, tk, device=DEV, generator=g) < 0.7
    if case["keep"] == "empty":  # the last batch item has no prompt
        holes[-1] = False
    return holes


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(BF16)

    def residual(*shape):  # a residual stream: some columns are far larger than the others
        heavy = torch.rand(shape[-1], device=DEV, generator=g) < 0.01
        return (torch.randn(*shape, device=DEV, generator=g) * torch.where(heavy, 20.0, 1.0)).to(BF16)

    if case["kind"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return dict(case=case, x=residual(rows, k), w=_held(normal(n, k, scale=k ** -0.5)),
                    bias=normal(n, scale=0.1) if case["bias"] else None)
    if case["kind"] == "ffn":
        b, t, d = case["batch"], case["tokens"], case["dim"]
        inner = 4 * d
        return dict(case=case, x=residual(b, t, d), f=normal(b, t, d), table=normal(9, d, scale=0.1),
                    emb=normal(b, 1, 9 * d, scale=0.3), w_in=_held(normal(inner, d, scale=d ** -0.5)),
                    w_out=_held(normal(d, inner, scale=inner ** -0.5)),
                    b_in=normal(inner, scale=0.1) if case["bias"] else None,
                    b_out=normal(d, scale=0.1) if case["bias"] else None)
    b, tq, tk, h = case["batch"], case["tq"], case["tk"], case["heads"]
    w = h * case["dim_head"]
    return dict(case=case, q=normal(b, tq, w, scale=1.5), k=normal(b, tk, w), v=normal(b, tk, w), keep=_lengths(case, g),
                logits=normal(b, tq, h) if case["gated"] else None)


# ------------------------------------------------------------------------- the operators --


def _plain_gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_product(x, held, bias):
    y = x @ _values(held, F32).t()
    return y if bias is None else y + bias.to(F32)


def _plain_ada(s, row):
    """bf16(table + embedding) of AdaLN row `row`, (B, 1, D)."""
    d = s["x"].shape[-1]
    return (s["table"][row].to(F32) + s["emb"][..., row * d:(row + 1) * d].to(F32)).to(BF16).to(F32)


def _plain_ffn(s):
    x = (s["x"].to(F32) + s["f"].to(F32) * _plain_ada(s, 2)).to(BF16)
    xf = x.to(F32)
    h = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS) * (1 + _plain_ada(s, 4)) + _plain_ada(s, 3)
    u = _plain_gelu(_plain_product(_rounded(h.reshape(-1, h.shape[-1])), s["w_in"], s["b_in"]))
    return x, _plain_product(_rounded(u), s["w_out"], s["b_out"]).to(BF16).view_as(x)


def _heads(x, h):
    b, t, w = x.shape
    return x.to(F32).view(b, t, h, w // h).transpose(1, 2).contiguous()


def _plain_attention(s):
    c = s["case"]
    h = c["heads"]
    q, k, v = (_heads(s[n], h) for n in ("q", "k", "v"))
    score = (q @ k.transpose(-1, -2).contiguous()) * c["dim_head"] ** -0.5
    if s["keep"] is not None:
        score = score.masked_fill(~s["keep"][:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    o = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)
    if s["logits"] is not None:
        o = o * (2 * torch.sigmoid(s["logits"].to(F32))).transpose(1, 2).unsqueeze(-1)
    return o.transpose(1, 2).reshape(s["q"].shape).to(BF16)


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        if kind == "linear":
            return _plain_product(_rounded(s["x"].to(F32)), s["w"], s["bias"]).to(BF16)
        return _plain_ffn(s) if kind == "ffn" else _plain_attention(s)
    import ltxk

    if kind == "linear":
        return ltxk.linear_fp8(s["x"], ltxk.Fp8Blocks(*s["w"]), s["bias"])
    if kind == "ffn":
        gate, shift, scale = (ltxk.AdaRef(s["table"], row, s["emb"]) for row in (2, 3, 4))
        x, h = ltxk.add_norm_modulate_fp8(s["x"], s["f"], gate=gate, shift=shift, scale=scale, eps=EPS)
        u = ltxk.linear_gelu_fp8(h, ltxk.Fp8Blocks(*s["w_in"]), s["b_in"])
        return x, ltxk.linear_fp8(u, ltxk.Fp8Blocks(*s["w_out"]), s["b_out"])
    return ltxk.cross_attention(s["q"], s["k"], s["v"], s["case"]["heads"], keep=s["keep"], logits=s["logits"])


# ----------------------------------------------------------------------- in 64 bits --


def _grid64(x):
    """x (rows, k) in fp64 on the grid of its blocks, written from the format: in a block whose largest magnitude is a,
    the step of a value of magnitude 2^p is 2^(p - 3), no finer than 2^(e - 9); halves go to the even neighbour."""
    rows, k = x.shape
    out = torch.zeros_like(x)
    whole = k // BLOCK * BLOCK
    pieces = [(0, whole, BLOCK)] if whole else []
    if k > whole:
        pieces.append((whole, k, k - whole))
    for lo, hi, width in pieces:
        b = x[:, lo:hi].reshape(rows, -1, width)
        a = b.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / 448))
        e = torch.where(a > torch.exp2(e) * 448, e + 1, e)      # log2 may round
        e = torch.where(a <= torch.exp2(e - 1) * 448, e - 1, e).clamp(min=-127)
        p = torch.floor(torch.log2(torch.where(b == 0, torch.ones_like(b), b.abs())))
        p = torch.where(b.abs() >= torch.exp2(p + 1), p + 1, p)
        p = torch.where(b.abs() < torch.exp2(p), p - 1, p)
        step = torch.exp2(torch.maximum(p - 3, e - 9))
        out[:, lo:hi] = (torch.round(b / step) * step).reshape(rows, -1)
    return out


def _product64(x, held, bias):
    y = torch.mm(x, _values(held, F64).t().contiguous())
    return y if bias is None else y + bias.to(F64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _product64(_grid64(s["x"].to(F64)), s["w"], s["bias"])
    if case["kind"] == "ffn":
        d = case["dim"]
        gate, shift, scale = ((s["table"][r].to(F64) + s["emb"][..., r * d:(r + 1) * d].to(F64)).to(BF16).to(F64)
                              for r in (2, 3, 4))
        x = s["x"].to(F64) + s["f"].to(F64) * gate
        r = x.to(BF16).to(F64)
        h = r / torch.sqrt(r.square().mean(-1, keepdim=True) + EPS) * (1 + scale) + shift
        u = _product64(_grid64(h.view(-1, d)), s["w_in"], s["b_in"])
        u = u * torch.special.expit(2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3))
        return x, _product64(_grid64(u), s["w_out"], s["b_out"]).view_as(x)
    h, dh = case["heads"], case["dim_head"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    for i in range(case["batch"]):
        kept = slice(None) if s["keep"] is None else s["keep"][i]
        k, v = s["k"][i][kept].to(F64), s["v"][i][kept].to(F64)
        if not k.shape[0]:
            continue
        for j in range(h):
            c = slice(j * dh, (j + 1) * dh)
            w = torch.softmax(s["q"][i, :, c].to(F64) @ k[:, c].t().contiguous() / math.sqrt(dh), -1)
            o = w @ v[:, c]
            if s["logits"] is not None:
                o = o * 2 * torch.sigmoid(s["logits"][i, :, j].to(F64)).unsqueeze(-1)
            out[i, :, c] = o
    return out


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k * (1 + 1 / BLOCK) + 2 * m * n, "flops": 2 * m * n * k}
    if case["kind"] == "ffn":
        m, d = case["batch"] * case["tokens"], case["dim"]
        return {"bytes": 8 * m * d + 8 * d * d * (1 + 1 / BLOCK), "flops": 16 * m * d * d}
    b, tq, w = case["batch"], case["tq"], case["heads"] * case["dim_head"]
    share = {"none": 1.0, "front": 0.55, "back": 0.55, "holes": 0.7, "empty": 0.7}[case["keep"]]  # of the keys, about
    keys = max(1.0, share * case["tk"])
    return {"bytes": 4 * b * w * (tq + keys), "flops": 4 * b * tq * keys * w}
