"""Cases of attention over packed sequences, and of attention for a batch that shares a prefix.

Both serve the language side of the framework: the states that the text connectors take come from a causal language
model with grouped heads, whose prompts have different lengths (a guidance batch holds at least two), begin with the same
instructions, and are continued token by token where the model is asked to write a prompt out.  Clips of different
lengths in one call are the same operator without the causal mask.

  packed   queries of sequences laid end to end, each over the keys of its own sequence (its newest ones, where keys of
           earlier calls stand before them), causal or not, in a window or not, several query heads a key head
  prefix   queries of a batch over keys that all of it shares, then over each item's own ones in a cache that is not full

Heads of 64 and 128 are the framework's own; 256 is a common size in language models.  Lengths of a case are drawn from
its `mix` alone, so that every seed has the same work.
"""
import math
import pathlib
import random
import sys

import torch

own = False

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "ltx-nv_amd"))

DEV = "cuda"
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _packed(name, seqs, shortest, longest, heads, kv_heads, dim, causal=True, window=0, cached=(0, 0), slack=0, mix=1):
    return dict(name=name, kind="packed", seqs=seqs, shortest=shortest, longest=longest, cached_least=cached[0],
                cached_most=cached[1], heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, window=window, slack=slack,
                mix=mix)


def _prefix(name, items, queries, prefix, shortest, longest, room, heads, kv_heads, dim, causal=True, mix=1):
    return dict(name=name, kind="prefix", items=items, queries=queries, prefix=prefix, shortest=shortest, longest=longest,
                room=room, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, mix=mix)


def listed():
    return [
        # Two short captions: the smallest call, latency counts.
        _packed("packed_captions", 2, 5, 126, 16, 8, 256),
        # The guidance batch's prompts, the negative one shorter.
        _packed("packed_guidance", 2, 333, 1024, 16, 8, 256),
        # The same model's layers that look back 1024 tokens, on long descriptions; a buffer that is not full.
        _packed("packed_window", 5, 700, 8192, 16, 8, 256, window=1024, slack=77),
        # A batch of prompts of all lengths.
        _packed("packed_prompts", 33, 17, 2048, 32, 8, 128),
        # One long document.
        _packed("packed_document", 1, 12288, 12288, 32, 8, 128),
        # Clips of different lengths through a video stream's self-attention: the largest call.
        _packed("packed_clips", 4, 4290, 6144, 32, 32, 128, causal=False),
        # A token of each of 64 sequences over the keys of its earlier ones.
        _packed("packed_tokens", 64, 1, 1, 32, 8, 128, cached=(100, 8192)),
        # Four continuations' next token after a short common prompt: latency counts.
        _prefix("prefix_captions", 4, 1, 333, 1, 126, 128, 16, 8, 256),
        # 64 continuations' next token after long common instructions.
        _prefix("prefix_tokens", 64, 1, 8192, 64, 1024, 1024, 32, 8, 128),
        # The same over a document, heads of 64.
        _prefix("prefix_document", 48, 1, 32768, 32, 2048, 2048, 32, 4, 64),
        # Five proposed tokens each, checked in one call.
        _prefix("prefix_proposals", 7, 5, 4290, 200, 1500, 1536, 16, 8, 256),
        # 16 prompts after common instructions, left-padded to 512 tokens.
        _prefix("prefix_prompts", 16, 512, 2048, 100, 512, 512, 32, 8, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if kv_heads * g <= 40])
    mix = rng.randrange(1 << 30)
    most = 1 << 30  # scores of a call, padding counted
    if rng.random() < 0.5:
        tokens = rng.random() < 0.3  # one token a sequence, over earlier keys
        seqs = _log_int(rng, 1, 128)
        longest = 1 if tokens else _log_int(rng, 1, max(1, min(8192, int((most / (seqs * heads)) ** 0.5))))
        room = max(2, min(16384, most // (seqs * heads * longest) - longest))
        cached = _log_int(rng, 2, room) if tokens or rng.random() < 0.2 else 0
        causal = tokens or rng.random() < 0.8
        return dict(kind="packed", seqs=seqs, shortest=rng.randint(0 if longest > 1 else 1, longest), longest=longest,
                    cached_least=rng.randint(0, cached), cached_most=cached, heads=heads, kv_heads=kv_heads, dim=dim,
                    causal=causal, window=_log_int(rng, 1, 4096) if causal and rng.random() < 0.3 else 0,
                    slack=rng.choice([0, 0, 0, 1, 7]), mix=mix)
    items = _log_int(rng, 1, 128)
    queries = rng.choice([1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 600)])
    keys = min(40000, most // (items * heads * queries))
    prefix = min(_log_int(rng, 1, 40000), keys) if rng.random() < 0.95 else 0
    room = queries + min(_log_int(rng, 1, 4096), max(1, keys - prefix))
    longest = rng.randint(queries, room)
    return dict(kind="prefix", items=items, queries=queries, prefix=prefix, shortest=rng.randint(0, longest),
                longest=longest, room=room, heads=heads, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.8, mix=mix)


# ------------------------------------------------------------------------------- lengths --


def _between(rng, count, lo, hi):
    """Lengths spread over the logarithm, both ends among them where there are two or more."""
    n = [lo, hi][:count] if count > 1 else [hi]
    return n + [min(hi, max(lo, _log_int(rng, lo + 1, hi + 1) - 1)) for _ in range(count - len(n))]


def _counts(case):
    """(queries, keys) of each sequence or item."""
    rng = random.Random(case["mix"])
    if case["kind"] == "prefix":
        return [case["queries"]] * case["items"], _between(rng, case["items"], case["shortest"], case["longest"])
    n = _between(rng, case["seqs"], case["shortest"], case["longest"])
    cached = _between(rng, case["seqs"], case["cached_least"], case["cached_most"])
    return n, [a + b for a, b in zip(n, cached)]


def _offsets(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


# ------------------------------------------------------------------------------- inputs --


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    queries, keys = _counts(case)
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):  # a tenth of the columns are larger, as projections have them
        wide = torch.where(torch.rand(shape[-1], device=DEV, generator=g) < 0.1, 2.0, 1.0)
        return (torch.randn(*shape, device=DEV, generator=g) * wide * scale).to(BF16)

    def ints(values):
        return torch.tensor(values, device=DEV, dtype=I32)

    if case["kind"] == "prefix":
        b, c = case["items"], case["room"]
        return dict(case=case, q=normal(b, case["queries"], h * d), k=normal(b, c, kvh * d), v=normal(b, c, kvh * d),
                    prefix_k=normal(case["prefix"], kvh * d), prefix_v=normal(case["prefix"], kvh * d), lengths=ints(keys))
    tq, tk = sum(queries), sum(keys)
    s = dict(case=case, offsets=ints(_offsets(queries)), k_offsets=ints(_offsets(keys)) if case["cached_most"] else None,
             q=normal(tq + case["slack"], h * d), out=None)
    rows = tk if case["cached_most"] else tq + case["slack"]
    s["k"], s["v"] = normal(rows, kvh * d), normal(rows, kvh * d)
    if case["slack"]:
        s["out"] = normal(tq + case["slack"], h * d)
    return s


# ------------------------------------------------------------------------- the operators --


def _softmax_weights(score, seen):
    """exp(score - its row's maximum) where seen, and its sum (at least a tiny number: rows that see nothing give zeros)."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    return p, p.sum(-1, keepdim=True).clamp(min=1e-30)


def _heads(x, kvh, d):
    """(N, T, KVH*G*D) as (N, KVH, G, T, D) in fp32."""
    n, t, w = x.shape
    return x.to(F32).view(n, t, kvh, w // (kvh * d), d).permute(0, 2, 3, 1, 4).contiguous()


def _plain_packed(s):
    c = s["case"]
    h, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    queries, keys = _counts(c)
    nq, nk = max(1, max(queries)), max(1, max(keys))
    qo = s["offsets"].long()
    ko = qo if s["k_offsets"] is None else s["k_offsets"].long()

    def padded(x, offsets, n):  # (S, n, W), and which of them are there
        at = offsets[:-1, None] + torch.arange(n, device=DEV)
        there = at < offsets[1:, None]
        if not x.shape[0]:
            return x.new_zeros(len(offsets) - 1, n, x.shape[1]), there, at
        return x[at.clamp(max=x.shape[0] - 1)], there, at

    q, q_there, at = padded(s["q"], qo, nq)
    k, k_there, _ = padded(s["k"], ko, nk)
    v, _, _ = padded(s["v"], ko, nk)
    pos = torch.arange(nq, device=DEV) + (ko.diff() - qo.diff())[:, None]      # (S, nq) among the keys
    seen = k_there[:, None, :].expand(-1, nq, -1)
    if c["causal"]:
        back = pos[:, :, None] - torch.arange(nk, device=DEV)
        seen = seen & (back >= 0)
        if c["window"]:
            seen = seen & (back < c["window"])
    q = _heads(q, kvh, d).reshape(len(queries), kvh, -1, d)                    # (S, KVH, G*nq, D)
    k, v = _heads(k, kvh, d).squeeze(2), _heads(v, kvh, d).squeeze(2)
    score = (q @ k.transpose(-1, -2).contiguous() * d ** -0.5).view(len(queries), kvh, h // kvh, nq, nk)
    p, total = _softmax_weights(score, seen[:, None, None])
    o = (p.view(len(queries), kvh, -1, nk) @ v).view(len(queries), kvh, h // kvh, nq, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(len(queries), nq, h * d).to(BF16)
    out = torch.zeros_like(s["q"]) if s["out"] is None else s["out"].clone()
    out[at[q_there]] = o[q_there]
    return out


def _plain_prefix(s):
    c = s["case"]
    h, kvh, d, t = c["heads"], c["kv_heads"], c["dim"], c["queries"]
    b, room, prefix = c["items"], c["room"], c["prefix"]
    q = _heads(s["q"], kvh, d)                                                 # (B, KVH, G, T, D)
    k, v = _heads(s["k"], kvh, d).squeeze(2), _heads(s["v"], kvh, d).squeeze(2)
    pk, pv = (_heads(x[None], kvh, d)[0].squeeze(1) for x in (s["prefix_k"], s["prefix_v"]))  # (KVH, P, D)
    n = s["lengths"].long()
    at = torch.arange(room, device=DEV)
    seen = (at < n[:, None])[:, None].expand(b, t, room)
    there = torch.ones(b, t, device=DEV, dtype=torch.bool)
    if c["causal"]:
        pos = n[:, None] - t + torch.arange(t, device=DEV)
        seen, there = seen & (at <= pos[..., None]), pos >= 0
    stacked = q.transpose(0, 1).reshape(kvh, -1, d)                            # (KVH, B*G*T, D)
    common = (stacked @ pk.transpose(-1, -2).contiguous()).view(kvh, b, h // kvh * t, prefix).transpose(0, 1)
    of_own = q.view(b, kvh, -1, d) @ k.transpose(-1, -2).contiguous()
    score = torch.cat([common, of_own], -1).view(b, kvh, h // kvh, t, prefix + room) * d ** -0.5
    seen = torch.cat([there[..., None].expand(b, t, prefix), seen], -1)
    p, total = _softmax_weights(score, seen[:, None, None])
    p = p.view(b, kvh, h // kvh * t, prefix + room)
    o = (p[..., :prefix].transpose(0, 1).reshape(kvh, b * (h // kvh) * t, prefix) @ pv).view(kvh, b, h // kvh * t, d).transpose(0, 1)
    o = (o + p[..., prefix:].contiguous() @ v).view(b, kvh, h // kvh, t, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, h * d).to(BF16)


def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_packed(s) if c["kind"] == "packed" else _plain_prefix(s)
    import ltxk

    if c["kind"] == "packed":
        return ltxk.packed_attention(s["q"], s["k"], s["v"], c["heads"], s["offsets"], kv_heads=c["kv_heads"],
                                     k_offsets=s["k_offsets"], causal=c["causal"], window=c["window"] or None, out=s["out"])
    return ltxk.prefix_attention(s["q"], s["k"], s["v"], s["prefix_k"], s["prefix_v"], c["heads"], kv_heads=c["kv_heads"],
                                 lengths=s["lengths"], causal=c["causal"])


# ----------------------------------------------------------------------- in 64 bits --


def _row_values(q, k, v, hi, lo, scale):
    """Each query of one head over keys lo .. hi - 1 of its own, q (n, D), k and v (m, D), all in fp64."""
    w = (q @ k.t().contiguous()) * scale
    j = torch.arange(k.shape[0], device=DEV)
    w = torch.where((j >= lo[:, None]) & (j < hi[:, None]), w, torch.full_like(w, -math.inf))
    w = torch.softmax(w, -1)
    return torch.where((hi > lo)[:, None], w.nan_to_num(0.0) @ v, torch.zeros_like(q))


def exact(case, seed):
    s = prepare(case, seed)
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    queries, keys = _counts(case)
    if sum(h * a * (b + case.get("prefix", 0)) * (d + 20) for a, b in zip(queries, keys)) > 3e12 or len(queries) * h > 6000:
        return None
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    if s.get("out") is not None:
        out.copy_(s["out"])
    qo, ko = _offsets(queries), _offsets(keys)
    for i, (n, m) in enumerate(zip(queries, keys)):
        if case["kind"] == "packed":
            q, k, v = s["q"][qo[i]:qo[i + 1]], s["k"][ko[i]:ko[i + 1]], s["v"][ko[i]:ko[i + 1]]
            to, p = out[qo[i]:qo[i + 1]], 0
        else:
            q, to, p = s["q"][i], out[i], case["prefix"]
            k, v = (torch.cat([x, y[i, :m]]) for x, y in ((s["prefix_k"], s["k"]), (s["prefix_v"], s["v"])))
        hi = torch.full((n,), p + m, device=DEV)
        lo = torch.zeros_like(hi)
        if case["causal"]:
            pos = torch.arange(m - n, m, device=DEV)
            hi = torch.where(pos >= 0, p + pos + 1, 0)
            if case.get("window"):
                lo = (pos + 1 - case["window"]).clamp(min=0)
        if not n or not k.shape[0]:
            continue
        k, v = k.to(F64), v.to(F64)
        for j in range(h):
            a, b = slice(j * d, (j + 1) * d), slice(j // (h // kvh) * d, (j // (h // kvh) + 1) * d)
            to[:, a] = _row_values(q[:, a].to(F64), k[:, b], v[:, b], hi, lo, 1 / math.sqrt(d))
    return out


def work(case):
    queries, keys = _counts(case)
    h, kvh, d, p = case["heads"], case["kv_heads"], case["dim"], case.get("prefix", 0)
    window = case.get("window") or (1 << 40)
    pairs = 0  # of a query and a key that it sees
    for n, m in zip(queries, keys):
        if not case["causal"]:
            pairs += n * (m + p)
            continue
        first = max(0, m - n)  # positions first .. m - 1 see min(position + 1, window) keys
        full = max(first, min(m, window))
        pairs += (full * (full + 1) - first * (first + 1)) // 2 + (m - full) * min(window, m) + (m - first) * p
    return {"bytes": 4 * d * (h * sum(queries) + kvh * (sum(keys) + p)), "flops": 4 * d * h * pairs}
