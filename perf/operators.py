"""Workloads of the serving operators: the 8-bit paged KV cache and the answers' log probabilities.

A program that serves many sequences keeps their keys and values in pages of a
few tokens each, in 8 bits (e4m3) with one scale for each page and kv head, and
reports how likely the tokens are that it answers with. Three kinds of case:

* ``append``: q/k norm and RoPE of a ragged batch's new tokens and the append
  of their keys and values to the pages (``launch_paged_append``);
* ``attend``: causal grouped-query attention of those tokens over the pages
  (``launch_paged_attention``);
* ``logprobs``: log probability of given tokens, entropy of the distribution
  and its top alternatives (``launch_token_logprobs``).

A case is a dict of plain values. ``prepare`` builds what the program holds
before the call, ``run`` makes one pass: with ``own`` through the framework's
entry points, otherwise in plain fp32 torch operations. ``exact`` computes the
same outputs in 64 bits, sequence by sequence.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
ROPE_THETA = 1_000_000.0
E4M3_MAX = 448.0
MIN_EXPONENT = -126  # the smallest scale is 2^-126


# -- cases ---------------------------------------------------------------------


def _append(name, batch, new, context, *, ragged, x, q_heads=32, kv_heads=8, head_dim=128, page=64, norm=True, lengths=1):
    return {"name": name, "kind": "append", "batch": batch, "new": new, "context": context, "ragged": ragged, "x": x,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "norm": norm,
            "lengths": lengths}


def _attend(name, batch, new, context, *, ragged, q, out, q_heads=32, kv_heads=8, head_dim=128, page=64, lengths=1):
    return {"name": name, "kind": "attend", "batch": batch, "new": new, "context": context, "ragged": ragged, "q": q,
            "out": out, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "lengths": lengths}


def _logprobs(name, rows, vocab, top, *, x, banned=0.0):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "x": x, "banned": banned}


def listed():
    return [
        # One sequence decoding: the smallest call, latency is all of it.
        _append("append_one", 1, 1, 600, ragged=False, x="f32"),
        # A decode step of many sequences at unlike positions, small pages.
        _append("append_batch", 48, 1, 4000, ragged=True, x="bf16", page=16),
        # Chunks of a few prompts of unlike lengths, heads without norms (seven q heads share a kv head).
        _append("append_ragged", 5, 700, 300, ragged=True, x="f16", q_heads=14, kv_heads=2, head_dim=64, page=32,
                norm=False),
        # Four long prompts at once.
        _append("append_prompt", 4, 2048, 0, ragged=False, x="f32"),
        # One sequence decoding inside a short conversation.
        _attend("attend_one", 1, 1, 600, ragged=False, q="f32", out="bf16"),
        # A decode step of many sequences of unlike lengths.
        _attend("attend_batch", 32, 1, 4000, ragged=True, q="bf16", out="bf16", page=16),
        # One token far into a very long document.
        _attend("attend_long", 1, 1, 131000, ragged=False, q="f32", out="f32", page=128),
        # A few tokens of each sequence to verify at once, wide heads.
        _attend("attend_verify", 16, 6, 3001, ragged=True, q="f16", out="f32", q_heads=16, kv_heads=4, head_dim=256),
        # The second chunk of a long prompt: attention against the chunk and what the cache already holds.
        _attend("attend_prompt", 1, 1531, 517, ragged=False, q="f32", out="bf16"),
        # The token just chosen and its five nearest alternatives.
        _logprobs("logprobs_one", 1, 151936, 5, x="f32"),
        # A decode step of many sequences under a grammar that bans most of an odd vocabulary.
        _logprobs("logprobs_batch", 48, 50257, 20, x="bf16", banned=0.7),
        # Scoring a whole text: every position's next token.
        _logprobs("logprobs_score", 1531, 151936, 0, x="f32"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


GEOMETRIES = [(32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 8, 128), (8, 1, 128), (14, 2, 64), (4, 4, 64), (16, 4, 256),
              (8, 4, 256), (20, 4, 128)]


def draw(rng):
    pick = rng.random()
    q_heads, kv_heads, head_dim = rng.choice(GEOMETRIES)
    heads = {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128]),
             "lengths": rng.randint(1, 1 << 20)}
    if pick < 0.3:
        if rng.random() < 0.5:
            batch, new = _log_int(rng, 1, 64), 1
        else:
            batch = _log_int(rng, 1, 8)
            new = _log_int(rng, 2, 6000 // batch)
        case = _append("", batch, new, rng.choice([0, _log_int(rng, 1, 4000)]), ragged=rng.random() < 0.7,
                       x=rng.choice(["f32", "bf16", "f16"]), norm=rng.random() < 0.7, **heads)
    elif pick < 0.7:
        kind = rng.random()
        if kind < 0.45:
            batch, new = _log_int(rng, 1, 40), 1
            context = _log_int(rng, 1, 100000 // batch)
        elif kind < 0.65:
            batch, new = _log_int(rng, 1, 16), rng.randint(2, 12)
            context = _log_int(rng, 1, 3000)
        else:
            batch = rng.choice([1, 1, 2, 3])
            new = _log_int(rng, 17, 1200 // batch)
            context = rng.choice([0, _log_int(rng, 1, 700)])
        case = _attend("", batch, new, context, ragged=rng.random() < 0.7, q=rng.choice(["f32", "bf16", "f16"]),
                       out=rng.choice(["f32", "bf16", "f16"]), **heads)
    else:
        vocab = _log_int(rng, 1000, 260000)
        case = _logprobs("", _log_int(rng, 1, max(1, min(1531, 200_000_000 // vocab))), vocab, rng.choice([0, 1, 5, 20, 32]),
                         x=rng.choice(["f32", "bf16", "f16"]), banned=rng.choice([0.0, 0.0, 0.3, 0.9]))
        if case["rows"] * vocab > 20_000_000 and case["top"]:
            case["top"] = 0
    del case["name"]
    return case


def _lengths(case):
    """(rows already cached, new tokens) of each sequence; the first is the longest of a ragged batch."""
    r = random.Random(case["lengths"])
    got = [(case["context"], case["new"])]
    for _ in range(case["batch"] - 1):
        got.append((r.randint(0, case["context"]), _log_int(r, 1, case["new"])) if case["ragged"] else got[0])
    return got


def work(case):
    """Bytes: each input read once and each output written once. Flops: products and sums of the definition."""
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["x"]] + case["rows"] * (8 + 8 + 12 * case["top"]), "flops": 5 * n}
    lengths = _lengths(case)
    tokens = sum(n for _, n in lengths)
    qh, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        x = tokens * (qh + 2 * kv) * d * SIZES[case["x"]]
        return {"bytes": x + tokens * (qh * d * 4 + 2 * kv * d + d * 4), "flops": 10 * tokens * (qh + kv) * d}
    rows = sum(c + n for c, n in lengths)
    seen = sum(n * c + n * (n + 1) // 2 for c, n in lengths)
    return {"bytes": 2 * rows * kv * d + 8 * (rows // case["page"] + 1) * kv
            + tokens * qh * d * (SIZES[case["q"]] + SIZES[case["out"]]), "flops": 4 * seen * qh * d}


# -- inputs --------------------------------------------------------------------


def _power_scale(amax):
    """The least power of two, from 2^-126 on, that brings amax within e4m3's 448 = 0.875 * 2^9."""
    mantissa, exponent = torch.frexp(amax)
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    exponent = torch.where(amax > 0, exponent, MIN_EXPONENT).clamp(min=MIN_EXPONENT)
    return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _history(g, pages, kv, rows, cols):
    """Filled pages: normal values whose size differs from page to page and head to head."""
    x = torch.randn(pages, kv, rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(pages, kv, 1, 1, generator=g, device="cuda"))
    scale = _power_scale(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(case=case, kind=case["kind"])
    if s.kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
        # A few likely tokens in each row, the given one among them as often as not.
        likely = torch.randint(vocab, (rows, 8), generator=g, device="cuda")
        x.scatter_(1, likely, 6 + 4 * torch.rand(rows, 8, generator=g, device="cuda"))
        s.tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, likely[:, 0],
                               torch.randint(vocab, (rows,), generator=g, device="cuda"))
        if case["banned"]:
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < case["banned"], -math.inf)
            x.scatter_(1, s.tokens[:, None], 5.0)
        s.logits = x.to(DTYPES[case["x"]])
        return s

    lengths = _lengths(case)
    qh, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    used = [-(-(c + n) // page) for c, n in lengths]
    # Sequences own pages spread over the pool; the table's entries behind the last page hold no page.
    pool = sum(used) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    s.page_table = torch.full((case["batch"], max(used) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        s.page_table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for _, n in lengths:
        starts.append(starts[-1] + n)
    s.tokens, s.longest = starts[-1], max(n for _, n in lengths)
    s.query_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s.context_lens = torch.tensor([c for c, _ in lengths], dtype=torch.int32, device="cuda")
    s.k_pages, s.k_scales = _history(g, pool, kv, page, d)
    s.v_pages, s.v_scales = _history(g, pool, kv, d, page)  # values lie transposed: head_dim rows of page columns
    if s.kind == "attend":
        s.q = _randn(g, DTYPES[case["q"]], s.tokens, qh, d)
        s.scaling = d**-0.5
        return s
    x = DTYPES[case["x"]]
    s.q = _randn(g, x, s.tokens, qh * d)
    s.k = _randn(g, x, s.tokens, kv * d)
    s.v = _randn(g, x, s.tokens, kv * d)
    s.q_norm = s.k_norm = None
    if case["norm"]:
        s.q_norm = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
        s.k_norm = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    positions = max(c + n for c, n in lengths)
    inv = 1.0 / (ROPE_THETA ** (torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d))
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    s.cos, s.sin = angle.cos().float(), angle.sin().float()
    return s


# -- one pass ------------------------------------------------------------------


def run(s):
    return _OWN[s.kind](s) if own else _PLAIN[s.kind](s)


def _own_append(s):
    from nanoquant_amd.runtime import shell_ops as ops

    cache = ops.PagedCache(s.k_pages, s.v_pages, s.k_scales, s.v_scales)
    q = ops.launch_paged_append(s.q, s.k, s.v, cache, q_heads=s.case["q_heads"], q_norm=s.q_norm, k_norm=s.k_norm,
                                eps=EPS, cos=s.cos, sin=s.sin, page_table=s.page_table, query_starts=s.query_starts,
                                context_lens=s.context_lens)
    return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages, "k_scales": s.k_scales, "v_scales": s.v_scales}


def _own_attend(s):
    from nanoquant_amd.runtime import shell_ops as ops

    cache = ops.PagedCache(s.k_pages, s.v_pages, s.k_scales, s.v_scales)
    return ops.launch_paged_attention(s.q, cache, page_table=s.page_table, query_starts=s.query_starts,
                                      context_lens=s.context_lens, scaling=s.scaling,
                                      out_dtype=DTYPES[s.case["out"]])


def _own_logprobs(s):
    from nanoquant_amd.runtime import shell_ops as ops

    return dict(ops.launch_token_logprobs(s.logits, s.tokens, top=s.case["top"])._asdict())


def _sequence_of(s):
    """Each token's sequence and its place among that sequence's new tokens."""
    token = torch.arange(s.tokens, device="cuda", dtype=torch.int32)
    seq = torch.bucketize(token, s.query_starts[1:], right=True)
    return seq, (token - s.query_starts[seq]).long()


def _rope(x, norm, cos, sin):
    if norm is not None:
        x = norm.float() * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS))
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    c = s.case
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    seq, place = _sequence_of(s)
    position = s.context_lens[seq].long() + place
    cos, sin = s.cos[position][:, None], s.sin[position][:, None]
    q = _rope(s.q.float().view(s.tokens, -1, d), s.q_norm, cos, sin)
    k = _rope(s.k.float().view(s.tokens, kv, d), s.k_norm, cos, sin)
    v = s.v.float().view(s.tokens, kv, d)
    where = s.page_table[seq, position // page].long()
    row = position % page
    # Each page's first new row: what lies before it stays, with the scale that it needs; a page begun at its first row is new.
    pages = s.k_pages.shape[0]
    first = torch.full((pages,), page, device="cuda").index_reduce_(0, where, row, "amin")
    touched = first < page
    kept = torch.arange(page, device="cuda") < first[:, None]
    _plain_store(k, s.k_pages, s.k_scales, where, row, first, touched, kept[:, None, :, None])
    _plain_store(v, s.v_pages.transpose(2, 3), s.v_scales, where, row, first, touched, kept[:, None, :, None])
    return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages, "k_scales": s.k_scales, "v_scales": s.v_scales}


def _plain_store(x, pages, scales, where, row, first, touched, kept):
    old = torch.where((first == 0)[:, None], 2.0**MIN_EXPONENT, scales)
    need = _power_scale(torch.zeros_like(scales).index_reduce_(0, where, x.abs().amax(-1), "amax"))
    new = torch.where(touched[:, None], torch.maximum(old, need), scales)
    moved = (pages.float() * (old / new)[:, :, None, None]).to(torch.float8_e4m3fn)
    moved = torch.where(kept & touched[:, None, None, None], moved.view(torch.uint8), pages.view(torch.uint8))
    moved[where, :, row] = (x / new[where][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    pages.view(torch.uint8).copy_(moved)
    scales.copy_(new)


def _plain_attend(s):
    c = s.case
    batch, kv, d = c["batch"], c["kv_heads"], c["head_dim"]
    group = c["q_heads"] // kv
    table = s.page_table.clamp(min=0).long()
    rows = table.shape[1] * c["page"]

    def gathered(pages, scales):
        x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        return x * scales[table][..., None, None]

    k = gathered(s.k_pages, s.k_scales).transpose(1, 2).reshape(batch, kv, rows, d)
    v = gathered(s.v_pages, s.v_scales).transpose(3, 4).transpose(1, 2).reshape(batch, kv, rows, d)
    place = torch.arange(s.longest, device="cuda")
    token = (s.query_starts[:-1, None] + place).clamp(max=s.tokens - 1)
    q = s.q.float()[token].view(batch, s.longest, kv, group, d).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(batch, kv, group * s.longest, d) @ k.transpose(2, 3)) * s.scaling
    scores = scores.view(batch, kv, group, s.longest, rows)
    seen = torch.arange(rows, device="cuda") <= (s.context_lens[:, None] + place)[..., None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p.view(batch, kv, group * s.longest, rows) @ v).view(batch, kv, group, s.longest, d)
    out = out / p.sum(-1, keepdim=True)
    seq, at = _sequence_of(s)
    out = out.permute(0, 3, 1, 2, 4)[seq, at]
    return out.reshape(s.tokens, c["q_heads"] * d).to(DTYPES[c["out"]])


def _plain_logprobs(s):
    x = s.logits.float()
    top = s.case["top"]
    centred = x - x.amax(-1, keepdim=True)
    weight = torch.exp(centred)
    total = weight.sum(-1)
    spread = torch.where(weight > 0, weight * centred, 0.0).sum(-1)
    log_total = torch.log(total)
    out = {"logprobs": centred.gather(1, s.tokens[:, None])[:, 0] - log_total, "entropy": log_total - spread / total}
    # The largest first, the lowest index first among equals: one whole number orders by both.
    bits = (centred + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = (order << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device="cuda")) if top else order[:, :0]
    ids = 0xFFFFFFFF - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
    out["top_ids"] = ids
    out["top_logprobs"] = centred.gather(1, ids) - log_total[:, None]
    return out


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}
_OWN = {"append": _own_append, "attend": _own_attend, "logprobs": _own_logprobs}


# -- the same outputs in 64 bits -------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](s)


def _power(exponent):
    """2 to a whole exponent, exactly."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """The e4m3 value nearest to x, ties to the even one: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    _, exponent = torch.frexp(x)
    step = _power((exponent - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_append(s):
    c = s.case
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    stored = {"k": s.k_pages.double(), "v": s.v_pages.double().transpose(2, 3).contiguous()}
    scales = {"k": s.k_scales.double(), "v": s.v_scales.double()}
    q_out = torch.empty(s.tokens, c["q_heads"], d, dtype=torch.float64, device="cuda")

    def turned(x, norm, position):
        x = x.double().view(x.shape[0], -1, d)
        if norm is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) * norm.double()
        cos, sin = s.cos[position].double()[:, None, :], s.sin[position].double()[:, None, :]
        low, high = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([low * cos - high * sin, high * cos + low * sin], dim=-1)

    for i, (context, new) in enumerate(_lengths(c)):
        begin = int(s.query_starts[i])
        rows = slice(begin, begin + new)
        position = torch.arange(context, context + new, device="cuda")
        q_out[rows] = turned(s.q[rows], s.q_norm, position)
        fresh = {"k": turned(s.k[rows], s.k_norm, position), "v": s.v[rows].double().view(new, kv, d)}
        for slot in range(context // page, (context + new - 1) // page + 1):
            at = int(s.page_table[i, slot])
            low, high = max(context, slot * page), min(context + new, (slot + 1) * page)
            begun = low - slot * page
            for name, x in fresh.items():
                x = x[low - context:high - context].transpose(0, 1)  # [kv, rows, d]
                amax = x.abs().amax((1, 2))
                exponent = torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(min=MIN_EXPONENT)
                before = scales[name][at] if begun else torch.full_like(amax, 2.0**MIN_EXPONENT)
                after = torch.maximum(before, _power(exponent))
                kept = stored[name][at, :, :begun] * (before / after)[:, None, None]
                stored[name][at, :, :begun] = _e4m3(kept)
                stored[name][at, :, begun:begun + high - low] = _e4m3(x / after[:, None, None])
                scales[name][at] = after
    return {"q": q_out, "k_pages": stored["k"], "v_pages": stored["v"].transpose(2, 3), "k_scales": scales["k"],
            "v_scales": scales["v"]}


def _exact_attend(s):
    c = s.case
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    out = torch.empty(s.tokens, kv, c["q_heads"] // kv, d, dtype=torch.float64, device="cuda")
    for i, (context, new) in enumerate(_lengths(c)):
        begin, rows = int(s.query_starts[i]), context + new
        at = s.page_table[i, :-(-rows // page)].long()
        k = s.k_pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * s.k_scales.double()[at][..., None, None]
        v = s.v_pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * s.v_scales.double()[at][..., None, None]
        seen = torch.arange(rows, device="cuda")[None] <= torch.arange(context, rows, device="cuda")[:, None]
        for head in range(kv):
            keys = k[:, head].reshape(-1, d)[:rows]
            values = v[:, head].transpose(1, 2).reshape(-1, d)[:rows]
            q = s.q[begin:begin + new].view(new, kv, -1, d)[:, head].double()
            for j in range(q.shape[1]):
                scores = (q[:, j] @ keys.T * s.scaling).masked_fill(~seen, -math.inf)
                out[begin:begin + new, head, j] = torch.softmax(scores, -1) @ values
    return out.view(s.tokens, -1)


def _exact_logprobs(s):
    top = s.case["top"]
    parts = {"logprobs": [], "entropy": [], "top_logprobs": []}
    for x, token in zip(s.logits.split(64), s.tokens.split(64)):
        x = x.double()
        log_p = x - torch.logsumexp(x, -1, keepdim=True)
        p = log_p.exp()
        parts["logprobs"].append(log_p.gather(1, token[:, None])[:, 0])
        parts["entropy"].append(-torch.where(p > 0, p * log_p, 0.0).sum(-1))
        parts["top_logprobs"].append(torch.sort(log_p, -1, descending=True).values[:, :top] if top else log_p[:, :0])
    return {**{name: torch.cat(x) for name, x in parts.items()}, "top_ids": None}
