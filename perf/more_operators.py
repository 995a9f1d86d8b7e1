"""Workloads of serving long conversations in bounded memory and traffic.

A program that serves many long conversations from the 8-bit paged KV cache
reads a prefix that they share once for all, keeps each within a number of
cache rows by evicting those that little attention falls on, and holds its
output projection in 4 bits. Four kinds of case:

* ``shared``: causal grouped-query attention of a ragged batch whose sequences
  hold the same first rows, with each row's log-sum-exp
  (``launch_shared_attention``);
* ``weigh``: how much attention every cached row gets from the tokens of a
  call, added to what it got before (``launch_attention_weights``);
* ``evict``: the rows that stay, the heaviest between the first and the newest,
  moved to fresh pages (``launch_paged_evict``);
* ``int4``: products with 4-bit weights and group scales
  (``launch_int4_projection``).

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
E4M3_MAX = 448.0
MIN_EXPONENT = -126  # the smallest scale is 2^-126


# -- cases ---------------------------------------------------------------------


def _shared(name, batch, new, prefix, context, *, ragged, q, out, q_heads=32, kv_heads=8, head_dim=128, page=64, lengths=1):
    """`prefix` shared rows, up to `context` cached rows of its own behind them and up to `new` tokens for each sequence."""
    return {"name": name, "kind": "shared", "batch": batch, "new": new, "prefix": prefix, "context": context,
            "ragged": ragged, "q": q, "out": out, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "lengths": lengths}


def _weigh(name, batch, new, context, first, *, ragged, q, q_heads=32, kv_heads=8, head_dim=128, page=64, lengths=1):
    return {"name": name, "kind": "weigh", "batch": batch, "new": new, "context": context, "first": first,
            "ragged": ragged, "q": q, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "lengths": lengths}


def _evict(name, batch, context, budget, first, recent, *, ragged, kv_heads=8, head_dim=128, page=64, lengths=1):
    return {"name": name, "kind": "evict", "batch": batch, "context": context, "budget": budget, "first": first,
            "recent": recent, "ragged": ragged, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "lengths": lengths}


def _int4(name, tokens, in_features, out_features, group, *, x, out, scale, zeros):
    return {"name": name, "kind": "int4", "tokens": tokens, "in": in_features, "outs": out_features, "group": group,
            "x": x, "out": out, "scale": scale, "zeros": zeros}


def listed():
    return [
        # Two short conversations under one system prompt: the smallest call, latency is all of it.
        _shared("shared_pair", 2, 1, 500, 90, ragged=True, q="f32", out="bf16"),
        # A decode step of many conversations about one long document.
        _shared("shared_batch", 32, 1, 16000, 700, ragged=True, q="bf16", out="bf16", page=16),
        # Chunks of unlike lengths, each behind the same instructions, wide heads.
        _shared("shared_chunks", 6, 300, 1001, 133, ragged=True, q="f16", out="f32", q_heads=16, kv_heads=4, head_dim=256,
                page=32),
        # One token of one conversation.
        _weigh("weigh_one", 1, 1, 700, 4, ragged=False, q="f32"),
        # A decode step of many conversations of unlike lengths, small pages.
        _weigh("weigh_batch", 32, 1, 4000, 4, ragged=True, q="bf16", page=16),
        # A prompt's second chunk, whose rows all count.
        _weigh("weigh_prompt", 1, 1531, 517, 0, ragged=False, q="bf16"),
        # One conversation that has outgrown its rows by a little.
        _evict("evict_one", 1, 1100, 1000, 4, 128, ragged=False),
        # Many conversations, most of them too long; the whole pages of their first rows stay where they are.
        _evict("evict_batch", 24, 6001, 2000, 133, 500, ragged=True, kv_heads=4, head_dim=64, page=32),
        # A very long document cut to a quarter.
        _evict("evict_long", 1, 131000, 32768, 4, 1024, ragged=False, page=128),
        # One token through a small model's gate projection.
        _int4("int4_gate", 1, 1152, 6912, 32, x="bf16", out="bf16", scale="bf16", zeros=False),
        # Several sequences' tokens through a down projection with zero points.
        _int4("int4_down", 11, 10240, 2560, 64, x="f16", out="f16", scale="f16", zeros=True),
        # The output projection of one token.
        _int4("int4_head", 1, 4096, 151936, 128, x="f32", out="f32", scale="f16", zeros=False),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


GEOMETRIES = [(32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 8, 128), (8, 1, 128), (14, 2, 64), (4, 4, 64), (16, 4, 256),
              (8, 4, 256), (20, 4, 128)]
IN_FEATURES = [1152, 2560, 4096, 4096, 6912, 10240, 14336]


def draw(rng):
    pick = rng.random()
    q_heads, kv_heads, head_dim = rng.choice(GEOMETRIES)
    heads = {"kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128]),
             "lengths": rng.randint(1, 1 << 20)}
    if pick < 0.3:
        if rng.random() < 0.6:
            batch, new = _log_int(rng, 2, 64), 1
            prefix = _log_int(rng, 64, 20000)
        else:
            batch = _log_int(rng, 2, 8)
            new, prefix = _log_int(rng, 2, 1200 // batch), _log_int(rng, 64, 1500)
        case = _shared("", batch, new, prefix, rng.choice([0, _log_int(rng, 1, 700)]), ragged=rng.random() < 0.8,
                       q=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16", "f16"]), q_heads=q_heads, **heads)
    elif pick < 0.55:
        if rng.random() < 0.6:
            batch, new = _log_int(rng, 1, 40), rng.choice([1, 1, 1, 4])
            context = _log_int(rng, 1, 100000 // batch)
        else:
            batch = rng.choice([1, 1, 2, 3])
            new, context = _log_int(rng, 5, 1200 // batch), rng.choice([0, _log_int(rng, 1, 700)])
        case = _weigh("", batch, new, context, rng.choice([0, 4, rng.randint(0, 64)]), ragged=rng.random() < 0.7,
                      q=rng.choice(["f32", "bf16", "f16"]), q_heads=q_heads, **heads)
    elif pick < 0.75:
        batch = _log_int(rng, 1, 40)
        context = _log_int(rng, 50, 130000 // batch)
        budget = max(8, round(context * rng.uniform(0.1, 0.98)))
        first = rng.choice([0, 4, rng.randint(0, budget // 4)])
        case = _evict("", batch, context, budget, min(first, budget), rng.randint(0, budget // 3), ragged=rng.random() < 0.7,
                      **heads)
    else:
        in_features = rng.choice(IN_FEATURES + [32 * rng.randint(1, 400)])
        outs = _log_int(rng, 16, min(151936, 600_000_000 // in_features))
        tokens = rng.choice([1, 1, 1, rng.randint(2, 16)])
        if in_features * outs > 100_000_000:
            tokens = 1
        case = _int4("", tokens, in_features, outs, rng.choice([32, 64, 128]), x=rng.choice(["f32", "bf16", "f16"]),
                     out=rng.choice(["f32", "bf16", "f16"]), scale=rng.choice(["f32", "bf16", "f16"]),
                     zeros=rng.random() < 0.5)
    del case["name"]
    return case


def _lengths(case):
    """(rows already cached, new tokens) of each sequence; the first is the longest of a ragged batch."""
    r = random.Random(case["lengths"])
    base, new = case.get("prefix", 0), case.get("new", 0)
    got = [(base + case["context"], new)]
    for _ in range(case["batch"] - 1):
        got.append((base + r.randint(0, case["context"]), _log_int(r, 1, new) if new else 0) if case["ragged"] else got[0])
    return got


def work(case):
    """Bytes: each input read once and each output written once. Flops: products and sums of the definition."""
    kind = case["kind"]
    if kind == "int4":
        t, k, n = case["tokens"], case["in"], case["outs"]
        groups = n * -(-k // case["group"])
        return {"bytes": n * k // 2 + groups * (SIZES[case["scale"]] + case["zeros"]) + t * k * SIZES[case["x"]]
                + t * n * SIZES[case["out"]], "flops": 2 * t * n * k}
    lengths = _lengths(case)
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    if kind == "evict":
        budget, first, recent = case["budget"], case["first"], case["recent"]
        longer = [c for c, _ in lengths if c > budget]
        moved = len(longer) * (budget - first // page * page)
        weighed = sum(c - first - recent for c in longer)
        return {"bytes": kv * (4 * moved * d + 4 * weighed + 8 * moved) + len(lengths) * kv * budget * 4, "flops": kv * weighed}
    tokens = sum(n for _, n in lengths)
    qh = case["q_heads"]
    rows = sum(c + n for c, n in lengths)
    if kind == "weigh":
        seen = sum(n * c + n * (n + 1) // 2 for c, n in lengths)
        return {"bytes": rows * kv * (d + 8) + tokens * qh * (d * SIZES[case["q"]] + 4), "flops": 2 * seen * qh * d}
    held = rows - (len(lengths) - 1) * case["prefix"]
    seen = sum(n * c + n * (n + 1) // 2 for c, n in lengths)
    return {"bytes": 2 * held * kv * d + 8 * (held // page + 1) * kv
            + tokens * qh * (d * (SIZES[case["q"]] + SIZES[case["out"]]) + 4), "flops": 4 * seen * qh * d}


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


def _received(g, *shape):
    """Attention that rows got so far: a few heavy ones, some that got none at all."""
    x = torch.exp(2.0 * torch.randn(*shape, generator=g, device="cuda"))
    return x.masked_fill_(torch.rand(*shape, generator=g, device="cuda") < 0.05, 0.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(case=case, kind=case["kind"])
    if s.kind == "int4":
        outs, groups = case["outs"], -(-case["in"] // case["group"])

        def nibbles():
            x = torch.randn(outs, case["in"] // 2, generator=g, device="cuda")
            return x.mul_(2.7).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)

        s.packed = nibbles() | (nibbles() << 4)
        s.scales = (0.01 * (0.5 + torch.rand(outs, groups, generator=g, device="cuda"))).to(DTYPES[case["scale"]])
        s.zeros = None
        if case["zeros"]:
            s.zeros = torch.randint(5, 12, (outs, groups), generator=g, device="cuda", dtype=torch.uint8)
        x = torch.randn(case["tokens"], case["in"], generator=g, device="cuda")
        # A few channels are much larger than the others.
        x *= torch.where(torch.rand(case["in"], generator=g, device="cuda") < 0.01, 30.0, 1.0)
        s.x = x.to(DTYPES[case["x"]])
        return s

    lengths = _lengths(case)
    batch, kv, d, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    rows = [c + n for c, n in lengths]
    used = [-(-r // page) for r in rows]
    # Sequences own pages spread over the pool; the table's entries behind the last page hold no page.
    shared = case.get("prefix", 0) // page
    fresh = -(-case["budget"] // page) - case["first"] // page if s.kind == "evict" else 0
    pool = shared + sum(used) - shared * batch + fresh * batch + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    s.page_table = torch.full((batch, max(used) + 1), -1, dtype=torch.int32, device="cuda")
    s.page_table[:, :shared] = order[:shared]
    at = shared
    for i, n in enumerate(used):
        s.page_table[i, shared:n] = order[at:at + n - shared]
        at += n - shared
    s.context_lens = torch.tensor([c for c, _ in lengths], dtype=torch.int32, device="cuda")
    s.k_pages, s.k_scales = _history(g, pool, kv, page, d)
    s.v_pages, s.v_scales = _history(g, pool, kv, d, page)  # values lie transposed: head_dim rows of page columns
    if s.kind == "evict":
        s.into = order[at:at + fresh * batch].view(batch, fresh).contiguous()
        s.weights = _received(g, pool, kv, page)
        return s
    starts = [0]
    for _, n in lengths:
        starts.append(starts[-1] + n)
    s.tokens, s.longest = starts[-1], max(n for _, n in lengths)
    s.query_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s.q = torch.randn(s.tokens, case["q_heads"], d, generator=g, device="cuda").to(DTYPES[case["q"]])
    s.scaling = d**-0.5
    if s.kind == "weigh":
        s.weights = _received(g, pool, kv, page)
        s.out = torch.zeros_like(s.weights)
        s.lse = _scores_lse(s)  # as the attention of the same call left it
    return s


def _scores_lse(s):
    """The attention's log-sum-exp, sequence by sequence."""
    kv, d, page = s.case["kv_heads"], s.case["head_dim"], s.case["page"]
    parts = []
    for i, (context, new) in enumerate(_lengths(s.case)):
        at = s.page_table[i, :-(-(context + new) // page)].long()
        k = s.k_pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * s.k_scales[at][..., None, None]
        k = k.transpose(0, 1).reshape(kv, -1, d)[:, :context + new].contiguous()
        begin = sum(n for _, n in _lengths(s.case)[:i])
        q = s.q[begin:begin + new].float().view(new, kv, -1, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
        scores = (torch.matmul(q, k.transpose(1, 2)) * s.scaling).view(kv, -1, new, context + new)
        row = torch.arange(context + new, device="cuda")
        scores.masked_fill_(row > row[context:, None], -math.inf)
        parts.append(torch.logsumexp(scores, -1).permute(2, 0, 1).reshape(new, -1))
    return torch.cat(parts)


# -- one pass ------------------------------------------------------------------


def run(s):
    return _OWN[s.kind](s) if own else _PLAIN[s.kind](s)


def _own_shared(s):
    from nanoquant_amd.runtime import shell_ops as ops

    cache = ops.PagedCache(s.k_pages, s.v_pages, s.k_scales, s.v_scales)
    lse = torch.empty(s.tokens, s.case["q_heads"], device="cuda")
    out = ops.launch_shared_attention(s.q, cache, page_table=s.page_table, query_starts=s.query_starts,
                                      context_lens=s.context_lens, shared_rows=s.case["prefix"], scaling=s.scaling,
                                      out_dtype=DTYPES[s.case["out"]], lse=lse)
    return {"out": out, "lse": lse}


def _own_weigh(s):
    from nanoquant_amd.runtime import shell_ops as ops

    cache = ops.PagedCache(s.k_pages, s.v_pages, s.k_scales, s.v_scales)
    return ops.launch_attention_weights(s.q, cache, s.lse, s.weights, page_table=s.page_table,
                                        query_starts=s.query_starts, context_lens=s.context_lens, scaling=s.scaling,
                                        first=s.case["first"], out=s.out)


def _own_evict(s):
    from nanoquant_amd.runtime import shell_ops as ops

    c = s.case
    cache = ops.PagedCache(s.k_pages, s.v_pages, s.k_scales, s.v_scales)
    got = ops.launch_paged_evict(cache, s.weights, page_table=s.page_table, context_lens=s.context_lens, into=s.into,
                                 budget=c["budget"], first=c["first"], recent=c["recent"])
    return _evicted(s, got.page_table, got.context_lens, got.rows)


def _evicted(s, page_table, context_lens, rows):
    return {"page_table": page_table, "context_lens": context_lens, "rows": rows, "k_pages": s.k_pages,
            "v_pages": s.v_pages, "k_scales": s.k_scales, "v_scales": s.v_scales, "weights": s.weights}


def _own_int4(s):
    from nanoquant_amd.runtime import shell_ops as ops

    return ops.launch_int4_projection(s.x, ops.Int4Matrix(s.packed, s.scales, s.zeros), out_dtype=DTYPES[s.case["out"]])


def _gathered(pages, scales, table):
    x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
    return x * scales[table][..., None, None]


def _sequence_of(s):
    """Each token's sequence and its place among that sequence's new tokens."""
    token = torch.arange(s.tokens, device="cuda", dtype=torch.int32)
    seq = torch.bucketize(token, s.query_starts[1:], right=True)
    return seq, (token - s.query_starts[seq]).long()


def _by_sequence(s, x):
    """Token rows as [batch, longest, ...]; places behind a sequence's tokens repeat others."""
    place = torch.arange(s.longest, device="cuda")
    return x[(s.query_starts[:-1, None] + place).clamp(max=s.tokens - 1)]


def _plain_shared(s):
    c = s.case
    batch, kv, d, page = c["batch"], c["kv_heads"], c["head_dim"], c["page"]
    group = c["q_heads"] // kv
    whole = c["prefix"] // page  # pages of the prefix; its last rows are each sequence's own
    head = s.page_table[0, :whole].long()
    k0 = _gathered(s.k_pages, s.k_scales, head).transpose(0, 1).reshape(kv, whole * page, d)
    v0 = _gathered(s.v_pages, s.v_scales, head).permute(1, 0, 3, 2).reshape(kv, whole * page, d)
    q0 = s.q.float().view(s.tokens, kv, group, d).transpose(0, 1).reshape(kv, s.tokens * group, d)
    s0 = (q0 @ k0.transpose(1, 2)) * s.scaling  # [kv, tokens * group, shared rows]

    table = s.page_table[:, whole:].clamp(min=0).long()
    rows = table.shape[1] * page
    k = _gathered(s.k_pages, s.k_scales, table).transpose(1, 2).reshape(batch, kv, rows, d)
    v = _gathered(s.v_pages, s.v_scales, table).transpose(3, 4).transpose(1, 2).reshape(batch, kv, rows, d)
    q = _by_sequence(s, s.q.float()).view(batch, s.longest, kv, group, d).permute(0, 2, 1, 3, 4)
    s1 = (q.reshape(batch, kv, s.longest * group, d) @ k.transpose(2, 3)) * s.scaling
    position = s.context_lens[:, None] - whole * page + torch.arange(s.longest, device="cuda")
    seen = torch.arange(rows, device="cuda") <= position[..., None]
    s1 = s1.view(batch, kv, s.longest, group, rows).masked_fill(~seen[:, None, :, None], -math.inf)

    seq, at = _sequence_of(s)
    m0 = s0.amax(-1).view(kv, s.tokens, group).transpose(0, 1) if whole else s0.new_full((s.tokens, kv, group), -math.inf)
    m = torch.maximum(m0, s1.amax(-1).transpose(1, 2)[seq, at])
    p0 = torch.exp(s0 - m.transpose(0, 1).reshape(kv, -1, 1))
    spread = s1.new_zeros(batch, s.longest, kv, group)
    spread[seq, at] = m
    p1 = torch.exp(s1 - spread.transpose(1, 2)[..., None])
    total = p0.sum(-1).view(kv, s.tokens, group).transpose(0, 1) + p1.sum(-1).transpose(1, 2)[seq, at]
    out = (p0 @ v0).view(kv, s.tokens, group, d).transpose(0, 1)
    out = out + (p1.view(batch, kv, -1, rows) @ v).view(batch, kv, s.longest, group, d).transpose(1, 2)[seq, at]
    out = out / total[..., None]
    return {"out": out.reshape(s.tokens, -1).to(DTYPES[c["out"]]), "lse": (m + torch.log(total)).reshape(s.tokens, -1)}


def _plain_weigh(s):
    c = s.case
    batch, kv, d, page = c["batch"], c["kv_heads"], c["head_dim"], c["page"]
    group = c["q_heads"] // kv
    table = s.page_table.clamp(min=0).long()
    rows = table.shape[1] * page
    k = _gathered(s.k_pages, s.k_scales, table).transpose(1, 2).reshape(batch, kv, rows, d)
    q = _by_sequence(s, s.q.float()).view(batch, s.longest, kv, group, d).permute(0, 2, 3, 1, 4)
    lse = _by_sequence(s, s.lse).view(batch, s.longest, kv, group).permute(0, 2, 3, 1)
    scores = (q.reshape(batch, kv, group * s.longest, d) @ k.transpose(2, 3)) * s.scaling
    p = torch.exp(scores.view(batch, kv, group, s.longest, rows) - lse[..., None])
    place = torch.arange(s.longest, device="cuda")
    row = torch.arange(rows, device="cuda")
    new = s.query_starts[1:] - s.query_starts[:-1]
    seen = (row <= (s.context_lens[:, None] + place)[..., None]) & (place < new[:, None])[..., None]
    got = p.masked_fill(~seen[:, None, None], 0.0).sum((2, 3))  # [batch, kv, rows]
    ends = s.context_lens + new
    b, r = torch.nonzero((row >= c["first"]) & (row < ends[:, None]), as_tuple=True)
    page_of = table[b, r // page]
    before = torch.where((r < s.context_lens[b])[:, None], s.weights[page_of, :, r % page], 0.0)
    s.out[page_of, :, r % page] = before + got[b, :, r]
    return s.out


def _plain_evict(s):
    c = s.case
    batch, kv, d, page = c["batch"], c["kv_heads"], c["head_dim"], c["page"]
    budget, first, recent = c["budget"], c["first"], c["recent"]
    table = s.page_table.clamp(min=0).long()
    held = table.shape[1] * page
    n = s.context_lens.long()[:, None, None]
    row = torch.arange(held, device="cuda")
    # Heaviest first, the lowest row first among equals: one whole number orders by both.
    weight = s.weights[table].transpose(1, 2).reshape(batch, kv, held)
    bits = (weight + 0.0).view(torch.int32).long()
    key = (bits << 32) + (0xFFFFFFFF - row)
    key = torch.where((row < first) | (row >= n - recent), (1 << 63) - 1, key)
    key = torch.where(row < n, key, -1 - row)
    rows = torch.topk(key, min(budget, held), dim=2).indices.sort(2).values
    if budget > held:
        rows = torch.nn.functional.pad(rows, (0, budget - held), value=held)
    longer = s.context_lens > budget
    rows = torch.where(rows < n, rows, -1)

    kept = first // page  # pages in front that stay as they are
    entries = -(-budget // page)
    stay = torch.nn.functional.pad(s.page_table, (0, max(0, entries - s.page_table.shape[1])), value=-1)[:, :entries]
    page_table = torch.where(longer[:, None], torch.cat((stay[:, :kept], s.into), 1), stay)
    moved = torch.nonzero(longer)[:, 0]
    if moved.numel():
        take = rows[moved, :, kept * page:]
        fill = (entries - kept) * page - take.shape[2]
        pages = table[moved[:, None, None], take // page]
        heads = torch.arange(kv, device="cuda")[None, :, None]
        into = s.into[moved].long()
        for stored, scales in ((s.k_pages, s.k_scales), (s.v_pages.transpose(2, 3), s.v_scales)):
            x = stored.view(torch.uint8)[pages, heads, take % page].view(torch.float8_e4m3fn).float()
            x = torch.nn.functional.pad(x * scales[pages, heads][..., None], (0, 0, 0, fill))
            x = x.view(moved.numel(), kv, -1, page, d)
            new = _power_scale(x.abs().amax((3, 4)))
            x = (x / new[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8).transpose(1, 2)
            old = stored.view(torch.uint8)[into]
            at = torch.arange(into.shape[1] * page, device="cuda").view(-1, 1, page, 1)
            stored.view(torch.uint8)[into] = torch.where(at < take.shape[2], x, old)
            scales[into] = new.transpose(1, 2)
        w = torch.nn.functional.pad(weight[moved].gather(2, take), (0, fill)).view(moved.numel(), kv, -1, page).transpose(1, 2)
        at = torch.arange(into.shape[1] * page, device="cuda").view(-1, 1, page)
        s.weights[into] = torch.where(at < take.shape[2], w, s.weights[into])
    return _evicted(s, page_table, s.context_lens.clamp(max=budget), rows.to(torch.int32))


def _plain_int4(s):
    c = s.case
    low, high = s.packed & 15, s.packed >> 4
    w = torch.stack((low, high), 2).view(c["outs"], c["in"]).float()
    zeros = 8.0 if s.zeros is None else s.zeros.float().repeat_interleave(c["group"], 1)[:, :c["in"]]
    w = (w - zeros) * s.scales.float().repeat_interleave(c["group"], 1)[:, :c["in"]]
    return (s.x.float() @ w.T).to(DTYPES[c["out"]])


_PLAIN = {"shared": _plain_shared, "weigh": _plain_weigh, "evict": _plain_evict, "int4": _plain_int4}
_OWN = {"shared": _own_shared, "weigh": _own_weigh, "evict": _own_evict, "int4": _own_int4}


# -- the same outputs in 64 bits -------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "weigh": _exact_weigh, "evict": _exact_evict, "int4": _exact_int4}[case["kind"]](s)


def _keys_values(s, i, rows, head, what):
    """fp64 rows [0, rows) of sequence i and one kv head."""
    pages = s.page_table[i, :-(-rows // s.case["page"])].long()
    stored, scales = (s.k_pages, s.k_scales) if what == "k" else (s.v_pages, s.v_scales)
    x = stored.view(torch.uint8)[pages, head].view(torch.float8_e4m3fn).double() * scales[pages, head].double()[:, None, None]
    if what == "v":
        x = x.transpose(1, 2)
    return x.reshape(-1, s.case["head_dim"])[:rows]


def _scores(s, i, begin, context, new, head):
    """fp64 scores [new, group, rows] of a sequence's tokens, -inf where a token does not see a row."""
    rows = context + new
    keys = _keys_values(s, i, rows, head, "k")
    q = s.q[begin:begin + new].view(new, s.case["kv_heads"], -1, s.case["head_dim"])[:, head].double()
    scores = torch.tensordot(q, keys, dims=([2], [1])) * s.scaling
    hidden = torch.arange(rows, device="cuda")[None] > torch.arange(context, rows, device="cuda")[:, None]
    return scores.masked_fill(hidden[:, None], -math.inf)


def _exact_shared(s):
    c = s.case
    kv, d = c["kv_heads"], c["head_dim"]
    out = torch.empty(s.tokens, kv, c["q_heads"] // kv, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(s.tokens, kv, c["q_heads"] // kv, dtype=torch.float64, device="cuda")
    begin = 0
    for i, (context, new) in enumerate(_lengths(c)):
        for head in range(kv):
            scores = _scores(s, i, begin, context, new, head)
            lse[begin:begin + new, head] = torch.logsumexp(scores, -1)
            values = _keys_values(s, i, context + new, head, "v")
            out[begin:begin + new, head] = torch.softmax(scores, -1) @ values
        begin += new
    return {"out": out.view(s.tokens, -1), "lse": lse.view(s.tokens, -1)}


def _exact_weigh(s):
    c = s.case
    kv, page, first = c["kv_heads"], c["page"], c["first"]
    out = s.out.double()
    begin = 0
    for i, (context, new) in enumerate(_lengths(c)):
        rows = torch.arange(min(first, context + new), context + new, device="cuda")
        pages = s.page_table[i].long()[rows // page]
        for head in range(kv):
            scores = _scores(s, i, begin, context, new, head)
            lse = s.lse[begin:begin + new].view(new, kv, -1)[:, head].double()
            got = (scores - lse[..., None]).exp().sum((0, 1))
            got[:context] += s.weights[s.page_table[i].long()[torch.arange(context, device="cuda") // page], head,
                                       torch.arange(context, device="cuda") % page].double()
            out[pages, head, rows % page] = got[first:]
        begin += new
    return out


def _power(exponent):
    """2 to a whole exponent, exactly."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """The e4m3 value nearest to x, ties to the even one: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    _, exponent = torch.frexp(x)
    step = _power((exponent - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_evict(s):
    c = s.case
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    budget, first, recent = c["budget"], c["first"], c["recent"]
    kept, entries = first // page, -(-budget // page)
    k, v = s.k_pages.double(), s.v_pages.double().transpose(2, 3).contiguous()
    scales = {"k": s.k_scales.double(), "v": s.v_scales.double()}
    weights = s.weights.double()
    table = torch.full((c["batch"], entries), -1, dtype=torch.int32, device="cuda")
    all_rows = torch.full((c["batch"], kv, budget), -1, dtype=torch.int32, device="cuda")
    for i, (n, _) in enumerate(_lengths(c)):
        width = min(entries, s.page_table.shape[1])
        table[i, :width] = s.page_table[i, :width]
        if n <= budget:
            all_rows[i, :, :n] = torch.arange(n, device="cuda", dtype=torch.int32)
            continue
        table[i, kept:] = s.into[i]
        at = s.page_table[i, :-(-n // page)].long()
        for head in range(kv):
            w = s.weights[at, head].reshape(-1)[:n]
            middle = torch.arange(first, n - recent, device="cuda")
            order = torch.sort(w[first:n - recent], descending=True, stable=True).indices
            chosen = middle[order[:budget - first - recent]]
            rows = torch.cat((torch.arange(first, device="cuda"), chosen.sort().values,
                              torch.arange(n - recent, n, device="cuda")))
            all_rows[i, head] = rows
            keys, values = _keys_values(s, i, n, head, "k"), _keys_values(s, i, n, head, "v")
            for slot in range(kept, entries):
                take = rows[slot * page:(slot + 1) * page]
                page_at = int(s.into[i, slot - kept])
                weights[page_at, head, :take.numel()] = w[take].double()
                for name, x, stored in (("k", keys[take], k), ("v", values[take], v)):
                    exponent = torch.ceil(torch.log2(x.abs().amax() / E4M3_MAX)).clamp(min=MIN_EXPONENT)
                    scale = _power(exponent)
                    scales[name][page_at, head] = scale
                    stored[page_at, head, :take.numel()] = _e4m3(x / scale)
    return {"page_table": table, "context_lens": s.context_lens.clamp(max=budget), "rows": all_rows, "k_pages": k,
            "v_pages": v.transpose(2, 3), "k_scales": scales["k"], "v_scales": scales["v"], "weights": weights}


def _exact_int4(s):
    c = s.case
    x = s.x.double()
    column = torch.arange(c["in"], device="cuda")
    group = column // c["group"]
    parts = []
    for first in range(0, c["outs"], 4096):
        rows = slice(first, first + 4096)
        packed = s.packed[rows]
        w = (packed[:, column // 2] >> (4 * (column % 2)).to(torch.uint8)) & 15
        w = w.double() - (8.0 if s.zeros is None else s.zeros[rows].double()[:, group])
        parts.append(x @ (w * s.scales[rows].double()[:, group]).T)
    return torch.cat(parts, 1)
