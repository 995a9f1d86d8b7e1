"""CPU oracle of the operators for long conversations — TEST INFRASTRUCTURE ONLY.

Log-sum-exp of attention over the 8-bit paged cache, the attention weight that
cached rows receive, eviction by it, and products with 4-bit weights, restated
from their definitions in 64 bits, sequence by sequence and row by row.
``tests/`` compare the HIP kernels with it. Pinned by closed forms in
tests/test_long_conversations_oracle.py. Caches and batches are those of
``oracle.serving``.
"""

from __future__ import annotations

import math

import torch

from oracle import serving as osv


def _rows(cache, name, entries, page, rows, head):
    """fp64 rows [0, rows) of one kv head of the pages `entries`, NaN where an entry names no page."""

    pages = cache[name].shape[0]
    d = cache["k"].shape[3]
    out = torch.full((rows, d), math.nan, dtype=torch.float64)
    for slot in range(-(-rows // page)):
        at = entries[slot]
        if 0 <= at < pages:
            stored = cache[name][at, head].double() * cache[name + "_scales"][at, head].double()
            stored = stored if name == "k" else stored.T
            n = min(page, rows - slot * page)
            out[slot * page:slot * page + n] = stored[:n]
    return out


def attention_lse(q, cache, table, spans, *, page, scaling):
    """fp64 log-sum-exps [tokens, q_heads]: NaN rows for nobody's tokens, -inf where a token's row has no place."""

    tokens, heads = q.shape[:2]
    kv = cache["k"].shape[1]
    lse = torch.full((tokens, heads), math.nan, dtype=torch.float64)
    held = len(table[0]) * page
    for b, (begin, end, context) in enumerate(spans):
        last = max(0, min(context + end - begin, held))
        for g in range(kv):
            keys = _rows(cache, "k", table[b], page, last, g)
            mine = slice(g * heads // kv, (g + 1) * heads // kv)
            for t in range(begin, end):
                row = context + t - begin
                lse[t, mine] = (torch.logsumexp(q[t, mine].double() @ keys[:row + 1].T * scaling, -1)
                                if 0 <= row < held else -math.inf)
    return lse


def attention_weights(q, cache, lse, weights, table, spans, *, page, scaling, first):
    """fp64 [pages, kv, page]: NaN-free copy of `weights` with what the rows from
    `first` on receive; and for each what an fp32 evaluation's rounding is relative
    to, sum p (1 + scaling |q| |k|), with a mask of the rows that were written."""

    out, spread = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    written = torch.zeros(weights.shape, dtype=torch.bool)
    kv, heads, pages = cache["k"].shape[1], q.shape[1], cache["k"].shape[0]
    held = len(table[0]) * page
    for b, (begin, end, context) in enumerate(spans):
        if end <= begin:
            continue
        last = max(0, min(context + end - begin, held))
        for g in range(kv):
            keys = _rows(cache, "k", table[b], page, last, g)
            mine = slice(g * heads // kv, (g + 1) * heads // kv)
            x = q[begin:end, mine].double()
            s = x @ keys.T * scaling
            reach = x.abs() @ keys.abs().T * scaling
            row, place = torch.arange(last), torch.arange(end - begin)
            seen = (row <= context + place[:, None])[:, None] & (context + place < held)[:, None, None]
            seen &= (context + place >= 0)[:, None, None]
            p = torch.where(seen, torch.exp(s - lse[begin:end, mine].double()[..., None]), 0.0)
            total, size = p.sum((0, 1)), torch.where(p > 0, p * (1 + reach), p).sum((0, 1))
            for r in range(min(first, last), last):
                at = table[b][r // page]
                if 0 <= at < pages:
                    before = float(weights[at, g, r % page]) if r < context else 0.0
                    out[at, g, r % page] = before + total[r]
                    spread[at, g, r % page] = size[r]
                    written[at, g, r % page] = True
    return out, spread, written


def evict(cache, weights, table, contexts, into, *, page, budget, first, recent):
    """The cache, weights, table, lengths and kept rows after an eviction."""

    cache = {name: x.clone().double() for name, x in cache.items()}
    source = {name: x.clone() for name, x in cache.items()}
    weights, old = weights.clone(), weights.clone()
    pages, kv = cache["k"].shape[:2]
    kept, entries, held = first // page, -(-budget // page), len(table[0]) * page
    tables, lengths, rows = [], [], []
    for b, context in enumerate(contexts):
        n = min(context, held)
        line = (table[b] + [-1] * entries)[:entries]
        if n <= budget:
            tables.append(line)
            lengths.append(context)
            rows.append([[r if r < n else -1 for r in range(budget)] for _ in range(kv)])
            continue
        tables.append(line[:kept] + into[b])
        lengths.append(budget)
        rows.append([])
        for g in range(kv):
            def weight(r):
                at = table[b][r // page]
                return float(old[at, g, r % page]) if 0 <= at < pages else math.nan
            def order(r):
                w = weight(r)
                return (0, 0.0, r) if math.isnan(w) else (1, -w, r)
            chosen = sorted(range(first, n - recent), key=order)[:budget - first - recent]
            stay = list(range(first)) + sorted(chosen) + list(range(n - recent, n))
            rows[-1].append(stay)
            for slot in range(kept, entries):
                to = into[b][slot - kept]
                if not 0 <= to < pages:
                    continue
                take = stay[slot * page:(slot + 1) * page]
                for name in ("k", "v"):
                    x = torch.stack([_rows(source, name, [table[b][r // page]], page, page, g)[r % page] for r in take])
                    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
                    scale = osv.scale_for(float(finite.max()))
                    cache[name + "_scales"][to, g] = scale
                    stored = cache[name][to, g] if name == "k" else cache[name][to, g].T
                    stored[:len(take)] = osv.e4m3(x / scale)
                weights[to, g, :len(take)] = torch.tensor([weight(r) for r in take])
    return cache, weights, tables, lengths, rows


def int4_dense(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, group: int) -> torch.Tensor:
    """fp64 [out, in] of 4-bit weights: byte j of a row holds columns 2 j (low bits) and 2 j + 1."""

    outs, half = packed.shape
    w = torch.empty(outs, 2 * half, dtype=torch.float64)
    w[:, 0::2] = (packed & 15).double()
    w[:, 1::2] = (packed >> 4).double()
    column = torch.arange(2 * half) // group
    zero = 8.0 if zeros is None else zeros.double()[:, column]
    return (w - zero) * scales.double()[:, column]
