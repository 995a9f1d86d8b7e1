"""Appends at positions that are no cache rows, and a run of the operators for long
conversations as a server makes it, on the GPU against their restatements."""

from __future__ import annotations

import pytest
import torch
from test_gpu_attention_weights import check_weights
from test_gpu_serving import DEV, EPS, Batch, _check_attention, _g, _rope_tables, _same_bytes, _say
from test_gpu_shared_attention import check_lse

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc
from oracle import serving as osv

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


@pytest.mark.parametrize("lengths,starts,q_heads,kv,d,page,dtype", [
    ([(20, 1)], [100], 4, 2, 64, 16, torch.float32),
    ([(15, 1), (16, 1), (0, 1), (47, 2)], [40, 16, 0, 3], 8, 2, 128, 16, torch.bfloat16),
    ([(5, 40), (30, 20)], [90, 20], 4, 4, 256, 32, torch.float16),
    ([(10, 30), (20, 30)], [-12, 100], 2, 1, 64, 16, torch.float32),     # tokens before and behind the tables
    ([(10, 3), (4, 2), (-2, 5)], [200, -50, 7], 2, 1, 128, 64, torch.float32),
])
def test_append_at_positions(lengths, starts, q_heads, kv, d, page, dtype):
    _say("append at", lengths, starts, q_heads, kv, d, page, dtype)
    b = Batch(lengths, kv=kv, d=d, page=page, seed=407, ahead=1, behind=2)
    q, k, v = (torch.randn(b.tokens, h, d, generator=_g(s)).to(dtype) for h, s in ((q_heads, 1), (kv, 2), (kv, 3)))
    qn, kn = (1 + 0.1 * torch.randn(d, generator=_g(4)) for _ in range(2))
    cos, sin = _rope_tables(130, d)
    rotated, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=page, q_norm=qn, k_norm=kn, eps=EPS,
                                   cos=cos, sin=sin, rope_starts=starts)
    cache, batch = b.device()
    out = torch.full((b.tokens, q_heads, d), 77.0, device=DEV)
    ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=q_heads, q_norm=qn.to(DEV), k_norm=kn.to(DEV),
                            eps=EPS, cos=cos.to(DEV), sin=sin.to(DEV), q_out=out,
                            rope_starts=torch.tensor(starts, dtype=torch.int32, device=DEV), **batch)
    assert torch.equal(cache.k_scales.cpu().double(), expected["k_scales"])
    assert torch.equal(cache.v_scales.cpu().double(), expected["v_scales"])
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    written = ~torch.isnan(rotated[:, 0, 0])
    assert (out.cpu()[~written] == 77.0).all()
    x = rotated[written]
    pair = torch.sqrt(x[..., :d // 2].pow(2) + x[..., d // 2:].pow(2)).repeat(1, 1, 2)
    assert ((out.cpu()[written].double() - x).abs() <= 8 * 2.0**-24 * 1.5 * pair).all()


def test_positions_that_are_cache_rows_change_nothing():
    b = Batch([(20, 30), (3, 1)], kv=2, d=128, page=16, seed=411)
    q, k, v = (torch.randn(b.tokens, h, 128, generator=_g(s)).to(DEV) for h, s in ((4, 1), (2, 2), (2, 3)))
    cos, sin = (x.to(DEV) for x in _rope_tables(60, 128))
    got = []
    for starts in (None, torch.tensor([20, 3], dtype=torch.int32, device=DEV)):
        cache, batch = b.device()
        out = ops.launch_paged_append(q, k, v, cache, q_heads=4, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin,
                                      rope_starts=starts, **batch)
        got.append([out, cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scales, cache.v_scales])
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_conversation_within_a_budget(dtype):
    """A shared prompt, tokens whose attention is added up, an eviction of all but
    the shared rows, the newest and the heaviest, and tokens at the positions that go on from there."""

    heads, kv, d, page, shared, budget, recent = 8, 2, 128, 16, 64, 112, 20
    g = _g(420)
    pages = 80
    order = torch.randperm(pages, generator=g).tolist()
    # Sequence b: the shared pages, then 8 of its own; 3 fresh ones for the eviction.
    table = [order[:4] + order[4 + 8 * b:12 + 8 * b] for b in range(3)]
    into = [order[40 + 3 * b:43 + 3 * b] for b in range(3)]
    cache = ops.paged_cache(pages, kv, page, d, DEV)
    weights = torch.zeros(pages, kv, page, device=DEV)
    host = {"k": torch.zeros(pages, kv, page, d), "v": torch.zeros(pages, kv, d, page), "k_scales": torch.zeros(pages, kv),
            "v_scales": torch.zeros(pages, kv)}
    cos, sin = _rope_tables(300, d)
    lengths, positions = [0, 0, 0], [0, 0, 0]

    def device(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def step(new, first):
        """`new[b]` tokens of each sequence; rows before `first` are not weighed."""

        nonlocal host
        spans, at = [], 0
        for n, c in zip(new, lengths):
            spans.append((at, at + n, c))
            at += n
        q, k, v = (torch.randn(at, h, d, generator=g).to(dtype) for h in (heads, kv, kv))
        batch = {"page_table": device(table), "query_starts": device([0] + [e for _, e, _ in spans]), "context_lens": device(lengths)}
        rotated = ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=heads, q_norm=None, k_norm=None,
                                          eps=EPS, cos=cos.to(DEV), sin=sin.to(DEV), rope_starts=device(positions),
                                          q_dtype=dtype, **batch)
        lse = torch.empty(at, heads, device=DEV)
        out = ops.launch_shared_attention(rotated, cache, shared_rows=shared if min(lengths) >= shared else 0,
                                          scaling=d**-0.5, lse=lse, out_dtype=torch.float32, **batch)
        before = weights.clone()
        ops.launch_attention_weights(rotated, cache, lse, weights, scaling=d**-0.5, first=first, **batch)
        _, host = osv.append(q, k, v, host, table, spans, page=page, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin,
                             rope_starts=positions)
        _same_bytes(cache.k, host["k"])
        _same_bytes(cache.v, host["v"])
        r = rotated.cpu()
        expected, spread, reach = osv.attention(r, host, table, spans, page=page, scaling=d**-0.5)
        rows = max(c + e - s for s, e, c in spans)
        _check_attention(out, expected, spread, reach, q_dtype=dtype, rows=rows, d=d)
        check_lse(lse, olc.attention_lse(r, host, table, spans, page=page, scaling=d**-0.5), reach, q_dtype=dtype, rows=rows, d=d)
        w, size, written = olc.attention_weights(r, host, lse.cpu(), before.cpu(), table, spans, page=page, scaling=d**-0.5, first=first)
        check_weights(weights, w, size, written, before.cpu(), q_dtype=dtype, d=d, lse=lse.cpu().double(), n=max(new) * heads // kv)
        for b, n in enumerate(new):
            lengths[b] += n
            positions[b] += n

    step([shared, 0, 0], shared)              # the shared prompt, appended once
    lengths[:], positions[:] = [shared] * 3, [shared] * 3
    step([40, 50, 9], shared)                 # each conversation's own question
    for _ in range(4):
        step([1, 1, 1], shared)
    step([5, 1, 0], shared)
    got = ops.launch_paged_evict(cache, weights, page_table=device(table), context_lens=device(lengths), into=device(into),
                                 budget=budget, first=shared, recent=recent)
    # The first sequences are cut, the last is short enough.
    assert lengths == [113, 119, 77]
    before = ops.PagedCache(*(x.clone() for x in cache))
    host, new_weights, tables, new_lengths, rows = olc.evict(host, weights.cpu(), table, lengths, into, page=page, budget=budget,
                                                             first=shared, recent=recent)
    _same_bytes(before.k, host["k"])
    _same_bytes(before.v, host["v"])
    assert got.page_table.tolist() == tables and got.context_lens.tolist() == new_lengths and got.rows.tolist() == rows
    assert torch.equal(cache.k_scales.cpu().double(), host["k_scales"].double())
    width = len(table[0])
    for b in range(3):
        free = [at for at in table[b] if at not in tables[b]]
        table[b] = (tables[b] + free)[:width]
    lengths[:] = new_lengths
    assert positions == [113, 119, 77]
    step([1, 1, 1], shared)
    step([6, 2, 1], shared)


def test_offsets_beyond_32_bits():
    """The last pages of a cache of 4.6 GB each for K and V give what the same pages
    give in a small one."""

    kv, d, page, pages, few = 8, 128, 64, 70000, 24
    g = torch.Generator(device=DEV).manual_seed(431)
    big, small = ops.paged_cache(pages, kv, page, d, DEV), ops.paged_cache(few, kv, page, d, DEV)
    for x, y in ((small.k, big.k), (small.v, big.v)):
        x.view(torch.uint8).copy_(torch.randint(0, 0x7f, x.shape, generator=g, device=DEV, dtype=torch.uint8))
        y.view(torch.uint8)[-few:] = x.view(torch.uint8)
    for x, y in ((small.k_scales, big.k_scales), (small.v_scales, big.v_scales)):
        x.fill_(2.0**-9)
        y.fill_(2.0**-9)
    weights = torch.rand(few, kv, page, generator=g, device=DEV)
    big_weights = torch.zeros(pages, kv, page, device=DEV)
    big_weights[-few:] = weights
    table = torch.arange(16, dtype=torch.int32, device=DEV).view(2, 8)
    table[1, :2] = table[0, :2]
    into = torch.arange(16, 24, dtype=torch.int32, device=DEV).view(2, 4)
    batch = {"query_starts": torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV),
             "context_lens": torch.tensor([500, 400], dtype=torch.int32, device=DEV)}
    q = torch.randn(3, 32, d, generator=g, device=DEV)
    results = []
    for cache, w, ahead in ((small, weights, 0), (big, big_weights, pages - few)):
        lse = torch.empty(3, 32, device=DEV)
        out = ops.launch_shared_attention(q, cache, page_table=table + ahead, shared_rows=128, scaling=0.05, lse=lse, **batch)
        ops.launch_attention_weights(q, cache, lse, w, page_table=table + ahead, scaling=0.05, first=128, **batch)
        got = ops.launch_paged_evict(cache, w, page_table=table + ahead, context_lens=batch["context_lens"], into=into + ahead,
                                     budget=300, first=70, recent=30)
        results.append([out, lse, got.page_table - ahead, got.rows, w[-few:], cache.k.view(torch.uint8)[-few:],
                        cache.v.view(torch.uint8)[-few:], cache.k_scales[-few:], cache.v_scales[-few:]])
    assert all(torch.equal(x, y) for x, y in zip(*results))
