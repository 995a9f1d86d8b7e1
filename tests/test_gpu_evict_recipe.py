"""Eviction in the order of steps that the integration guide gives: the rows of the call that
has just run count, and tokens to come get pages behind the new table."""

from __future__ import annotations

import pytest
import torch
from test_gpu_serving import DEV, EPS, _check_attention, _g, _rope_tables, _same_bytes

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc
from oracle import serving as osv

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


def test_tokens_after_an_eviction_to_whole_pages():
    heads, kv, d, page, prefix, budget, recent = 4, 2, 64, 16, 32, 96, 20
    g = _g(931)
    pages = torch.randperm(60, generator=g).tolist()
    table = [pages[:2] + pages[2 + 8 * b:10 + 8 * b] for b in range(2)]
    free, spare = [pages[20 + 4 * b:24 + 4 * b] for b in range(2)], [pages[30 + b:31 + b] for b in range(2)]
    cache, weights = ops.paged_cache(60, kv, page, d, DEV), torch.zeros(60, kv, page, device=DEV)
    host = {"k": torch.zeros(60, kv, page, d), "v": torch.zeros(60, kv, d, page), "k_scales": torch.zeros(60, kv),
            "v_scales": torch.zeros(60, kv)}
    cos, sin = _rope_tables(300, d)

    def device(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def append(new, lengths, positions, table):
        nonlocal host
        spans = [(sum(new[:b]), sum(new[:b + 1]), lengths[b]) for b in range(2)]
        q, k, v = (torch.randn(sum(new), h, d, generator=g) for h in (heads, kv, kv))
        batch = {"page_table": device(table), "query_starts": device([0, new[0], sum(new)]), "context_lens": device(lengths)}
        out = torch.full((sum(new), heads, d), 77.0, device=DEV)
        ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=heads, q_norm=None, k_norm=None, eps=EPS,
                                cos=cos.to(DEV), sin=sin.to(DEV), q_out=out, rope_starts=device(positions), **batch)
        _, host = osv.append(q, k, v, host, table, spans, page=page, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin,
                             rope_starts=positions)
        _same_bytes(cache.k, host["k"])
        return out, batch, spans

    append([prefix, 0], [0, 0], [0, 0], table)
    append([70, 20], [prefix, prefix], [prefix, prefix], table)
    cached = [prefix + 70, prefix + 20]
    q, batch, _ = append([3, 1], cached, cached, table)
    lse = torch.empty(4, heads, device=DEV)
    ops.launch_shared_attention(q, cache, shared_rows=prefix, scaling=d**-0.5, lse=lse, **batch)
    ops.launch_attention_weights(q, cache, lse, weights, scaling=d**-0.5, first=prefix, **batch)
    held = batch["context_lens"] + batch["query_starts"].diff()
    positions = held.tolist()
    old = weights.cpu()
    cut = ops.launch_paged_evict(cache, weights, page_table=batch["page_table"], context_lens=held, into=device(free), budget=budget,
                                 first=prefix, recent=recent)
    host, _, tables, lengths, rows = olc.evict(host, old, table, positions, free, page=page, budget=budget, first=prefix, recent=recent)
    assert cut.rows.tolist() == rows and cut.page_table.tolist() == tables
    assert cut.rows[0, :, -1].tolist() == [104, 104]  # the call's last token is among those that stayed
    # All entries are in use: a token of the first sequence has no place in this table.
    assert lengths == [budget, 53] and budget == cut.page_table.shape[1] * page
    before = cache.k.view(torch.uint8).clone()
    nowhere, _, _ = append([1, 0], lengths, positions, tables)
    assert (nowhere == 77.0).all() and torch.equal(cache.k.view(torch.uint8), before)
    wider = torch.cat((cut.page_table, device(spare)), 1).tolist()
    q, batch, spans = append([1, 1], cut.context_lens.tolist(), positions, wider)
    out = ops.launch_paged_attention(q, cache, scaling=d**-0.5, out_dtype=torch.float32, **batch)
    r = q.cpu()
    _check_attention(out, *osv.attention(r, host, wider, spans, page=page, scaling=d**-0.5), q_dtype=torch.float32, rows=budget + 1, d=d)
