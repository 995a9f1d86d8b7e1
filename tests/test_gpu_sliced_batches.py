"""Batches taken in several calls by slices of query_starts, context_lens and the page table, with the
same q, outputs, log-sum-exps and weights: groups of other prefixes, a prompt apart from single tokens, a long
sequence evicted by itself."""

from __future__ import annotations

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_attention_weights import check_weights
from test_gpu_serving import DEV, Batch, _check_attention, _filled, _say
from test_gpu_shared_attention import check_lse

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc
from oracle import serving as osv

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


def part(batch, first, last):
    """Sequences [first, last) of a batch."""
    return {"page_table": batch["page_table"][first:last], "query_starts": batch["query_starts"][first:last + 1],
            "context_lens": batch["context_lens"][first:last]}


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
def test_groups_with_prefixes_of_their_own(q_dtype):
    _say("prefix groups", q_dtype)
    d, page, prefixes = 128, 32, ((0, 3, 128), (3, 5, 256), (5, 6, 0))
    lengths = [(200, 1), (150, 2), (131, 1), (300, 1), (280, 1), (70, 90)]
    b = Batch(lengths, kv=2, d=d, page=page, seed=961)
    for first, last, shared in prefixes:
        for line in b.table[first:last]:
            line[:shared // page] = b.table[first][:shared // page]
    _filled(b, 962)
    for line, (_, _, context) in zip(b.table, b.spans):
        for at in line[:-(-context // page)]:
            for stored in (b.k_bytes[at], b.v_bytes[at]):
                stored[(stored & 0x7f) == 0x7f] = 0x31
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, 8, d, generator=generator(963)).to(q_dtype)
    cache, batch = b.device()
    out, lse = torch.full((b.tokens, 8 * d), 9.0, device=DEV), torch.full((b.tokens, 8), 9.0, device=DEV)
    for first, last, shared in prefixes:
        ops.launch_shared_attention(q.to(DEV), cache, shared_rows=shared, scaling=d**-0.5, out=out, lse=lse, **part(batch, first, last))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    _check_attention(out, expected, spread, reach, q_dtype=q_dtype, rows=302, d=d)
    check_lse(lse, olc.attention_lse(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5), reach, q_dtype=q_dtype, rows=302, d=d)


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
def test_attention_weights_of_a_prompt_and_of_single_tokens(q_dtype):
    _say("prompt apart", q_dtype)
    d, page = 64, 16
    b = shared_batch([(100, 160)] + [(30 + 7 * i, 1) for i in range(20)], 0, kv=2, d=d, page=page, seed=971)
    q = torch.randn(b.tokens, 8, d, generator=generator(972)).to(q_dtype)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5).float()
    start = torch.rand(b.k_bytes.shape[0], 2, page, generator=generator(973))
    expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=page, scaling=d**-0.5, first=3)
    cache, batch = b.device()
    for cuts in ((0, 21), (0, 1, 21), (0, 1, 9, 21)):
        weights = start.to(DEV)
        for first, last in zip(cuts, cuts[1:]):
            ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), weights, scaling=d**-0.5, first=3, **part(batch, first, last))
        check_weights(weights, expected, spread, written, start, q_dtype=q_dtype, d=d, lse=lse.double(), n=640)


def test_evictions_in_one_call_and_in_two():
    d, page, budget = 64, 16, 100
    results = []
    for cuts in ((0, 4), (0, 1, 4)):
        b = Batch([(900, 0), (130, 0), (60, 0), (210, 0)], kv=2, d=d, page=page, seed=981, spare=40)
        cache, batch = b.device()
        used = {at for line in b.table for at in line if at >= 0}
        free = [at for at in range(b.k_bytes.shape[0]) if at not in used][:4 * 6]
        into = torch.tensor(free, dtype=torch.int32, device=DEV).view(4, 6)
        weights = torch.rand(b.k_bytes.shape[0], 2, page, generator=generator(982)).to(DEV)
        got = []
        for first, last in zip(cuts, cuts[1:]):
            one = part(batch, first, last)
            got.append(ops.launch_paged_evict(cache, weights, page_table=one["page_table"], context_lens=one["context_lens"],
                                              into=into[first:last], budget=budget, first=20, recent=30))
        results.append([torch.cat(x) for x in zip(*got)] + [cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scales,
                                                             cache.v_scales, weights])
    assert all(torch.equal(x, y) for x, y in zip(*results))
