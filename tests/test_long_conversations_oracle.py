"""The restatement of the operators for long conversations against closed forms (no GPU needed)."""

from __future__ import annotations

import math

import torch

from oracle import long_conversations as olc
from oracle import serving as osv


def _cache(pages, kv, page, d, seed):
    g = torch.Generator().manual_seed(seed)
    return {"k": osv.e4m3(torch.randn(pages, kv, page, d, generator=g)), "v": osv.e4m3(torch.randn(pages, kv, d, page, generator=g)),
            "k_scales": torch.ones(pages, kv).double(), "v_scales": torch.ones(pages, kv).double()}


def test_lse_and_weights_are_torchs():
    cache, q = _cache(3, 2, 16, 64, 1), torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(2))
    table, spans = [[2, 0, 1]], [(0, 3, 20)]
    lse = olc.attention_lse(q, cache, table, spans, page=16, scaling=0.125)
    keys = cache["k"][[2, 0, 1]].transpose(0, 1).reshape(2, 48, 64)
    total = torch.zeros(2, 48, dtype=torch.float64)
    for t in range(3):
        for h in range(4):
            s = keys[h // 2, :21 + t] @ q[t, h].double() * 0.125
            assert torch.allclose(lse[t, h], torch.logsumexp(s, 0))
            total[h // 2, :21 + t] += torch.softmax(s, 0)
    start = torch.rand(3, 2, 16)
    got, _, written = olc.attention_weights(q, cache, lse, start, table, spans, page=16, scaling=0.125, first=5)
    rows = got[[2, 0, 1]].transpose(0, 1).reshape(2, 48)
    old = start[[2, 0, 1]].transpose(0, 1).reshape(2, 48).double()
    assert torch.allclose(rows[:, 5:20], old[:, 5:20] + total[:, 5:20])
    assert torch.allclose(rows[:, 20:23], total[:, 20:23])
    assert torch.equal(rows[:, :5], old[:, :5]) and torch.equal(rows[:, 23:], old[:, 23:])
    assert int(written.sum()) == 2 * 18


def test_eviction_keeps_the_heaviest_and_the_lowest_of_equals():
    cache = _cache(6, 1, 16, 64, 3)
    weights = torch.zeros(6, 1, 16)
    weights[0, 0, 3], weights[1, 0, 2], weights[1, 0, 9] = 5.0, math.nan, 2.0  # rows 3, 18 and 25
    after, moved, tables, lengths, rows = olc.evict(cache, weights, [[0, 1, 2]], [40], [[4]], page=16, budget=8, first=1, recent=2)
    assert rows == [[[0, 1, 2, 3, 18, 25, 38, 39]]]  # of the rest, with weights of zero, 1 and 2
    assert tables == [[4]] and lengths == [8]
    keys = cache["k"][[0, 1, 2], 0].reshape(48, 64)[rows[0][0]]
    scale = float(after["k_scales"][4, 0])
    assert scale == osv.scale_for(float(keys.abs().max()))
    assert torch.equal(after["k"][4, 0, :8] * scale, osv.e4m3(keys / scale) * scale)
    assert torch.equal(after["k"][4, 0, 8:], cache["k"][4, 0, 8:])
    assert math.isnan(float(moved[4, 0, 4])) and moved[4, 0, 5] == 2.0


def test_a_short_sequence_keeps_everything():
    cache, weights = _cache(4, 2, 16, 64, 4), torch.rand(4, 2, 16)
    after, same, tables, lengths, rows = olc.evict(cache, weights, [[3, 1]], [17], [[0, 2]], page=16, budget=20, first=0, recent=0)
    assert tables == [[3, 1]] and lengths == [17] and rows[0][1] == list(range(17)) + [-1] * 3
    assert torch.equal(same, weights) and torch.equal(after["k"], cache["k"])


def test_4_bit_weights():
    packed = torch.tensor([[0x21, 0xF8]], dtype=torch.uint8).repeat(1, 8)
    dense = olc.int4_dense(packed, torch.tensor([[2.0]]), None, 32)
    assert dense[0, :4].tolist() == [-14.0, -12.0, 0.0, 14.0]
    assert olc.int4_dense(packed, torch.tensor([[1.0]]), torch.tensor([[3]]), 32)[0, :4].tolist() == [-2.0, -1.0, 5.0, 12.0]
