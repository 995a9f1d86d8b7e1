"""Eviction from the 8-bit paged cache on the GPU against its restatement
(oracle/long_conversations.py): rows, tables, lengths, stored values, scales and
weights all equal it. A moved value is byte * scale exactly in fp64 there; the
kernel's product is exact in fp32 for scales that are powers of two and rounded to odd
from fp64 for others, so that one e4m3 rounding is all there is."""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_serving import DEV, Batch, _filled, _g, _same_bytes, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


def evict_batch(contexts, *, kv, d, page, budget, first, seed, extra_entries=1):
    """A batch, weights with ties and the free pages that its rows may go to."""

    slots = -(-budget // page) - first // page
    b = Batch([(c, 0) for c in contexts], kv=kv, d=d, page=page, seed=seed, spare=len(contexts) * slots + 2,
              extra_entries=extra_entries)
    used = {at for line in b.table for at in line}
    free = [at for at in range(b.k_bytes.shape[0]) if at not in used]
    into = [free[i * slots:(i + 1) * slots] for i in range(len(contexts))]
    g = _g(seed + 1)
    weights = torch.exp(2 * torch.randn(b.k_bytes.shape[0], kv, page, generator=g))
    weights[torch.rand(weights.shape, generator=g) < 0.2] = 0.0
    weights[torch.rand(weights.shape, generator=g) < 0.2] = 1.5
    return b, weights, into


def run_and_check(b, weights, into, *, page, budget, first, recent):
    contexts = [c for _, _, c in b.spans]
    expected, new_weights, tables, lengths, rows = olc.evict(b.host(), weights, b.table, contexts, into, page=page,
                                                             budget=budget, first=first, recent=recent)
    cache, batch = b.device()
    slots = -(-budget // page) - first // page
    device_into = torch.tensor(into, dtype=torch.int32, device=DEV).reshape(len(contexts), slots)
    device_weights = weights.to(DEV)
    got = ops.launch_paged_evict(cache, device_weights, page_table=batch["page_table"], context_lens=batch["context_lens"],
                                 into=device_into, budget=budget, first=first, recent=recent)
    assert got.page_table.tolist() == tables
    assert got.context_lens.tolist() == lengths
    assert got.rows.tolist() == rows
    assert batch["context_lens"].tolist() == contexts
    for name in ("k_scales", "v_scales"):
        x, y = getattr(cache, name).cpu().double(), expected[name]
        assert torch.equal(torch.nan_to_num(x, nan=-1.0), torch.nan_to_num(y, nan=-1.0))
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    assert torch.equal(torch.nan_to_num(device_weights.cpu(), nan=-1.0), torch.nan_to_num(new_weights, nan=-1.0))
    return cache, got


CASES = [
    # contexts, budget, first, recent, kv heads, head_dim, page
    ([1], 1, 0, 0, 1, 64, 16),                                # nothing to do
    ([2], 1, 0, 0, 1, 64, 16),
    ([17, 16, 15, 0], 16, 0, 0, 2, 64, 16),                   # one too many, just enough, fewer, none
    ([100, 40, 33], 33, 4, 7, 2, 128, 16),
    ([200, 100], 64, 33, 20, 2, 64, 16),                      # whole pages in front stay
    ([200, 100], 64, 32, 32, 2, 64, 32),                      # all of it first and recent rows
    ([90], 32, 32, 0, 1, 64, 16),                             # the first rows alone: no page is written
    ([90], 40, 0, 40, 1, 128, 16),                            # the newest alone
    ([700, 650, 20], 300, 10, 50, 3, 256, 64),
    ([1300], 1299, 0, 1, 2, 128, 128),
    ([3000, 100], 140, 5, 9, 1, 64, 128),
    ([5000], 2500, 100, 100, 1, 64, 32),
    ([60, 61, 62], 1000, 0, 0, 1, 64, 16),                    # a budget beyond the page table
]


@pytest.mark.parametrize("contexts,budget,first,recent,kv,d,page", CASES)
def test_paged_evict(contexts, budget, first, recent, kv, d, page):
    _say("evict", contexts, budget, first, recent, kv, d, page)
    b, weights, into = evict_batch(contexts, kv=kv, d=d, page=page, budget=budget, first=first, seed=312)
    run_and_check(b, weights, into, page=page, budget=budget, first=first, recent=recent)


@pytest.mark.parametrize("what", ["equal", "nan", "inf", "negative", "zeros", "denormal"])
def test_weights_of_any_kind(what):
    _say("evict weights", what)
    b, weights, into = evict_batch([300, 150], kv=2, d=64, page=16, budget=100, first=3, seed=321)
    g = _g(322)
    some = torch.rand(weights.shape, generator=g) < 0.1
    if what == "equal":
        weights.fill_(0.25)
    elif what == "nan":
        weights[some] = math.nan
        weights[torch.rand(weights.shape, generator=g) < 0.05] = -math.nan
    elif what == "inf":
        weights[some] = math.inf
        weights[torch.rand(weights.shape, generator=g) < 0.5] = -math.inf
    elif what == "negative":
        weights = torch.randn(weights.shape, generator=g)
    elif what == "zeros":
        weights = torch.where(some, -0.0, 0.0)
    else:
        weights = 1e-42 * torch.rand(weights.shape, generator=g)
    run_and_check(b, weights, into, page=16, budget=100, first=3, recent=11)


@pytest.mark.parametrize("what", ["scales", "zero", "tiny", "large", "nan", "entry", "into"])
def test_caches_of_any_kind(what):
    _say("evict cache", what)
    b, weights, into = evict_batch([260, 90], kv=2, d=128, page=16, budget=77, first=17, seed=331)
    if what == "scales":
        b.scales = 0.01 * torch.rand(b.scales.shape, generator=_g(332))
    elif what == "zero":
        b.scales[:, b.table[0][1:9]] = 0.0
    elif what == "tiny":
        b.scales = torch.pow(2.0, torch.randint(-126, -115, b.scales.shape, generator=_g(333)).float())
    elif what == "large":
        b.scales = torch.pow(2.0, torch.randint(110, 119, b.scales.shape, generator=_g(334)).float())
    elif what == "nan":
        b.k_bytes[b.table[0][4]] = 0x7f
        b.v_bytes[b.table[0][5], 1, 7, 3] = 0xff
    elif what == "entry":
        b.table[0][3], b.table[0][11] = -7, 5000
    else:
        into[0][1] = -3
        into[1][2] = 9000
    run_and_check(b, weights, into, page=16, budget=77, first=17, recent=8)


def test_lengths_that_have_no_place():
    """A negative length is no rows; one beyond the table is the table's rows."""

    b, weights, into = evict_batch([40, 40], kv=1, d=64, page=16, budget=20, first=0, seed=341, extra_entries=0)
    b.spans = [(0, 0, -5), (0, 0, 4000)]
    _, got = run_and_check(b, weights, into, page=16, budget=20, first=0, recent=3)
    assert got.context_lens.tolist() == [-5, 20]


def test_sources_that_sequences_share_stay():
    """Two sequences over the same pages: each has its own rows afterwards."""

    b, weights, into = evict_batch([200, 180], kv=2, d=64, page=16, budget=90, first=40, seed=351)
    b.table[1] = b.table[0][:]
    run_and_check(b, weights, into, page=16, budget=90, first=40, recent=10)


def test_outputs_and_workspace_of_the_callers():
    b, weights, into = evict_batch([9000, 40], kv=2, d=64, page=64, budget=100, first=3, seed=356, extra_entries=400)
    cache, batch = b.device()
    into = torch.tensor(into, dtype=torch.int32, device=DEV)
    w = weights.to(DEV)
    args = {"page_table": batch["page_table"], "context_lens": batch["context_lens"], "into": into, "budget": 100, "first": 3}
    expected = ops.launch_paged_evict(cache, w, **args)
    size = ops.paged_evict_workspace_bytes(2, cache, batch["page_table"].shape[1], 100)
    assert size > 0
    out = ops.Evicted(*(torch.full_like(x, -9) for x in expected))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.launch_paged_evict(cache, w, out=out, workspace=torch.empty(size, dtype=torch.uint8, device=DEV), **args)
    side.synchronize()
    assert all(x is y for x, y in zip(got, out)) and all(torch.equal(x, y) for x, y in zip(got, expected))
    with pytest.raises(ValueError, match="outputs"):
        ops.launch_paged_evict(cache, w, out=out._replace(rows=out.rows[:1]), **args)


def test_many_sequences():
    g = _g(360)
    contexts = torch.randint(0, 90, (150,), generator=g).tolist()
    contexts[7] = 700
    b, weights, into = evict_batch(contexts, kv=2, d=64, page=16, budget=40, first=2, seed=361)
    run_and_check(b, weights, into, page=16, budget=40, first=2, recent=5)


def test_captured_calls_replay_with_other_lengths_and_weights():
    b, weights, into = evict_batch([400, 300], kv=2, d=64, page=32, budget=128, first=4, seed=371)
    cache, batch = b.device()
    into = torch.tensor(into, dtype=torch.int32, device=DEV)
    w = weights.to(DEV)
    args = {"page_table": batch["page_table"], "context_lens": batch["context_lens"], "into": into, "budget": 128, "first": 4,
            "recent": 16}
    ops.launch_paged_evict(cache, w, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.launch_paged_evict(cache, w, **args)
    for seed, contexts in ((1, [400, 300]), (2, [129, 128]), (3, [300, 10])):
        batch["context_lens"].copy_(torch.tensor(contexts, dtype=torch.int32))
        w.copy_(torch.rand(w.shape, generator=_g(seed)))
        kept = w.clone()
        eager = ops.launch_paged_evict(cache, w, **args)
        pages = [x.clone().view(torch.uint8) for x in cache[:2]] + [x.clone() for x in cache[2:]] + [w.clone()]
        w.copy_(kept)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager))
        after = [x.view(torch.uint8) for x in cache[:2]] + [*cache[2:], w]
        assert all(torch.equal(x, y) for x, y in zip(pages, after))


@pytest.mark.parametrize("contexts,kv,page,budget,first,recent,kind", [
    ([20000, 9000, 8193], 2, 64, 5000, 10, 300, "spread"),
    ([70001], 3, 128, 20000, 4, 64, "spread"),                # parts of a sequence's rows
    ([33000, 8300, 8192, 24577], 2, 64, 8192, 0, 8192, "spread"),
    ([40001, 16390], 2, 32, 9000, 5, 0, "few"),
    ([70001], 3, 128, 20000, 4, 64, "equal"),
    ([40000, 100], 1, 16, 39999, 0, 0, "few"),
    ([33000], 128, 64, 1000, 0, 20, "spread"),                 # more rows than registers hold keys
    ([30000], 130, 64, 900, 7, 0, "few"),
    ([8192], 2, 32, 4000, 0, 0, "spread"),
])
def test_long_sequences(contexts, kv, page, budget, first, recent, kind):
    """Rows against torch's stable sort; the values that moved are the values they were."""

    _say("evict long", contexts, kv, page, budget, first, recent, kind)
    d = 64
    g = torch.Generator(device=DEV).manual_seed(381)
    used = [-(-c // page) for c in contexts]
    slots = -(-budget // page) - first // page
    pages = sum(used) + len(contexts) * slots
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(contexts), max(used)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    into = order[at:].view(len(contexts), slots).contiguous()
    cache = ops.paged_cache(pages, kv, page, d, DEV)
    for x, scale in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x.view(torch.uint8).copy_(torch.randint(0x20, 0x70, x.shape, generator=g, device=DEV, dtype=torch.uint8))
        scale.fill_(2.0**-5)
    weights = torch.rand(pages, kv, page, generator=g, device=DEV)
    if kind == "equal":
        weights.fill_(1.0)
    elif kind == "few":
        weights = torch.randint(0, 3, weights.shape, generator=g, device=DEV).float()
    before, old = ops.PagedCache(*(x.clone() for x in cache)), weights.clone()
    lens = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    got = ops.launch_paged_evict(cache, weights, page_table=table, context_lens=lens, into=into, budget=budget, first=first,
                                 recent=recent)

    def rows_of(c, w, line, n):
        """A sequence's rows as values and weights: [kv, n, d] twice, [kv, n]."""
        at = line[:-(-n // page)].long()
        k = c.k.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * c.k_scales[at][..., None, None]
        v = c.v.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * c.v_scales[at][..., None, None]
        return (k.transpose(0, 1).reshape(kv, -1, d)[:, :n], v.permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :n],
                w[at].transpose(0, 1).reshape(kv, -1)[:, :n])

    for b, n in enumerate(contexts):
        cut = min(n, budget)
        k, v, w = rows_of(before, old, table[b], n)
        keep = torch.arange(n, device=DEV).expand(kv, n)
        if n > budget:
            mid = torch.sort(w[:, first:n - recent], dim=1, descending=True, stable=True).indices[:, :budget - first - recent] + first
            keep = torch.cat((keep[:, :first], mid.sort(1).values, keep[:, n - recent:]), 1)
        assert torch.equal(got.rows[b, :, :cut].long(), keep)
        assert (got.rows[b, :, cut:] == -1).all()
        new = rows_of(cache, weights, got.page_table[b], cut)
        index = keep[..., None].expand(kv, cut, d)
        assert torch.equal(new[0], k.gather(1, index)) and torch.equal(new[1], v.gather(1, index))
        assert torch.equal(new[2], w.gather(1, keep))
    assert got.context_lens.tolist() == [min(n, budget) for n in contexts]
