"""Attention over sequences that hold the same first rows, on the GPU against its
64-bit restatement (oracle/serving.py, oracle/long_conversations.py).

Bounds: outputs as for ``launch_paged_attention`` (tests/test_gpu_serving.py). A
log-sum-exp is off by what a score is, 2^-24 (parts D + 8) scaling sum |q| |k|, by
the relative error of its sum, 2^-24 (n / 16 + 64) and the hardware exponentials'
and logarithm's 2^-22 each, and by one rounding.
"""

from __future__ import annotations

import math

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_serving import DEV, _check_attention, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc
from oracle import serving as osv

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def check_lse(got, expected, reach, *, q_dtype, rows, d):
    u = 2.0**-24
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(expected))
    flat = torch.isinf(expected)
    assert torch.equal(got[flat], expected[flat])
    ok = ~flat & ~torch.isnan(expected)
    bound = u * (PARTS[q_dtype] * d + 8) * reach + u * (rows / 16 + 64) + 2 * 2.0**-22 + u * expected.abs()
    worst = float(((got - expected).abs() / bound)[ok].max()) if ok.any() else 0.0
    assert worst <= 1, worst


def run_and_check(b, shared_rows, q, q_heads, *, page, d, out_dtype):
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    cache, batch = b.device()
    out = torch.full((b.tokens, q_heads * d), 9.0, dtype=out_dtype, device=DEV)
    got_lse = torch.full((b.tokens, q_heads), 9.0, device=DEV)
    args = {"shared_rows": shared_rows, "scaling": d**-0.5, **batch}
    ops.launch_shared_attention(q.to(DEV), cache, out=out, lse=got_lse, **args)
    torch.cuda.synchronize()
    mine = torch.zeros(b.tokens, dtype=torch.bool)
    for begin, end, _ in b.spans:
        mine[begin:end] = True
    assert (out.cpu()[~mine] == 9.0).all() and (got_lse.cpu()[~mine] == 9.0).all()
    rows = max(c + e - s for s, e, c in b.spans)
    _check_attention(out[mine.to(DEV)], expected[mine], spread[mine], reach[mine], q_dtype=q.dtype, rows=rows, d=d)
    check_lse(got_lse[mine.to(DEV)], lse[mine], reach[mine], q_dtype=q.dtype, rows=rows, d=d)
    again = ops.launch_shared_attention(q.to(DEV), cache, out_dtype=out_dtype, **args)
    again, first = (torch.nan_to_num(x.cpu()[mine], nan=77.0) for x in (again, out))
    assert torch.equal(again, first)  # a fixed order, with and without lse
    return out, got_lse


CASES = [
    # lengths, shared rows, q heads, kv heads, head_dim, page
    ([(0, 1)], 0, 4, 2, 64, 16),                                    # nothing cached, nothing shared
    ([(100, 1), (70, 1)], 64, 4, 2, 64, 16),                        # one shared tile
    ([(64, 1), (64, 1), (64, 1)], 64, 8, 2, 128, 64),               # only the new row is a sequence's own
    ([(500, 1), (590, 1), (501, 1)], 500, 8, 2, 128, 64),           # shared rows that end inside a page
    ([(700, 1), (650, 3), (649, 0), (700, 2)], 640, 6, 2, 128, 32), # a sequence without tokens
    ([(300, 1), (20, 1), (0, 2), (400, 1)], 256, 8, 2, 64, 16),     # sequences that see only some shared rows
    ([(260, 9), (300, 17), (256, 1)], 256, 4, 1, 256, 128),
    ([(200, 40), (250, 33)], 192, 4, 2, 128, 64),                   # slots full of one sequence's rows
    ([(130, 70), (140, 130)], 128, 8, 2, 64, 16),                   # prompts behind a shared prefix
    ([(1500, 1), (1310, 1), (1280, 2)], 1290, 34, 2, 64, 16),       # more heads to a group than an MFMA has columns
    ([(2000, 1)], 1984, 8, 2, 128, 32),                             # one sequence
    ([(15, 1), (90, 1)], 40, 4, 2, 128, 16),                        # less than a tile
    ([(520, 3), (512, 3)], 512, 5, 1, 256, 16),
]
DTYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
          (torch.float32, torch.float16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)]


@pytest.mark.parametrize("q_dtype,out_dtype", DTYPES)
@pytest.mark.parametrize("lengths,shared,q_heads,kv,d,page", CASES)
def test_shared_attention(lengths, shared, q_heads, kv, d, page, q_dtype, out_dtype):
    _say("shared", lengths, shared, q_heads, kv, d, page, q_dtype, out_dtype)
    b = shared_batch(lengths, shared, kv=kv, d=d, page=page, seed=112, ahead=1, behind=2)
    q = torch.randn(b.tokens, q_heads, d, generator=generator(114)).to(q_dtype)
    run_and_check(b, shared, q, q_heads, page=page, d=d, out_dtype=out_dtype)


@pytest.mark.parametrize("batch,kv,d,shared,page", [(64, 2, 64, 200, 16), (65, 2, 128, 130, 64), (63, 1, 256, 64, 16),
                                                    (150, 2, 128, 320, 32), (300, 1, 64, 64, 64)])
def test_many_sequences(batch, kv, d, shared, page):
    """As many sequences as a wave looks up at once, one less and more."""

    _say("shared many", batch, kv, d, shared, page)
    g = generator(120)
    lengths = [(shared + int(c), int(n)) for c, n in zip(torch.randint(0, 90, (batch,), generator=g),
                                                         torch.randint(0, 3, (batch,), generator=g))]
    lengths[0] = (shared + 400, 1)
    lengths[batch // 2] = (3, 2)
    b = shared_batch(lengths, shared, kv=kv, d=d, page=page, seed=121, ahead=2, behind=1, extra_entries=5)
    q = torch.randn(b.tokens, 2 * kv, d, generator=generator(123)).to(torch.bfloat16)
    run_and_check(b, shared, q, 2 * kv, page=page, d=d, out_dtype=torch.float32)


def test_without_shared_rows_it_is_paged_attention():
    for lengths, q_heads in (([(600, 1), (30, 4)], 8), ([(64, 200)], 4), ([(5, 3)] * 40, 8)):
        b = shared_batch(lengths, 0, kv=2, d=128, page=64, seed=131)
        q = torch.randn(b.tokens, q_heads, 128, generator=generator(132)).to(DEV)
        cache, batch = b.device()
        lse = torch.empty(b.tokens, q_heads, device=DEV)
        got = ops.launch_shared_attention(q, cache, shared_rows=0, scaling=0.1, lse=lse, out_dtype=torch.float32, **batch)
        plain = ops.launch_paged_attention(q, cache, scaling=0.1, out_dtype=torch.float32, **batch)
        assert torch.allclose(got, plain, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("what", ["k", "v", "q", "inf", "entry", "lowest"])
def test_values_that_are_not_finite(what):
    """NaN and infinities reach the tokens that see them, and no others."""

    _say("shared not finite", what)
    lengths, shared = [(200, 2), (130, 1), (60, 1), (128, 1)], 128
    b = shared_batch(lengths, shared, kv=2, d=64, page=16, seed=141)
    q = torch.randn(b.tokens, 4, 64, generator=generator(142))
    if what == "k":
        b.k_bytes[b.table[0][6], 1, 5, 3] = 0x7f      # a shared row (101) that sequence 2 does not see
    elif what == "v":
        b.v_bytes[b.table[0][6], 0, 7, 5] = 0xff
        b.v_bytes[b.table[0][12], 0, 9, 9] = 0x7f     # row 201: the second token of sequence 0 alone
    elif what == "q":
        q[1, 2, 5] = math.nan
    elif what == "inf":
        q[2, 1, 5] = math.inf
    elif what == "entry":
        b.table[3][8] = 4000                          # the page of its own row
    else:
        q[0, 0] = -3e38
    run_and_check(b, shared, q, 4, page=16, d=64, out_dtype=torch.float32)


def test_rows_without_a_place():
    """Tokens outside the page table give zeros and a log-sum-exp of -inf."""

    b = shared_batch([(-2, 4), (78, 4), (66, 1)], 64, kv=1, d=64, page=16, seed=151, extra_entries=0)
    assert len(b.table[0]) * 16 == 96 or len(b.table[0]) * 16 == 80
    b.spans[1] = (*b.spans[1][:2], len(b.table[0]) * 16 - 2)
    q = torch.randn(b.tokens, 2, 64, generator=generator(152))
    out, lse = run_and_check(b, 64, q, 2, page=16, d=64, out_dtype=torch.float32)
    for t in (0, 1, 6, 7):
        assert (out[t] == 0).all() and (lse[t] == -math.inf).all()


def test_work_on_another_stream_with_a_workspace_of_the_callers():
    b = shared_batch([(500, 1), (410, 3), (330, 1)], 320, kv=2, d=128, page=32, seed=165)
    q = torch.randn(b.tokens, 8, 128, generator=generator(166)).to(DEV)
    cache, batch = b.device()
    args = {"shared_rows": 320, "scaling": 0.1, **batch}
    here = ops.launch_shared_attention(q, cache, **args)
    size = ops.shared_attention_workspace_bytes(b.tokens, 3, 8, cache, batch["page_table"].shape[1], 320)
    assert size > 0
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        there = ops.launch_shared_attention(q, cache, workspace=torch.empty(size, dtype=torch.uint8, device=DEV), **args)
    side.synchronize()
    assert torch.equal(here, there)
    with pytest.raises(ValueError, match="lse"):
        ops.launch_shared_attention(q, cache, lse=torch.empty(b.tokens, 9, device=DEV), **args)
    with pytest.raises(ValueError, match="shared_rows"):
        ops.launch_shared_attention(q, cache, **{**args, "shared_rows": 10**6})


def test_captured_calls_replay_with_other_lengths():
    """Two graphs with workspaces of their own, and other lengths under one capture."""

    page, d, shared = 32, 128, 320
    b = shared_batch([(500, 1), (410, 1), (330, 1)], shared, kv=2, d=d, page=page, seed=161)
    q = torch.randn(b.tokens, 8, d, generator=generator(162)).to(DEV)
    cache, batch = b.device()
    args = {"shared_rows": shared, "scaling": d**-0.5, "out_dtype": torch.float32, **batch}
    ops.launch_shared_attention(q, cache, **args)
    graphs = []
    for _ in range(2):
        graph, lse = torch.cuda.CUDAGraph(), torch.empty(b.tokens, 8, device=DEV)
        with torch.cuda.graph(graph):
            out = ops.launch_shared_attention(q, cache, lse=lse, **args)
        graphs.append((graph, out, lse))
    for contexts in ([500, 410, 330], [321, 340, 400], [500, 320, 10]):
        batch["context_lens"].copy_(torch.tensor(contexts, dtype=torch.int32))
        lse = torch.empty(b.tokens, 8, device=DEV)
        eager = ops.launch_shared_attention(q, cache, lse=lse, **args)
        for graph, out, got in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for x, y in ((out, eager), (got, lse)):  # sequences over rows that hold no numbers give NaN
                assert torch.equal(torch.nan_to_num(x, nan=77.0), torch.nan_to_num(y, nan=77.0))
