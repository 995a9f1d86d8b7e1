"""The attention that cached rows receive, on the GPU against its 64-bit
restatement (oracle/long_conversations.py).

Bounds: a weight's exponent is off by 2^-24 (parts D + 8) scaling sum |q| |k| (the
score), 2^-24 of lse twice (its factor log2 e, the subtraction) and 2^-24 of the score again;
the hardware exponential adds 2^-22; n sums add 2^-24 each of the total at most,
old weight and output 2^-24 of theirs.
"""

from __future__ import annotations

import math

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_serving import DEV, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def check_weights(got, expected, spread, written, start, *, q_dtype, d, lse, n):
    u = 2.0**-24
    got = got.cpu()
    assert torch.equal(got[~written], start[~written])
    top = float(lse[torch.isfinite(lse)].abs().max()) if torch.isfinite(lse).any() else 0.0
    got, expected, spread = got.double()[written], expected[written], spread[written]
    assert torch.equal(torch.isnan(got), torch.isnan(expected))
    ok = ~torch.isnan(expected)
    bound = (u * (PARTS[q_dtype] * d + 9) + 2.0**-22 + 4 * u * top + u * (n + 64)) * spread + 2 * u * expected.abs() + 1e-36
    worst = float(((got - expected).abs() / bound)[ok].max()) if ok.any() else 0.0
    assert worst <= 1, worst


CASES = [
    # lengths, first, shared rows, q heads, kv heads, head_dim, page
    ([(0, 1)], 0, 0, 4, 2, 64, 16),
    ([(63, 1), (64, 1), (65, 1)], 0, 0, 8, 2, 128, 64),
    ([(600, 1)], 4, 0, 8, 2, 128, 64),
    ([(130, 5), (0, 3), (77, 0), (1, 1)], 3, 0, 6, 2, 128, 32),      # a sequence without tokens, one shorter than `first`
    ([(33, 40)], 17, 0, 5, 1, 64, 32),
    ([(0, 130), (61, 70)], 0, 0, 8, 4, 128, 128),
    ([(300, 17), (20, 2)], 5, 0, 4, 4, 256, 64),
    ([(5, 66)], 0, 0, 2, 2, 256, 16),
    ([(129, 2), (200, 1)], 100, 0, 34, 2, 64, 16),                   # more heads to a group than an MFMA has columns
    ([(300, 1), (280, 1), (299, 2)], 256, 256, 8, 2, 64, 16),        # rows of shared pages stay as they are
    ([(20, 1)], 21, 0, 4, 2, 64, 16),                                # no row from `first` on
    ([(20, 1)], 4000, 0, 4, 2, 64, 16),
    ([(10, 300)], 0, 0, 8, 2, 128, 16),
]


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,first,shared,q_heads,kv,d,page", CASES)
def test_attention_weights(lengths, first, shared, q_heads, kv, d, page, q_dtype):
    _say("weights", lengths, first, q_heads, kv, d, page, q_dtype)
    b = shared_batch(lengths, shared, kv=kv, d=d, page=page, seed=212, ahead=1, behind=2)
    q = torch.randn(b.tokens, q_heads, d, generator=generator(213)).to(q_dtype)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5).float()
    start = torch.rand(b.k_bytes.shape[0], kv, page, generator=generator(214))
    expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=page,
                                                      scaling=d**-0.5, first=first)
    cache, batch = b.device()
    weights = start.to(DEV)
    args = {"scaling": d**-0.5, "first": first, **batch}
    apart = torch.full_like(weights, 5.0)
    ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), weights, out=apart, **args)
    assert torch.equal(weights.cpu(), start)
    got = ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), weights, **args)
    assert got is weights
    n = max(e - s for s, e, _ in b.spans) * (q_heads // kv)
    check_weights(weights, expected, spread, written, start, q_dtype=q_dtype, d=d, lse=lse.double(), n=n)
    assert torch.equal(apart.cpu()[written], weights.cpu()[written]) and (apart.cpu()[~written] == 5.0).all()


def test_many_sequences_and_wide_tables():
    g = generator(220)
    lengths = [(int(c), int(n)) for c, n in zip(torch.randint(0, 90, (150,), generator=g), torch.randint(0, 3, (150,), generator=g))]
    lengths[70] = (2000, 1)
    b = shared_batch(lengths, 0, kv=2, d=64, page=16, seed=221, extra_entries=300)
    q = torch.randn(b.tokens, 8, 64, generator=generator(222)).to(torch.bfloat16)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=16, scaling=0.125).float()
    start = torch.rand(b.k_bytes.shape[0], 2, 16, generator=generator(223))
    expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=16, scaling=0.125, first=2)
    cache, batch = b.device()
    got = ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), start.to(DEV), scaling=0.125, first=2, **batch)
    check_weights(got, expected, spread, written, start, q_dtype=torch.bfloat16, d=64, lse=lse.double(), n=8)


def test_with_the_attentions_own_lse_a_token_gives_one_for_each_head():
    """A row's weights over the cache sum to its q heads' count, whatever the types."""

    for q_dtype in (torch.float32, torch.bfloat16, torch.float16):
        b = shared_batch([(700, 1), (90, 3)], 0, kv=2, d=128, page=32, seed=231)
        q = torch.randn(b.tokens, 8, 128, generator=generator(232)).to(q_dtype).to(DEV)
        cache, batch = b.device()
        lse = torch.empty(b.tokens, 8, device=DEV)
        ops.launch_shared_attention(q, cache, shared_rows=0, scaling=0.1, lse=lse, **batch)
        got = ops.launch_attention_weights(q, cache, lse, torch.zeros(b.k_bytes.shape[0], 2, 32, device=DEV), scaling=0.1, **batch)
        for i, tokens in enumerate((1, 3)):
            pages = [at for at in b.table[i] if at >= 0]
            assert torch.allclose(got[pages].sum((0, 2)).cpu(), torch.full((2,), 4.0 * tokens), rtol=2e-6)


@pytest.mark.parametrize("what", ["k", "q", "entry", "place", "large"])
def test_values_and_rows_out_of_the_ordinary(what):
    _say("weights out of the ordinary", what)
    lengths = [(200, 2), (60, 1)]
    if what == "place":
        lengths = [(-2, 4), (92, 6)]
    b = shared_batch(lengths, 0, kv=2, d=64, page=16, seed=241, extra_entries=0 if what == "place" else 1)
    if what == "place":
        b.spans[1] = (*b.spans[1][:2], len(b.table[0]) * 16 - 2)
    q = torch.randn(b.tokens, 4, 64, generator=generator(242))
    if what == "k":
        b.k_bytes[b.table[0][12], 1, 9, 5] = 0x7f    # row 201: the second token alone sees it
    elif what == "q":
        q[1, 2, 5] = math.nan
    elif what == "entry":
        b.table[0][3] = 4000
    elif what == "large":
        q[0] = 3e5
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=16, scaling=0.125).float()
    start = torch.rand(b.k_bytes.shape[0], 2, 16, generator=generator(243))
    expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=16, scaling=0.125, first=0)
    cache, batch = b.device()
    got = ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), start.to(DEV), scaling=0.125, **batch)
    check_weights(got, expected, spread, written, start, q_dtype=torch.float32, d=64, lse=lse.double(), n=4)


def test_captured_calls_replay_with_other_lengths():
    b = shared_batch([(500, 1), (410, 1)], 0, kv=2, d=128, page=32, seed=251)
    q = torch.randn(b.tokens, 8, 128, generator=generator(252)).to(DEV)
    cache, batch = b.device()
    lse = torch.full((b.tokens, 8), 3.0, device=DEV)
    start = torch.rand(b.k_bytes.shape[0], 2, 32, generator=generator(253)).to(DEV)
    out = start.clone()
    ops.launch_attention_weights(q, cache, lse, start, scaling=0.1, out=out, **batch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.launch_attention_weights(q, cache, lse, start, scaling=0.1, out=out, **batch)
    for contexts in ([500, 410], [20, 400], [500, 0]):
        batch["context_lens"].copy_(torch.tensor(contexts, dtype=torch.int32))
        eager = ops.launch_attention_weights(q, cache, lse, start, scaling=0.1, out=start.clone(), **batch)
        out.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("q_dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 256)])
def test_many_rows_of_waves_with_tiles_of_their_own(q_dtype, d):
    """Under a wide page table tens of tokens are not taken in turn."""

    _say("weights not in turn", q_dtype, d)
    b = shared_batch([(100, 40), (3, 30)], 0, kv=2, d=d, page=128, seed=261, ahead=1, behind=1, extra_entries=200)
    q = torch.randn(b.tokens, 8, d, generator=generator(262)).to(q_dtype)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=128, scaling=d**-0.5).float()
    start = torch.rand(b.k_bytes.shape[0], 2, 128, generator=generator(263))
    expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=128, scaling=d**-0.5, first=7)
    cache, batch = b.device()
    got = ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), start.to(DEV), scaling=d**-0.5, first=7, **batch)
    check_weights(got, expected, spread, written, start, q_dtype=q_dtype, d=d, lse=lse.double(), n=160)


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,page,extra", [
    ([(150, 2), (70, 1)], 32, 0),         # few query rows under a short table
    ([(150, 2), (70, 1)], 128, 520),      # and under a wide one
    ([(150, 9), (70, 10)], 32, 0),        # tens of query rows
    ([(150, 41), (70, 30)], 128, 30),     # taken in turn, in tiles of 64 rows
    ([(150, 41), (70, 30)], 16, 0),       # and of 32
])
def test_each_size_of_tile(lengths, page, extra, d, q_dtype):
    _say("weights by tiles", lengths, page, extra, d, q_dtype)
    b = shared_batch(lengths, 0, kv=2, d=d, page=page, seed=271, ahead=1, behind=1, extra_entries=extra)
    q = torch.randn(b.tokens, 8, d, generator=generator(272)).to(q_dtype)
    lse = olc.attention_lse(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5).float()
    start = torch.rand(b.k_bytes.shape[0], 2, page, generator=generator(273))
    cache, batch = b.device()
    for first in (0, 83):
        expected, spread, written = olc.attention_weights(q, b.host(), lse, start, b.table, b.spans, page=page, scaling=d**-0.5, first=first)
        got = ops.launch_attention_weights(q.to(DEV), cache, lse.to(DEV), start.to(DEV), scaling=d**-0.5, first=first, **batch)
        check_weights(got, expected, spread, written, start, q_dtype=q_dtype, d=d, lse=lse.double(), n=164)
