"""Paged attention where scores are far larger than fp32's steps resolve: the largest
score's weight is 1 however large the score is, as in fp32 arithmetic."""

from __future__ import annotations

import pytest
import torch
from test_gpu_serving import DEV, Batch, _filled, _g, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import serving as osv

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


@pytest.mark.parametrize("size", [1e6, 1e12, 3e38])
@pytest.mark.parametrize("lengths,d", [([(200, 2), (40, 1)], 64), ([(130, 40)], 128), ([(1500, 1)], 128), ([(300, 3)], 256)])
def test_scores_beyond_what_fp32_resolves(lengths, d, size):
    """One row's score is above all others by far more than rounding takes off it
    (scores differ by a few per cent of themselves, rounding takes 2^-22 of them): the output is that row's V."""

    _say("large scores", lengths, d, size)
    b = Batch(lengths, kv=2, d=d, page=32, seed=171)
    _filled(b, 172)
    b.scales *= 2.0**-3
    q = torch.empty(b.tokens, 4, d).fill_(-size)
    q[1::2] *= 0.5
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=32, scaling=d**-0.5)
    cache, batch = b.device()
    got = ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out_dtype=torch.float32, **batch).cpu()
    got = got.view(expected.shape)
    assert not torch.isnan(got).any()
    # Rows whose two largest scores lie further apart than rounding moves them: one row is the output.
    u = 2.0**-24
    for t, (begin, end, context) in ((t, s) for s in b.spans for t in range(s[0], s[1])):
        for h in range(4):
            i = b.spans.index((begin, end, context))
            keys = torch.cat([b.host()["k"][at, h // 2] * b.host()["k_scales"][at, h // 2] for at in b.table[i]
                              if at >= 0])[:context + t - begin + 1]
            top = (keys @ q[t, h].double() * d**-0.5).topk(2).values
            if top[0] - top[1] > 200 + 4 * u * (3 * d + 8) * reach[t, h]:
                assert torch.allclose(got[t, h].double(), expected[t, h], rtol=2.0**-22, atol=0)
