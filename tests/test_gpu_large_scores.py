"""Attention over the 8-bit cache where every query row's largest score is far above the
next one by construction, at sizes that fp32 does not resolve: the output is that row's V."""

from __future__ import annotations

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_serving import DEV, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


@pytest.mark.parametrize("size", [1e6, 1e12, 1e30, 1e37])
@pytest.mark.parametrize("lengths,shared,d", [([(200, 2), (170, 1)], 0, 64), ([(130, 40)], 0, 128), ([(1500, 1)], 0, 128),
                                              ([(300, 3)], 0, 256), ([(400, 1), (390, 1), (450, 2)], 320, 128)])
def test_the_largest_score_has_a_weight_of_1(lengths, shared, d, size):
    """Row 90's keys are 128 in every dimension, the others' at most 120 with either sign, and q is one
    value: row 90's score is the largest for all query rows, the next at most 15/16 of it, more than 10^4
    below. The other weights are 0, so the output is V of row 90."""

    _say("separate scores", lengths, shared, d, size)
    b = shared_batch(lengths, shared, kv=2, d=d, page=32, seed=901)
    b.k_bytes = torch.randint(0, 0x70, b.k_bytes.shape, generator=generator(902), dtype=torch.uint8) \
        | (torch.randint(0, 2, b.k_bytes.shape, generator=generator(903), dtype=torch.uint8) << 7)  # up to 120
    b.scales[0] = 2.0**-12
    for line in b.table:
        b.k_bytes[line[2], :, 90 % 32] = 0x70  # 128
    q = torch.full((b.tokens, 4, d), size)
    cache, batch = b.device()
    args = {"scaling": d**-0.5, **batch}
    assert float(q[0, 0].double().sum()) * 2.0**-12 * d**-0.5 * (128 - 120) > 1e4
    v = torch.stack([b.v_bytes[line[2], :, :, 90 % 32].view(torch.float8_e4m3fn).double() * b.scales[1][line[2]].double()[:, None]
                     for line in b.table])  # [batch, kv, d]
    expected = torch.cat([v[i][None].repeat_interleave(2, 1).expand(e - s, 4, d) for i, (s, e, _) in enumerate(b.spans)])
    for dtype in (torch.float32, torch.bfloat16):
        for got in (ops.launch_paged_attention(q.to(DEV), cache, out_dtype=dtype, **args),
                    ops.launch_shared_attention(q.to(DEV), cache, shared_rows=shared, out_dtype=dtype, **args)):
            got = got.cpu().view(b.tokens, 4, d).double()
            if dtype == torch.bfloat16:  # V's four bits fit: a weight of 16 bits rounds back to them
                assert torch.equal(got, expected)
            else:  # the product, its sum's inverse and theirs: 2^-24 each
                assert torch.allclose(got, expected, rtol=2.0**-22, atol=0)
