"""Forms of the serving operators beside those of tests/test_gpu_serving.py, against the
same 64-bit restatement (oracle/serving.py).

Bounds. fp32 queries: two fp16 parts are within 2^-23 of every value down to 2^-28 of
the head's largest (three values in four are exact); products and sums of fp32 as in
tests/test_gpu_serving.py, whose bound for fp32 queries (2^-24 (3 D + 8) of sum |q| |k|)
holds 2^-23 for the parts and D + 6 roundings of 2^-24 many times over. Where a score
is one product alone, it is held to the parts' 2^-23 and the roundings of that product,
of its scales and of the subtraction: 2^-24 * 8 of it.
"""

from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import serving as osv
from test_gpu_serving import DEV, Batch, _filled, _g, _same_bytes, _say

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


@pytest.mark.parametrize("d,tokens,extra", [(64, 1, 1), (64, 9, 1), (64, 70, 260), (128, 1, 1), (128, 9, 12), (128, 70, 260),
                                            (256, 2, 1), (256, 40, 1)])
@pytest.mark.parametrize("light", [-3, -12, -16, -20, -24, -28])
def test_paged_attention_light_query_values_beside_a_heavy_one(d, tokens, extra, light):
    """K is 0 where the query is heavy, and 1 in one light dimension, another for each
    row: the weights hang on the light values' last bits. One token, a few and a chunk."""

    _say("light values", d, tokens, extra, light)
    page = 64
    b = Batch([(100, tokens)], kv=1, d=d, page=page, seed=93, extra_entries=extra)
    _filled(b, 94)
    b.k_bytes.zero_()
    for row in range(100 + tokens):
        b.k_bytes[b.table[0][row // page], 0, row % page, 1 + row % (d - 1)] = 0x38  # 1.0
    b.scales[0] = 2.0 ** (5 - light)
    q = (1.9 + 0.1 * torch.rand(tokens, 4, d, generator=_g(95))) * 2.0**light  # scores from 60.8 to 64
    q[:, :, 0] = 1.0
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=1.0)
    cache, at = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=1.0, out_dtype=torch.float32, **at).cpu().double()
    u = 2.0**-24
    # A weight: its score's error and the maximum's, an exponential's and a part's step; sums over the rows.
    bound = (2 * u * 8 * reach[..., None] + u * ((100 + tokens) / 16 + 64 + 2)) * spread + u * expected.abs()
    assert ((out.view(expected.shape) - expected).abs() / bound).max() <= 1


def test_paged_append_rounds_k_once_below_the_least_normal_number():
    """At the smallest scale, 2^-126, e4m3's borders between bytes 0, 1, 2 and 3 are
    fp32 subnormals. K = x + y of fp64, its rotation's sum: x on such a border, y too
    little for fp32 to hold beside it, on either side. The byte is that of the exact sum."""

    d, page = 64, 16
    borders = [2.0**-136, 3 * 2.0**-136, 5 * 2.0**-136, 2.0**-135 + 2.0**-137]  # the last is no border
    b = Batch([(0, 8)], kv=1, d=d, page=page, seed=96)
    k = torch.zeros(8, 1, d, dtype=torch.float64)
    sin = torch.zeros(8, d // 2)
    for t in range(8):
        for j, border in enumerate(borders):
            k[t, 0, j] = border * (1 if t % 4 < 2 else -1)
            k[t, 0, j + d // 2] = 2.0**-140
            sin[t, j] = 2.0**-30 * (1 if t % 2 else -1)  # K = border -+ 2^-170
    k = k.float()
    v = torch.zeros(8, 1, d)
    cos = torch.ones(8, d // 2)
    _, expected = osv.append(k, k, v, b.host(), b.table, b.spans, page=page, q_norm=None, k_norm=None, eps=0.0, cos=cos, sin=sin)
    cache, batch = b.device()
    ops.launch_paged_append(k.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=1, q_norm=None, k_norm=None, eps=0.0,
                            cos=cos.to(DEV), sin=sin.to(DEV), **batch)
    _same_bytes(cache.k, expected["k"])
    assert len(set(expected["k"][b.table[0][0], 0, :8, 0].abs().tolist())) == 2  # both sides of the first border
