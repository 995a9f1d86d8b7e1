"""Pins of the serving operators' oracle (oracle/serving.py) by torch's own
conversions and softmax, on the CPU."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving as osv


def test_e4m3_is_torchs_conversion_for_every_byte_and_between():
    values = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    finite = values[torch.isfinite(values)].sort().values
    between = torch.cat([finite, (finite[1:] + finite[:-1]) / 2, finite * 0.9371, finite * 1.03]).clamp(-448, 448)
    assert torch.equal(osv.e4m3(between).float(), between.to(torch.float8_e4m3fn).float())
    assert torch.isnan(osv.e4m3(torch.tensor([math.nan, math.inf, -math.inf]))).all()


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (0.0, 2.0**-126), (1e-45, 2.0**-126),
                                        (3.4e38, 2.0**120)])
def test_scale_is_the_least_power_of_two(amax, scale):
    assert osv.scale_for(amax) == scale


def test_append_then_attention_is_attention_over_the_rounded_rows():
    g = torch.Generator().manual_seed(5)
    page, kv, d, tokens = 16, 2, 64, 21
    cache = {"k": torch.zeros(3, kv, page, d), "v": torch.zeros(3, kv, d, page), "k_scales": torch.zeros(3, kv),
             "v_scales": torch.zeros(3, kv)}
    q, k, v = (torch.randn(tokens, h, d, generator=g) for h in (4, kv, kv))
    cos, sin = torch.ones(64, d // 2), torch.zeros(64, d // 2)
    table, spans = [[2, 0]], [(0, tokens, 0)]
    rotated, cache = osv.append(q, k, v, cache, table, spans, page=page, q_norm=None, k_norm=None, eps=0.0, cos=cos, sin=sin)
    assert torch.equal(rotated, q.double())  # a turn by no angle
    stored = (cache["k"] * cache["k_scales"][..., None, None])[[2, 0]].transpose(0, 1).reshape(kv, 2 * page, d)[:, :tokens]
    assert ((stored - k.transpose(0, 1).double()).abs() <= 2.0**-4 * k.transpose(0, 1).abs() + 2.0**-10 * cache["k_scales"].max()).all()
    out, _, _ = osv.attention(rotated, cache, table, spans, page=page, scaling=0.1)
    value = (cache["v"] * cache["v_scales"][..., None, None])[[2, 0]].transpose(0, 1).transpose(2, 3).reshape(kv, 2 * page, d)
    for t in (0, 7, 20):
        p = torch.softmax(rotated[t, 3] @ stored[1, :t + 1].T * 0.1, -1)
        assert torch.allclose(out[t, 3], p @ value[1, :t + 1], rtol=1e-12, atol=1e-14)


def test_token_logprobs_are_log_softmax():
    x = torch.randn(3, 17, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
    x[1, 4] = -math.inf
    x[2, 3] = x[2, 9] = 5.0
    lp, h, ids, top = osv.token_logprobs(x, torch.tensor([2, 4, 17]), 3)
    expected = torch.log_softmax(x, -1)
    assert torch.allclose(lp[:2], expected[[0, 1], [2, 4]]) and torch.isnan(lp[2])
    assert torch.allclose(h, torch.distributions.Categorical(logits=x).entropy(), atol=1e-12)
    assert ids[2, :2].tolist() == [3, 9] and torch.allclose(top, expected.gather(1, ids))
