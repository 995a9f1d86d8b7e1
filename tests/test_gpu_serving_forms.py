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

import functools

import pytest
import torch

from conftest import gpu_available
from nanoquant_amd import synthetic as syn
from nanoquant_amd.runtime import shell_ops as ops
from nanoquant_amd.runtime.decoder_shell import PackedDecoder
from oracle import serving as osv
from oracle.nq_oracle import relative_l2
from test_gpu_serving import (DEV, EPS, HALF_STEP, SMALL, Batch, _check_attention, _filled, _g, _rope_tables, _same_bytes,
                              _say)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


# One call or more for each form that a call can take (tests/serving_plan.py; test_serving_plan.py
# holds this list to it): rows of a slot, waves that share them or not, one launch or two.
ATTENTIONS = [
    # lengths, q heads, kv heads, head_dim, page, table entries behind the longest sequence
    *(case for d in (64, 128) for case in (
        ([(130, 1), (63, 2), (0, 1)], 8, 2, d, 16, 1),                             # 16 rows, eight waves
        ([(i * 7 % 300, 1 + i % 3) for i in range(70)], 8, 4, d, 32, 1),           # 16 rows, the chip is full
        ([(1500, 2), (20, 3), (0, 1)], 8, 2, d, 64, 1),                            # ... split
        ([(i * 11 % 200, 5 + i % 3) for i in range(40)], 16, 4, d, 32, 1),         # 32 rows
        ([(1500, 10), (20, 12), (0, 8)], 8, 2, d, 64, 50),                         # ... split
        ([(37, 70), (0, 65), (5, 66), (100, 65)], 66, 33, d, 128, 128),            # 128 rows
        ([(700, 90), (0, 70), (33, 65)], 8, 4, d, 128, 122),                       # ... split
    )),
    ([(130, 1), (63, 2), (0, 1)], 8, 2, 256, 16, 1),
    ([(1500, 2), (20, 3), (0, 1)], 8, 2, 256, 64, 1),
    ([(i * 31 % 300, 39 + i % 3) for i in range(11)], 8, 8, 256, 32, 1),
    ([(1500, 30), (20, 33), (0, 28)], 8, 2, 256, 64, 1),
]

DTYPES = [(q, out) for q in (torch.float32, torch.bfloat16, torch.float16) for out in (torch.float32, torch.bfloat16, torch.float16)]


@functools.lru_cache(maxsize=2)
def _case(at: int, full: bool):
    """The batch, the queries (24 bits, or few enough for every type) and their attention."""

    lengths, q_heads, kv, d, page, extra = ATTENTIONS[at]
    b = Batch(lengths, kv=kv, d=d, page=page, seed=97, ahead=1, behind=2, extra_entries=extra)
    _filled(b, 98)
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, q_heads, d, generator=_g(99))
    if not full:
        q = (q * 32).round() / 32
    return b, q, osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)


@pytest.mark.parametrize("at", range(len(ATTENTIONS)))
@pytest.mark.parametrize("full", [True, False])
def test_paged_attention_in_every_form(at, full):
    """Each form with each type of q and of the output."""

    lengths, q_heads, kv, d, page, _ = ATTENTIONS[at]
    b, q, (expected, spread, reach) = _case(at, full)
    cache, batch = b.device()
    mine = ~torch.isnan(expected[:, 0, 0])
    assert mine.sum() == b.spans[-1][1] - 1
    for q_dtype, out_dtype in DTYPES:
        if full != (q_dtype == torch.float32):
            continue
        _say("form", at, q_dtype, out_dtype)
        assert torch.equal(q.to(q_dtype).float(), q)
        out = torch.full((b.tokens, q_heads * d), 9.0, dtype=out_dtype, device=DEV)
        ops.launch_paged_attention(q.to(q_dtype).to(DEV), cache, scaling=d**-0.5, out=out, **batch)
        assert (out.cpu()[~mine] == 9.0).all()
        _check_attention(out[mine.to(DEV)], expected[mine], spread[mine], reach[mine], q_dtype=q_dtype,
                         rows=max(c + n for c, n in lengths), d=d)


@pytest.mark.parametrize("dtype,norm_dtype,out_dtype,in_place", [
    (torch.float32, torch.bfloat16, torch.bfloat16, False), (torch.float32, torch.float16, torch.float16, False),
    (torch.bfloat16, torch.bfloat16, torch.bfloat16, True), (torch.float16, torch.float32, torch.float16, True),
    (torch.float32, torch.float32, torch.float32, True), (torch.bfloat16, torch.float16, torch.float16, False),
    (torch.float16, torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, None, torch.bfloat16, True)])
@pytest.mark.parametrize("d,q_heads,kv,page", [(64, 9, 3, 16), (128, 5, 5, 64), (256, 6, 2, 32)])
def test_paged_append_with_16_bit_norms_and_outputs(d, q_heads, kv, page, dtype, norm_dtype, out_dtype, in_place):
    """Norm weights and rotated queries of every type, and queries rotated in place."""

    _say("append", d, dtype, norm_dtype, out_dtype, in_place)
    b = Batch([(page - 3, 7), (0, 1), (2 * page, page + 2)], kv=kv, d=d, page=page, seed=100, ahead=1, behind=2)
    q, k, v = (torch.randn(b.tokens, h, d, generator=_g(s)).to(dtype) for h, s in ((q_heads, 101), (kv, 102), (kv, 103)))
    qn, kn = (None if norm_dtype is None else (1 + 0.1 * torch.randn(d, generator=_g(s))).to(norm_dtype) for s in (104, 105))
    cos, sin = _rope_tables(4 * page, d)
    rotated, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=page, q_norm=qn, k_norm=kn, eps=EPS, cos=cos, sin=sin)
    cache, batch = b.device()
    into = q.to(DEV)
    out = into if in_place else torch.full((b.tokens, q_heads, d), 7.0, dtype=out_dtype, device=DEV)
    got = ops.launch_paged_append(into, k.to(DEV), v.to(DEV), cache, q_heads=q_heads, q_norm=None if qn is None else qn.to(DEV),
                                  k_norm=None if kn is None else kn.to(DEV), eps=EPS, cos=cos.to(DEV), sin=sin.to(DEV),
                                  q_out=out, **batch)
    assert got is out
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    assert torch.equal(cache.k_scales.cpu().double(), expected["k_scales"])
    written = ~torch.isnan(rotated[:, 0, 0])
    assert torch.equal(out.cpu()[~written], q[~written] if in_place else torch.full_like(out.cpu()[~written], 7.0))
    # 8 fp32 roundings relative to the rotated pair, and the output's own.
    x, half = rotated[written], d // 2
    pair = torch.sqrt(x[..., :half].pow(2) + x[..., half:].pow(2)).repeat(1, 1, 2)
    bound = 8 * 2.0**-24 * 1.5 * pair + HALF_STEP[out_dtype] * x.abs() + (2.0**-25 if out_dtype == torch.float16 else 0.0)
    assert ((out.cpu()[written].double() - x).abs() <= bound).all()


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


@pytest.mark.parametrize("rise", [2.0, 4.0, -4.0])
@pytest.mark.parametrize("d,tokens,extra,scale", [(64, 1, 1, 1.0), (128, 9, 12, 1.0), (128, 70, 250, 1.0), (256, 9, 1, 1.0),
                                                  (64, 70, 250, 1.25)])
def test_paged_attention_values_near_the_top_of_fp32(d, tokens, extra, scale, rise):
    """Values of 2^123 with scores that rise from tile to tile by less than a running
    maximum may lag behind: a weight times its value stays below 2^128."""

    _say("large values", d, tokens, extra, scale, rise)
    page = 64
    b = Batch([(1000, tokens)], kv=1, d=d, page=page, seed=106, extra_entries=extra)
    b.k_bytes.zero_()
    b.k_bytes[..., 1] = 0x70  # 128: rows that weigh nothing, but for one in each page
    b.v_bytes[:] = 0x38       # 1.0
    for i, at in enumerate(b.table[0][:-(-(1000 + tokens) // page)]):
        b.k_bytes[at, :, 0, :2] = torch.tensor([min(i, 16), 0], dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    b.scales[0], b.scales[1] = 1.0, scale * 2.0**123
    q = torch.zeros(tokens, 4, d)
    q[:, :, 0], q[:, :, 1] = rise, -8.0
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=1.0)
    cache, at = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=1.0, out_dtype=torch.float32, **at)
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=1000 + tokens, d=d)


def test_paged_attention_takes_a_narrower_table_as_a_copy():
    """What a call sees does not hang on the table's width; a view of some of its columns is refused."""

    b = Batch([(300, 3), (20, 1), (0, 9)], kv=2, d=128, page=16, seed=107, extra_entries=900)
    _filled(b, 108)
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, 8, 128, generator=_g(109))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=16, scaling=0.1)
    cache, batch = b.device()
    narrow = batch["page_table"][:, :20]
    with pytest.raises(ValueError, match="contiguous"):
        ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, **{**batch, "page_table": narrow})
    for table in (batch["page_table"], narrow.contiguous()):
        out = ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, out_dtype=torch.float32, **{**batch, "page_table": table})
        _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=303, d=128)


def test_calls_on_two_streams_at_once():
    """Each call's workspace is its own: splits of two calls in flight do not meet."""

    batches = [Batch([(2000 + 500 * i, 2), (30, 1)], kv=2, d=64, page=64, seed=110 + i) for i in range(2)]
    inputs = []
    for i, b in enumerate(batches):
        _filled(b, 112 + i)
        b.scales *= 2.0**-3
        cache, batch = b.device()
        inputs.append((torch.randn(b.tokens, 8, 64, generator=_g(114 + i)).to(DEV), cache, batch))
    alone = [ops.launch_paged_attention(q, cache, scaling=0.125, **batch) for q, cache, batch in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    together = []
    for _ in range(20):
        for stream, (q, cache, batch) in zip(streams, inputs):
            with torch.cuda.stream(stream):
                together.append(ops.launch_paged_attention(q, cache, scaling=0.125, **batch))
    torch.cuda.synchronize()
    for i, out in enumerate(together):
        assert torch.equal(out, alone[i % 2]), i


def test_decoder_protocol_with_the_8_bit_cache():
    """forward_step, prompt and decode steps, gives the logits of prefill."""

    weights = syn.synthetic_decoder(SMALL, seed=syn.BASE_SEED + 84, random_norms=True)
    decoder = PackedDecoder(SMALL, weights, device="cuda", max_positions=150, activation_dtype=torch.float32,
                            cache_dtype=torch.float8_e4m3fn)
    ids = torch.randint(0, SMALL.vocab, (66,), generator=_g(116)).to(DEV)
    decoder.reset()
    expected = [decoder.prefill(ids[:63]).clone()]
    for i in range(63, 66):
        expected.append(decoder.prefill(ids[i:i + 1], start=i).clone())
    cache, got = None, []
    for at, n in ((0, 63), (63, 1), (64, 1), (65, 1)):
        where = torch.arange(at, at + n, device=DEV)
        step = decoder.forward_step(input_ids=ids[None, at:at + n], attention_mask=torch.ones(1, at + n, device=DEV),
                                    position_ids=where[None], cache_position=where, cache=cache, max_cache_length=150,
                                    workload="decode" if n == 1 else "prefill", deterministic=True)
        cache = step.cache
        got.append(step.logits.view(-1).clone())
    assert torch.equal(got[0], expected[0])
    # Decode steps fold norms and sums into the linears: 2e-5 relative a linear, e4m3 steps of K and V (8e-3 over three layers).
    for a, e in zip(got[1:], expected[1:]):
        assert relative_l2(a.cpu(), e.cpu()) < 8e-3


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn])
def test_decoder_passes_wait_for_nothing(cache):
    """A prompt on the device, its pass, decode steps and their scores: the host waits for none."""

    weights = syn.synthetic_decoder(SMALL, seed=syn.BASE_SEED + 85, random_norms=True)
    decoder = PackedDecoder(SMALL, weights, device=DEV, max_positions=150, cache_dtype=cache)
    ids = torch.randint(0, SMALL.vocab, (70,), generator=_g(117)).to(DEV)

    def passes():
        tokens = decoder.generate_greedy(ids, 20)
        scored, answer = decoder.generate_greedy_scored(ids, 20, top=2)
        return tokens, scored, answer, decoder.score(ids, top=2), decoder.prefill(ids[:33]).clone()

    first = passes()
    before = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        second = passes()
    finally:
        torch.cuda.set_sync_debug_mode(before)
    for a, b in zip(first, second):
        for x, y in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
            assert torch.equal(x, y)
