"""Products with 4-bit weights on the GPU against their 64-bit restatement
(oracle/long_conversations.py).

Bounds: x enters within 2^-23 (1.01) of its group's largest value. A group's digit sums are exact; each becomes
fp32, meets the scale and the digit's power (three roundings) and is added to its
lane's, 2^-24 each of what the digits' sizes add up to: |x| + 2^-7 of the group's
largest value for each column. Lanes, waves and groups of a chunk add 3 (128 / group) 4
more. The output is rounded once.
"""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_serving import DEV, HALF_STEP, _g, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


def matrix(outs, ins, group, scale_dtype, zeros, seed):
    g = _g(seed)
    groups = -(-ins // group)
    packed = torch.randint(0, 256, (outs, ins // 2), generator=g, dtype=torch.uint8)
    scales = (0.01 * (0.5 + torch.rand(outs, groups, generator=g))).to(scale_dtype)
    z = torch.randint(0, 16, (outs, groups), generator=g, dtype=torch.uint8) if zeros else None
    return ops.Int4Matrix(packed, scales, z)


def by_group(x, ins, group):
    """Each column's largest |x| of its group."""
    padded = torch.nn.functional.pad(x.abs(), (0, -ins % group)).view(x.shape[0], -1, group)
    return padded.amax(-1).repeat_interleave(group, 1)[:, :ins]


def check(got, x, m, group):
    outs, ins = m.shape
    w = olc.int4_dense(m.packed, m.scales, m.zeros, group)
    x = x.double()
    expected, top = x @ w.T, by_group(x, ins, group)
    sizes = (x.abs() + 2.0**-7 * top) @ w.abs().T
    adds = 3 + -(-ins // 128) + 3 * (128 // group) * 4
    bound = 1.01 * 2.0**-23 * (top @ w.abs().T) + 2.0**-24 * adds * sizes + HALF_STEP[got.dtype] * expected.abs() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + 2.0**-25
    worst = float(((got.cpu().double() - expected).abs() / bound).max())
    assert worst <= 1, worst


SHAPES = [
    # tokens, in, out, group
    (1, 32, 1, 32), (1, 32, 16, 128), (1, 64, 17, 64), (2, 96, 5, 32), (1, 128, 33, 128), (3, 160, 40, 64), (5, 256, 48, 128),
    (6, 1152, 100, 128), (1, 1152, 6912, 32), (2, 2560, 31, 64), (4, 4096, 257, 32), (16, 4096, 64, 128), (7, 10240, 40, 64),
    (1, 14336, 72, 128), (33, 224, 20, 32), (70, 480, 19, 128), (17, 32, 15, 64), (1, 4096, 4099, 128), (12, 992, 300, 64),
]


@pytest.mark.parametrize("x_dtype,out_dtype,scale_dtype,zeros", [
    (torch.float32, torch.float32, torch.float16, False), (torch.bfloat16, torch.bfloat16, torch.bfloat16, True),
    (torch.float16, torch.float16, torch.float32, True), (torch.float32, torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, torch.float32, False)])
@pytest.mark.parametrize("tokens,ins,outs,group", SHAPES)
def test_int4_projection(tokens, ins, outs, group, x_dtype, out_dtype, scale_dtype, zeros):
    _say("int4", tokens, ins, outs, group, x_dtype, out_dtype, scale_dtype, zeros)
    m = matrix(outs, ins, group, scale_dtype, zeros, 501)
    x = torch.randn(tokens, ins, generator=_g(502))
    x *= torch.where(torch.rand(ins, generator=_g(503)) < 0.02, 40.0, 1.0)
    x = x.to(x_dtype)
    out = torch.full((tokens + 1, outs), 9.0, dtype=out_dtype, device=DEV)
    got = ops.launch_int4_projection(x.to(DEV), m.to(DEV), out=out[:tokens])
    check(got, x, m, group)
    assert (out[tokens] == 9.0).all()
    again = ops.launch_int4_projection(x.to(DEV), m.to(DEV), out_dtype=out_dtype)
    assert torch.equal(again, got)


def test_every_nibble_is_its_value_at_every_place():
    """One column of one token at a time: x = 1 there gives the weight back."""

    m = matrix(48, 256, 64, torch.float32, True, 511)
    w = olc.int4_dense(m.packed, m.scales, m.zeros, 64)
    got = ops.launch_int4_projection(torch.eye(256).to(DEV), m.to(DEV)).cpu().double()
    assert torch.allclose(got, w.T, rtol=3 * 2.0**-24, atol=0)


@pytest.mark.parametrize("tokens,ins,outs,group", [(6, 12288, 300, 32), (6, 28672, 37, 32), (30, 14336, 300, 128)])
def test_slices_whose_workgroups_hold_more_than_64_kb(tokens, ins, outs, group):
    """Eight waves around digits of many chunks: 71 to 75 KB of LDS."""

    _say("int4 lds", tokens, ins, outs, group)
    m = matrix(outs, ins, group, torch.float16, True, 511)
    x = torch.randn(tokens, ins, generator=_g(512))
    got = ops.launch_int4_projection(x.to(DEV), m.to(DEV))
    check(got, x, m, group)
    assert torch.equal(ops.launch_int4_projection(x.to(DEV), m.to(DEV)), got)


@pytest.mark.parametrize("size", [1e-38, 1e-30, 2.0**-100, 1.0, 3e37, "ulp"])
def test_sizes(size):
    """Values near fp32's ends, and largest values just below a power of two."""

    _say("int4 sizes", size)
    m = matrix(40, 256, 128, torch.float32, False, 521)
    x = torch.rand(3, 256, generator=_g(522)) + 0.5
    if size == "ulp":
        x = torch.full((3, 256), 2.0 - 2.0**-23)
        x[1] = -x[1]
        x[2, ::2] = 127.5
        x[2, 1::2] = -127.998
    else:
        x *= size
    if size == 1e-38:  # below 2^-122 nothing is left, 2^-123 of it at most is off
        got = ops.launch_int4_projection(x.to(DEV), m.to(DEV)).cpu().double()
        w = olc.int4_dense(m.packed, m.scales, m.zeros, 128)
        assert ((got - x.double() @ w.T).abs() <= 1.01 * 2.0**-123 * w.abs().sum(1) + 2.0**-20 * (x.double() @ w.abs().T)).all()
        return
    check(ops.launch_int4_projection(x.to(DEV), m.to(DEV)), x, m, 128)


def test_tokens_that_hold_no_number_give_nan_alone():
    m = matrix(40, 384, 64, torch.float16, True, 531)
    x = torch.randn(5, 384, generator=_g(532))
    x[1, 200], x[3, 5], x[4, 383] = math.nan, math.inf, -math.inf
    got = ops.launch_int4_projection(x.to(DEV), m.to(DEV))
    assert torch.isnan(got[[1, 3, 4]]).all()
    check(got[[0, 2]], x[[0, 2]], m, 64)


def test_zeros_of_any_value_and_scales_that_are_zero_or_negative():
    m = matrix(33, 256, 32, torch.float32, True, 541)
    m.zeros.copy_(torch.randint(0, 256, m.zeros.shape, generator=_g(542), dtype=torch.uint8))
    m.scales[::3] = 0.0
    m.scales[1::3] *= -1
    x = torch.randn(3, 256, generator=_g(543))
    check(ops.launch_int4_projection(x.to(DEV), m.to(DEV)), x, m, 32)


@pytest.mark.parametrize("outs,ins,group", [(1, 32, 32), (16, 64, 32), (1000, 256, 64), (50257, 128, 128), (1000, 14336, 64)])
def test_partials_select_the_first_largest(outs, ins, group):
    m = matrix(outs, ins, group, torch.float16, False, 551)
    if outs > 900:
        m.packed[700] = m.packed[37]
        m.scales[700] = m.scales[37]
    x = torch.randn(1, ins, generator=_g(552))
    if outs > 900:  # the two equal rows are the largest
        w = olc.int4_dense(m.packed, m.scales, m.zeros, group)
        x = (x * 0.01 + w[37].float()[None] * 20).float()
    partials = torch.zeros(ops.int4_projection_partials(outs), dtype=torch.int64, device=DEV)
    logits = ops.launch_int4_projection(x.to(DEV), m.to(DEV), partials=partials)
    token = torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.launch_greedy_select_partials(partials, token_out=token)
    row = logits[0].cpu()
    assert int(token) == int((row == row.max()).nonzero()[0])
    if outs > 900:
        assert int(token) == 37


def test_rounding_to_4_bits():
    for group, ins in ((32, 96), (64, 96), (128, 288)):
        w = torch.randn(70, ins, generator=_g(561)).to(DEV)
        w[3] = 0.0
        m = ops.int4_matrix(w, group)
        back = olc.int4_dense(m.packed.cpu(), m.scales.cpu(), None, group)
        # Half a step of the group's scale, and 2^-11 of the value for the scale's own rounding (a step of it at the ends).
        step = m.scales.cpu().double().repeat_interleave(group, 1)[:, :ins]
        assert ((back - w.cpu().double()).abs() <= step * (0.5 + 8 * 2.0**-11) + 1e-12).all()
        assert (back[3] == 0).all()


def test_captured_calls_replay_with_other_inputs():
    m = matrix(300, 4096, 128, torch.float16, False, 571).to(DEV)
    x = torch.randn(4, 4096, generator=_g(572)).to(DEV)
    ops.launch_int4_projection(x, m)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.launch_int4_projection(x, m)
        graphs.append((graph, out))
    for seed in (1, 2, 3):
        x.copy_(torch.randn(4, 4096, generator=_g(seed)))
        eager = ops.launch_int4_projection(x, m)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_at_any_address(dtype):
    """x, scales, zeros and outputs that begin between their type's vectors."""

    m = matrix(50, 160, 32, dtype, True, 581)

    def moved(t):
        flat = torch.zeros(t.numel() + 3, dtype=t.dtype, device=DEV)
        flat[3:] = t.reshape(-1).to(DEV)
        return flat[3:].view(t.shape)

    x = torch.randn(3, 160, generator=_g(582)).to(dtype)
    at = ops.Int4Matrix(m.packed.to(DEV), moved(m.scales), moved(m.zeros))
    out = moved(torch.zeros(3, 50, dtype=dtype))
    check(ops.launch_int4_projection(moved(x), at, out=out), x, m, 32)


def test_work_on_another_stream_with_a_workspace_of_the_callers():
    m = matrix(300, 10240, 64, torch.float16, False, 591).to(DEV)
    x = torch.randn(9, 10240, generator=_g(592)).to(DEV)
    here = ops.launch_int4_projection(x, m)
    size = ops.int4_projection_workspace_bytes(9, m)
    assert size > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = ops.launch_int4_projection(x, m, workspace=torch.empty(size, dtype=torch.uint8, device=DEV))
    side.synchronize()
    assert torch.equal(here, there)


@pytest.mark.parametrize("tokens,ins,outs,group", [(1, 128, 40, 128), (5, 128, 40, 128), (9, 160, 33, 64), (3, 128, 200, 32),
                                                   (1, 4096, 64, 32), (11, 10240, 48, 64)])
def test_fp32_values_beside_one_that_meets_no_weight(tokens, ins, outs, group):
    """A column 10^5 times the others whose weights are all at the zero point: fp32 x is read to 2^-31
    of it, and nothing of it is in the result. A value's digits add up to 3.02 times it at most (1.502 to 0.498 where the
    highest is 1), whatever its neighbours are."""

    _say("int4 outlier", tokens, ins, outs, group)
    m = matrix(outs, ins, group, torch.float32, False, 601)
    column = 37 + 64 * (ins // 128 // 2)
    m.packed[:, column // 2] = (m.packed[:, column // 2] & 15) | 0x80
    x = torch.randn(tokens, ins, generator=_g(602))
    x[:, column] = 1e5
    w = olc.int4_dense(m.packed, m.scales, m.zeros, group)
    assert (w[:, column] == 0).all()
    got = ops.launch_int4_projection(x.to(DEV), m.to(DEV)).cpu().double()
    expected, top = x.double() @ w.T, by_group(x.double(), ins, group)
    adds = 3 + -(-ins // 128) + 3 * (128 // group) * 4
    sizes = 3.02 * (x.double().abs() @ w.abs().T)  # the column itself has no weight
    bound = 1.01 * 2.0**-31 * (top @ w.abs().T) + 2.0**-24 * adds * sizes + HALF_STEP[torch.float32] * expected.abs()
    worst = float(((got - expected).abs() / bound).max())
    assert worst <= 1, worst
