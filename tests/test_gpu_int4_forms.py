"""Products with 4-bit weights in every form that a call can take: tiles of their own or shared by
four waves, slices of the rows, digits in several stages, workgroups that walk over
several tiles (tests/test_int4_plan.py asks which of these SHAPES reach). The definition is formed on
the device in 64 bits; bounds as in tests/test_gpu_int4.py."""

from __future__ import annotations

import pytest
import torch
from test_gpu_int4 import by_group, check, matrix
from test_gpu_serving import DEV, HALF_STEP, _g, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

SHAPES = [
    # tokens, in, out, group
    (31, 1024, 16400, 128), (7, 2048, 16400, 32), (4, 2048, 32784, 32), (33, 288, 16948, 128),  # stages, passes, a short last one
    (1, 10944, 32951, 32), (5, 2592, 33544, 128), (6, 1952, 34248, 64),
    (1, 64, 12304, 32), (1, 64, 32752, 32), (3, 96, 12466, 32), (7, 32, 6240, 32), (14, 64, 13218, 128), (9, 32, 12332, 128),  # shared, walking
    (1, 11360, 24715, 64), (2, 5792, 24749, 32), (3, 3840, 24908, 32),  # slices, walking
    (1, 32160, 11271, 32), (8, 24800, 3, 128), (6, 30784, 18, 64), (5, 31552, 20, 32),  # slices in stages
    (4, 30688, 27, 32), (4, 36320, 20, 32),  # 87 KB of LDS (bf16), 103 (fp32)
    (1, 32, 32814, 32), (1, 32, 49268, 32), (2, 32, 49224, 32), (3, 32, 49379, 32), (7, 64, 24866, 32),
]


def dense(m, group):
    """fp64 [out, in] on the matrix's device."""
    w = torch.stack((m.packed & 15, m.packed >> 4), 2).view(m.packed.shape[0], -1).double()
    column = torch.arange(w.shape[1], device=w.device) // group
    zero = 8.0 if m.zeros is None else m.zeros.double()[:, column]
    return (w - zero) * m.scales.double()[:, column]


@pytest.mark.parametrize("x_dtype,scale_dtype,zeros", [(torch.float32, torch.float16, True), (torch.bfloat16, torch.float32, False)])
@pytest.mark.parametrize("tokens,ins,outs,group", SHAPES)
def test_every_form(tokens, ins, outs, group, x_dtype, scale_dtype, zeros):
    _say("int4 forms", tokens, ins, outs, group, x_dtype)
    m = matrix(outs, ins, group, scale_dtype, zeros, 801)
    x = torch.randn(tokens, ins, generator=_g(802))
    x *= torch.where(torch.rand(ins, generator=_g(803)) < 0.02, 40.0, 1.0)
    x = x.to(x_dtype)
    at, x_at = m.to(DEV), x.to(DEV)
    partials = torch.zeros(ops.int4_projection_partials(outs), dtype=torch.int64, device=DEV) if tokens == 1 else None
    out = torch.full((tokens + 1, outs), 9.0, device=DEV)
    got = ops.launch_int4_projection(x_at, at, out=out[:tokens], partials=partials)
    assert (out[tokens] == 9.0).all()
    assert torch.equal(ops.launch_int4_projection(x_at, at), got)
    if tokens == 1:
        token = torch.zeros(1, dtype=torch.int64, device=DEV)
        ops.launch_greedy_select_partials(partials, token_out=token)
        assert int(token) == int((got[0] == got[0].max()).nonzero()[0])
    top = by_group(x_at.double(), ins, group)
    adds = 3 + -(-ins // 128) + 3 * (128 // group) * 4
    for first in range(0, outs, 8192):
        rows = slice(first, first + 8192)
        w = dense(ops.Int4Matrix(*(None if t is None else t[rows] for t in at)), group)
        expected, size = x_at.double() @ w.T, w.abs().T.contiguous()
        bound = (1.01 * 2.0**-23 * (top @ size) + 2.0**-24 * adds * ((x_at.double().abs() + 2.0**-7 * top) @ size)
                 + HALF_STEP[torch.float32] * expected.abs() + 1e-30)
        worst = float(((got[:, rows].double() - expected).abs() / bound).max())
        assert worst <= 1, (first, worst)
    few = slice(max(0, outs - 40), outs)  # and against the oracle
    check(got[:, few], x, ops.Int4Matrix(*(None if t is None else t[few] for t in m)), group)
