"""Rounding a matrix to 4 bits (no GPU needed): the scale that is taken, and what is refused."""

from __future__ import annotations

import math

import pytest
import torch

from nanoquant_amd.runtime import shell_ops as ops
from oracle import long_conversations as olc


def _dense(m, group):
    return olc.int4_dense(m.packed, m.scales, m.zeros, group)


def test_the_larger_scale_is_taken_so_that_both_ends_are_held():
    w = torch.zeros(3, 64)
    w[0, 0], w[0, 1] = 7.0, -4.0     # 7 to 7, -4 to -4
    w[1, 0], w[1, 1] = 3.5, -8.0     # -8 to -8
    w[2, 5] = -16.0                  # a group without values above 0
    m = ops.int4_matrix(w, 64, torch.float32)
    assert m.scales[:, 0].tolist() == [1.0, 1.0, 2.0]
    assert _dense(m, 64)[0, :2].tolist() == [7.0, -4.0]
    assert _dense(m, 64)[1, :2].tolist() == [4.0, -8.0]  # 3.5 to the even 4
    assert _dense(m, 64)[2, 5] == -16.0


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("row", [0, 8191, 8192, 9000])
def test_weights_that_are_not_finite_are_refused(value, row):
    w = torch.ones(9001, 32)
    w[row, 31] = value
    with pytest.raises(ValueError, match="finite"):
        ops.int4_matrix(w, 32)


def test_scales_beyond_their_type_are_refused():
    w = torch.ones(2, 128)
    w[1, 100] = 5e5  # / 7 is beyond fp16's 65504
    with pytest.raises(ValueError, match="float16"):
        ops.int4_matrix(w, 128)
    for dtype in (torch.bfloat16, torch.float32):
        m = ops.int4_matrix(w, 128, dtype)
        assert abs(float(_dense(m, 128)[1, 100]) - 5e5) <= 5e5 * torch.finfo(dtype).eps / 2 * 1.01
    w[1, 100] = 4.5e5
    assert bool(torch.isfinite(ops.int4_matrix(w, 128).scales).all())


def test_groups_of_zeros_stay_zero():
    assert (_dense(ops.int4_matrix(torch.zeros(5, 96), 64), 64) == 0).all()
