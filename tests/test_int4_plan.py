"""The layout of 4-bit products, on the CPU: the restated plan is the library's, a workgroup's
LDS is bounded, and the GPU tests reach every form."""

from __future__ import annotations

import random

import pytest
import test_gpu_int4
import test_gpu_int4_forms
from int4_plan import plan, workspace_bytes

from nanoquant_amd.runtime import _native

# (waves, share, slices, several stages, several tiles): all that calls can reach.
FLOWS = {(4, 4, False, False, False), (4, 4, False, False, True), (4, 1, False, False, False), (4, 1, False, False, True),
         (4, 1, False, True, False), (4, 1, True, False, False), (4, 1, True, False, True), (4, 1, True, True, False),
         (8, 1, True, False, False), (8, 1, True, True, False)}
DIGITS = (3, 4)  # of 16-bit x, of fp32 x


def _calls(seed, count):
    rng = random.Random(seed)
    for _ in range(count):
        yield (min(65535, round(2 ** rng.uniform(0, 16))), round(2 ** rng.uniform(0, 18)), 32 * round(2 ** rng.uniform(0, 11)),
               rng.choice([32, 64, 128]))


def test_the_restated_plan_is_the_librarys():
    flows = set()
    for tokens, outs, ins, group in _calls(11, 40000):
        got = _native.load().nq_int4_projection_workspace_bytes(tokens, outs, ins, group)
        assert got == -1 or got == workspace_bytes(tokens, outs, ins, group), (tokens, outs, ins, group)
        flows |= {plan(tokens, outs, ins, group, digits).form[2:] for digits in DIGITS}
    assert flows == FLOWS


def test_slices_and_stages_cover_the_rows_and_lds_holds_them():
    for tokens, outs, ins, group in _calls(12, 20000):
        for digits in DIGITS:
            p = plan(tokens, outs, ins, group, digits)
            chunks = -(-ins // 128)
            assert (p.slices - 1) * p.slice < chunks <= p.slices * p.slice and 1 <= p.stage <= p.slice
            assert p.slices <= 16 and p.blocks * p.passes * (16 // (128 // group) // digits) >= tokens
            assert p.lds <= (88 if digits == 3 else 104) * 1024


@pytest.mark.parametrize("digits", DIGITS)
def test_the_gpu_tests_reach_every_form(digits):
    plans = [plan(tokens, outs, ins, group, digits)
             for tokens, ins, outs, group in test_gpu_int4.SHAPES + test_gpu_int4_forms.SHAPES]
    assert {p.form[2:] for p in plans} == FLOWS
    assert {p.blocks for p in plans} == {1, 2, 3, 6}
    assert {p.blocks for p in plans if p.stage < p.slice and p.slices == 1} >= {1, 3, 6}
    assert {p.passes for p in plans if p.stage < p.slice and p.slices == 1} >= {1, 2}
    assert max(p.lds for p in plans) >= (85 if digits == 3 else 101) * 1024


def test_a_text_scored_by_rows_takes_stages():
    """256 rows of a large output projection: no slices, several passes and stages, as in SHAPES."""

    for digits in DIGITS:
        p = plan(256, 151936, 4096, 128, digits)
        assert p.slices == 1 and p.stage < p.slice and p.passes > 1 and p.blocks == 6


def test_partials_of_sizes_at_the_limits():
    count = _native.load().nq_int4_projection_partials
    assert [count(n) for n in (1, 16, 17, 0x7FFFFFFF)] == [1, 1, 2, 1 << 27]
    assert [count(n) for n in (0, -1, 0x80000000, (1 << 63) - 1)] == [-1] * 4
