"""How nq_int4_projection lays a call out (plan_int4 in nanoquant_amd/csrc/nq_int4.hip),
restated from its rules. tests/test_int4_plan.py holds it to the library's workspace sizes
and asks it which forms the GPU tests reach."""

from __future__ import annotations

from typing import NamedTuple

CHUNK, MOST_WAVES, WALKERS, MOST_SLICES = 128, 2048, 768, 16
BUDGET = {3: 60 * 1024, 4: 78 * 1024}  # by digits
AT_ONCE = 4


def _up(a: int, b: int) -> int:
    return -(-a // b)


def lds_bytes(waves: int, tokens: int, digits: int, blocks: int, groups: int, stage: int) -> int:
    each_wave = 16 * 16 * 4 + 16 * 17 + AT_ONCE * groups * 20
    return 64 + tokens * digits * (stage * CHUNK + 64) + stage * blocks * 16 * 8 + waves * each_wave * 4


class Plan(NamedTuple):
    digits: int
    waves: int
    blocks: int
    passes: int
    share: int    # waves that share a tile of 16 rows
    slices: int
    slice: int    # chunks of one
    stage: int    # chunks whose digits LDS holds at once
    walkers: int  # workgroups of a pass and slice
    tiles: int
    lds: int

    @property
    def form(self) -> tuple[int, int, int, int, bool, bool, bool]:
        """What decides which code runs: digits, blocks, waves, share, whether there are slices, several
        stages, several tiles to a workgroup."""
        return (self.digits, self.blocks, self.waves, self.share, self.slices > 1, self.stage < self.slice,
                self.walkers * (self.waves // self.share) < self.tiles)


def plan(tokens: int, outs: int, ins: int, group: int, digits: int) -> Plan:
    groups = CHUNK // group
    each = 16 // groups // digits
    wanted, chunks, tiles = _up(tokens, each), _up(ins, CHUNK), _up(outs, 16)
    at_once = _up(wanted, _up(wanted, 6))
    blocks = at_once if at_once <= 3 else 6
    passes = _up(wanted, blocks)
    held = min(tokens, blocks * each)
    fixed = lds_bytes(4, held, digits, blocks, groups, 0)
    most = min(chunks, max(1, (BUDGET[digits] - min(fixed, BUDGET[digits])) // (lds_bytes(4, held, digits, blocks, groups, 1) - fixed)))
    work = tiles * passes
    slices, waves, share = 1, 4, 1 if work >= MOST_WAVES else 4
    if most < chunks and work < MOST_WAVES:
        share, waves = 1, 8 if blocks == 6 else 4
        slices = min(MOST_SLICES, chunks, max(_up(MOST_WAVES, work), 1))
    length = _up(chunks, slices)
    slices = _up(chunks, length)
    stages = _up(length, most)
    stage = _up(length, stages)
    all_ = _up(tiles, waves // share)
    walkers = min(all_, max(1, WALKERS // (passes * slices))) if stages == 1 else all_
    return Plan(digits, waves, blocks, passes, share, slices, length, stage, walkers, tiles,
                lds_bytes(waves, held, digits, blocks, groups, stage))


def workspace_bytes(tokens: int, outs: int, ins: int, group: int) -> int:
    """Whatever the type of x."""
    plans = [plan(tokens, outs, ins, group, digits) for digits in (3, 4)]
    return max(0 if p.slices == 1 else p.slices * tokens * outs * 4 for p in plans)
