"""How nq_paged_attention lays a call out (plan_attention in
nanoquant_amd/csrc/nq_paged_attention.hip), restated from its rules: which form of the
kernel runs, over how many slots and splits. tests/test_serving_plan.py holds it to
the library's workspace sizes and asks it which forms the GPU tests reach."""

from __future__ import annotations

from typing import NamedTuple

TILE, OWN_ROWS = 64, 128
FULL, SHORT, MEDIUM, VERY_LONG, SKEW, MOST_SPLITS = 256, 12, 64, 256, 96, 128
MOST_PARTIALS = 1 << 30


class Plan(NamedTuple):
    head_dim: int
    rows: int      # query rows of a slot
    shared: bool   # whether a slot's waves share its rows
    waves: int
    slots: int
    splits: int
    least: int     # cache tiles that a split takes at least

    def active(self, visible: int) -> int:
        """Splits of a sequence whose last token sees that many rows."""
        tiles = _up(visible, TILE)
        return 1 if self.splits == 1 else max(_up(tiles, max(_up(tiles, self.splits), self.least)), 1)

    @property
    def form(self) -> tuple[int, int, bool, int, bool]:
        """What decides which code runs: all but the counts, and whether there is a join."""
        return self.head_dim, self.rows, self.shared, self.waves, self.splits > 1


def _up(a: int, b: int) -> int:
    return -(-a // b)


def plan(tokens: int, batch: int, q_heads: int, kv_heads: int, head_dim: int, cache_rows: int) -> Plan:
    rows = tokens * (q_heads // kv_heads)
    mean, tiles, narrow = _up(rows, batch), _up(cache_rows, TILE), head_dim < 256

    def work(of: int) -> int:
        return batch * _up(mean, of) * kv_heads

    shared = not narrow or rows <= 64 * batch or (
        work(OWN_ROWS) < (1024 if head_dim == 64 else 352) and (mean <= OWN_ROWS or tiles < VERY_LONG))
    if not shared:
        slot = OWN_ROWS
    else:
        slot = 16 if rows <= 16 * batch or (work(16) < FULL and tiles <= (MEDIUM if narrow else SHORT)) else 32
    slots = rows // slot + batch
    units = slots * kv_heads
    full = units >= FULL
    least = 4 if shared and units * ((tiles + 7) // 8) < 512 else 8
    waves = 8 if shared and narrow and slot == 16 and not full and tiles <= SHORT else 4
    target = 256 if not narrow and slot == 32 else 512
    if shared and (waves == 8 or (full and narrow)):
        target = 0
    splits = target // work(slot)
    alone = _up(mean, slot) * kv_heads
    if full and shared and batch > 1 and alone < FULL:
        splits = max(splits, min(tiles // SKEW, 16, 512 // alone))
    splits = min(splits, _up(tiles, least), MOST_SPLITS, MOST_PARTIALS // (units * slot * (head_dim + 2) * 4))
    return Plan(head_dim, slot, shared, waves, slots, max(splits, 1), least)


# (head_dim, rows, shared, waves, joined): all that calls can reach.
FORMS = {(d, *form) for d in (64, 128) for form in (
    (16, True, 8, False), (16, True, 4, False), (16, True, 4, True), (32, True, 4, False), (32, True, 4, True),
    (128, False, 4, False), (128, False, 4, True))} | {
    (256, rows, True, 4, joined) for rows in (16, 32) for joined in (False, True)}


def workspace_bytes(p: Plan, kv_heads: int) -> int:
    return 0 if p.splits == 1 else p.slots * p.splits * kv_heads * p.rows * (p.head_dim + 2) * 4
