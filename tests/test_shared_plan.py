"""How nq_shared_attention splits the rows behind the shared ones, by its workspace (no GPU needed)."""

from __future__ import annotations

import random

import pytest

from nanoquant_amd.runtime import _native

BOUND = 1 << 30


def _up(a: int, b: int) -> int:
    return -(-a // b)


def splits(tokens, batch, q_heads, kv_heads, head_dim, page, table_pages, shared):
    """(splits of a sequence's own rows, of the shared rows) of a call that shares rows, restated
    from plan_shared in nanoquant_amd/csrc/nq_shared_attention.hip; the workspace that they take."""
    rows, grain = tokens * (q_heads // kv_heads), max(page, 64)
    skip = shared // grain * grain
    tiles, own_tiles, mean = skip // 64, _up(table_pages * page - skip, 64), _up(rows, batch)
    assert tiles and mean <= 64 and batch > 1
    slot = 16 if rows <= 16 else 32
    blocks, slots = _up(rows, slot), rows // slot + batch
    both = max(1, min(256 // (blocks * kv_heads), _up(tiles, 4), 64))
    both = _up(tiles, _up(tiles, both))
    skew = min(own_tiles // 96, 16, 512 // (_up(mean, slot) * kv_heads))
    each = kv_heads * slot * (head_dim + 2) * 4
    own = max(1, min(max(512 // (slots * kv_heads), skew), _up(own_tiles, 4), 64, (BOUND // each - blocks * both) // slots))
    return own, both, (slots * own + blocks * both) * each


def _bytes(*call):
    return _native.load().nq_shared_attention_workspace_bytes(*call)


@pytest.mark.parametrize("batch,heads,kv,d,own,expected", [
    (32, 32, 8, 128, 700, 1), (32, 32, 8, 128, 6000, 1), (32, 32, 8, 128, 20000, 3), (32, 32, 8, 128, 100000, 16),
    (16, 32, 8, 128, 100000, 16), (2, 32, 8, 128, 100000, 32), (128, 16, 4, 256, 50000, 8),
])
def test_long_histories_behind_shared_rows_are_split(batch, heads, kv, d, own, expected):
    call = (batch, batch, heads, kv, d, 64, (4096 + own + 63) // 64, 4096)
    got, _, need = splits(*call)
    assert got == expected and _bytes(*call) == need


def test_the_restated_splits_are_the_librarys_and_bounded():
    rng = random.Random(21)
    seen = 0
    for _ in range(20000):
        heads, kv, d = rng.choice([(32, 8, 128), (8, 1, 128), (14, 2, 64), (4, 4, 64), (16, 4, 256), (64, 64, 128)])
        batch = round(2 ** rng.uniform(1, 12))
        tokens = round(batch * 2 ** rng.uniform(-1, 3))
        page, shared = rng.choice([16, 64, 128]), round(2 ** rng.uniform(7, 15))
        call = (tokens, batch, heads, kv, d, page, _up(shared, page) + round(2 ** rng.uniform(0, 12)), shared)
        if tokens * (heads // kv) > 64 * batch:
            continue
        got = _bytes(*call)
        assert got <= BOUND
        need = splits(*call)[2]
        if got >= 0 and need <= BOUND:
            assert got == need, call
            seen += 1
    assert seen > 10000
