"""The layout of paged attention calls, on the CPU: the restated plan is the library's,
and a call's workspace is bounded."""

from __future__ import annotations

import ctypes
import random

import pytest
from serving_plan import FORMS, MOST_PARTIALS, plan, workspace_bytes
from test_gpu_serving_forms import ATTENTIONS, DTYPES

from nanoquant_amd.runtime import _native

GEOMETRIES = [(32, 8, 128), (16, 8, 128), (8, 1, 128), (32, 32, 128), (64, 64, 128), (14, 2, 64), (4, 4, 64), (34, 2, 64),
              (16, 4, 256), (8, 8, 256), (64, 8, 256)]


def _bytes(tokens, batch, q_heads, kv_heads, head_dim, page, entries):
    return _native.load().nq_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, head_dim, page, entries)


def test_the_restated_plan_is_the_librarys():
    rng = random.Random(5)
    forms = set()
    for _ in range(20000):
        q_heads, kv, d = rng.choice(GEOMETRIES)
        batch = round(2 ** rng.uniform(0, 10))
        tokens = min(round(batch * 2 ** rng.uniform(-1, 13)) + 1, 0x3FFFFFFF // q_heads)
        page = rng.choice([16, 32, 64, 128])
        entries = round(2 ** rng.uniform(0, 20 - (page.bit_length() - 1)))
        p = plan(tokens, batch, q_heads, kv, d, page * entries)
        got = _bytes(tokens, batch, q_heads, kv, d, page, entries)
        assert got == -1 or got == workspace_bytes(p, kv), (tokens, batch, q_heads, kv, d, page, entries, p)
        forms.add(p.form)
    assert forms == FORMS


def test_the_gpu_tests_reach_every_form_with_every_type():
    forms = set()
    for lengths, q_heads, kv, d, page, extra in ATTENTIONS:
        width = max(-(-(c + n) // page) for c, n in lengths) + extra
        p = plan(sum(n for _, n in lengths) + 3, len(lengths), q_heads, kv, d, width * page)
        active = {p.active(c + n) for c, n in lengths}
        assert p.splits == 1 or (max(active) > 1 and min(active) == 1), "some sequences are split, others not"
        forms.add(p.form)
    assert forms == FORMS
    assert {q for q, _ in DTYPES} == {out for _, out in DTYPES} and len(set(DTYPES)) == 9


@pytest.mark.parametrize("tokens,batch,q_heads,kv,d,rows,most", [
    (32768, 1, 16, 4, 256, 131072, 0),             # one long prompt of 256-wide heads: its slots fill the chip
    (32768, 1, 16, 4, 256, 32768, 0),
    (32768, 1, 32, 8, 128, 131072, 0),
    (8192, 4, 16, 4, 256, 131072, 0),              # each of four prompts does
    (4096, 256, 32, 8, 128, 131072, MOST_PARTIALS),  # 16 tokens each
    (512, 512, 32, 8, 128, 131072, MOST_PARTIALS),   # a decode step
    (4096, 4096, 64, 64, 128, 1 << 20, MOST_PARTIALS),
])
def test_workspace_of_calls_that_fill_the_chip(tokens, batch, q_heads, kv, d, rows, most):
    assert 0 <= _bytes(tokens, batch, q_heads, kv, d, 64, rows // 64) <= most


def test_no_workspace_is_larger_than_the_bound():
    rng = random.Random(6)
    for _ in range(20000):
        q_heads, kv, d = rng.choice(GEOMETRIES)
        batch = round(2 ** rng.uniform(0, 16))
        tokens = min(round(2 ** rng.uniform(0, 22)), 0x3FFFFFFF // q_heads)
        assert _bytes(tokens, batch, q_heads, kv, d, 64, round(2 ** rng.uniform(0, 16))) <= MOST_PARTIALS


# -- launches: at most 2^32 - 1 threads --------------------------------------------

A = 4096  # an address: checks end before it is read


def _kv(**changes):
    kv = _native.PagedKv(A, A, A, A, 8, 2, 128, 16, 0, A, 4, A, A, 3)
    for name, value in changes.items():
        setattr(kv, name, value)
    return kv


@pytest.mark.parametrize("changes,tokens,q_heads", [
    ({"batch": 1 << 21, "page_size": 128, "head_dim": 64}, 3, 4),      # slots of pages, 1024 threads each
    ({"batch": 1 << 23, "page_size": 16}, 3, 4),                       # 128 threads each
    ({"batch": 1, "page_size": 16}, 0xFFFFFF, 64),                     # groups of q heads
])
def test_append_refuses_what_no_launch_holds(changes, tokens, q_heads):
    status = _native.load().nq_paged_append(A, A, A, 0, tokens, q_heads, None, None, 0, 1e-6, A, A, 64,
                                            ctypes.byref(_kv(**changes)), A, 0, None)
    assert status == -3


@pytest.mark.parametrize("changes,tokens,q_heads", [
    ({"batch": 1 << 23}, 3, 4),
    ({"batch": 1 << 23, "head_dim": 256}, 3, 4),
    ({"batch": 1 << 18, "kv_heads": 64}, 3, 64),
])
def test_attention_refuses_what_no_launch_holds(changes, tokens, q_heads):
    kv = _kv(**changes)
    assert _bytes(tokens, kv.batch, q_heads, kv.kv_heads, kv.head_dim, 16, 4) == -1
    status = _native.load().nq_paged_attention(A, 0, tokens, q_heads, ctypes.byref(kv), 0.1, A, 0, A, 1 << 40, None)
    assert status == -3


def test_token_logprobs_refuse_what_no_launch_holds():
    lib = _native.load()
    assert lib.nq_token_logprobs_workspace_bytes(8388607, 64, 1) > 0  # 512 threads to a row's join
    assert lib.nq_token_logprobs_workspace_bytes(0xFFFFFF, 64, 0) == 0  # 256, and no join
    for rows in (8388608, 0xFFFFFF):
        assert lib.nq_token_logprobs_workspace_bytes(rows, 64, 1) == -1
        assert lib.nq_token_logprobs(A, 0, rows, 64, 64, A, 1, A, A, A, A, A, 1 << 50, None) == -3
