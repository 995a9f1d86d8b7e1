"""What the operators for long conversations refuse, before any device work: the
C entry points' statuses and the Python wrappers' ValueErrors (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from nanoquant_amd.runtime import _native
from nanoquant_amd.runtime import shell_ops as ops

A = 4096  # an address: checks end before it is read


def _kv(**changes):
    kv = _native.PagedKv(A, A, A, A, 8, 2, 128, 16, 0, A, 4, A, A, 3)
    for name, value in changes.items():
        setattr(kv, name, value)
    return kv


def _shared(kv, *, q=A, dtype=0, tokens=3, q_heads=4, shared=0, scaling=0.1, out=A, out_dtype=0, lse=A, workspace=A, size=1 << 40):
    return _native.load().nq_shared_attention(q, dtype, tokens, q_heads, ctypes.byref(kv), shared, scaling, out, out_dtype, lse,
                                              workspace, size, None)


def _weigh(kv, *, q=A, dtype=0, tokens=3, q_heads=4, scaling=0.1, lse=A, first=0, weights=A, out=A):
    return _native.load().nq_attention_weights(q, dtype, tokens, q_heads, ctypes.byref(kv), scaling, lse, first, weights, out, None)


def _evict(kv, *, weights=A, into=A, budget=40, first=0, recent=0, table=2 * A, lens=2 * A, rows=A, workspace=A, size=1 << 40):
    return _native.load().nq_paged_evict(ctypes.byref(kv), weights, into, budget, first, recent, table, lens, rows, workspace, size,
                                         None)


CACHES = [
    ({"k_pages": None}, -1), ({"v_scales": None}, -1), ({"page_table": None}, -1), ({"context_lens": None}, -1),
    ({"head_dim": 96}, -3), ({"page_size": 8}, -3), ({"page_size": 48}, -3), ({"page_size": 256}, -3), ({"num_pages": 0}, -3),
    ({"kv_heads": 0}, -3), ({"batch": 0}, -3), ({"table_pages": 0}, -3), ({"table_pages": 1 << 28}, -3), ({"v_pages": A + 8}, -4),
]


@pytest.mark.parametrize("call", [_shared, _weigh, _evict])
@pytest.mark.parametrize("changes,status", CACHES)
def test_caches(call, changes, status):
    assert call(_kv(**changes)) == status


@pytest.mark.parametrize("call", [_shared, _weigh])
def test_calls_with_tokens_need_their_starts(call):
    assert call(_kv(query_starts=None)) == -1
    assert call(_kv(kv_heads=3)) == -3  # q heads no multiple


@pytest.mark.parametrize("arguments,status", [
    ({"q": None}, -1), ({"out": None}, -1), ({"scaling": 0.0}, -1), ({"scaling": float("nan")}, -1), ({"dtype": 4}, -2),
    ({"out_dtype": 3}, -2), ({"tokens": 0}, -3), ({"q_heads": 3}, -3), ({"shared": -1}, -3), ({"shared": 65}, -3), ({"q": A + 8}, -4),
    ({"out": A + 4}, -4),
])
def test_shared_attention(arguments, status):
    assert _shared(_kv(), **arguments) == status


def test_shared_attention_workspace():
    lib = _native.load()
    need = lib.nq_shared_attention_workspace_bytes(32, 32, 8, 2, 128, 64, 100, 5000)
    assert 0 < need <= 1 << 30
    kv = _kv(page_size=64, table_pages=100, batch=32)
    arguments = {"tokens": 32, "q_heads": 8, "shared": 5000}
    assert _shared(kv, size=need - 1, **arguments) == -5
    assert _shared(kv, workspace=None, **arguments) == -1
    assert _shared(kv, workspace=A + 4, **arguments) == -4
    assert lib.nq_shared_attention_workspace_bytes(32, 32, 8, 2, 96, 64, 100, 0) == -1


@pytest.mark.parametrize("tokens,batch,q_heads,kv,d,pages,shared", [
    (64, 64, 32, 8, 128, 512, 20000), (4096, 4096, 64, 64, 128, 2048, 100000), (100000, 100000, 4, 4, 256, 64, 4000),
    (16384, 256, 32, 8, 128, 2048, 100000), (1, 1, 8, 1, 64, 4096, 200000), (32768, 2, 32, 8, 128, 1024, 30000)])
def test_shared_attention_workspace_is_bounded(tokens, batch, q_heads, kv, d, pages, shared):
    assert 0 <= _native.load().nq_shared_attention_workspace_bytes(tokens, batch, q_heads, kv, d, 64, pages, shared) <= 1 << 30


@pytest.mark.parametrize("arguments,status", [
    ({"q": None}, -1), ({"lse": None}, -1), ({"weights": None}, -1), ({"out": None}, -1), ({"scaling": float("inf")}, -1),
    ({"dtype": 3}, -2), ({"tokens": 0}, -3), ({"q_heads": 0}, -3), ({"first": -1}, -3), ({"q": A + 4}, -4),
])
def test_attention_weights(arguments, status):
    assert _weigh(_kv(), **arguments) == status


@pytest.mark.parametrize("arguments,status", [
    ({"weights": None}, -1), ({"into": None}, -1), ({"table": None}, -1), ({"lens": None}, -1), ({"rows": None}, -1),
    ({"table": A}, -1), ({"lens": A}, -1),  # in place of what the call reads
    ({"budget": 0}, -3), ({"first": -1}, -3), ({"recent": -1}, -3), ({"first": 41}, -3), ({"first": 20, "recent": 21}, -3),
    ({"budget": 1 << 30}, -3),
])
def test_paged_evict(arguments, status):
    assert _evict(_kv(), **arguments) == status


def test_paged_evict_workspace():
    lib = _native.load()
    assert lib.nq_paged_evict_workspace_bytes(1, 2, 64, 100, 500) == 0
    assert lib.nq_paged_evict_workspace_bytes(1, 2, 64, 512, 500) == 0
    need = lib.nq_paged_evict_workspace_bytes(1, 2, 64, 1000, 500)
    assert need == 2 * 8 * 3 * 2048 * 4  # 64000 rows in parts of 8192
    kv = _kv(page_size=64, table_pages=1000, batch=1)
    assert _evict(kv, budget=500, size=need - 1) == -5
    assert _evict(kv, budget=500, workspace=None) == -1
    assert _evict(kv, budget=500, workspace=A + 4) == -4
    assert lib.nq_paged_evict_workspace_bytes(1 << 23, 4, 16, 10, 500) == -1  # no launch holds it


def _int4(*, x=A, dtype=0, tokens=2, packed=A, scales=A, scale_dtype=1, outs=100, ins=256, group=64, y=A, y_dtype=0, partials=None,
          workspace=A, size=1 << 40):
    return _native.load().nq_int4_projection(x, dtype, tokens, packed, scales, scale_dtype, None, outs, ins, group, y, y_dtype,
                                             partials, workspace, size, None)


@pytest.mark.parametrize("arguments,status", [
    ({"x": None}, -1), ({"packed": None}, -1), ({"scales": None}, -1), ({"y": None}, -1), ({"dtype": 3}, -2),
    ({"scale_dtype": 4}, -2), ({"y_dtype": 3}, -2), ({"tokens": 0}, -3), ({"tokens": 65536}, -3), ({"outs": 0}, -3),
    ({"ins": 0}, -3), ({"ins": 40}, -3), ({"ins": 1 << 25}, -3), ({"group": 16}, -3), ({"partials": A}, -3), ({"packed": A + 8}, -4),
    ({"tokens": 1, "partials": A + 4}, -4),
])
def test_int4_projection(arguments, status):
    assert _int4(**arguments) == status


def test_int4_projection_workspace():
    lib = _native.load()
    assert lib.nq_int4_projection_workspace_bytes(1, 151936, 4096, 128) == 0
    need = lib.nq_int4_projection_workspace_bytes(11, 2560, 10240, 64)
    assert need > 0 and need % (11 * 2560 * 4) == 0
    shape = {"tokens": 11, "outs": 2560, "ins": 10240}
    assert _int4(size=need - 1, **shape) == -5
    assert _int4(workspace=None, **shape) == -1
    assert _int4(workspace=A + 8, **shape) == -4
    assert lib.nq_int4_projection_partials(33) == 3 and lib.nq_int4_projection_partials(0) == -1


def test_append_at_positions_and_greedy_partials():
    lib = _native.load()
    assert lib.nq_paged_append_at(None, A, A, 0, 3, 4, A, A, 0, 1e-6, A, A, 64, ctypes.byref(_kv()), A, A, 0, None) == -1
    assert lib.nq_paged_append_at(A, A, A, 0, 3, 4, A, A, 0, 1e-6, A, A, 0, ctypes.byref(_kv()), A, A, 0, None) == -3
    assert lib.nq_greedy_select_partials(None, 4, A, None, 0, None, None, None) == -1
    assert lib.nq_greedy_select_partials(A, 0, A, None, 0, None, None, None) == -3
    assert lib.nq_greedy_select_partials(A, 4, A, A, 10, None, None, None) == -1


def test_wrappers_refuse_host_tensors_and_bad_geometry():
    cache = ops.paged_cache(4, 2, 16, 64, "cpu")
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    batch = {"page_table": table, "query_starts": torch.zeros(2, dtype=torch.int32), "context_lens": lens}
    q, weights = torch.zeros(1, 4, 64), torch.zeros(4, 2, 16)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_shared_attention(q, cache, shared_rows=0, scaling=0.1, **batch)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_attention_weights(q, cache, torch.zeros(1, 4), weights, scaling=0.1, **batch)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_paged_evict(cache, weights, page_table=table, context_lens=lens, into=table, budget=20)
    m = ops.int4_matrix(torch.randn(8, 64), 32)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_int4_projection(torch.zeros(1, 64), m)
    with pytest.raises(ValueError, match="input"):
        ops.launch_int4_projection(torch.zeros(1, 32), m)
    with pytest.raises(ValueError, match="scales"):
        ops.launch_int4_projection(torch.zeros(1, 64), m._replace(scales=torch.zeros(8, 7)))
    with pytest.raises(ValueError, match="zeros"):
        ops.launch_int4_projection(torch.zeros(1, 64), m._replace(zeros=torch.zeros(8, 2)))
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.launch_int4_projection(torch.zeros(1, 64), m._replace(packed=torch.zeros(8, 20, dtype=torch.uint8)))
    for weight, group in ((torch.zeros(4, 40), 32), (torch.zeros(4, 64), 48), (torch.zeros(64), 32)):
        with pytest.raises(ValueError, match="4-bit"):
            ops.int4_matrix(weight, group)
