"""What the serving operators refuse, before any device work: the Python
wrappers' ValueErrors and the C entry points' statuses (no GPU needed)."""

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


def _append(kv, *, q=A, dtype=0, tokens=3, q_heads=4, q_norm=A, k_norm=A, norm_dtype=0, eps=1e-6, rope=64, q_out=A, q_out_dtype=0):
    return _native.load().nq_paged_append(q, A, A, dtype, tokens, q_heads, q_norm, k_norm, norm_dtype, eps, A, A, rope,
                                          ctypes.byref(kv), q_out, q_out_dtype, None)


def _attend(kv, *, q=A, dtype=0, tokens=3, q_heads=4, scaling=0.1, out=A, out_dtype=0, workspace=A, size=1 << 40):
    return _native.load().nq_paged_attention(q, dtype, tokens, q_heads, ctypes.byref(kv), scaling, out, out_dtype, workspace,
                                             size, None)


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("changes,status", [
    ({"k_pages": None}, -1), ({"v_scales": None}, -1), ({"page_table": None}, -1), ({"query_starts": None}, -1),
    ({"context_lens": None}, -1), ({"head_dim": 96}, -3), ({"page_size": 8}, -3), ({"page_size": 48}, -3),
    ({"page_size": 256}, -3), ({"num_pages": 0}, -3), ({"kv_heads": 0}, -3), ({"kv_heads": 3}, -3), ({"batch": 0}, -3),
    ({"table_pages": 0}, -3), ({"table_pages": 1 << 28}, -3), ({"table_pages": 1 << 26}, -3), ({"v_pages": A + 8}, -4),
])
def test_cache_and_batch(call, changes, status):
    assert call(_kv(**changes)) == status


@pytest.mark.parametrize("arguments,status", [
    ({"q": None}, -1), ({"q_norm": None}, -1), ({"q_out": None}, -1), ({"eps": -1.0}, -1), ({"eps": float("nan")}, -1),
    ({"dtype": 3}, -2), ({"norm_dtype": 4}, -2), ({"q_out_dtype": 3}, -2), ({"tokens": 0}, -3), ({"tokens": 1 << 24}, -3),
    ({"q_heads": 5}, -3), ({"rope": 0}, -3),
])
def test_append(arguments, status):
    assert _append(_kv(), **arguments) == status


@pytest.mark.parametrize("arguments,status", [
    ({"q": None}, -1), ({"out": None}, -1), ({"scaling": 0.0}, -1), ({"scaling": float("inf")}, -1),
    ({"scaling": float("nan")}, -1), ({"dtype": 4}, -2), ({"out_dtype": 3}, -2), ({"tokens": 0}, -3), ({"q_heads": 0}, -3),
    ({"q_heads": 3}, -3), ({"q": A + 8}, -4), ({"out": A + 4}, -4),
])
def test_attention(arguments, status):
    assert _attend(_kv(), **arguments) == status


def test_attention_workspace():
    lib = _native.load()
    need = lib.nq_paged_attention_workspace_bytes(1, 1, 8, 2, 128, 64, 2000)
    assert need > 0
    kv = _kv(page_size=64, table_pages=2000, batch=1)
    assert _attend(kv, tokens=1, q_heads=8, size=need - 1) == -5
    assert _attend(kv, tokens=1, q_heads=8, workspace=None) == -1
    assert lib.nq_paged_attention_workspace_bytes(1, 1, 8, 2, 96, 64, 10) == -1
    assert lib.nq_paged_attention_workspace_bytes(0, 1, 8, 2, 128, 64, 10) == -1
    assert lib.nq_paged_attention_workspace_bytes(1, 1, 8, 3, 128, 64, 10) == -1


@pytest.mark.parametrize("arguments,status", [
    ({"logits": None}, -1), ({"top_ids": None}, -1), ({"workspace": None}, -1), ({"dtype": 3}, -2), ({"rows": 0}, -3),
    ({"vocab": 0}, -3), ({"stride": 8999}, -3), ({"top": 33}, -3), ({"top": -1}, -3), ({"vocab": 4, "stride": 4, "top": 5}, -3),
    ({"vocab": 1 << 31, "stride": 1 << 31}, -3), ({"logits": A + 2}, -4), ({"size": 8}, -5),
])
def test_token_logprobs(arguments, status):
    a = {"logits": A, "dtype": 0, "rows": 2, "vocab": 9000, "stride": 9000, "top": 5, "top_ids": A, "workspace": A, "size": 1 << 30}
    a.update(arguments)
    assert _native.load().nq_token_logprobs(a["logits"], a["dtype"], a["rows"], a["vocab"], a["stride"], A, a["top"], A, A,
                                            a["top_ids"], A, a["workspace"], a["size"], None) == status


def test_wrappers_refuse_host_tensors_and_bad_geometry():
    cache = ops.paged_cache(4, 2, 16, 64, "cpu")
    assert cache.k.shape == (4, 2, 16, 64) and cache.v.shape == (4, 2, 64, 16) and cache.k_scales.shape == (4, 2)
    batch = {"page_table": torch.zeros(1, 2, dtype=torch.int32), "query_starts": torch.zeros(2, dtype=torch.int32),
             "context_lens": torch.zeros(1, dtype=torch.int32)}
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_paged_attention(torch.zeros(1, 4, 64), cache, scaling=0.1, **batch)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_paged_append(torch.zeros(1, 256), torch.zeros(1, 128), torch.zeros(1, 128), cache, q_heads=4, q_norm=None,
                                k_norm=None, eps=0.0, cos=torch.zeros(8, 32), sin=torch.zeros(8, 32), **batch)
    with pytest.raises(ValueError, match="CUDA/HIP"):
        ops.launch_token_logprobs(torch.zeros(1, 10), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="alternatives"):
        ops.launch_token_logprobs(torch.zeros(1, 10), torch.zeros(1, dtype=torch.int64), top=11)
    with pytest.raises(ValueError, match="adjacent"):
        ops.launch_token_logprobs(torch.zeros(10, 4).T, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="adjacent"):
        ops.launch_token_logprobs(torch.zeros(1, 10).expand(3, 10), torch.zeros(3, dtype=torch.int64))
    for geometry in ((0, 1, 16, 64), (1, 1, 24, 64), (1, 1, 16, 80), (1, 0, 16, 64)):
        with pytest.raises(ValueError, match="geometry"):
            ops.paged_cache(*geometry, "cpu")


@pytest.mark.parametrize("tokens,batch", [(1, 2), (3, 70), (64, 65), (1, 100000)])
def test_a_batch_may_have_more_sequences_than_tokens(tokens, batch):
    for head_dim in (64, 128, 256):
        for table_pages in (1, 100, 4000):
            assert _native.load().nq_paged_attention_workspace_bytes(tokens, batch, 4, 4, head_dim, 64, table_pages) >= 0
