"""Launch wrappers of the decoder-shell kernels (``include/nqamd_shell.h``).

Each function validates its tensors the way the reference's launch helpers do
(src/nanoquant/runtime/cuda_kernels.py:493-544,644-815: ``ValueError`` for a
wrong dtype, device, geometry or layout), then enqueues the HIP kernel on the
current stream. Outputs and workspaces come from torch's caching allocator
unless the caller passes them, so every call can be captured in a HIP graph.
Token positions are device int32 tensors (``position[0]`` = cache row of the
first token) so a captured step replays at every position.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from nanoquant_amd.runtime import _native

_FLOAT = (torch.float32, torch.float16, torch.bfloat16)


def _check_device(name: str, device: torch.device, *tensors: torch.Tensor | None) -> None:
    if device.type != "cuda":
        raise ValueError(f"{name} requires CUDA/HIP tensors")
    index = device.index
    for tensor in tensors:
        if tensor is None:
            continue
        if tensor.get_device() != index:  # -1 on the CPU; half the time of comparing devices
            raise ValueError(f"{name} inputs must share one device")
        if not tensor.is_contiguous():
            raise ValueError(f"{name} requires contiguous tensors")


def _check_float(name: str, *tensors: torch.Tensor | None) -> None:
    for tensor in tensors:
        if tensor is not None and tensor.dtype not in _FLOAT:
            raise ValueError(f"{name} tensor dtype {tensor.dtype} is not F32/F16/BF16")


def _position(name: str, position: torch.Tensor, device: torch.device) -> None:
    if position.dtype != torch.int32 or position.numel() < 1 or position.device != device:
        raise ValueError(f"{name} position must be a device int32 tensor")


def _stream(device: torch.device) -> int:
    return _native.current_stream_handle(device)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def launch_embedding(
    ids: torch.Tensor, table: torch.Tensor, *, scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """fp32 rows ``table[ids]`` (``* scale``). Mirrors ``launch_bfloat16_embedding``
    (src/nanoquant/runtime/cuda_kernels.py:644-681) for any float table. With
    ``slots`` (fp32 ``[*ids, hidden / 16]``) it also writes each row's sums of
    squares per 16 columns, the statistics a ``rmsnorm`` input kind of
    ``linear_batch_fused`` reads."""

    if ids.dtype != torch.int64 or table.ndim != 2:
        raise ValueError("embedding requires int64 ids and a 2-D table")
    _check_float("embedding", table)
    _check_device("embedding", ids.device, ids, table, scale, out)
    if scale is not None and (scale.dtype != torch.float32 or scale.numel() != 1):
        raise ValueError("embedding scale must be one fp32 value")
    vocab, hidden = table.shape
    if out is None:
        out = torch.empty((*ids.shape, hidden), dtype=torch.float32, device=ids.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != (*ids.shape, hidden):
        raise ValueError("embedding output must be fp32 [*ids, hidden]")
    if slots is None:
        status = _native.load().nq_embedding(
            ids.data_ptr(), ids.numel(), table.data_ptr(), _native.dtype_code(table.dtype), vocab, hidden,
            _ptr(scale), out.data_ptr(), _stream(ids.device),
        )
        _native.check("nq_embedding", status)
        return out
    _check_device("embedding", ids.device, slots)
    if hidden % 16 or slots.dtype != torch.float32 or tuple(slots.shape) != (*ids.shape, hidden // 16) \
            or not slots.is_contiguous():
        raise ValueError("embedding slots must be contiguous fp32 [*ids, hidden / 16] (hidden % 16 == 0)")
    status = _native.load().nq_embedding_slots(
        ids.data_ptr(), ids.numel(), table.data_ptr(), _native.dtype_code(table.dtype), vocab, hidden,
        _ptr(scale), out.data_ptr(), slots.data_ptr(), _stream(ids.device),
    )
    _native.check("nq_embedding_slots", status)
    return out


def launch_add_rmsnorm(
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    *,
    delta: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``residual += delta`` (in place, optional), then
    ``out = weight * (residual * rsqrt(mean(residual^2) + eps))`` per row."""

    if residual.dtype != torch.float32:
        raise ValueError("rmsnorm residual must be fp32")
    _check_float("rmsnorm", weight, delta)
    _check_device("rmsnorm", residual.device, residual, weight, delta, out)
    hidden = residual.shape[-1]
    if weight.numel() != hidden or (delta is not None and delta.shape != residual.shape):
        raise ValueError("rmsnorm geometry is incompatible")
    if out is None:
        out = torch.empty(residual.shape, dtype=out_dtype, device=residual.device)
    elif out.shape != residual.shape or out.dtype not in _FLOAT:
        raise ValueError("rmsnorm output geometry is incompatible")
    rows = residual.numel() // hidden
    status = _native.load().nq_add_rmsnorm(
        residual.data_ptr(), _ptr(delta), _native.dtype_code(delta.dtype) if delta is not None else 0,
        weight.data_ptr(), _native.dtype_code(weight.dtype), float(eps), rows, hidden, out.data_ptr(),
        _native.dtype_code(out.dtype), _stream(residual.device),
    )
    _native.check("nq_add_rmsnorm", status)
    return out


def launch_qk_norm_rope_cache(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    q_heads: int,
    kv_heads: int,
    head_dim: int,
    q_norm: torch.Tensor | None,
    k_norm: torch.Tensor | None,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    position: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Per-head RMSNorm + RoPE of q and k, KV-cache append; returns the rotated q
    (fp32 ``[tokens, q_heads, head_dim]``). Mirrors ``launch_decode_rope`` and
    ``launch_cache_prefix_update`` (src/nanoquant/runtime/cuda_kernels.py:715-815)."""

    device = q.device
    tokens = q.numel() // (q_heads * head_dim)
    for name, t, heads in (("q", q, q_heads), ("k", k, kv_heads), ("v", v, kv_heads)):
        if t.dtype != torch.float32 or t.numel() != tokens * heads * head_dim:
            raise ValueError(f"{name} must be fp32 [tokens, {heads} * {head_dim}]")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm must be given together")
    if q_norm is not None and (q_norm.numel() != head_dim or k_norm.numel() != head_dim or q_norm.dtype != k_norm.dtype):
        raise ValueError("q/k norm weights must be [head_dim] of one dtype")
    _check_float("qk norm", q_norm, k_norm, k_cache)
    _check_device("qk rope", device, q, k, v, q_norm, k_norm, cos, sin, position, k_cache, v_cache, q_out)
    _position("qk rope", position, device)
    max_positions = k_cache.shape[-2]
    expected = (kv_heads, max_positions, head_dim)
    if tuple(k_cache.shape) != expected or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("KV cache must be [kv_heads, max_positions, head_dim] for K and V")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or tuple(cos.shape) != (max_positions, head_dim // 2) or sin.shape != cos.shape:
        raise ValueError("RoPE tables must be fp32 [max_positions, head_dim / 2]")
    if q_out is None:
        q_out = torch.empty((tokens, q_heads, head_dim), dtype=torch.float32, device=device)
    elif q_out.dtype != torch.float32 or q_out.numel() != tokens * q_heads * head_dim:
        raise ValueError("q_out must be fp32 [tokens, q_heads, head_dim]")
    status = _native.load().nq_qk_norm_rope_cache(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), tokens, q_heads, kv_heads, head_dim, _ptr(q_norm),
        _ptr(k_norm), _native.dtype_code(q_norm.dtype) if q_norm is not None else 0, float(eps),
        cos.data_ptr(), sin.data_ptr(), position.data_ptr(), max_positions, q_out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), _native.dtype_code(k_cache.dtype), _stream(device),
    )
    _native.check("nq_qk_norm_rope_cache", status)
    return q_out


def attention_workspace_bytes(tokens: int, q_heads: int, head_dim: int, max_positions: int) -> int:
    return int(_native.load().nq_attention_workspace_bytes(tokens, q_heads, head_dim, max_positions))


def launch_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    position: torch.Tensor,
    scaling: float,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal grouped-query attention of ``q`` (fp32 ``[tokens, q_heads, D]``) over
    cache rows ``[0, position + t]``. Mirrors ``launch_decode_attention``
    (src/nanoquant/runtime/cuda_kernels.py:493-544) for any GQA geometry."""

    device = q.device
    if q.dtype != torch.float32 or q.ndim != 3:
        raise ValueError("attention query must be fp32 [tokens, q_heads, head_dim]")
    tokens, q_heads, head_dim = q.shape
    kv_heads, max_positions = k_cache.shape[0], k_cache.shape[1]
    if k_cache.ndim != 3 or k_cache.shape[2] != head_dim or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("attention cache geometry is incompatible")
    _check_float("attention", k_cache)
    _check_device("attention", device, q, k_cache, v_cache, position, out, workspace)
    _position("attention", position, device)
    if out is None:
        out = torch.empty((tokens, q_heads * head_dim), dtype=out_dtype, device=device)
    elif out.numel() != tokens * q_heads * head_dim or out.dtype not in _FLOAT:
        raise ValueError("attention output geometry is incompatible")
    need = attention_workspace_bytes(tokens, q_heads, head_dim, max_positions)
    if need < 0:
        raise ValueError("attention geometry was rejected")
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = _native.load().nq_attention(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _native.dtype_code(k_cache.dtype), tokens, q_heads,
        kv_heads, head_dim, position.data_ptr(), max_positions, float(scaling), out.data_ptr(),
        _native.dtype_code(out.dtype), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream(device),
    )
    _native.check("nq_attention", status)
    return out


def decode_attention_workspace_bytes(q_heads: int, kv_heads: int, head_dim: int, cache_dtype: torch.dtype,
                                     max_positions: int) -> int:
    return int(_native.load().nq_decode_attention_workspace_bytes(
        q_heads, kv_heads, head_dim, _native.dtype_code(cache_dtype), max_positions))


def _decode_attention_checks(q, k, v, q_heads, kv_heads, head_dim, q_norm, k_norm, cos, sin, position, k_cache,
                             v_cache, out, workspace) -> tuple[int, torch.Tensor]:
    """Validate one-token attention operands; returns (max_positions, workspace)."""

    device = q.device
    for name, t, heads in (("q", q, q_heads), ("k", k, kv_heads), ("v", v, kv_heads)):
        if t.dtype != torch.float32 or t.numel() != heads * head_dim:
            raise ValueError(f"{name} must be fp32 [{heads} * {head_dim}] (one token)")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm must be given together")
    if q_norm is not None and (q_norm.numel() != head_dim or k_norm.numel() != head_dim or q_norm.dtype != k_norm.dtype):
        raise ValueError("q/k norm weights must be [head_dim] of one dtype")
    _check_float("decode attention", q_norm, k_norm, k_cache)
    _check_device("decode attention", device, q, k, v, q_norm, k_norm, cos, sin, position, k_cache, v_cache, out,
                  workspace)
    _position("decode attention", position, device)
    max_positions = k_cache.shape[-2]
    if tuple(k_cache.shape) != (kv_heads, max_positions, head_dim) or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("KV cache must be [kv_heads, max_positions, head_dim] for K and V")
    if cos.dtype != torch.float32 or tuple(cos.shape) != (max_positions, head_dim // 2) or sin.shape != cos.shape:
        raise ValueError("RoPE tables must be fp32 [max_positions, head_dim / 2]")
    need = decode_attention_workspace_bytes(q_heads, kv_heads, head_dim, k_cache.dtype, max_positions)
    if need < 0:
        raise ValueError("decode attention geometry was rejected")
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    return max_positions, workspace


def launch_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    q_heads: int,
    kv_heads: int,
    head_dim: int,
    q_norm: torch.Tensor | None,
    k_norm: torch.Tensor | None,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    position: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scaling: float,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """One decode token: q/k RMSNorm + RoPE, KV append at ``position`` and
    causal GQA attention, fused into one kernel where the geometry allows."""

    device = q.device
    max_positions, workspace = _decode_attention_checks(q, k, v, q_heads, kv_heads, head_dim, q_norm, k_norm, cos,
                                                        sin, position, k_cache, v_cache, out, workspace)
    if out is None:
        out = torch.empty(q_heads * head_dim, dtype=out_dtype, device=device)
    elif out.numel() != q_heads * head_dim or out.dtype not in _FLOAT:
        raise ValueError("decode attention output geometry is incompatible")
    status = _native.load().nq_decode_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_heads, kv_heads, head_dim, _ptr(q_norm), _ptr(k_norm),
        _native.dtype_code(q_norm.dtype) if q_norm is not None else 0, float(eps), cos.data_ptr(), sin.data_ptr(),
        position.data_ptr(), max_positions, k_cache.data_ptr(), v_cache.data_ptr(),
        _native.dtype_code(k_cache.dtype), float(scaling), out.data_ptr(), _native.dtype_code(out.dtype),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_decode_attention", status)
    return out


def decode_attention_partials_supported(q_heads: int, kv_heads: int, head_dim: int, cache_dtype: torch.dtype) -> bool:
    """Whether one-token attention runs as pass 1 + merge (the form whose
    partials ``launch_decode_attention_partials`` leaves in the workspace):
    head_dim * cache element bytes <= 256 and 1, 2, 4 or 8 q heads per kv head."""

    if q_heads <= 0 or kv_heads <= 0 or q_heads % kv_heads:
        return False
    element = 4 if cache_dtype == torch.float32 else 2
    return head_dim in (64, 128, 256) and head_dim * element <= 256 and q_heads // kv_heads in (1, 2, 4, 8)


def launch_decode_attention_partials(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    q_heads: int,
    kv_heads: int,
    head_dim: int,
    q_norm: torch.Tensor | None,
    k_norm: torch.Tensor | None,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    position: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scaling: float,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Pass 1 of ``launch_decode_attention`` alone (nq_decode_attention_partials):
    returns the workspace, which holds every cache block's partial (max, sum,
    acc) for a projection with ``input_kind="attention"`` to merge."""

    device = q.device
    max_positions, workspace = _decode_attention_checks(q, k, v, q_heads, kv_heads, head_dim, q_norm, k_norm, cos,
                                                        sin, position, k_cache, v_cache, None, workspace)
    status = _native.load().nq_decode_attention_partials(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_heads, kv_heads, head_dim, _ptr(q_norm), _ptr(k_norm),
        _native.dtype_code(q_norm.dtype) if q_norm is not None else 0, float(eps), cos.data_ptr(), sin.data_ptr(),
        position.data_ptr(), max_positions, k_cache.data_ptr(), v_cache.data_ptr(),
        _native.dtype_code(k_cache.dtype), float(scaling),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_decode_attention_partials", status)
    return workspace


def launch_silu_mul(
    gate: torch.Tensor, up: torch.Tensor, *, out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16
) -> torch.Tensor:
    """``silu(gate) * up`` (fp32 inputs)."""

    if gate.dtype != torch.float32 or up.dtype != torch.float32 or gate.shape != up.shape:
        raise ValueError("silu_mul requires fp32 gate and up of one shape")
    _check_device("silu_mul", gate.device, gate, up, out)
    if out is None:
        out = torch.empty(gate.shape, dtype=out_dtype, device=gate.device)
    elif out.shape != gate.shape or out.dtype not in _FLOAT:
        raise ValueError("silu_mul output geometry is incompatible")
    status = _native.load().nq_silu_mul(
        gate.data_ptr(), up.data_ptr(), gate.numel(), out.data_ptr(), _native.dtype_code(out.dtype),
        _stream(gate.device),
    )
    _native.check("nq_silu_mul", status)
    return out


def output_projection_workspace_bytes(vocab: int, hidden: int) -> int:
    return int(_native.load().nq_output_projection_workspace_bytes(vocab, hidden))


def launch_output_projection(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    logits: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 logits of one token through a bf16 ``[vocab, hidden]`` matrix; also
    returns the workspace holding the argmax partials for
    ``launch_greedy_select``. Mirrors ``launch_bfloat16_output_projection``
    (src/nanoquant/runtime/cuda_kernels.py:684-712) for one token."""

    if weight.dtype != torch.bfloat16 or weight.ndim != 2:
        raise ValueError("output projection requires a bf16 [vocab, hidden] matrix")
    if x.dtype not in (torch.float32, torch.bfloat16) or x.numel() != weight.shape[1]:
        raise ValueError("output projection input must be one F32/BF16 row of width hidden")
    _check_device("output projection", x.device, x, weight, logits, workspace)
    vocab, hidden = weight.shape
    if logits is None:
        logits = torch.empty(vocab, dtype=torch.float32, device=x.device)
    elif logits.dtype != torch.float32 or logits.numel() != vocab:
        raise ValueError("logits must be fp32 [vocab]")
    need = output_projection_workspace_bytes(vocab, hidden)
    if need < 0:
        raise ValueError("output projection geometry was rejected")
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    status = _native.load().nq_output_projection(
        x.data_ptr(), _native.dtype_code(x.dtype), weight.data_ptr(), vocab, hidden, logits.data_ptr(),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(x.device),
    )
    _native.check("nq_output_projection", status)
    return logits, workspace


def launch_greedy_select(
    workspace: torch.Tensor,
    vocab: int,
    hidden: int,
    *,
    token_out: torch.Tensor,
    history: torch.Tensor | None = None,
    step: torch.Tensor | None = None,
    position: torch.Tensor | None = None,
) -> torch.Tensor:
    """Greedy token (lowest index among equal maxima, like ``torch.argmax``) from
    the partials of ``launch_output_projection``, written to ``token_out[0]``;
    optionally appended to ``history`` at ``step`` and advancing ``position``."""

    after = _greedy_outputs(workspace, token_out, history, step, position)
    status = _native.load().nq_greedy_select(workspace.data_ptr(), vocab, hidden, *after)
    _native.check("nq_greedy_select", status)
    return token_out


def launch_greedy_select_partials(
    partials: torch.Tensor,
    *,
    token_out: torch.Tensor,
    history: torch.Tensor | None = None,
    step: torch.Tensor | None = None,
    position: torch.Tensor | None = None,
) -> torch.Tensor:
    """``launch_greedy_select`` from the int64 partials of ``launch_int4_projection``."""

    if partials.dtype is not torch.int64 or partials.ndim != 1 or not partials.numel():
        raise ValueError("greedy select partials must be int64 [count]")
    after = _greedy_outputs(partials, token_out, history, step, position)
    status = _native.load().nq_greedy_select_partials(partials.data_ptr(), partials.numel(), *after)
    _native.check("nq_greedy_select_partials", status)
    return token_out


def _greedy_outputs(workspace, token_out, history, step, position) -> tuple:
    """Checks of what a greedy selection writes; its arguments in C."""

    device = workspace.device
    if token_out.dtype != torch.int64 or token_out.numel() < 1:
        raise ValueError("token_out must be an int64 tensor")
    if (history is None) != (step is None):
        raise ValueError("history and step must be given together")
    if history is not None and (history.dtype != torch.int64 or step.dtype != torch.int32):
        raise ValueError("history must be int64 and step int32")
    if position is not None:
        _position("greedy select", position, device)
    _check_device("greedy select", device, workspace, token_out, history, step, position)
    return (token_out.data_ptr(), _ptr(history), 0 if history is None else history.numel(), _ptr(step), _ptr(position),
            _stream(device))


# -- 4-bit weights ---------------------------------------------------------------


class Int4Matrix(NamedTuple):
    """A ``[out, in]`` matrix of 4-bit weights: uint8 ``packed`` ``[out, in / 2]``, byte j of a
    row holding column 2 j in its low bits and 2 j + 1 in its high ones, ``scales`` F32/F16/BF16
    ``[out, ceil(in / group)]`` with groups of 32, 64 or 128 columns, and uint8
    ``zeros`` of that shape (None: 8). A weight is ``scale * (nibble - zero)``."""

    packed: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None = None

    @property
    def shape(self) -> tuple[int, int]:
        return self.packed.shape[0], 2 * self.packed.shape[1]

    def to(self, device: torch.device | str) -> "Int4Matrix":
        return Int4Matrix(*(None if t is None else t.to(device).contiguous() for t in self))


_INT4_GROUPS = (32, 64, 128)


def int4_matrix(weight: torch.Tensor, group: int = 128, scale_dtype: torch.dtype = torch.float16) -> Int4Matrix:
    """``weight`` ``[out, in]`` rounded to 4 bits: for each group of columns the larger of
    the scales that bring its largest value to 7 and its lowest to -8. A weight that is not
    finite, or a group whose scale is beyond ``scale_dtype``, is refused. Once, before serving
    (the check waits for the device)."""

    if weight.ndim != 2 or weight.shape[1] % 32 or group not in _INT4_GROUPS or scale_dtype not in _FLOAT:
        raise ValueError("4-bit weights need [out, in] with in a multiple of 32 and groups of 32, 64 or 128")
    outs, ins = weight.shape
    groups = -(-ins // group)
    packed = torch.empty(outs, ins // 2, dtype=torch.uint8, device=weight.device)
    scales = torch.empty(outs, groups, dtype=scale_dtype, device=weight.device)
    for first in range(0, outs, 8192):
        w = torch.nn.functional.pad(weight[first:first + 8192].float(), (0, groups * group - ins)).view(-1, groups, group)
        scale = torch.maximum(w.amax(-1) / 7, -w.amin(-1) / 8).to(scale_dtype)
        scales[first:first + 8192] = scale
        scale = scale.float()
        q = torch.where(scale[..., None] > 0, w / scale[..., None], 0.0).round_().clamp_(-8, 7).add_(8).nan_to_num_().to(torch.uint8)
        q = q.view(q.shape[0], -1)[:, :ins]
        packed[first:first + 8192] = q[:, 0::2] | (q[:, 1::2] << 4)
    # A weight that is NaN or infinite makes its group's scale so.
    if not bool(torch.isfinite(scales).all()):
        raise ValueError(f"4-bit weights need finite values whose groups' scales {scale_dtype} holds")
    return Int4Matrix(packed, scales)


def int4_projection_workspace_bytes(tokens: int, weight: Int4Matrix) -> int:
    outs, ins = weight.shape
    return int(_native.load().nq_int4_projection_workspace_bytes(tokens, outs, ins, _int4_group(weight)))


def int4_projection_partials(out_features: int) -> int:
    return int(_native.load().nq_int4_projection_partials(out_features))


def _int4_group(weight: Int4Matrix) -> int:
    """The group that the scales' shape says (the widest, where a narrower one would be the same)."""

    ins, groups = 2 * weight.packed.shape[1], weight.scales.shape[1]
    for group in reversed(_INT4_GROUPS):
        if -(-ins // group) == groups:
            return group
    raise ValueError("4-bit scales must be [out, ceil(in / group)] with groups of 32, 64 or 128")


def launch_int4_projection(
    x: torch.Tensor,
    weight: Int4Matrix,
    *,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
    partials: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x @ W.T`` of F32/F16/BF16 ``x`` ``[tokens, in]`` and 4-bit weights, for a few
    tokens (nq_int4_projection): fp32 sums, rounded once to ``out``. For one
    token ``partials`` (int64 ``[int4_projection_partials(out)]``) get what
    ``launch_greedy_select_partials`` chooses by. Beside ``launch_output_projection``, at a
    quarter of its weight's bytes (src/nanoquant/runtime/cuda_kernels.py:684-712)."""

    device = x.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_int4_projection(x, weight, out=out, out_dtype=out_dtype, partials=partials, workspace=workspace)
    packed, scales, zeros = weight
    if packed.dtype is not torch.uint8 or packed.ndim != 2 or packed.shape[1] % 16 or not packed.numel():
        raise ValueError("4-bit weights must be uint8 [out, in / 2] with in a multiple of 32")
    outs, ins = weight.shape
    if scales.dtype not in _FLOAT or scales.ndim != 2 or scales.shape[0] != outs:
        raise ValueError("4-bit scales must be F32/F16/BF16 [out, ceil(in / group)]")
    group = _int4_group(weight)
    if zeros is not None and (zeros.dtype is not torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("4-bit zeros must be uint8 of the scales' shape")
    if x.ndim != 2 or x.dtype not in _FLOAT or not x.shape[0] or x.shape[1] != ins:
        raise ValueError("4-bit projection input must be F32/F16/BF16 [tokens, in]")
    _check_device("4-bit projection", device, x, packed, scales, zeros, out, partials, workspace)
    tokens = x.shape[0]
    if out is None:
        out = torch.empty(tokens, outs, dtype=out_dtype, device=device)
    elif out.shape != (tokens, outs):
        raise ValueError("4-bit projection output must be [tokens, out]")
    if out.dtype not in _FLOAT:
        raise ValueError("4-bit projection output must be F32/F16/BF16")
    lib = _native.load()
    if partials is not None and (tokens != 1 or partials.dtype is not torch.int64
                                 or partials.shape != (lib.nq_int4_projection_partials(outs),)):
        raise ValueError("4-bit projection partials are those of one token: int64 [int4_projection_partials(out)]")
    need = lib.nq_int4_projection_workspace_bytes(tokens, outs, ins, group)
    if need < 0:
        raise ValueError("4-bit projection geometry was rejected")
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = lib.nq_int4_projection(
        x.data_ptr(), _native.DTYPE_CODES[x.dtype], tokens, packed.data_ptr(), scales.data_ptr(),
        _native.DTYPE_CODES[scales.dtype], _ptr(zeros), outs, ins, group, out.data_ptr(), _native.DTYPE_CODES[out.dtype],
        _ptr(partials), _ptr(workspace), 0 if workspace is None else workspace.numel() * workspace.element_size(),
        _stream(device),
    )
    _native.check("nq_int4_projection", status)
    return out


# -- serving: ragged batches over an 8-bit paged cache ---------------------------


class PagedCache(NamedTuple):
    """An 8-bit paged KV cache (``nq_paged_kv`` in ``include/nqamd_shell.h``): K
    ``[pages, kv_heads, page_size, head_dim]`` and V, transposed,
    ``[pages, kv_heads, head_dim, page_size]``, float8_e4m3fn values that stand
    for value * scale, with one fp32 scale ``[pages, kv_heads]`` each."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


_PAGE_SIZES = (16, 32, 64, 128)
_HEAD_DIMS = (64, 128, 256)


def paged_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, device: torch.device | str) -> PagedCache:
    """An empty paged cache. ``page_size`` is 16, 32, 64 or 128, ``head_dim`` 64, 128 or 256."""

    if pages < 1 or kv_heads < 1 or page_size not in _PAGE_SIZES or head_dim not in _HEAD_DIMS:
        raise ValueError("paged cache geometry is unsupported")

    def zeros(*shape: int) -> torch.Tensor:
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

    scales = torch.zeros((2, pages, kv_heads), dtype=torch.float32, device=device)
    return PagedCache(zeros(pages, kv_heads, page_size, head_dim), zeros(pages, kv_heads, head_dim, page_size),
                      scales[0], scales[1])


def _paged_kv(name: str, device: torch.device, cache: PagedCache, page_table: torch.Tensor,
              query_starts: torch.Tensor | None, context_lens: torch.Tensor) -> _native.PagedKv:
    """Checks of the cache and the batch; the C descriptor of both. A call without
    tokens has no query_starts."""

    k, v, k_scales, v_scales = cache
    _check_device(name, device, k, v, k_scales, v_scales, page_table, query_starts, context_lens)
    if k.dtype is not torch.float8_e4m3fn or v.dtype is not torch.float8_e4m3fn or k.ndim != 4:
        raise ValueError(f"{name} cache pages must be 4-D float8_e4m3fn")
    pages, kv_heads, page_size, head_dim = k.shape
    scales = (pages, kv_heads)
    if v.shape != (pages, kv_heads, head_dim, page_size):
        raise ValueError(f"{name} cache must be K [pages, kv_heads, page_size, head_dim], V [pages, kv_heads, head_dim, page_size]")
    if page_size not in _PAGE_SIZES or head_dim not in _HEAD_DIMS or not pages or not kv_heads:
        raise ValueError(f"{name} page size must be 16, 32, 64 or 128 and head_dim 64, 128 or 256")
    if k_scales.dtype is not torch.float32 or v_scales.dtype is not torch.float32 or k_scales.shape != scales \
            or v_scales.shape != scales:
        raise ValueError(f"{name} cache scales must be fp32 [pages, kv_heads]")
    if page_table.dtype is not torch.int32 or context_lens.dtype is not torch.int32 \
            or (query_starts is not None and query_starts.dtype is not torch.int32):
        raise ValueError(f"{name} page_table, query_starts and context_lens must be int32")
    shape = page_table.shape
    if len(shape) != 2 or not shape[0] or not shape[1] or context_lens.shape != (shape[0],) \
            or (query_starts is not None and query_starts.shape != (shape[0] + 1,)):
        raise ValueError(f"{name} takes page_table [batch, pages], query_starts [batch + 1] and context_lens [batch]")
    return _native.PagedKv(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages, kv_heads,
                           head_dim, page_size, 0, page_table.data_ptr(), shape[1], _ptr(query_starts),
                           context_lens.data_ptr(), shape[0])


def _elsewhere(device: torch.device) -> bool:
    """Whether another device than `device` is current. A default stream's handle
    is the same on every device and a launch goes to the current one's."""

    return device.type == "cuda" and torch._C._cuda_getDevice() != device.index


def launch_paged_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cache: PagedCache,
    *,
    q_heads: int,
    q_norm: torch.Tensor | None,
    k_norm: torch.Tensor | None,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    page_table: torch.Tensor,
    query_starts: torch.Tensor,
    context_lens: torch.Tensor,
    q_out: torch.Tensor | None = None,
    q_dtype: torch.dtype = torch.float32,
    rope_starts: torch.Tensor | None = None,
) -> torch.Tensor:
    """Per-head RMSNorm + RoPE of a ragged batch's q and k and the append of k and
    v to an 8-bit paged cache; returns the rotated q ``[tokens, q_heads,
    head_dim]``. Tokens ``query_starts[b] .. query_starts[b + 1]`` are sequence
    b's, at cache rows ``context_lens[b] ..``, in the pages ``page_table[b]``
    (nq_paged_append). ``rope_starts`` (int32 ``[batch]``) are the positions that
    the sequences' tokens begin at where those are not their cache rows, as after
    ``launch_paged_evict`` (nq_paged_append_at). Mirrors ``launch_decode_rope`` and
    ``launch_cache_prefix_update`` (src/nanoquant/runtime/cuda_kernels.py:715-815)
    for many sequences."""

    device = q.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_paged_append(
                q, k, v, cache, q_heads=q_heads, q_norm=q_norm, k_norm=k_norm, eps=eps, cos=cos, sin=sin,
                page_table=page_table, query_starts=query_starts, context_lens=context_lens, q_out=q_out, q_dtype=q_dtype,
                rope_starts=rope_starts)
    _check_device("paged append", device, q, k, v, q_norm, k_norm, cos, sin, q_out, rope_starts)
    kv = _paged_kv("paged append", device, cache, page_table, query_starts, context_lens)
    kv_heads, head_dim = kv.kv_heads, kv.head_dim
    if q_heads < 1 or q_heads % kv_heads:
        raise ValueError("paged append q heads must be a multiple of the cache's kv heads")
    size = q.numel()
    tokens = size // (q_heads * head_dim)
    rows = tokens * kv_heads * head_dim
    if tokens < 1 or size != tokens * q_heads * head_dim or k.numel() != rows or v.numel() != rows:
        raise ValueError("paged append takes q [tokens, q_heads * head_dim], k and v [tokens, kv_heads * head_dim]")
    dtype = q.dtype
    if dtype not in _FLOAT or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("paged append q, k and v must share one of F32/F16/BF16")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm must be given together")
    norm_code = 0
    if q_norm is not None:
        if q_norm.numel() != head_dim or k_norm.numel() != head_dim or q_norm.dtype != k_norm.dtype \
                or q_norm.dtype not in _FLOAT:
            raise ValueError("q/k norm weights must be [head_dim] of one of F32/F16/BF16")
        norm_code = _native.DTYPE_CODES[q_norm.dtype]
    table = cos.shape
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(table) != 2 \
            or table[1] * 2 != head_dim or not table[0] or sin.shape != table:
        raise ValueError("RoPE tables must be fp32 [positions, head_dim / 2]")
    if rope_starts is not None and (rope_starts.dtype is not torch.int32 or rope_starts.shape != context_lens.shape):
        raise ValueError("paged append rope_starts must be int32 [batch]")
    if q_out is None:
        q_out = torch.empty(tokens, q_heads, head_dim, dtype=q_dtype, device=device)
    elif q_out.numel() != tokens * q_heads * head_dim:
        raise ValueError("q_out must be [tokens, q_heads, head_dim]")
    if q_out.dtype not in _FLOAT:
        raise ValueError("q_out must be F32/F16/BF16")
    status = _native.load().nq_paged_append_at(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.DTYPE_CODES[dtype], tokens, q_heads, _ptr(q_norm),
        _ptr(k_norm), norm_code, eps, cos.data_ptr(), sin.data_ptr(), table[0], ctypes.byref(kv), _ptr(rope_starts),
        q_out.data_ptr(), _native.DTYPE_CODES[q_out.dtype], _stream(device),
    )
    _native.check("nq_paged_append_at", status)
    return q_out


def paged_attention_workspace_bytes(tokens: int, batch: int, q_heads: int, cache: PagedCache, table_pages: int) -> int:
    _pages, kv_heads, page_size, head_dim = cache.k.shape
    return int(_native.load().nq_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, head_dim, page_size,
                                                                 table_pages))


def launch_paged_attention(
    q: torch.Tensor,
    cache: PagedCache,
    *,
    page_table: torch.Tensor,
    query_starts: torch.Tensor,
    context_lens: torch.Tensor,
    scaling: float,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal grouped-query attention of a ragged batch's ``q`` (F32/F16/BF16
    ``[tokens, q_heads, head_dim]``) over an 8-bit paged cache that holds the
    tokens' own rows too (``launch_paged_append`` with the same batch): the
    token at cache row r attends rows ``[0, r]`` of its sequence
    (nq_paged_attention). One token a sequence or a whole prompt each. Mirrors
    ``launch_decode_attention`` (src/nanoquant/runtime/cuda_kernels.py:493-544)
    for many sequences."""

    device = q.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_paged_attention(
                q, cache, page_table=page_table, query_starts=query_starts, context_lens=context_lens, scaling=scaling,
                out=out, out_dtype=out_dtype, workspace=workspace)
    if q.ndim != 3 or q.dtype not in _FLOAT:
        raise ValueError("paged attention query must be F32/F16/BF16 [tokens, q_heads, head_dim]")
    _check_device("paged attention", device, q, out, workspace)
    kv = _paged_kv("paged attention", device, cache, page_table, query_starts, context_lens)
    tokens, q_heads, head_dim = q.shape
    if head_dim != kv.head_dim or not tokens or not q_heads or q_heads % kv.kv_heads:
        raise ValueError("paged attention query geometry does not match the cache")
    if not 0.0 < scaling < float("inf"):
        raise ValueError("paged attention scaling must be positive and finite")
    if out is None:
        out = torch.empty(tokens, q_heads * head_dim, dtype=out_dtype, device=device)
    elif out.numel() != q.numel():
        raise ValueError("paged attention output geometry is incompatible")
    if out.dtype not in _FLOAT:
        raise ValueError("paged attention output must be F32/F16/BF16")
    lib = _native.load()
    need = lib.nq_paged_attention_workspace_bytes(tokens, kv.batch, q_heads, kv.kv_heads, head_dim, kv.page_size,
                                                  kv.table_pages)
    if need < 0:
        raise ValueError("paged attention geometry was rejected")
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = lib.nq_paged_attention(
        q.data_ptr(), _native.DTYPE_CODES[q.dtype], tokens, q_heads, ctypes.byref(kv), scaling, out.data_ptr(),
        _native.DTYPE_CODES[out.dtype], _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_paged_attention", status)
    return out


# -- serving: long conversations in bounded memory and traffic ---------------------


def shared_attention_workspace_bytes(tokens: int, batch: int, q_heads: int, cache: PagedCache, table_pages: int,
                                     shared_rows: int) -> int:
    _pages, kv_heads, page_size, head_dim = cache.k.shape
    return int(_native.load().nq_shared_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, head_dim, page_size,
                                                                  table_pages, shared_rows))


def launch_shared_attention(
    q: torch.Tensor,
    cache: PagedCache,
    *,
    page_table: torch.Tensor,
    query_starts: torch.Tensor,
    context_lens: torch.Tensor,
    shared_rows: int,
    scaling: float,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    lse: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """``launch_paged_attention`` for a batch whose sequences hold the same first
    ``shared_rows`` cache rows: the first ``shared_rows // page_size`` entries of
    every part of the page table name the same pages (sequence 0's are read),
    and their keys and values are read once for many sequences
    (nq_shared_attention). ``lse`` (fp32 ``[tokens, q_heads]``) gets each query
    row's log-sum-exp, which ``launch_attention_weights`` takes. With
    ``shared_rows=0`` nothing is shared. Mirrors ``launch_decode_attention``
    (src/nanoquant/runtime/cuda_kernels.py:493-544) for many sequences."""

    device = q.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_shared_attention(
                q, cache, page_table=page_table, query_starts=query_starts, context_lens=context_lens,
                shared_rows=shared_rows, scaling=scaling, out=out, out_dtype=out_dtype, lse=lse, workspace=workspace)
    if q.ndim != 3 or q.dtype not in _FLOAT:
        raise ValueError("shared attention query must be F32/F16/BF16 [tokens, q_heads, head_dim]")
    _check_device("shared attention", device, q, out, lse, workspace)
    kv = _paged_kv("shared attention", device, cache, page_table, query_starts, context_lens)
    tokens, q_heads, head_dim = q.shape
    if head_dim != kv.head_dim or not tokens or not q_heads or q_heads % kv.kv_heads:
        raise ValueError("shared attention query geometry does not match the cache")
    if not 0.0 < scaling < float("inf"):
        raise ValueError("shared attention scaling must be positive and finite")
    if not 0 <= shared_rows <= kv.table_pages * kv.page_size:
        raise ValueError("shared attention shared_rows must lie within the page table")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (tokens, q_heads)):
        raise ValueError("shared attention lse must be fp32 [tokens, q_heads]")
    if out is None:
        out = torch.empty(tokens, q_heads * head_dim, dtype=out_dtype, device=device)
    elif out.numel() != q.numel():
        raise ValueError("shared attention output geometry is incompatible")
    if out.dtype not in _FLOAT:
        raise ValueError("shared attention output must be F32/F16/BF16")
    lib = _native.load()
    need = lib.nq_shared_attention_workspace_bytes(tokens, kv.batch, q_heads, kv.kv_heads, head_dim, kv.page_size,
                                                   kv.table_pages, shared_rows)
    if need < 0:
        raise ValueError("shared attention geometry was rejected")
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = lib.nq_shared_attention(
        q.data_ptr(), _native.DTYPE_CODES[q.dtype], tokens, q_heads, ctypes.byref(kv), shared_rows, scaling,
        out.data_ptr(), _native.DTYPE_CODES[out.dtype], _ptr(lse), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_shared_attention", status)
    return out


def launch_attention_weights(
    q: torch.Tensor,
    cache: PagedCache,
    lse: torch.Tensor,
    weights: torch.Tensor,
    *,
    page_table: torch.Tensor,
    query_starts: torch.Tensor,
    context_lens: torch.Tensor,
    scaling: float,
    first: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Adds the attention that each cached row from ``first`` on receives from the
    call's tokens to ``weights`` (fp32 ``[pages, kv_heads, page_size]``, in place
    unless ``out`` is given; rows that the call brought start at 0), after
    ``launch_shared_attention`` with the same arrays, whose ``lse`` it takes
    (nq_attention_weights). ``launch_paged_evict`` decides by these weights. Pages
    that sequences share hold rows before ``first`` alone. The reference keeps
    every row (src/nanoquant/runtime/transformers_generation.py:262-418)."""

    device = q.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_attention_weights(
                q, cache, lse, weights, page_table=page_table, query_starts=query_starts, context_lens=context_lens,
                scaling=scaling, first=first, out=out)
    if q.ndim != 3 or q.dtype not in _FLOAT:
        raise ValueError("attention weights query must be F32/F16/BF16 [tokens, q_heads, head_dim]")
    _check_device("attention weights", device, q, lse, weights, out)
    kv = _paged_kv("attention weights", device, cache, page_table, query_starts, context_lens)
    tokens, q_heads, head_dim = q.shape
    if head_dim != kv.head_dim or not tokens or not q_heads or q_heads % kv.kv_heads:
        raise ValueError("attention weights query geometry does not match the cache")
    if not 0.0 < scaling < float("inf"):
        raise ValueError("attention weights scaling must be positive and finite")
    if lse.dtype is not torch.float32 or lse.shape != (tokens, q_heads):
        raise ValueError("attention weights lse must be fp32 [tokens, q_heads]")
    if out is None:
        out = weights
    shape = (kv.num_pages, kv.kv_heads, kv.page_size)
    if weights.dtype is not torch.float32 or out.dtype is not torch.float32 or weights.shape != shape or out.shape != shape:
        raise ValueError("attention weights must be fp32 [pages, kv_heads, page_size]")
    if first < 0:
        raise ValueError("attention weights begin at a row from 0 on")
    status = _native.load().nq_attention_weights(
        q.data_ptr(), _native.DTYPE_CODES[q.dtype], tokens, q_heads, ctypes.byref(kv), scaling, lse.data_ptr(), first,
        weights.data_ptr(), out.data_ptr(), _stream(device),
    )
    _native.check("nq_attention_weights", status)
    return out


class Evicted(NamedTuple):
    """``launch_paged_evict``'s result: the sequences' new int32 page table ``[batch,
    ceil(budget / page_size)]`` and lengths ``[batch]``, and the old row of each
    row that stayed, int32 ``[batch, kv_heads, budget]`` (-1 behind the last)."""

    page_table: torch.Tensor
    context_lens: torch.Tensor
    rows: torch.Tensor


def paged_evict_workspace_bytes(batch: int, cache: PagedCache, table_pages: int, budget: int) -> int:
    _pages, kv_heads, page_size, _head_dim = cache.k.shape
    return int(_native.load().nq_paged_evict_workspace_bytes(batch, kv_heads, page_size, table_pages, budget))


def launch_paged_evict(
    cache: PagedCache,
    weights: torch.Tensor,
    *,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    into: torch.Tensor,
    budget: int,
    first: int = 0,
    recent: int = 0,
    out: Evicted | None = None,
    workspace: torch.Tensor | None = None,
) -> Evicted:
    """Cuts every sequence with more than ``budget`` cached rows to that many: its
    ``first`` rows, its ``recent`` newest and, for each kv head, of those between
    the heaviest by ``weights`` (``launch_attention_weights``). The rows that stay
    move in their order to the free pages ``into`` (int32 ``[batch, ceil(budget /
    page_size) - first // page_size]``), but for the whole pages of the first rows, which stay where
    they are (nq_paged_evict). ``context_lens`` are the rows that the sequences hold by now, those
    of the call whose attention was added last among them. The new table has no entries behind the
    budget: pages for tokens to come go behind them. The keys keep the positions they were rotated at:
    ``launch_paged_append`` takes those of the next tokens as ``rope_starts``. The reference
    keeps every row (src/nanoquant/runtime/transformers_generation.py:262-418)."""

    device = cache.k.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_paged_evict(cache, weights, page_table=page_table, context_lens=context_lens, into=into,
                                      budget=budget, first=first, recent=recent, out=out, workspace=workspace)
    _check_device("paged evict", device, weights, into, workspace)
    batch = page_table.shape[0] if page_table.ndim == 2 else 0
    kv = _paged_kv("paged evict", device, cache, page_table, None, context_lens)
    if weights.dtype is not torch.float32 or weights.shape != (kv.num_pages, kv.kv_heads, kv.page_size):
        raise ValueError("paged evict weights must be fp32 [pages, kv_heads, page_size]")
    if budget < 1 or first < 0 or recent < 0 or first + recent > budget:
        raise ValueError("paged evict keeps at least one row, and first and recent rows within its budget")
    entries = -(-budget // kv.page_size)
    slots = entries - first // kv.page_size
    if into.dtype is not torch.int32 or into.shape != (batch, slots):
        raise ValueError("paged evict into must be int32 [batch, ceil(budget / page_size) - first // page_size]")
    if out is None:
        out = Evicted(into.new_empty(batch, entries), into.new_empty(batch), into.new_empty(batch, kv.kv_heads, budget))
    else:
        _check_device("paged evict", device, *out)
        if any(x.dtype is not torch.int32 for x in out) or out.page_table.shape != (batch, entries) \
                or out.context_lens.shape != (batch,) or out.rows.shape != (batch, kv.kv_heads, budget):
            raise ValueError("paged evict outputs must be int32 [batch, pages], [batch] and [batch, kv_heads, budget]")
    lib = _native.load()
    need = lib.nq_paged_evict_workspace_bytes(batch, kv.kv_heads, kv.page_size, kv.table_pages, budget)
    if need < 0:
        raise ValueError("paged evict geometry was rejected")
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = lib.nq_paged_evict(
        ctypes.byref(kv), weights.data_ptr(), into.data_ptr() if slots else None, budget, first, recent,
        out.page_table.data_ptr(), out.context_lens.data_ptr(), out.rows.data_ptr(), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_paged_evict", status)
    return out


# -- how likely the answers are ---------------------------------------------------


class TokenLogprobs(NamedTuple):
    """``launch_token_logprobs``' result: fp32 ``[rows]`` log probability of each
    row's token and entropy of its distribution, int64 and fp32 ``[rows, top]``
    likeliest tokens and their log probabilities, likeliest first."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs_workspace_bytes(rows: int, vocab: int, top: int) -> int:
    return int(_native.load().nq_token_logprobs_workspace_bytes(rows, vocab, top))


def launch_token_logprobs(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    *,
    top: int = 0,
    out: TokenLogprobs | None = None,
    workspace: torch.Tensor | None = None,
) -> TokenLogprobs:
    """Log probability of ``tokens[r]`` under ``softmax(logits[r])``, the entropy of
    that distribution and its ``top`` (0 to 32) likeliest tokens, the lowest id
    first among equals (nq_token_logprobs). ``logits`` is F32/F16/BF16 ``[rows,
    vocab]``; its rows may lie further apart than vocab."""

    device = logits.device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return launch_token_logprobs(logits, tokens, top=top, out=out, workspace=workspace)
    if logits.ndim != 2 or logits.dtype not in _FLOAT:
        raise ValueError("token logprobs take F32/F16/BF16 logits [rows, vocab]")
    rows, vocab = logits.shape
    if not rows or not vocab:
        raise ValueError("token logprobs need at least one row and one token")
    stride = logits.stride(0) if rows > 1 else vocab
    if (vocab > 1 and logits.stride(1) != 1) or stride < vocab:
        raise ValueError("token logprobs need rows of adjacent logits that do not overlap")
    if tokens.dtype != torch.int64 or tokens.shape != (rows,):
        raise ValueError("token logprobs take int64 tokens [rows]")
    if not 0 <= top <= 32 or top > vocab:
        raise ValueError("token logprobs give 0 to 32 alternatives, at most the vocabulary")
    if device.type != "cuda" or tokens.device != device:
        raise ValueError("token logprobs require CUDA/HIP tensors on one device")
    if out is None:
        _check_device("token logprobs", device, tokens, workspace)
        logprobs = torch.empty(rows, dtype=torch.float32, device=device)
        out = TokenLogprobs(logprobs, torch.empty_like(logprobs), tokens.new_empty(rows, top), logprobs.new_empty(rows, top))
    else:
        _check_device("token logprobs", device, tokens, *out, workspace)
        if out.logprobs.dtype != torch.float32 or out.entropy.dtype != torch.float32 or out.top_ids.dtype != torch.int64 \
                or out.top_logprobs.dtype != torch.float32 or out.logprobs.shape != (rows,) \
                or out.entropy.shape != (rows,) or out.top_ids.shape != (rows, top) \
                or out.top_logprobs.shape != (rows, top):
            raise ValueError("token logprobs outputs must be fp32 [rows] twice, int64 and fp32 [rows, top]")
    lib = _native.load()
    need = lib.nq_token_logprobs_workspace_bytes(rows, vocab, top)
    if need < 0:
        raise ValueError("token logprobs geometry was rejected")
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    status = lib.nq_token_logprobs(
        logits.data_ptr(), _native.DTYPE_CODES[logits.dtype], rows, vocab, stride, tokens.data_ptr(), top,
        out.logprobs.data_ptr(), out.entropy.data_ptr(), _ptr(out.top_ids if top else None),
        _ptr(out.top_logprobs if top else None), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(), _stream(device),
    )
    _native.check("nq_token_logprobs", status)
    return out
