"""CPU oracle of the serving operators — TEST INFRASTRUCTURE ONLY.

The 8-bit paged KV cache's append, attention over it, and token log
probabilities, restated from their definitions in 64 bits, sequence by sequence
and page by page. ``tests/`` compare the HIP kernels with it. Pinned by closed
forms in tests/test_serving_oracle.py (torch's own e4m3 conversion, softmax and
log_softmax on small inputs).

The cache is a dict of ``k`` [pages, kv, page, D], ``v`` [pages, kv, D, page]
(e4m3 values as fp64, before their scale) and ``k_scales`` / ``v_scales``
[pages, kv]. A batch is a list of (first token, end token, cached rows) and a
list of each sequence's table entries.
"""

from __future__ import annotations

import math

import torch
from torch.nn import functional as F

from oracle import decoder_shell as ods

MIN_EXPONENT = -126


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each |x| <= 448, ties to even, NaN for what is
    not finite."""

    x = x.double()
    out = torch.full_like(x, math.nan)
    ok = torch.isfinite(x)
    exponent = torch.frexp(x[ok]).exponent.double()  # |x| in [2^(e - 1), 2^e)
    step = torch.pow(2.0, (exponent - 4).clamp(min=-9))
    out[ok] = torch.round(x[ok] / step) * step
    return out


def scale_for(amax: float) -> float:
    """The least power of two from 2^-126 on with amax <= 448 * scale."""

    exponent = MIN_EXPONENT
    while amax > math.ldexp(448.0, exponent):
        exponent += 1
    return math.ldexp(1.0, exponent)


def norm_rope(x: torch.Tensor, weight: torch.Tensor | None, eps: float, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """fp64 RMSNorm (optional) and rotate-half RoPE of [heads, D] at one position."""

    x = x.double()
    if weight is not None:
        x = weight.double() * x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    half = x.shape[-1] // 2
    a, b, c, s = x[:, :half], x[:, half:], cos.double(), sin.double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def finite_amax(x: torch.Tensor) -> torch.Tensor:
    return torch.where(torch.isfinite(x), x.abs(), 0.0).amax((1, 2))


def append(q, k, v, cache, table, spans, *, page, q_norm, k_norm, eps, cos, sin, rope_starts=None):
    """Rotated q (fp64, NaN rows where no token writes) and the cache afterwards;
    `rope_starts` are the sequences' first positions where those are not cache rows."""

    cache = {name: x.clone().double() for name, x in cache.items()}
    pages, d = cache["k"].shape[0], cache["k"].shape[3]
    tokens, kv = q.shape[0], cache["k"].shape[1]
    q_out = torch.full((tokens, q.shape[1], d), math.nan, dtype=torch.float64)
    rows_held = len(table[0]) * page
    for b, (begin, end, context) in enumerate(spans):
        new: dict[int, list[tuple[int, torch.Tensor, torch.Tensor]]] = {}
        for t in range(begin, end):
            row = context + t - begin
            at = row if rope_starts is None else rope_starts[b] + t - begin
            if row < 0 or row >= rows_held or at < 0 or at >= cos.shape[0]:
                continue
            q_out[t] = norm_rope(q[t], q_norm, eps, cos[at], sin[at])
            new.setdefault(row // page, []).append(
                (row % page, norm_rope(k[t], k_norm, eps, cos[at], sin[at]), v[t].double()))
        for slot, rows in new.items():
            at = table[b][slot]
            if at < 0 or at >= pages:
                continue
            first = rows[0][0]
            for name, pick in (("k", 1), ("v", 2)):
                values = torch.stack([r[pick] for r in rows], 1)  # [kv, rows, D]
                stored = cache[name][at] if name == "k" else cache[name][at].transpose(1, 2)
                amax = finite_amax(values)
                for g in range(kv):
                    scale = scale_for(float(amax[g]))
                    if first:
                        old = float(cache[name + "_scales"][at, g])
                        scale = max(scale, old)
                        if scale != old:
                            stored[g, :first] = e4m3(stored[g, :first] * (old / scale))
                    cache[name + "_scales"][at, g] = scale
                    for (r, *_), x in zip(rows, values[g]):
                        stored[g, r] = e4m3(x / scale)
    return q_out, cache


def attention(q, cache, table, spans, *, page, scaling):
    """fp64 outputs [tokens, q_heads, D] (NaN rows for nobody's tokens), and for each
    output sum p |v| and for each row the largest scaling * sum |q| |k|: what the
    rounding of an fp32 evaluation is relative to."""

    kv, d = cache["k"].shape[1], cache["k"].shape[3]
    tokens, heads = q.shape[0], q.shape[1]
    out = torch.full((tokens, heads, d), math.nan, dtype=torch.float64)
    spread, reach = out.clone(), torch.zeros(tokens, heads, dtype=torch.float64)
    k_all = cache["k"].double() * cache["k_scales"].double()[..., None, None]
    v_all = cache["v"].double().transpose(2, 3) * cache["v_scales"].double()[..., None, None]
    rows_held = len(table[0]) * page
    for b, (begin, end, context) in enumerate(spans):
        last = min(context + end - begin, rows_held)
        keys, values = [], []
        for slot in range(-(-last // page) if last > 0 else 0):
            at = table[b][slot]
            bad = at < 0 or at >= k_all.shape[0]
            keys.append(torch.full_like(k_all[0], math.nan) if bad else k_all[at])
            values.append(torch.full_like(v_all[0], math.nan) if bad else v_all[at])
        for t in range(begin, end):
            row = context + t - begin
            if row < 0 or row >= rows_held:
                out[t], spread[t] = 0.0, 0.0
                continue
            ks = torch.cat(keys, 1)[:, :row + 1]
            vs = torch.cat(values, 1)[:, :row + 1]
            for h in range(heads):
                g = h // (heads // kv)
                x = q[t, h].double()
                p = torch.softmax(ks[g] @ x * scaling, 0)
                out[t, h], spread[t, h] = p @ vs[g], p @ vs[g].abs()
                reach[t, h] = (ks[g].abs() @ x.abs()).max() * scaling
    return out, spread, reach


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int):
    """fp64 log probabilities, entropy, top ids and log probabilities."""

    x = logits.double()
    log_p = x - torch.logsumexp(x, -1, keepdim=True)
    log_p = torch.where(torch.isnan(x).any(-1, keepdim=True) | (x == math.inf).any(-1, keepdim=True)
                        | (x == -math.inf).all(-1, keepdim=True), math.nan, log_p)
    vocab = x.shape[1]
    picked = torch.stack([log_p[r, t] if 0 <= t < vocab else torch.tensor(math.nan, dtype=torch.float64)
                          for r, t in enumerate(tokens.tolist())])
    p = log_p.exp()
    entropy = -torch.where(p == 0, 0.0, p * log_p).sum(-1)
    ids = []
    for row in x.tolist():
        order = sorted(range(vocab), key=lambda i: (0 if math.isnan(row[i]) else 1,
                                                    0.0 if math.isnan(row[i]) else -row[i], i))
        ids.append(order[:top])
    ids = torch.tensor(ids, dtype=torch.int64).reshape(x.shape[0], top)
    return picked, entropy, ids, log_p.gather(1, ids)


class PagedOracleDecoder(ods.OracleDecoder):
    """``OracleDecoder`` whose KV cache is the 8-bit paged one: pages of `page`
    rows in table order, appended call by call."""

    def __init__(self, geometry, weights, *, max_positions: int, page: int) -> None:
        self.page = page
        super().__init__(geometry, weights, max_positions=max_positions)

    def reset(self) -> None:
        g, pages = self.g, -(-self.max_positions // self.page)
        self.table = [list(range(pages))]
        self.caches = [{"k": torch.zeros(pages, g.kv_heads, self.page, g.head_dim),
                        "v": torch.zeros(pages, g.kv_heads, g.head_dim, self.page),
                        "k_scales": torch.zeros(pages, g.kv_heads), "v_scales": torch.zeros(pages, g.kv_heads)}
                       for _ in range(g.layers)]

    def forward(self, ids: torch.Tensor, start: int) -> torch.Tensor:
        g, w, t = self.g, self.w, ids.numel()
        h = w.embed[ids.long()].float()
        spans = [(0, t, start)]
        for i, layer in enumerate(w.layers):
            lin = self.linears[i]
            x = ods.rms_norm(h, layer.input_norm, g.eps)
            q, k, v = (lin[role](x).view(t, -1, g.head_dim) for role in ("q_proj", "k_proj", "v_proj"))
            # q and k have norms of their own
            kn = layer.k_norm
            q = torch.stack([norm_rope(q[j], layer.q_norm, g.eps, self.cos[start + j], self.sin[start + j]) for j in range(t)])
            _, self.caches[i] = append(k, k, v, self.caches[i], self.table, spans, page=self.page, q_norm=kn, k_norm=kn,
                                       eps=g.eps, cos=self.cos, sin=self.sin)
            attn, _, _ = attention(q, self.caches[i], self.table, spans, page=self.page, scaling=g.head_dim**-0.5)
            h = h + lin["o_proj"](attn.reshape(t, -1).float())
            x = ods.rms_norm(h, layer.post_norm, g.eps)
            h = h + lin["down_proj"](F.silu(lin["gate_proj"](x)) * lin["up_proj"](x))
        return ods.rms_norm(h, w.final_norm, g.eps) @ w.lm_head.float().T
