"""The serving operators on the GPU against their 64-bit restatement
(oracle/serving.py): append to the 8-bit paged cache, attention over it, token
log probabilities, and a run of them as a serving step makes it.

Bounds, derived from the kernels' arithmetic:

* stored bytes and scales equal the oracle's: K is normed and rotated in fp64
  (a byte could differ only within 2^-50 of a border), V is scaled exactly;
* rotated q: fp32 products and one fused sum, 8 roundings of at most 2^-24 of
  |x| |cos| + |y| |sin|;
* attention: products are exact, a score is a sum of D parts products in fp32,
  so it is off by at most 2^-24 (parts D + 8) scaling sum |q| |k|; a weight by
  that twice (the maximum's too) relative to itself, 2^-17 or 2^-24 for its
  parts, and the sums over n rows add 2^-24 (n / 16 + 64); the output, a mean of
  v by these weights, by the sum of these relative to sum p |v|, and it is
  rounded once to its type (eps / 2);
* log probabilities: a weight e^d is off by 2^-22 (hardware exponential and its
  product) + 2^-23 |d| relative, sums add 2^-24 (64 + 10) on their way through a
  lane, a wave and a row; so log S is off by 2^-24 (96 + 4 E|d|), the entropy by
  that and the same relative to E|d| and E d^2, each result by a half step.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import gpu_available
from nanoquant_amd import synthetic as syn
from nanoquant_amd.runtime import shell_ops as ops
from nanoquant_amd.runtime.decoder_shell import PAGE_ROWS, DecoderShellConfig, DecoderShellError, PackedDecoder
from oracle import decoder_shell as ods
from oracle import serving as osv
from oracle.nq_oracle import operands_from_state, relative_l2

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = torch.device("cuda", 0)
EPS = 1e-6
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _g(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def _say(*parts) -> None:
    print("[case]", *parts, flush=True)


def _rope_tables(rows: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


class Batch:
    """A ragged batch over a pool of pages in no order: (cached rows, new tokens) of each sequence."""

    def __init__(self, lengths, *, kv, d, page, seed, spare=2, ahead=0, behind=0, extra_entries=1):
        g = _g(seed)
        self.kv, self.d, self.page = kv, d, page
        used = [max(0, -(-(c + n) // page)) for c, n in lengths]
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=g).tolist()
        width = max(max(used), 1) + extra_entries
        self.table, at = [], 0
        for n in used:
            self.table.append(order[at:at + n] + [-7] * (width - n))
            at += n
        self.spans, first = [], ahead
        for c, n in lengths:
            self.spans.append((first, first + n, c))
            first += n
        self.tokens = first + behind
        # Every byte of the pool is something, NaN among them; scales are powers of two.
        bytes_ = torch.randint(0, 256, (2, pages, kv, page * d), generator=g, dtype=torch.uint8)
        scales = torch.pow(2.0, torch.randint(-10, -6, (2, pages, kv), generator=g).float())
        self.k_bytes, self.v_bytes = bytes_[0].view(pages, kv, page, d).clone(), bytes_[1].view(pages, kv, d, page).clone()
        self.scales = scales
        # The rows that sequences hold already are numbers.
        for b, (c, _) in enumerate(lengths):
            for row in range(max(0, c)):
                at = self.table[b][row // page]
                for stored in (self.k_bytes[at, :, row % page, :], self.v_bytes[at, :, :, row % page]):
                    stored[(stored & 0x7f) == 0x7f] = 0x31

    def host(self):
        return {"k": self.k_bytes.view(torch.float8_e4m3fn).double(), "v": self.v_bytes.view(torch.float8_e4m3fn).double(),
                "k_scales": self.scales[0].double(), "v_scales": self.scales[1].double()}

    def device(self):
        cache = ops.PagedCache(self.k_bytes.to(DEV).view(torch.float8_e4m3fn), self.v_bytes.to(DEV).view(torch.float8_e4m3fn),
                               self.scales[0].contiguous().to(DEV), self.scales[1].contiguous().to(DEV))
        return cache, self.batch()

    def batch(self):
        starts = [self.spans[0][0]] + [e for _, e, _ in self.spans]
        return {"page_table": torch.tensor(self.table, dtype=torch.int32, device=DEV),
                "query_starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
                "context_lens": torch.tensor([c for _, _, c in self.spans], dtype=torch.int32, device=DEV)}


def _same_bytes(got: torch.Tensor, expected: torch.Tensor) -> None:
    """Values of e4m3 tensors equal, NaN where NaN (a stored NaN's sign is free)."""

    got = got.cpu().view(torch.uint8).view(torch.float8_e4m3fn).double()
    nan = torch.isnan(expected)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], expected[~nan])


APPENDS = [
    # lengths, q heads, kv heads, head_dim, page, dtype, norm
    ([(0, 1)], 4, 2, 64, 16, torch.float32, True),                      # the first token of all
    ([(15, 1), (16, 1), (0, 1), (47, 1)], 8, 2, 128, 16, torch.bfloat16, True),   # a page's last and first row
    ([(63, 2), (5, 0), (0, 130), (64, 64)], 6, 2, 128, 64, torch.float16, True),  # an empty sequence, whole pages
    ([(3, 40), (100, 33)], 4, 4, 256, 32, torch.float32, False),
    ([(127, 3), (1, 255)], 7, 1, 64, 128, torch.bfloat16, False),
    ([(9, 17)], 3, 1, 256, 16, torch.float16, True),
]


@pytest.mark.parametrize("lengths,q_heads,kv,d,page,dtype,norm", APPENDS)
def test_paged_append(lengths, q_heads, kv, d, page, dtype, norm):
    _say("append", lengths, q_heads, kv, d, page, dtype)
    g = _g(31)
    b = Batch(lengths, kv=kv, d=d, page=page, seed=7, ahead=1, behind=2)
    # Sizes unlike from token to token: some pages keep their scale, others grow.
    size = torch.pow(2.0, torch.randint(-6, 7, (b.tokens, 1, 1), generator=g).float())
    q, k, v = (((torch.randn(b.tokens, h, d, generator=g) * size)).to(dtype) for h in (q_heads, kv, kv))
    qn, kn = ((1 + 0.1 * torch.randn(d, generator=g)) if norm else None for _ in range(2))
    cos, sin = _rope_tables(max(c + n for c, n in lengths) + 3, d)
    rotated, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=page, q_norm=qn, k_norm=kn, eps=EPS,
                                   cos=cos, sin=sin)
    cache, batch = b.device()
    q_out = torch.full((b.tokens, q_heads, d), 77.0, device=DEV)
    ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=q_heads, q_norm=None if qn is None else qn.to(DEV),
                            k_norm=None if kn is None else kn.to(DEV), eps=EPS, cos=cos.to(DEV), sin=sin.to(DEV),
                            q_out=q_out, **batch)
    assert torch.equal(cache.k_scales.cpu().double(), expected["k_scales"])
    assert torch.equal(cache.v_scales.cpu().double(), expected["v_scales"])
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    written = ~torch.isnan(rotated[:, 0, 0])
    assert written.sum() == b.spans[-1][1] - 1  # all but the token ahead and those behind
    assert (q_out.cpu()[~written] == 77.0).all()
    # 8 roundings of the two products' sizes: their root sum is at most sqrt 2 of the pair's length.
    x = rotated[written]
    half = d // 2
    pair = torch.sqrt(x[..., :half].pow(2) + x[..., half:].pow(2)).repeat(1, 1, 2)
    assert ((q_out.cpu()[written].double() - x).abs() <= 8 * 2.0**-24 * 1.5 * pair).all()


def test_paged_append_stores_what_is_not_finite_as_nan():
    b = Batch([(2, 3)], kv=1, d=64, page=16, seed=8)
    q = torch.randn(3, 1, 64, generator=_g(1))
    k, v = torch.randn(3, 1, 64, generator=_g(2)), torch.randn(3, 1, 64, generator=_g(3))
    v[0, 0, 5], v[1, 0, 6], v[2, 0, 7] = math.inf, -math.inf, math.nan
    k[1, 0, 3] = math.inf
    cos, sin = torch.ones(8, 32), torch.zeros(8, 32)
    _, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=16, q_norm=None, k_norm=None, eps=0.0, cos=cos, sin=sin)
    cache, batch = b.device()
    ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=1, q_norm=None, k_norm=None, eps=0.0,
                            cos=cos.to(DEV), sin=sin.to(DEV), **batch)
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    assert torch.equal(cache.v_scales.cpu().double(), expected["v_scales"])


@pytest.mark.parametrize("size", [0.0, 1e-44, 1e-30, 1e38])
def test_paged_append_sizes(size):
    """Zeros, values below every scale, and values near the top of fp32."""

    b = Batch([(0, 5)], kv=2, d=64, page=16, seed=9)
    k, v = (size * (0.5 + torch.rand(5, 2, 64, generator=_g(s))) for s in (4, 5))
    cos, sin = torch.ones(8, 32), torch.zeros(8, 32)
    _, expected = osv.append(k, k, v, b.host(), b.table, b.spans, page=16, q_norm=None, k_norm=None, eps=0.0, cos=cos, sin=sin)
    cache, batch = b.device()
    ops.launch_paged_append(k.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=2, q_norm=None, k_norm=None, eps=0.0,
                            cos=cos.to(DEV), sin=sin.to(DEV), **batch)
    assert torch.equal(cache.k_scales.cpu().double(), expected["k_scales"])
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])


def test_paged_append_token_by_token_is_the_append_at_once():
    """The scale only grows and rows move by powers of two: one token at a time
    leaves the bytes of one call, but for values that a grown scale makes
    subnormal, which are rounded twice (at most a step of the subnormals apart)."""

    n, kv, d, page = 50, 2, 128, 32
    q, k, v = (torch.randn(n, h, d, generator=_g(s)) for h, s in ((4, 1), (kv, 2), (kv, 3)))
    cos, sin = (x.to(DEV) for x in _rope_tables(n, d))
    caches = []
    for parts in ([n], [1] * n, [7, 30, 13]):
        b = Batch([(0, n)], kv=kv, d=d, page=page, seed=10)
        cache, batch = b.device()
        at = 0
        for m in parts:
            batch["context_lens"].fill_(at)
            batch["query_starts"].copy_(torch.tensor([0, m], dtype=torch.int32))
            ops.launch_paged_append(q[at:at + m].to(DEV), k[at:at + m].to(DEV), v[at:at + m].to(DEV), cache, q_heads=4,
                                    q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin, **batch)
            at += m
        caches.append(cache)
        pages = b.table[0][:2]
    for other in caches[1:]:
        for name in ("k", "v"):
            assert torch.equal(getattr(other, name + "_scales"), getattr(caches[0], name + "_scales"))
            x, y = (getattr(c, name)[pages].cpu().view(torch.uint8).view(torch.float8_e4m3fn).float() for c in (other, caches[0]))
            if name == "v":
                x, y = x.transpose(2, 3), y.transpose(2, 3)
            x, y = (t.transpose(1, 2).reshape(2 * page, kv, d)[:n] for t in (x, y))
            assert ((x - y).abs() <= torch.where(y.abs() > 2.0**-6, 0.0, 2.0**-9)).all()


def test_paged_append_rows_without_a_place():
    """Negative rows, rows behind the table or the RoPE tables, table entries that
    name no page: nothing of the cache changes for them."""

    b = Batch([(-2, 5), (30, 6), (0, 2)], kv=1, d=64, page=16, seed=11, extra_entries=0)
    assert len(b.table[0]) == 3
    b.table[2][0] = 99  # no page
    q, k, v = (torch.randn(b.tokens, h, 64, generator=_g(s)) for h, s in ((2, 1), (1, 2), (1, 3)))
    cos, sin = _rope_tables(33, 64)  # rows 33, 34, 35 of the second sequence have none
    rotated, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=16, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin)
    cache, batch = b.device()
    out = ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=2, q_norm=None, k_norm=None, eps=EPS,
                                  cos=cos.to(DEV), sin=sin.to(DEV), q_out=torch.full((b.tokens, 2, 64), 5.0, device=DEV), **batch)
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])
    off = torch.isnan(rotated[:, 0, 0])
    assert off.tolist() == [True, True] + [False] * 6 + [True] * 3 + [False] * 2
    assert (out.cpu()[off] == 5.0).all()


# -- attention -------------------------------------------------------------------


def _filled(b: Batch, seed: int) -> None:
    """Numbers in the new tokens' rows too, as an append leaves them."""

    g = _g(seed)
    for i, (begin, end, context) in enumerate(b.spans):
        for row in range(max(0, context), context + end - begin):
            if row // b.page < len(b.table[i]) and 0 <= b.table[i][row // b.page] < b.k_bytes.shape[0]:
                at = b.table[i][row // b.page]
                for stored in (b.k_bytes[at, :, row % b.page, :], b.v_bytes[at, :, :, row % b.page]):
                    stored.copy_(torch.randint(0, 127, stored.shape, generator=g, dtype=torch.uint8)
                                 | (torch.randint(0, 2, stored.shape, generator=g, dtype=torch.uint8) << 7))


def _check_attention(got, expected, spread, reach, *, q_dtype, rows, d) -> None:
    parts = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[q_dtype]
    out_dtype = got.dtype
    got = got.cpu().double().view(expected.shape)
    nan = torch.isnan(expected)
    assert torch.equal(torch.isnan(got), nan)
    u = 2.0**-24
    relative = 2 * u * (parts * d + 8) * reach[..., None] + (u if out_dtype == torch.float32 else 2.0**-17) + u * (rows / 16 + 64)
    bound = relative * spread + HALF_STEP[out_dtype] * expected.abs() + 1e-30
    if out_dtype == torch.float16:
        bound = bound + 2.0**-25  # its subnormals
    error = (got - expected).abs()
    worst = float((error / bound)[~nan].max()) if (~nan).any() else 0.0
    assert worst <= 1, worst


ATTENTIONS = [
    # lengths, q heads, kv heads, head_dim, page
    ([(0, 1)], 4, 2, 64, 16),
    ([(600, 1)], 8, 2, 128, 64),
    ([(0, 1), (63, 1), (64, 1), (700, 1), (15, 1)], 8, 2, 128, 16),
    ([(130, 5), (0, 3), (77, 0), (1, 1)], 6, 2, 128, 32),
    ([(33, 40)], 5, 1, 64, 32),                # seven rows over a tile's edge
    ([(0, 130), (61, 70)], 8, 4, 128, 128),    # whole prompts
    ([(129, 2), (200, 1)], 34, 2, 64, 16),     # more heads to a group than an MFMA has columns
    ([(300, 17)], 4, 4, 256, 64),
    ([(5, 66)], 2, 2, 256, 16),
    # Caches long enough to be split, few query rows and many.
    ([(1500, 1), (20, 1)], 8, 2, 128, 64),
    ([(1300, 6), (40, 2), (0, 1)], 8, 2, 128, 32),
    ([(900, 3), (1000, 1)], 8, 2, 256, 64),
    ([(1100, 40)], 4, 1, 64, 32),
    ([(1000, 30)], 4, 2, 256, 16),
]


@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float32), (torch.float32, torch.float16)])
@pytest.mark.parametrize("lengths,q_heads,kv,d,page", ATTENTIONS)
def test_paged_attention(lengths, q_heads, kv, d, page, q_dtype, out_dtype):
    _say("attention", lengths, q_heads, kv, d, page, q_dtype, out_dtype)
    b = Batch(lengths, kv=kv, d=d, page=page, seed=12, ahead=1, behind=2)
    _filled(b, 13)
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, q_heads, d, generator=_g(14)).to(q_dtype)
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    cache, batch = b.device()
    out = torch.full((b.tokens, q_heads * d), 9.0, dtype=out_dtype, device=DEV)
    ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out=out, **batch)
    mine = ~torch.isnan(expected[:, 0, 0])
    assert mine.sum() == b.spans[-1][1] - 1
    assert (out.cpu()[~mine] == 9.0).all()
    rows = max(c + n for c, n in lengths)
    _check_attention(out[mine.to(DEV)], expected[mine], spread[mine], reach[mine], q_dtype=q_dtype, rows=rows, d=d)
    again = ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out_dtype=out_dtype, **batch)
    assert torch.equal(again[mine.to(DEV)], out[mine.to(DEV)])  # a fixed order


@pytest.mark.parametrize("batch,kv,d,page,extra", [(140, 2, 64, 16, 0), (140, 2, 128, 64, 40), (70, 4, 64, 128, 100),
                                                   (150, 1, 128, 16, 3), (200, 2, 256, 16, 1)])
def test_paged_attention_many_sequences(batch, kv, d, page, extra):
    """More sequences than a wave looks up at once, enough to fill the chip, with
    page tables much wider than the caches."""

    _say("many sequences", batch, kv, d, page, extra)
    g = _g(60)
    lengths = [(int(c), int(n)) for c, n in zip(torch.randint(0, 90, (batch,), generator=g), torch.randint(0, 3, (batch,), generator=g))]
    lengths[batch // 2] = (600, 1)
    b = Batch(lengths, kv=kv, d=d, page=page, seed=61, extra_entries=extra)
    _filled(b, 62)
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, 2 * kv, d, generator=_g(63)).to(torch.bfloat16)
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    cache, at = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out_dtype=torch.float32, **at)
    _check_attention(out, expected, spread, reach, q_dtype=torch.bfloat16, rows=601, d=d)


def test_paged_append_many_sequences():
    g = _g(64)
    lengths = [(int(c), int(n)) for c, n in zip(torch.randint(0, 40, (4200,), generator=g), torch.randint(0, 3, (4200,), generator=g))]
    b = Batch(lengths, kv=1, d=64, page=16, seed=65)
    q, k, v = (torch.randn(b.tokens, 1, 64, generator=_g(s)) for s in (66, 67, 68))
    cos, sin = _rope_tables(48, 64)
    _, expected = osv.append(q, k, v, b.host(), b.table, b.spans, page=16, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin)
    cache, at = b.device()
    ops.launch_paged_append(q.to(DEV), k.to(DEV), v.to(DEV), cache, q_heads=1, q_norm=None, k_norm=None, eps=EPS,
                            cos=cos.to(DEV), sin=sin.to(DEV), **at)
    assert torch.equal(cache.k_scales.cpu().double(), expected["k_scales"])
    _same_bytes(cache.k, expected["k"])
    _same_bytes(cache.v, expected["v"])


@pytest.mark.parametrize("lengths", [[(70, 1)], [(200, 30)], [(18, 5)], [(20, 1)]])
def test_paged_attention_scales_of_any_kind(lengths):
    """A cache from elsewhere: scales that are no powers of two, and zeros, also in
    the last page."""

    b = Batch(lengths, kv=2, d=128, page=16, seed=69)
    _filled(b, 70)
    b.scales = 0.01 * torch.rand(b.scales.shape, generator=_g(71))
    b.scales[:, b.table[0][1]] = 0.0
    q = torch.randn(b.tokens, 4, 128, generator=_g(72))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=16, scaling=0.1)
    cache, at = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, out_dtype=torch.float32, **at)
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=230, d=128)


def test_paged_attention_every_byte_is_its_value():
    """One row a query attends alone gives that row's value back: all 256 bytes."""

    d, page = 256, 16
    b = Batch([(0, 1)], kv=1, d=d, page=page, seed=15)
    at = b.table[0][0]
    b.k_bytes[at] = 0
    b.v_bytes[at, 0, :, 0] = torch.arange(256, dtype=torch.uint8)
    b.scales[1] = 2.0**-4
    cache, batch = b.device()
    out = ops.launch_paged_attention(torch.randn(1, 1, d, generator=_g(1)).to(DEV), cache, scaling=1.0,
                                     out_dtype=torch.float32, **batch)
    expected = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float() * 2.0**-4
    nan = torch.isnan(expected)
    assert torch.equal(torch.isnan(out[0].cpu()), nan)
    assert torch.equal(out[0].cpu()[~nan], expected[~nan])


@pytest.mark.parametrize("batch,d,new", [(63, 64, (0, 1, 1, 3)), (64, 128, (1, 0, 9, 2, 33)), (64, 256, (6, 1, 0, 4, 9)),
                                         (65, 64, (0, 1, 9, 2)), (5, 64, (40, 0, 25, 18, 50)), (5, 256, (30, 0, 25, 18, 50)),
                                         (129, 64, (0, 1, 1, 9)), (200, 128, (1, 1, 0, 1)), (4098, 64, (1, 0, 0, 0, 0, 0, 2))])
def test_paged_attention_uneven_batches(batch, d, new):
    """Sequences without tokens or rows, of one slot and several, among ones that are split."""

    _say("uneven", batch, d, new)
    contexts = (700, 0, 33, 2000 if batch < 6 else 900, 1) if batch < 1000 else (20, 0, 33, 9, 1)
    lengths = [(contexts[i * i % 5] if i % 3 else 0, new[i % len(new)]) for i in range(batch - 1)] + [(1200, new[0])]
    b = Batch(lengths, kv=2, d=d, page=32, seed=83, ahead=2, behind=1)
    _filled(b, 84)
    b.scales *= 2.0**-3
    q = torch.randn(b.tokens, 8, d, generator=_g(85)).to(torch.bfloat16)
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=32, scaling=d**-0.5)
    cache, at = b.device()
    out = torch.full((b.tokens, 8 * d), 9.0, dtype=torch.float32, device=DEV)
    ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out=out, **at)
    mine = ~torch.isnan(expected[:, 0, 0])
    assert (out.cpu()[~mine] == 9.0).all()
    rows = max(c + n for c, n in lengths)
    _check_attention(out[mine.to(DEV)], expected[mine], spread[mine], reach[mine], q_dtype=torch.bfloat16, rows=rows, d=d)


@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float32)])
@pytest.mark.parametrize("what", ["numbers", "k", "v", "scales"])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attention_chunks_under_a_very_wide_table(d, what, q_dtype, out_dtype):
    """Slots whose waves have rows of their own, split and not, with NaN that some of
    their rows see and with scales that are no powers of two."""

    _say("wide table", d, what, q_dtype, out_dtype)
    page, lengths = 128, [(2600, 70), (0, 41), (100, 130)]
    b = Batch(lengths, kv=2, d=d, page=page, seed=86, ahead=1, behind=1, extra_entries=110)
    _filled(b, 87)
    b.scales *= 2.0**-3
    if what == "k":
        b.k_bytes[b.table[0][2620 // page], 1, 2620 % page, 3] = 0x7f
    if what == "v":
        b.v_bytes[b.table[0][2620 // page], 0, d - 5, 2620 % page] = 0xff
        b.v_bytes[b.table[2][0], 1, 7, 101] = 0x7f
    if what == "scales":
        b.scales *= 1 + torch.rand(b.scales.shape, generator=_g(88))
    q = torch.randn(b.tokens, 8, d, generator=_g(89)).to(q_dtype)
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    cache, at = b.device()
    out = torch.full((b.tokens, 8 * d), 9.0, dtype=out_dtype, device=DEV)
    ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out=out, **at)
    mine = torch.arange(b.tokens)[1:-1]
    assert (out[0] == 9.0).all() and (out[-1] == 9.0).all()
    assert torch.isnan(expected[mine]).any() == (what in ("k", "v"))
    _check_attention(out[mine.to(DEV)], expected[mine], spread[mine], reach[mine], q_dtype=q_dtype, rows=2670, d=d)


@pytest.mark.parametrize("rise", [0.5, 2.0, 4.0, 5.0, -3.0])
@pytest.mark.parametrize("tokens,extra", [(1, 1), (9, 1), (70, 250)])
def test_paged_attention_scores_that_rise_from_tile_to_tile(tokens, extra, rise):
    """By less than a running maximum may lag behind, and by more."""

    d, page = 64, 64
    b = Batch([(1000, tokens)], kv=1, d=d, page=page, seed=90, extra_entries=extra)
    _filled(b, 91)
    b.k_bytes.zero_()
    b.scales[0] = 1.0
    for i, at in enumerate(b.table[0][:-(-(1000 + tokens) // page)]):
        b.k_bytes[at, :, :, 0] = torch.tensor(min(i, 16), dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    q = torch.randn(tokens, 4, d, generator=_g(92))
    q[:, :, 0] = rise
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=1.0)
    cache, at = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=1.0, out_dtype=torch.float32, **at)
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=1000 + tokens, d=d)


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("lengths,row", [([(0, 70)], 40), ([(90, 6)], 93), ([(10, 3)], 12), ([(200, 2)], 17)])
def test_paged_attention_nan_reaches_those_who_see_it(lengths, row, what):
    d, page, kv = 128, 16, 2
    b = Batch(lengths, kv=kv, d=d, page=page, seed=16)
    _filled(b, 17)
    at = b.table[0][row // page]
    if what == "k":
        b.k_bytes[at, 1, row % page, 3] = 0x7f
    else:
        b.v_bytes[at, 1, 77, row % page] = 0xff
    q = torch.randn(b.tokens, 4, d, generator=_g(18))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=0.01)
    cache, batch = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=0.01, out_dtype=torch.float32, **batch)
    assert torch.isnan(expected).any()
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=300, d=d)


def test_paged_attention_infinite_and_nan_queries_stay_their_own():
    d, page = 64, 16
    b = Batch([(40, 3)], kv=1, d=d, page=page, seed=19)
    _filled(b, 20)
    q = torch.randn(3, 2, d, generator=_g(21))
    q[0, 0, 5], q[1, 1, 6], q[2, 0, 7] = math.inf, math.nan, -math.inf
    cache, batch = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, out_dtype=torch.float32, **batch).cpu().view(3, 2, d)
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=0.1)
    for t, h in ((0, 1), (1, 0), (2, 1)):
        _check_attention(out[t, h], expected[t, h], spread[t, h], reach[t, h], q_dtype=torch.float32, rows=43, d=d)
    for t, h in ((0, 0), (1, 1), (2, 0)):
        assert torch.isnan(out[t, h]).all()


@pytest.mark.parametrize("magnitude", [1e-30, 1e-3, 300.0])
def test_paged_attention_query_magnitudes(magnitude):
    d, page = 128, 32
    b = Batch([(150, 2)], kv=1, d=d, page=page, seed=25)
    _filled(b, 26)
    b.scales[0] = 2.0**-9
    q = magnitude * torch.randn(2, 4, d, generator=_g(27))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=d**-0.5)
    cache, batch = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=d**-0.5, out_dtype=torch.float32, **batch)
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=152, d=d)


def test_paged_attention_light_rows_beside_a_heavy_one():
    """Rows of weight e^-12 whose values are 2^14 times the heavy row's."""

    d, page = 64, 64
    b = Batch([(190, 1)], kv=1, d=d, page=page, seed=28)
    pages = b.table[0][:3]
    for at in pages:
        b.k_bytes[at] = 0x00
        b.v_bytes[at] = 0x78  # 256
    b.k_bytes[pages[0], 0, 0, 0] = 0x38
    b.v_bytes[pages[0], 0, :, 0] = 0x08  # 2^-6
    b.scales[:] = 1.0
    q = torch.zeros(1, 1, d)
    q[0, 0, 0] = 12.0
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=page, scaling=1.0)
    cache, batch = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=1.0, out_dtype=torch.float32, **batch)
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=191, d=d)


def test_paged_attention_rows_outside_the_table_and_missing_pages():
    b = Batch([(-1, 3), (30, 4), (20, 1)], kv=1, d=64, page=16, seed=29, extra_entries=0)
    b.table = [row[:2] for row in b.table]  # rows 32, 33 of the second sequence have no entry
    _filled(b, 30)
    b.table[2][0] = -5  # rows that no page holds
    q = torch.randn(b.tokens, 2, 64, generator=_g(31))
    expected, spread, reach = osv.attention(q, b.host(), b.table, b.spans, page=16, scaling=0.1)
    cache, batch = b.device()
    out = ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, out_dtype=torch.float32, **batch)
    assert (out.cpu()[[0, 5, 6]] == 0).all() and torch.isnan(out[7]).all()
    _check_attention(out, expected, spread, reach, q_dtype=torch.float32, rows=32, d=64)


def test_starts_out_of_order_stay_in_bounds():
    """Starts that fall, lie outside the tokens or before them name no token twice
    outside the buffers; outputs of such a batch are unspecified."""

    b = Batch([(0, 8), (3, 8), (0, 8)], kv=1, d=64, page=16, seed=32)
    q = torch.randn(24, 1, 64, generator=_g(33), dtype=torch.float32)
    cos, sin = (x.to(DEV) for x in _rope_tables(32, 64))
    for starts in ([5, -3, 900, 2], [24, 16, 8, 0], [0, 0, 0, 2**31 - 1], [-9, -8, -7, -6]):
        _say("starts", starts)
        cache, batch = b.device()
        batch["query_starts"].copy_(torch.tensor(starts, dtype=torch.int32))
        ops.launch_paged_append(q.to(DEV), q.to(DEV), q.to(DEV), cache, q_heads=1, q_norm=None, k_norm=None, eps=EPS,
                                cos=cos, sin=sin, **batch)
        ops.launch_paged_attention(q.to(DEV), cache, scaling=0.1, **batch)
        torch.cuda.synchronize()


# -- log probabilities -------------------------------------------------------------


def _check_logprobs(got, logits, tokens, top) -> None:
    lp, h, ids, tops = osv.token_logprobs(logits.cpu(), tokens.cpu(), top)
    x = logits.cpu().double()
    p = torch.softmax(x, -1)
    d = torch.where(p > 0, x - x.amax(-1, keepdim=True), 0.0).abs()
    e1, e2 = (p * d).sum(-1), (p * d * d).sum(-1)
    u = 2.0**-24
    log_s = u * (96 + 4 * e1)
    for name, value, expected, bound in (
            ("logprobs", got.logprobs, lp, log_s + u * lp.abs()),
            ("entropy", got.entropy, h, log_s + u * (96 * e1 + 4 * e2) + e1 * log_s + u * h.abs()),
            ("top", got.top_logprobs, tops, log_s[:, None] + u * tops.abs())):
        value = value.cpu().double()
        nan = torch.isnan(expected)
        assert torch.equal(torch.isnan(value), nan), name
        low = expected == -math.inf
        assert torch.equal(value == -math.inf, low), name
        ok = ~nan & ~low
        assert ((value - expected).abs()[ok] <= bound[ok]).all(), (name, float((value - expected).abs()[ok].max()))
    assert torch.equal(got.top_ids.cpu(), ids)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 5, 3), (3, 63, 32), (2, 2048, 20), (5, 2055, 1), (1, 50257, 32),
                                            (4, 8191, 0), (130, 8200, 7)])
def test_token_logprobs(rows, vocab, top, dtype):
    _say("logprobs", rows, vocab, top, dtype)
    x = (2.5 * torch.randn(rows, vocab, generator=_g(40))).to(dtype)
    tokens = torch.randint(vocab, (rows,), generator=_g(41))
    _check_logprobs(ops.launch_token_logprobs(x.to(DEV), tokens.to(DEV), top=top), x, tokens, top)


def test_token_logprobs_large_parts():
    """Enough rows that a lane takes 32 values; ties in plenty (16-bit logits of few values)."""

    x = torch.randint(-3, 4, (600, 9001), generator=_g(42)).to(torch.bfloat16)
    tokens = torch.randint(9001, (600,), generator=_g(43))
    got = ops.launch_token_logprobs(x.to(DEV), tokens.to(DEV), top=20)
    pick = torch.tensor([0, 1, 299, 598, 599])
    part = ops.TokenLogprobs(*(t.cpu()[pick] for t in got))
    _check_logprobs(part, x[pick], tokens[pick], 20)


@pytest.mark.parametrize("stride,offset", [(1000, 0), (1003, 1), (1021, 5)])
def test_token_logprobs_rows_apart(stride, offset):
    flat = torch.randn(7 * stride + offset, generator=_g(44)).to(torch.bfloat16).to(DEV)
    x = flat[offset:].as_strided((7, 997), (stride, 1), offset)
    tokens = torch.randint(997, (7,), generator=_g(45))
    _check_logprobs(ops.launch_token_logprobs(x, tokens.to(DEV), top=5), x, tokens, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_ties_in_plenty(dtype):
    """More equal values than are ranked at once: the lowest ids come first, also
    where the values above them lie behind."""

    vocab = 40003
    x = torch.zeros(7, vocab)
    x[1, 39990:40000] = 1.0                        # a few above, at the end
    x[2, ::2] = -math.inf                          # every other banned
    x[3] = torch.randint(-2, 3, (vocab,), generator=_g(47)).float()
    x[4] = -math.inf
    x[4, 17::1024] = 2.0                           # one to a block of 1024, and these alone
    x[5, 5:] = -math.inf                           # five equal ones, the rest banned
    x[6] = torch.arange(vocab) // 2000             # steps
    x = x.to(dtype)
    tokens = torch.tensor([0, 1, 3, 4, 17, 2, vocab - 1])
    for top in (1, 20, 32):
        _check_logprobs(ops.launch_token_logprobs(x.to(DEV), tokens.to(DEV), top=top), x, tokens, top)


def test_token_logprobs_special_rows():
    x = torch.randn(12, 5000, generator=_g(46))
    x[0, :4990] = -math.inf                 # few tokens allowed
    x[1, :] = -math.inf                     # none
    x[2, 1234] = math.nan
    x[3, 99] = math.inf
    x[4, :] = 1.5                           # all equal: the lowest ids
    x[5, ::2] = 0.0
    x[5, 1::2] = -0.0                       # equal too
    x[6, 2500:] = -math.inf
    x[7, 4321] = 90.0                       # nearly certain
    x[8, :] = torch.arange(5000) * 0.01     # the largest in one place
    x[9, :] = -torch.arange(5000) * 0.01
    x[10, 17] = -math.nan
    x[11, 1:] = -math.inf                   # certain: entropy 0
    tokens = torch.tensor([4995, 3, 5, 6, 7, 8, 4000, 4321, 4999, 5000, -1, 0])
    got = ops.launch_token_logprobs(x.to(DEV), tokens.to(DEV), top=32)
    _check_logprobs(got, x, tokens, 32)
    assert got.logprobs[11] == 0 and got.entropy[11] == 0
    assert got.top_ids[1].tolist() == list(range(32)) == got.top_ids[4].tolist() == got.top_ids[5].tolist()


# -- together ------------------------------------------------------------------------


def test_a_captured_serving_step_replays_with_other_lengths():
    """Append, attention and log probabilities captured once; every replay, with
    other lengths and pages, is the eager call."""

    kv, d, page, heads = 2, 128, 16, 8
    b = Batch([(100, 1), (31, 1), (0, 1)], kv=kv, d=d, page=page, seed=50, extra_entries=4, spare=12)
    spare = [i for i in range(b.k_bytes.shape[0]) if not any(i in row for row in b.table)]
    for row in b.table:
        row[row.index(-7)] = spare.pop()
    cache, batch = b.device()
    eager_cache, _ = b.device()
    cos, sin = (x.to(DEV) for x in _rope_tables(200, d))
    q, k, v = (torch.randn(3, h * d, generator=_g(s)).to(DEV) for h, s in ((heads, 52), (kv, 53), (kv, 54)))
    tokens = torch.tensor([1, 2, 3], device=DEV)

    def step(c):
        rotated = ops.launch_paged_append(q, k, v, c, q_heads=heads, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin, **batch)
        x = ops.launch_paged_attention(rotated, c, scaling=d**-0.5, out_dtype=torch.float32, **batch)
        return x, ops.launch_token_logprobs(x, tokens, top=4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, lp = step(cache)
    step(eager_cache)
    for i in range(5):
        batch["context_lens"].add_(1)
        q.add_(0.1)
        v.mul_(1.3)
        graph.replay()
        torch.cuda.synchronize()
        ex, elp = step(eager_cache)
        torch.cuda.synchronize()
        assert torch.equal(x, ex), i
        for got, expected in zip(lp, elp):
            assert torch.equal(got, expected), i
        assert torch.equal(cache.k.view(torch.uint8), eager_cache.k.view(torch.uint8))
        assert torch.equal(cache.v.view(torch.uint8), eager_cache.v.view(torch.uint8))


def test_offsets_beyond_32_bits():
    """Pages that lie more than 2^32 bytes into the pool."""

    kv, d, page, pages = 8, 128, 64, 66000
    k = torch.empty(pages, kv, page, d, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.empty(pages, kv, d, page, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.ones(2, pages, kv, device=DEV)
    far = ops.PagedCache(k, v, scales[0], scales[1])
    near = ops.paged_cache(4, kv, page, d, DEV)
    q, kn, vn = (torch.randn(70, h * d, generator=_g(s)).to(DEV) for h, s in ((16, 73), (kv, 74), (kv, 75)))
    cos, sin = (x.to(DEV) for x in _rope_tables(80, d))
    out = []
    for cache, table in ((far, [65999, 65990]), (near, [3, 1])):
        at = {"page_table": torch.tensor([table], dtype=torch.int32, device=DEV),
              "query_starts": torch.tensor([0, 70], dtype=torch.int32, device=DEV),
              "context_lens": torch.zeros(1, dtype=torch.int32, device=DEV)}
        rotated = ops.launch_paged_append(q, kn, vn, cache, q_heads=16, q_norm=None, k_norm=None, eps=EPS, cos=cos, sin=sin, **at)
        out.append(ops.launch_paged_attention(rotated, cache, scaling=0.1, **at))
        out.append(ops.launch_paged_attention(rotated[69:], cache, scaling=0.1, **{
            **at, "query_starts": torch.tensor([0, 1], dtype=torch.int32, device=DEV),
            "context_lens": torch.full((1,), 69, dtype=torch.int32, device=DEV)}))
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])
    del k, v, far
    stride = (1 << 31) + 5
    wide = torch.empty(2 * stride, dtype=torch.bfloat16, device=DEV).as_strided((2, 5000), (stride, 1))
    rows = torch.randn(2, 5000, generator=_g(76)).to(torch.bfloat16)
    wide.copy_(rows)
    tokens = torch.tensor([4999, 3])
    _check_logprobs(ops.launch_token_logprobs(wide, tokens.to(DEV), top=8), rows, tokens, 8)


def test_work_on_another_stream():
    b = Batch([(100, 30)], kv=2, d=64, page=16, seed=55)
    _filled(b, 56)
    q = torch.randn(30, 4, 64, generator=_g(57)).to(DEV)
    cache, batch = b.device()
    here = ops.launch_paged_attention(q, cache, scaling=0.1, **batch)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = ops.launch_paged_attention(q, cache, scaling=0.1, **batch)
        lp = ops.launch_token_logprobs(there.float(), torch.zeros(30, dtype=torch.int64, device=DEV), top=2)
    side.synchronize()
    assert torch.equal(here, there)
    assert torch.equal(lp.top_ids, ops.launch_token_logprobs(here.float(), torch.zeros(30, dtype=torch.int64, device=DEV), top=2).top_ids)


# -- the decoder ---------------------------------------------------------------------

SMALL = DecoderShellConfig(layers=3, hidden=256, intermediate=768, q_heads=4, kv_heads=2, head_dim=64, vocab=1000)


def _decoder(act, **arguments):
    weights = syn.synthetic_decoder(SMALL, seed=syn.BASE_SEED + 81, random_norms=True)
    return weights, PackedDecoder(SMALL, weights, device=DEV, max_positions=150, activation_dtype=act,
                                  cache_dtype=torch.float8_e4m3fn, **arguments)


def test_decoder_with_the_8_bit_cache_matches_the_oracle():
    """Logits against the oracle decoder with the same cache, teacher-forced. The
    linears differ by 2e-5 relative, which moves about 16 * 2e-5 of the stored
    values to the neighbouring e4m3 value, 1/8 away at most: sqrt(3.2e-4) / 8 =
    2.2e-3 of K and of V, and over three layers sqrt(3) * 2 * 2.2e-3 = 8e-3."""

    weights, decoder = _decoder(torch.float32)
    prompt = torch.randint(0, SMALL.vocab, (70,), generator=_g(81))
    tokens = decoder.generate_greedy(prompt.to(DEV), 8, use_graph=False).tolist()
    geometry = ods.ShellGeometry(SMALL.layers, SMALL.hidden, SMALL.intermediate, SMALL.q_heads, SMALL.kv_heads,
                                 SMALL.head_dim, SMALL.vocab, SMALL.eps, SMALL.rope_theta)
    ow = ods.ShellWeights(weights.embed, weights.lm_head, weights.final_norm,
                          [ods.LayerWeights(l.input_norm, l.post_norm, l.q_norm, l.k_norm,
                                            {r: operands_from_state(st) for r, st in l.linears.items()})
                           for l in weights.layers])
    oracle = osv.PagedOracleDecoder(geometry, ow, max_positions=150, page=PAGE_ROWS)
    expected = [oracle.forward(prompt, 0)[-1]]
    for i, token in enumerate(tokens[:-1]):
        expected.append(oracle.forward(torch.tensor([token]), 70 + i)[-1])
    decoder.reset()
    got = [decoder.prefill(prompt.to(DEV)).cpu().clone()]
    for i, token in enumerate(tokens[:-1]):
        got.append(decoder.prefill(torch.tensor([token]), start=70 + i).cpu().clone())
    for step, (a, e) in enumerate(zip(got, expected)):
        assert relative_l2(a, e) < 8e-3, step
        assert int(a.argmax()) == tokens[step]


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fuse", [True, False])
def test_decoder_with_the_8_bit_cache_graph_and_eager_agree(act, fuse):
    _, decoder = _decoder(act, fuse_decode=fuse)
    prompt = torch.randint(0, SMALL.vocab, (60,), generator=_g(82)).to(DEV)
    eager = decoder.generate_greedy(prompt, 21, use_graph=False).tolist()
    assert decoder.generate_greedy(prompt, 21).tolist() == eager
    tokens, scores = decoder.generate_greedy_scored(prompt, 21, top=3)
    assert tokens.tolist() == eager
    eager_tokens, eager_scores = decoder.generate_greedy_scored(prompt, 21, top=3, use_graph=False)
    assert eager_tokens.tolist() == eager
    for a, b in zip(scores, eager_scores):
        assert torch.equal(a, b)
    assert torch.equal(scores.top_ids[:, 0], tokens)
    assert torch.equal(scores.top_logprobs[:, 0], scores.logprobs)


@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float32])
def test_decoder_scores_a_text_as_its_logits_do(cache):
    weights = syn.synthetic_decoder(SMALL, seed=syn.BASE_SEED + 83, random_norms=True)
    decoder = PackedDecoder(SMALL, weights, device=DEV, max_positions=300, activation_dtype=torch.float32, cache_dtype=cache)
    ids = torch.randint(0, SMALL.vocab, (290,), generator=_g(83))
    got = decoder.score(ids, top=5)
    assert torch.equal(decoder.logits, decoder.prefill(ids))
    logits = []
    _, buffers = decoder._prefill(ids, 0)
    for row in range(289):
        logits.append(ops.launch_output_projection(buffers.final[row], decoder.lm_head)[0])
    _check_logprobs(got, torch.stack(logits), ids[1:], 5)
    with pytest.raises(DecoderShellError):
        decoder.score(ids[:1])
    with pytest.raises(DecoderShellError):
        decoder.score(ids, top=33)
