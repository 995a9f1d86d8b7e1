// Causal grouped-query attention over an 8-bit paged cache (layout: nq_paged.hip).
//
// A query row is one (token, q head) of a kv head's group: row r of a sequence
// is token r / group, head r % group, so that the rows which share a kv head
// fill the 16 columns of v_mfma_f32_16x16x32_bf16 whatever the group. Per TILE
// cache rows a wave forms S^T = K Q^T (A = 16 cache rows, B = 16 query rows),
// a running softmax over its columns, and O^T += V^T P^T. S^T leaves a lane
// with TILE / 4 cache rows of one query row; assigning cache row TILE / 4 g + 4 t
// + i to row 4 g + i of the t-th score tile makes them consecutive rows, which is
// what the second product's B operand wants, so P never leaves its registers.
// V lies transposed in the cache, so its A operand is as many consecutive bytes.
//
// Precision: an e4m3 byte is exact in bf16 and in fp16. bf16 and fp16 queries
// enter as they are; an fp32 query row enters as two fp16 parts after a power of
// two that brings its largest value to 2^14..2^15. The second part holds 2^12 times
// what the first leaves, and meets K times 2^-12, so that it has 11 bits of its own
// however small the value is: together they are within 2^-23 of every value down to
// 2^-28 of the largest (three values in four are exact), and within 2^-51 of the
// largest below. Unscaled, the second part would be subnormal from 2^-16 of the
// largest down and leave 15 bits at 2^-24, 11 at 2^-28; scaling it costs prompts 5%
// (1531 tokens after 517: 102.6 us, 97 unscaled), single tokens nothing. The
// weights enter the second product as two bf16 parts (16 bits, 2^-17 of a weight
// at most) for 16-bit outputs, whose own rounding is 2^-9 or 2^-12, and as three
// for fp32 outputs. Scales: K's multiplies the fp32 score; V's goes into the
// widening of its bytes (a power of two; any other multiplies the fp32 weight).
#pragma once

#include "nq_paged.h"

namespace nq {
namespace paged {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;  // cache rows that splits are counted in
constexpr float kSlack = 6.0f;  // what weights are relative to lies this far above a new maximum

struct AttnArgs {
    Pages p;
    const void* q;
    void* out;
    float* partial;    // [items][kv_heads][rows][2] (max, sum), then the same of [head_dim]
    float* partial_o;
    float scale;       // scaling * log2(e): scores are kept in base 2
    int32_t out_dtype, q_heads, group, slots, splits, least;  // least: cache tiles a split takes at least
};

// A call whose sequences hold the same first rows, or that wants each row's
// log-sum-exp. Workgroups [0, blocks) take the shared rows [0, skip), a multiple of
// the page and of kTile, for the query rows of all sequences together; the others take what lies
// behind them, sequence by sequence. All leave their shares to the join, the shared ones' behind
// the others' slots * splits items.
struct SharedArgs : AttnArgs {
    float* lse;                          // [tokens][q_heads], may be null
    int32_t skip, blocks, shared_splits, shared_per;  // shared_per: tiles of a split of the shared rows
};

template <bool SEGMENTS>
using ArgsOf = std::conditional_t<SEGMENTS, SharedArgs, AttnArgs>;

// Cache tiles of each split, and splits that have any, of a sequence whose last
// token sees `visible` rows.
struct SplitPlan {
    int per, active;
};

__device__ __forceinline__ SplitPlan split_plan(int visible, int splits, int least) {
    if (splits == 1) return {0x1ffffff, 1};
    const int tiles = (visible + kTile - 1) / kTile;
    const int per = max((tiles + splits - 1) / splits, least);
    return {per, max((tiles + per - 1) / per, 1)};
}

// A sequence's share of the work: items of `rows` query rows (a slot) and one of
// its splits, the splits of a slot next to each other.
struct Work {
    Found f;
    SplitPlan plan;
    int64_t first, local;  // the sequence's first item; the item's (a token's slot's first item's) place in it
};

// The work that item `at`, or (TOKEN) token `at` and its q head `head` of a group,
// belongs to. Up to 64 sequences' items follow each other without gaps, a lane
// counting each sequence's: workgroups go to the chip's dies and to their parts in
// turn, so that empty ones among the others leave parts with nothing to do
// (16 ragged sequences of up to 6 tokens after 3000 rows: 21.3 us, 30.8 with
// the search's empty ones; 16 of 12 tokens: 41, 58). More sequences have one slot
// more each than they may need, and all of a slot's splits, found by search (256 of
// up to 1000 rows: 73 us; counted in two rounds 77).
// Cache rows before `skip` are not these items'.
template <bool TOKEN>
__device__ __forceinline__ Work find(const Pages& p, int64_t at, int head, int group, int rows, int splits, int least,
                                     int skip = 0) {
    const int cache_rows = (p.table_pages << p.page_shift) - skip;
    const auto plan_of = [&](int context, int begin, int end) {
        const int64_t seen = static_cast<int64_t>(context) + (end - begin) - skip;
        return split_plan(static_cast<int>(min(max(seen, int64_t{0}), static_cast<int64_t>(cache_rows))), splits, least);
    };
    Work w;
    int stride;
    if (p.batch > kWave) {
        const auto slot_of = [&](int i, int begin) { return static_cast<int64_t>(begin) * group / rows + i; };
        const int64_t slot = TOKEN ? at : static_cast<uint32_t>(at) / static_cast<uint32_t>(splits);
        w.f = sequence_at(p, slot, [&](int i, int begin) { return TOKEN ? static_cast<int64_t>(begin) : slot_of(i, begin); });
        w.plan = plan_of(w.f.context, w.f.span.begin, w.f.span.end);
        w.first = slot_of(w.f.b, w.f.span.begin) * splits;
        stride = splits;
    } else {
        const int lane = threadIdx.x & (kWave - 1), b = min(lane, p.batch - 1);
        const int start = p.starts[b], stop = p.starts[b + 1], context = p.contexts[b];
        const int begin = min(max(start, 0), p.tokens), end = min(max(stop, begin), p.tokens);
        const SplitPlan plan = plan_of(context, begin, end);
        const uint32_t slots = static_cast<uint32_t>((end - begin) * group + rows - 1) / static_cast<uint32_t>(rows);
        const uint32_t count = lane < p.batch ? slots * plan.active : 0, upto = running_sum(count);
        // Of a prompt's rows the last see the most: the last items go first.
        if (!TOKEN) at = static_cast<uint32_t>(__builtin_amdgcn_readlane(upto, kWave - 1)) - 1 - at;
        const uint64_t before = __ballot(lane < p.batch && (TOKEN ? begin <= at : static_cast<int64_t>(upto) <= at));
        const int hit = TOKEN ? (before ? 63 - __builtin_clzll(before) : 0) : min(__popcll(before), p.batch - 1);
        const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, hit); };
        w.f = {hit, of(context), {of(begin), of(end)}};
        w.plan = {of(plan.per), of(plan.active)};
        w.first = static_cast<uint32_t>(of(static_cast<int>(upto - count)));
        stride = w.plan.active;
    }
    if constexpr (TOKEN) {
        const uint32_t row = static_cast<uint32_t>(max(static_cast<int>(at) - w.f.span.begin, 0)) * group + head;
        w.local = static_cast<int64_t>(row / static_cast<uint32_t>(rows)) * stride;
    } else {
        w.local = at - w.first;
    }
    return w;
}

// What a slot of a sequence, from query row `row0` on, holds.
struct SlotSpan {
    int b, begin, context;  // sequence, its first token, rows cached before the call
    int row0, rows;         // the slot's first query row in its sequence; rows it holds
    int visible;            // cache rows [0, visible) that some row of the slot sees
};

__device__ __forceinline__ SlotSpan slot_span(const Pages& p, const Found& f, int64_t row0, int group, int rows) {
    SlotSpan o;
    o.b = f.b;
    o.begin = f.span.begin;
    o.context = f.context;
    const int64_t all = static_cast<int64_t>(f.span.end - f.span.begin) * group;
    o.row0 = static_cast<int>(row0 < 0 || row0 >= all ? 0 : row0);
    o.rows = static_cast<int>(row0 < 0 || row0 >= all ? 0 : min(static_cast<int64_t>(rows), all - row0));
    const int64_t last = static_cast<int64_t>(o.context) + (o.row0 + o.rows - 1) / group;
    o.visible = o.rows == 0 || last < 0
                    ? 0 : static_cast<int>(min(last + 1, static_cast<int64_t>(p.table_pages) << p.page_shift));
    return o;
}

// The sequence of a token, for each lane its own: the last one that begins at or
// before it. With starts that are not in order some sequence comes out; its span
// decides whether it has the token.
__device__ __forceinline__ Found lane_sequence(const Pages& p, int token) {
    const auto span_of = [&](int b) {
        const int start = p.starts[b], stop = p.starts[b + 1];
        const int begin = min(max(start, 0), p.tokens);
        return Span{begin, min(max(stop, begin), p.tokens)};
    };
    if (p.batch <= kWave) {
        const int b = min(static_cast<int>(threadIdx.x & (kWave - 1)), p.batch - 1), context = p.contexts[b];
        const Span span = span_of(b);
        int hit = 0;
#pragma unroll
        for (int step = kWave / 2; step > 0; step /= 2) {
            const int begin = __shfl(span.begin, min(hit + step, kWave - 1), kWave);
            if (hit + step < p.batch && begin <= token) hit += step;
        }
        return {hit, __shfl(context, hit, kWave), {__shfl(span.begin, hit, kWave), __shfl(span.end, hit, kWave)}};
    }
    int low = 0, high = p.batch;  // the last b in [low, high) whose start is at most `token`
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (min(max(p.starts[mid], 0), p.tokens) <= token) low = mid;
        else high = mid;
    }
    return {low, p.contexts[low], span_of(low)};
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// log(2^m l): of a sum of weights relative to 2^m. In fp64, or a large m would cost
// the logarithm's last bits.
__device__ __forceinline__ float log_of_sum(float m, float l) {
    return static_cast<float>((static_cast<double>(m) + __builtin_amdgcn_logf(l)) * 0.6931471805599453);
}

// Max / sum over the four 16-lane rows of a wave (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float rows_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

__device__ __forceinline__ float rows_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// Eight e4m3 bytes times a power of two as bf16 (exact).
__device__ __forceinline__ bf16x8 widen(uint32_t a, uint32_t b, float power) {
    const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, false);
    const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, true);
    const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, false);
    const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, true);
    return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

__device__ __forceinline__ uint32_t high_halves(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

__device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// PARTS bf16 parts of eight values: each but the last cuts 8 bits off what the
// ones before left (exact), the last rounds (the third of three is exact).
template <int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&part)[PARTS]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        uint32_t w[4];
        if (s == PARTS - 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x2 y = {static_cast<__bf16>(rest[2 * j]), static_cast<__bf16>(rest[2 * j + 1])};
                w[j] = __builtin_bit_cast(uint32_t, y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = high_halves(rest[2 * j], rest[2 * j + 1]);
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = rest[j] - cut(rest[j]);
        }
        const u32x4 v = {w[0], w[1], w[2], w[3]};
        part[s] = __builtin_bit_cast(bf16x8, v);
    }
}

// The first product's operands: K's bytes widened to the query's 16-bit type, for
// fp32 queries times 2^7 (below fp16's 65504, and normal when 2^12 lower too).
template <int QT>
struct Query {
    static constexpr bool kHalf = QT != NQ_DTYPE_BF16;  // fp16 operands
    static constexpr int kParts = QT == NQ_DTYPE_F32 ? 2 : 1;
    static constexpr int kLift = QT == NQ_DTYPE_F32 ? 7 : 0;
};

constexpr int kPartShift = 12;  // powers of two between an fp32 query's parts

template <int QT>
__device__ __forceinline__ u32x4 widen_k(uint32_t a, uint32_t b) {
    if constexpr (Query<QT>::kHalf) {
        constexpr float up = 1 << Query<QT>::kLift;
        const f16x2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, up, false),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, up, true),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, up, false),
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, up, true)};
        return u32x4{__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                     __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3])};
    } else {
        return __builtin_bit_cast(u32x4, widen(a, b, 1.0f));
    }
}

// K as the second part of an fp32 query meets it (exact).
__device__ __forceinline__ u32x4 lowered(u32x4 k) {
    const f16x8 down = static_cast<_Float16>(1.0f / (1 << kPartShift));
    return __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, k) * down);
}

template <int QT>
__device__ __forceinline__ f32x4 mfma_k(u32x4 k, u32x4 q, f32x4 c) {
    if constexpr (Query<QT>::kHalf)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

// A lane's share of a query row, STEPS times eight values at `at` + 64 (c / 2) +
// 8 (c & 1), as parts; returns the power of two that their products with the
// widened K have to be multiplied by (1 but for fp32).
template <int QT, int STEPS>
__device__ __forceinline__ float load_query(const void* q, int64_t at, bool on, u32x4 (&part)[STEPS][Query<QT>::kParts]) {
    if constexpr (QT != NQ_DTYPE_F32) {
#pragma unroll
        for (int c = 0; c < STEPS; ++c)
            part[c][0] = on ? *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(q) + at + 64 * (c / 2) + 8 * (c & 1))
                            : u32x4{0, 0, 0, 0};
        return 1.0f;
    } else {
        f32x4 x[STEPS][2];
        float most = 0.0f;
#pragma unroll
        for (int c = 0; c < STEPS; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[c][h] = on ? *reinterpret_cast<const f32x4*>(static_cast<const float*>(q) + at + 64 * (c / 2) + 8 * (c & 1) + 4 * h)
                             : f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(x[c][h][j]));
            }
        most = rows_max(most);
        // 2^e <= the largest value < 2^(e + 1); from 2^-100 on, so that 2^(14 - e) is a number.
        const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100);
        const float up = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            f16x8 high, low;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[c][j >> 2][j & 3] * up;
                high[j] = static_cast<_Float16>(y);
                // What is not finite has no remainder.
                const float rest = (y - static_cast<float>(high[j])) * (1 << kPartShift);
                low[j] = fabsf(y) < INFINITY ? static_cast<_Float16>(rest) : static_cast<_Float16>(0.0f);
            }
            part[c][0] = __builtin_bit_cast(u32x4, high);
            part[c][1] = __builtin_bit_cast(u32x4, low);
        }
        return __uint_as_float(static_cast<uint32_t>(e - 14 - Query<QT>::kLift + 127) << 23);
    }
}

// Byte mask of the first n of 16 bytes, dword i.
__device__ __forceinline__ uint32_t first_bytes(int n, int i) {
    const int k = n - 4 * i;
    return k >= 4 ? 0xffffffffu : (k <= 0 ? 0u : (1u << (8 * k)) - 1u);
}

// 0x80 in each byte of w that is an e4m3 NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

__device__ __forceinline__ void store4(void* out, int dtype, int64_t at, const float (&v)[4]) {
    if (dtype == NQ_DTYPE_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (dtype == NQ_DTYPE_BF16) {
            const bf16x2 h = {static_cast<__bf16>(v[2 * i]), static_cast<__bf16>(v[2 * i + 1])};
            w[i] = __builtin_bit_cast(uint32_t, h);
        } else {
            const f16x2 h = {static_cast<_Float16>(v[2 * i]), static_cast<_Float16>(v[2 * i + 1])};
            w[i] = __builtin_bit_cast(uint32_t, h);
        }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(w[0], w[1]);
}

// One workgroup of WAVES waves: a slot of query rows of one kv head over one
// split of the cache. SHARED: the waves hold the same 16 NT rows and take the
// split's tiles in turn; otherwise each wave has 16 NT rows of its own and all take
// every tile. Where registers are short, q's parts wait in LDS (in registers they
// would leave room for one wave to a SIMD, and nothing would fill the matrix unit
// during a softmax).
//
// Single tokens after long caches are bound by the cache's bytes: 268 MB of one
// sequence at 4.8 TB/s (a copy reaches 5.04), 153 MB of 32 ragged sequences at 4.1 with the
// launch. Prompts are bound by the vector unit, which widens K and V, and takes
// exponentials and parts of the weights (4096 bf16 tokens of 32/8 heads of 128: 231
// to 237 us for 1.4e11 multiplications and additions; the vector unit works in 71% of the
// SIMDs' cycles, the matrix unit in 43%). Of some 600 vector instructions a tile 128
// widen K and V: waves that have rows of their own each do that for themselves,
// four times a workgroup, and heads of 128 spill 71 to 74 registers there.
template <int D, int QT, int PP, int NT, int TILE, bool SHARED, int WAVES, bool SEGMENTS>
__global__ __launch_bounds__(WAVES* kWave, D == 256 && NT == 2 ? 1 : 2) void k_paged_attention(const ArgsOf<SEGMENTS> a) {
    constexpr int kRows = (SHARED ? 1 : WAVES) * 16 * NT;
    constexpr int kChunks = D / 64, kDims = D / 16;
    constexpr int kBlock = TILE / 4;   // consecutive cache rows of a lane: of V, and of the scores
    constexpr int kScores = TILE / 16, kSteps = TILE / 32, kWords = kBlock / 4;
    constexpr bool kEarly = SHARED;    // the next K before the softmax, with registers of its own
    constexpr bool kInLds = !SHARED || NT > 1 || D == 256;  // where q's parts wait
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1), n = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int g = blockIdx.x % p.kv_heads;
    const int unit = blockIdx.x / p.kv_heads;
    bool all = false;  // of the shared rows, for all sequences
    int split, skip = 0;
    int64_t item;
    SplitPlan plan;
    SlotSpan s;
    if constexpr (SEGMENTS) all = static_cast<int>(blockIdx.x) < a.blocks;
    if (all) {
        if constexpr (SEGMENTS) {
            const int nth = unit / a.shared_splits;
            split = unit - nth * a.shared_splits;
            item = static_cast<int64_t>(a.slots) * a.splits + unit;
            plan = {a.shared_per, a.shared_splits};
            const int row0 = nth * kRows, rows = p.tokens * a.group;
            s = {0, 0, 0, row0, min(kRows, rows - row0), a.skip};
        }
    } else {
        Work w;
        if constexpr (SEGMENTS) {
            skip = a.skip;
            w = find<false>(p, unit - a.blocks / p.kv_heads, 0, a.group, kRows, a.splits, a.least, skip);
        } else {
            w = find<false>(p, unit, 0, a.group, kRows, a.splits, a.least);
        }
        item = w.first + w.local;
        if (w.local < 0 || item >= static_cast<int64_t>(a.slots) * a.splits) return;  // none, or query_starts out of order
        const uint32_t local = static_cast<uint32_t>(w.local), stride = p.batch > kWave ? a.splits : w.plan.active;
        const uint32_t nth = local / stride;
        split = static_cast<int>(local - nth * stride);
        if (split >= w.plan.active) return;
        plan = w.plan;
        s = slot_span(p, w.f, static_cast<int64_t>(nth) * kRows, a.group, kRows);
        if (s.rows == 0) return;
    }
    const int page = 1 << p.page_shift, cache_rows = p.table_pages << p.page_shift;

    // This wave's query rows: row numbers, positions (-1: sees nothing), q.
    constexpr int QP = Query<QT>::kParts, kQSteps = 2 * kChunks;
    // LDS: q's parts, of the wave or of all; where the waves share rows, their shares later.
    constexpr int kQFrags = kInLds ? kQSteps * NT * QP : 0, kQCopies = SHARED ? 1 : WAVES;
    constexpr int kJoinFrags = SHARED ? WAVES * kDims * NT : 0;
    __shared__ u32x4 lds[kQFrags * kQCopies > kJoinFrags ? kQFrags * kQCopies : kJoinFrags][kWave];
    u32x4(*q_lds)[kWave] = lds + (SHARED ? 0 : wave * kQFrags);
    u32x4 q_regs[kQSteps][QP];
    const int wave_row = SHARED ? 0 : wave * 16 * NT;
    int row[NT], pos[NT];
    float q_scale[NT];
    int64_t out_at[NT];
    int low_pos = 0x7fffffff, high_pos = -1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        row[t] = wave_row + 16 * t + n;
        const bool on = row[t] < s.rows;
        const int r = on ? s.row0 + row[t] : 0;
        const int place = r / a.group, head = g * a.group + r - place * a.group;
        if (all) {
            const Found f = lane_sequence(p, place);
            const bool has = on && place >= f.span.begin && place < f.span.end;
            pos[t] = has ? row_of(f.context, place - f.span.begin, cache_rows) : -1;
        } else {
            pos[t] = on ? row_of(s.context, place, cache_rows) : -1;
        }
        out_at[t] = (static_cast<int64_t>(s.begin + place) * a.q_heads + head) * D;
        q_scale[t] = a.scale * load_query<QT, kQSteps>(a.q, out_at[t] + 16 * grp, on, q_regs);
        if (kInLds && (!SHARED || wave == 0)) {
#pragma unroll
            for (int c = 0; c < kQSteps; ++c)
#pragma unroll
                for (int x = 0; x < QP; ++x) q_lds[(c * NT + t) * QP + x][lane] = q_regs[c][x];
        }
        int lo = on ? pos[t] : 0x7fffffff, hi = pos[t];
#pragma unroll
        for (int m = 1; m < 16; m *= 2) {
            lo = min(lo, __shfl_xor(lo, m, kWave));
            hi = max(hi, __shfl_xor(hi, m, kWave));
        }
        low_pos = min(low_pos, __builtin_amdgcn_readfirstlane(lo));
        high_pos = max(high_pos, __builtin_amdgcn_readfirstlane(hi));
    }
    // Rows of its own: a lane reads back what it wrote itself.
    if constexpr (kInLds && SHARED) __syncthreads();

    f32x4 acc[kDims][NT];
    float m_run[NT], l_run[NT];
    uint32_t nan_at[NT][(kDims + 7) / 8] = {};  // a bit for each output that a NaN of V reaches behind a mask
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m_run[t] = -INFINITY;
        l_run[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[d][t] = f32x4{0, 0, 0, 0};
    }

    const int first_tile = skip / TILE;
    const int tile_end = min(first_tile + (split + 1) * plan.per * (kTile / TILE), (min(high_pos + 1, s.visible) + TILE - 1) / TILE);
    const int step = SHARED ? WAVES : 1;
    const int tile_begin = first_tile + split * plan.per * (kTile / TILE) + (SHARED ? wave : 0);
    // Table entries of this lane's blocks of kBlock rows: block n / 4 for K, grp
    // for the scores' scales and for V. What no query sees takes the last entry
    // in use. All loads of the loop are unconditional and in one order (entries,
    // scales, K, V), or a wait for the oldest becomes a wait for all: behind the
    // last tile they read that tile again, from the L2.
    const int32_t* table = p.table + static_cast<int64_t>(s.b) * p.table_pages;
    const int last_row = max(s.visible - 1, 0);
    const auto page_at = [&](int tile, int block) { return table[min(tile * TILE + kBlock * block, last_row) >> p.page_shift]; };
    // An entry that names no page reads page 0 too, with a scale of NaN.
    const auto base_of = [&](int id) {
        return static_cast<int64_t>(static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pages) ? id : 0) * p.kv_heads + g;
    };
    u32x4 kf[kScores][kChunks];
    uint32_t vf[kDims][kWords];
    float k_scale = 0.0f, v_scale = 0.0f;
    const auto load_scales = [&](int id) {
        const int64_t at = base_of(id);
        k_scale = p.k_scales[at];
        v_scale = p.v_scales[at];
    };
    const auto load_k = [&](int tile, int id) {
        const uint8_t* at = p.k + (base_of(id) * page + ((tile * TILE + kBlock * (n >> 2)) & (page - 1)) + (n & 3)) * D + 16 * grp;
#pragma unroll
        for (int t = 0; t < kScores; ++t)
#pragma unroll
            for (int c = 0; c < kChunks; ++c) kf[t][c] = *reinterpret_cast<const u32x4*>(at + 4 * t * D + 64 * c);
    };
    const auto load_v = [&](int tile, int id) {
        const uint8_t* at = p.v + (base_of(id) * D + n) * page + ((tile * TILE + kBlock * grp) & (page - 1));
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            typedef uint32_t words __attribute__((ext_vector_type(kWords)));
            const words w = *reinterpret_cast<const words*>(at + static_cast<int64_t>(16 * d) * page);
#pragma unroll
            for (int i = 0; i < kWords; ++i) vf[d][i] = w[i];
        }
    };
    // K and V of the next tile are on their way while this one is worked on,
    // their table entries a tile ahead of that.
    int id_k = page_at(tile_begin, n >> 2), id_v = page_at(tile_begin, grp);
    int next_k = page_at(tile_begin + step, n >> 2), next_v = page_at(tile_begin + step, grp);
    if (tile_begin < tile_end) {
        load_scales(id_v);
        __builtin_amdgcn_sched_barrier(0);
        load_k(tile_begin, id_k);
        __builtin_amdgcn_sched_barrier(0);
        load_v(tile_begin, id_v);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (int tile = tile_begin; tile < tile_end; tile += step) {
        const int base = tile * TILE;
        const bool more = tile + step < tile_end;
        const int then = more ? tile + step : tile;
        const bool bad = static_cast<uint32_t>(id_v) >= static_cast<uint32_t>(p.pages);
        const float ks = bad ? __builtin_nanf("") : k_scale, vs = bad ? 1.0f : v_scale;
        if (more) {
            id_k = next_k;
            id_v = next_v;
        }
        next_k = page_at(tile + 2 * step, n >> 2);
        next_v = page_at(tile + 2 * step, grp);
        __builtin_amdgcn_sched_barrier(0);

        f32x4 sc[kScores][NT];
#pragma unroll
        for (int t = 0; t < kScores; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u) sc[t][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kQSteps; ++c) {
            u32x4 qf[NT][QP];
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int x = 0; x < QP; ++x)
                    qf[u][x] = kInLds ? q_lds[kInLds ? (c * NT + u) * QP + x : 0][lane] : q_regs[c][x];
#pragma unroll
            for (int t = 0; t < kScores; ++t) {
                const u32x4 k = widen_k<QT>(kf[t][c / 2][2 * (c & 1)], kf[t][c / 2][2 * (c & 1) + 1]);
                if constexpr (QP == 2) {
                    const u32x4 low = lowered(k);
#pragma unroll
                    for (int u = 0; u < NT; ++u) sc[t][u] = mfma_k<QT>(low, qf[u][1], sc[t][u]);
                }
#pragma unroll
                for (int u = 0; u < NT; ++u) sc[t][u] = mfma_k<QT>(k, qf[u][0], sc[t][u]);
            }
        }

        // Many query rows (not early): K's registers serve the softmax meanwhile, and
        // the SIMD's other wave fills the wait for the next ones.
        const auto load_next_k = [&] {
            __builtin_amdgcn_sched_barrier(0);
            load_scales(id_v);
            __builtin_amdgcn_sched_barrier(0);
            load_k(then, id_k);
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (kEarly) load_next_k();

        // What the scores and the weights are multiplied by. A power of two for V, as
        // the append writes, goes into its widening instead.
        const uint32_t v_bits = __float_as_uint(vs);
        const bool v_power = (v_bits & 0x807fffffu) == 0 && v_bits - 1u < 0x7f7fffffu;
        const float v_up = v_power ? vs : 1.0f;
        float f[NT], weight_up[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            f[u] = ks * q_scale[u];
            weight_up[u] = v_power ? 1.0f : vs;
        }

        const bool masked = base + TILE > low_pos + 1;  // uniform: some row of the wave does not see them all
        if (masked) {
            // Rows that nobody sees may have any scale: the scores are multiplied here, for all query rows of
            // the wave. (So the last bits of a result hang on the positions of the rows beside it, never on their values.)
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const int seen = pos[u] + 1 - (base + kBlock * grp);
#pragma unroll
                for (int j = 0; j < kBlock; ++j)
                    sc[j >> 2][u][j & 3] = j < seen ? sc[j >> 2][u][j & 3] * f[u] : -INFINITY;
                f[u] = 1.0f;
                if (seen <= 0) weight_up[u] = 1.0f;
            }
        }

        bf16x8 pf[NT][kSteps][PP];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float x[kBlock], top = sc[0][u][0];
#pragma unroll
            for (int j = 1; j < kBlock; ++j) top = fmaxf(top, sc[j >> 2][u][j & 3]);
            // What weights are relative to need not be the largest score: it moves
            // only where a weight would pass 1, seldom after the first tiles, to 2^kSlack
            // above the score, and the accumulators with it (4096 tokens of 16/4 heads
            // of 256: 343 us, 364 where they follow every new maximum). Weights
            // never pass 1, so that values near fp32's largest stay what they are.
            const float m_tile = rows_max(top * f[u]);
            if (const bool grows = m_tile > m_run[u]; __ballot(grows)) {
                const float m_new = grows ? m_tile + kSlack : m_run[u];
                const float keep = exp2_hw(m_run[u] - (m_new == -INFINITY ? 0.0f : m_new));
                l_run[u] *= keep;
#pragma unroll
                for (int d = 0; d < kDims; ++d) acc[d][u] *= keep;
                m_run[u] = m_new;
            }
            // Nothing seen so far (or only -inf): subtract 0, the weights are 0.
            const float m_use = m_run[u] == -INFINITY ? 0.0f : m_run[u];
            // The fused subtraction sees what rounding took off the largest score: half a
            // step of it, which is no number to raise 2 to where scores pass 2^30. They
            // are rounded first there, so that the largest has the weight that it has in fp32: by query
            // row, so that one row's scores change no bit of another's result.
            if (const bool large = fabsf(m_use) > 0x1p24f; __ballot(large)) {
#pragma unroll
                for (int j = 0; j < kBlock; ++j) sc[j >> 2][u][j & 3] *= large ? f[u] : 1.0f;
                f[u] = large ? 1.0f : f[u];
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                x[j] = exp2_hw(fmaf(sc[j >> 2][u][j & 3], f[u], -m_use));
                sum += x[j];
            }
            l_run[u] += sum;
            if (__ballot(weight_up[u] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < kBlock; ++j) x[j] *= weight_up[u];
            }
#pragma unroll
            for (int h = 0; h < kSteps; ++h) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = x[8 * h + j];
                split8<PP>(y, pf[u][h]);
            }
        }
        if (masked) {
            // Bytes of V rows that nobody sees may be anything. Among those
            // that only some see, a NaN must not meet a weight of zero: it is
            // taken out and given back to the queries that do see its row.
            const int seen_rows = high_pos + 1 - (base + kBlock * grp);
            uint32_t any = 0;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    vf[d][i] &= first_bytes(seen_rows, i);
                    any |= nan_bytes(vf[d][i]);
                }
            if (__ballot(any != 0)) {
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    bf16x8 see[kSteps];
#pragma unroll
                    for (int h = 0; h < kSteps; ++h)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            see[h][j] = static_cast<__bf16>(base + kBlock * grp + 8 * h + j <= pos[u] ? 1.0f : 0.0f);
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        uint32_t one[kWords];  // e4m3 1.0 where V holds NaN
#pragma unroll
                        for (int i = 0; i < kWords; ++i) one[i] = (nan_bytes(vf[d][i]) >> 7) * 0x38u;
                        f32x4 hits = {0, 0, 0, 0};
#pragma unroll
                        for (int h = 0; h < kSteps; ++h)
                            hits = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(one[2 * h], one[2 * h + 1], 1.0f), see[h], hits, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (hits[i] > 0.0f) nan_at[u][d / 8] |= 1u << (4 * (d % 8) + i);
                    }
                }
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int i = 0; i < kWords; ++i) vf[d][i] &= ~((nan_bytes(vf[d][i]) >> 7) * 0xffu);
            }
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int h = 0; h < kSteps; ++h) {
                const bf16x8 v = widen(vf[d][2 * h], vf[d][2 * h + 1], v_up);
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int x = PP - 1; x >= 0; --x)
                        acc[d][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[u][h][x], acc[d][u], 0, 0, 0);
            }
        if constexpr (!kEarly) load_next_k();
        __builtin_amdgcn_sched_barrier(0);
        load_v(then, id_v);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        l_run[u] = rows_sum(l_run[u]);
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (nan_at[u][d / 8] >> (4 * (d % 8) + i) & 1u) acc[d][u][i] = __builtin_nanf("");
    }

    // Output o of query row t, or its share for the merge.
    const auto put = [&](int t, int d, const f32x4& o, float m, float l) {
        if (row[t] >= s.rows) return;
        bool whole = plan.active <= 1;
        if constexpr (SEGMENTS) whole = whole && a.blocks == 0;
        if (whole) {
            const float inv = pos[t] < 0 ? 0.0f : 1.0f / l;
            if constexpr (SEGMENTS) {
                if (a.lse && d == 0 && grp == 0) a.lse[out_at[t] / D] = pos[t] < 0 ? -INFINITY : log_of_sum(m, l);
            }
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = pos[t] < 0 ? 0.0f : o[i] * inv;
            store4(a.out, a.out_dtype, out_at[t] + 16 * d + 4 * grp, v);
        } else {
            const int64_t at = (item * p.kv_heads + g) * kRows + row[t];
            if (d == 0 && grp == 0) {
                a.partial[2 * at] = m;
                a.partial[2 * at + 1] = l;
            }
            *reinterpret_cast<f32x4*>(a.partial_o + at * D + 16 * d + 4 * grp) = o;
        }
    };
    if constexpr (SHARED) {
        // The waves' shares of the same rows meet in LDS; each wave joins some of the
        // dimensions, the shares in wave order.
        __shared__ float join_ml[WAVES][2][16 * NT];
        if constexpr (kInLds) __syncthreads();  // q's parts are read
        if (grp == 0) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                join_ml[wave][0][16 * u + n] = m_run[u];
                join_ml[wave][1][16 * u + n] = l_run[u];
            }
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int u = 0; u < NT; ++u) lds[(wave * kDims + d) * NT + u][lane] = __builtin_bit_cast(u32x4, acc[d][u]);
        __syncthreads();
        if (wave >= kDims) return;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float weight[WAVES], m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m_all = fmaxf(m_all, join_ml[w][0][16 * u + n]);
            const float m_use = m_all == -INFINITY ? 0.0f : m_all;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                weight[w] = exp2_hw(join_ml[w][0][16 * u + n] - m_use);
                l_all += weight[w] * join_ml[w][1][16 * u + n];
            }
#pragma unroll
            for (int d = wave; d < kDims; d += WAVES) {
                f32x4 o = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) o += weight[w] * __builtin_bit_cast(f32x4, lds[(w * kDims + d) * NT + u][lane]);
                put(u, d, o, m_all, l_all);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int d = 0; d < kDims; ++d) put(u, d, acc[d][u], m_run[u], l_run[u]);
    }
}

// Host side: grid and rows of a slot for a call, and its launch.
struct AttnPlan {
    int rows, slots, splits, least, waves;
    bool shared;
};

// Cache rows that a wave takes at once where the registers hold them.
template <int D>
constexpr int kRowsAtOnce = D == 256 ? 32 : 64;

constexpr int kOwnRows = 128;  // of a slot whose waves have rows of their own, 32 each

template <int D>
int launch_paged_attention(const AttnArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream);

// The same with shared rows apart or log-sum-exps.
template <int D, int QT, int PP>
int launch_shared_as(const SharedArgs& a, const AttnPlan& plan, hipStream_t stream) {
    const int64_t blocks = static_cast<int64_t>(plan.slots) * plan.splits * a.p.kv_heads + a.blocks;
    const dim3 grid(static_cast<unsigned>(blocks)), block(4 * kWave);
    constexpr int kTileRows = kRowsAtOnce<D>;
    if (plan.rows == 16) {
        hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 1, kTileRows, true, 4, true>), grid, block, 0, stream, a);
    } else if (plan.shared) {
        hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 2, 32, true, 4, true>), grid, block, 0, stream, a);
    } else if constexpr (D < 256) {
        hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 2, kTileRows, false, 4, true>), grid, block, 0, stream, a);
    }
    return nq::launch_status();
}

template <int D, int QT, int PP>
int launch_attention_as(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream) {
    const int64_t blocks = static_cast<int64_t>(plan.slots) * plan.splits * a.p.kv_heads;  // launchable: checked with the workspace
    const dim3 grid(static_cast<unsigned>(blocks)), block(static_cast<unsigned>(plan.waves * kWave));
    constexpr int kTileRows = kRowsAtOnce<D>;
    if (plan.shared && plan.waves == 4) {
        if (plan.rows == 32)
            hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 2, 32, true, 4, false>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 1, kTileRows, true, 4, false>), grid, block, 0, stream, a);
    } else if constexpr (D < 256) {
        if (plan.shared)
            hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 1, kTileRows, true, 8, false>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((k_paged_attention<D, QT, PP, 2, kTileRows, false, 4, false>), grid, block, 0, stream, a);
    }
    return nq::launch_status();
}

template <int D, int QT>
int launch_attention_out(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream) {
    return a.out_dtype == NQ_DTYPE_F32 ? launch_attention_as<D, QT, 3>(a, plan, stream)
                                       : launch_attention_as<D, QT, 2>(a, plan, stream);
}

template <int D>
int launch_attention_for(const AttnArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream) {
    switch (q_dtype) {
        case NQ_DTYPE_F32: return launch_attention_out<D, NQ_DTYPE_F32>(a, plan, stream);
        case NQ_DTYPE_F16: return launch_attention_out<D, NQ_DTYPE_F16>(a, plan, stream);
        default: return launch_attention_out<D, NQ_DTYPE_BF16>(a, plan, stream);
    }
}

template <int D, int QT>
int launch_shared_out(const SharedArgs& a, const AttnPlan& plan, hipStream_t stream) {
    return a.out_dtype == NQ_DTYPE_F32 ? launch_shared_as<D, QT, 3>(a, plan, stream)
                                       : launch_shared_as<D, QT, 2>(a, plan, stream);
}

template <int D>
int launch_shared_for(const SharedArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream) {
    switch (q_dtype) {
        case NQ_DTYPE_F32: return launch_shared_out<D, NQ_DTYPE_F32>(a, plan, stream);
        case NQ_DTYPE_F16: return launch_shared_out<D, NQ_DTYPE_F16>(a, plan, stream);
        default: return launch_shared_out<D, NQ_DTYPE_BF16>(a, plan, stream);
    }
}

template <int D>
int launch_shared_attention(const SharedArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream);

// The layout of a call without shared rows (nq_paged_attention.hip).
AttnPlan plan_attention(int64_t tokens, int64_t batch, int q_heads, int kv_heads, int head_dim, int64_t cache_rows);

}  // namespace paged
}  // namespace nq
