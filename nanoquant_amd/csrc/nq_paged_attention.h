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
// Precision: an e4m3 byte is exact in bf16. q enters as one bf16 part, two or
// three (bf16 / fp16 / fp32: 8, 16, 24 bits: exact), so scores carry fp32
// rounding only. The weights enter the second product as two bf16 parts (16
// bits, 2^-17 of a weight at most) for 16-bit outputs, whose own rounding is
// 2^-9 or 2^-12, and as three for fp32 outputs. Scales: K's multiplies the
// fp32 score, V's the fp32 weight before it is split.
#pragma once

#include "nq_paged.h"

namespace nq {
namespace paged {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;  // cache rows that splits are counted in

struct AttnArgs {
    Pages p;
    const void* q;
    void* out;
    float* partial;    // [slots][splits][kv_heads][rows][2] (max, sum), then the same of [head_dim]
    float* partial_o;
    float scale;       // scaling * log2(e): scores are kept in base 2
    int32_t out_dtype, q_heads, group, slots, splits, least;  // least: cache tiles a split takes at least
};

// What a slot of `rows` query rows holds, the same for the attention and the merge.
struct SlotSpan {
    int b, begin, context;  // sequence, its first token, rows cached before the call
    int row0, rows;         // the slot's first query row in its sequence; rows it holds
    int visible;            // cache rows [0, visible) that some row of the slot sees
};

__device__ __forceinline__ int64_t first_slot_of(int b, int begin, int group, int rows) {
    return static_cast<int64_t>(begin) * group / rows + b;
}

__device__ __forceinline__ SlotSpan slot_span(const Pages& p, const Found& f, int64_t slot, int group, int rows) {
    SlotSpan o;
    o.b = f.b;
    o.begin = f.span.begin;
    o.context = f.context;
    const int64_t row0 = (slot - first_slot_of(f.b, f.span.begin, group, rows)) * rows;
    const int64_t all = static_cast<int64_t>(f.span.end - f.span.begin) * group;
    o.row0 = static_cast<int>(row0 < 0 || row0 >= all ? 0 : row0);
    o.rows = static_cast<int>(row0 < 0 || row0 >= all ? 0 : min(static_cast<int64_t>(rows), all - row0));
    const int64_t last = static_cast<int64_t>(o.context) + (o.row0 + o.rows - 1) / group;
    o.visible = o.rows == 0 || last < 0
                    ? 0 : static_cast<int>(min(last + 1, static_cast<int64_t>(p.table_pages) << p.page_shift));
    return o;
}

// Cache tiles of each split, and splits that have any.
struct SplitPlan {
    int tiles, per, active;
};

__device__ __forceinline__ SplitPlan split_plan(int visible, int splits, int least) {
    SplitPlan s;
    s.tiles = (visible + kTile - 1) / kTile;
    s.per = max((s.tiles + splits - 1) / splits, least);
    s.active = (s.tiles + s.per - 1) / s.per;
    return s;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

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

// Eight e4m3 bytes as bf16 (exact).
__device__ __forceinline__ bf16x8 widen(uint32_t a, uint32_t b) {
    const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
    const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
    const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

__device__ __forceinline__ uint32_t high_halves(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

__device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// PARTS bf16 parts of eight values: each but the last cuts 8 bits off what the
// ones before left (exact), the last rounds (the third of three is exact). An
// infinite or NaN value is its own first part and leaves nothing.
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

// q parts: 3 from fp32, 2 from fp16, 1 from bf16.
template <int QP>
__device__ __forceinline__ void load_q8(const void* q, int64_t at, bool on, bf16x8 (&part)[QP]) {
    if constexpr (QP == 1) {
        u32x4 v = {0, 0, 0, 0};
        if (on) v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(q) + at);
        part[0] = __builtin_bit_cast(bf16x8, v);
    } else {
        float x[8];
        if constexpr (QP == 2) {
            typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
            f16x8 v = {};
            if (on) v = *reinterpret_cast<const f16x8*>(static_cast<const _Float16*>(q) + at);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = static_cast<float>(v[j]);
        } else {
            f32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (on) {
                a = *reinterpret_cast<const f32x4*>(static_cast<const float*>(q) + at);
                b = *reinterpret_cast<const f32x4*>(static_cast<const float*>(q) + at + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = a[j];
                x[4 + j] = b[j];
            }
        }
        split8<QP>(x, part);
        // What is not finite has no remainder.
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!(fabsf(x[j]) < INFINITY))
#pragma unroll
                for (int s = 1; s < QP; ++s) part[s][j] = static_cast<__bf16>(0.0f);
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
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 h = {static_cast<_Float16>(v[2 * i]), static_cast<_Float16>(v[2 * i + 1])};
            w[i] = __builtin_bit_cast(uint32_t, h);
        }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(w[0], w[1]);
}

// Waves of a SIMD that the registers are held to.
template <int D>
constexpr int kWavesFor = D == 256 ? 1 : 2;
template <int D>
constexpr int kTileFor = D == 256 ? 32 : 64;

// One workgroup of four waves: a slot of query rows of one kv head over one
// split of the cache. SHARED: the waves hold the same 16 NT rows and take the
// split's tiles in turn (few query rows: the cache's bytes are the work);
// otherwise each wave holds 16 NT rows of its own and all take every tile.
template <int D, int QP, int PP, int NT, int TILE, bool SHARED>
__global__ __launch_bounds__(256, kWavesFor<D>) void k_paged_attention(const AttnArgs a) {
    constexpr int kRows = (SHARED ? 1 : 4) * 16 * NT;
    constexpr int kChunks = D / 64, kDims = D / 16;
    constexpr int kBlock = TILE / 4;   // consecutive cache rows of a lane: of V, and of the scores
    constexpr int kScores = TILE / 16, kSteps = TILE / 32, kWords = kBlock / 4;
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1), n = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int g = blockIdx.x % p.kv_heads;
    const int rest = blockIdx.x / p.kv_heads;
    const int split = rest % a.splits, slot = rest / a.splits;
    const Found found = sequence_at(p, slot, [&](int i, int begin) { return first_slot_of(i, begin, a.group, kRows); });
    const SlotSpan s = slot_span(p, found, slot, a.group, kRows);
    if (s.rows == 0) return;
    const int page = 1 << p.page_shift, cache_rows = p.table_pages << p.page_shift;
    const SplitPlan plan = split_plan(s.visible, a.splits, a.least);
    if (split > 0 && split >= plan.active) return;

    // This wave's query rows: row numbers, positions (-1: sees nothing), q.
    const int wave_row = SHARED ? 0 : wave * 16 * NT;
    int row[NT], pos[NT];
    int64_t out_at[NT];
    bf16x8 qf[NT][2 * kChunks][QP];
    int low_pos = 0x7fffffff, high_pos = -1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        row[t] = wave_row + 16 * t + n;
        const bool on = row[t] < s.rows;
        const int r = on ? s.row0 + row[t] : 0;
        const int place = r / a.group, head = g * a.group + r - place * a.group;
        pos[t] = on ? row_of(s.context, place, cache_rows) : -1;
        out_at[t] = (static_cast<int64_t>(s.begin + place) * a.q_heads + head) * D;
#pragma unroll
        for (int c = 0; c < 2 * kChunks; ++c)
            load_q8<QP>(a.q, out_at[t] + 64 * (c / 2) + 16 * grp + 8 * (c & 1), on, qf[t][c]);
        int lo = on ? pos[t] : 0x7fffffff, hi = pos[t];
#pragma unroll
        for (int m = 1; m < 16; m *= 2) {
            lo = min(lo, __shfl_xor(lo, m, kWave));
            hi = max(hi, __shfl_xor(hi, m, kWave));
        }
        low_pos = min(low_pos, __builtin_amdgcn_readfirstlane(lo));
        high_pos = max(high_pos, __builtin_amdgcn_readfirstlane(hi));
    }

    f32x4 acc[kDims][NT];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m_run[t] = -INFINITY;
        l_run[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[d][t] = f32x4{0, 0, 0, 0};
    }

    const int tile_end = min((split + 1) * plan.per * (kTile / TILE), (min(high_pos + 1, s.visible) + TILE - 1) / TILE);
    const int step = SHARED ? 4 : 1;
    const int tile_begin = split * plan.per * (kTile / TILE) + (SHARED ? wave : 0);
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
        const float ks = bad ? __builtin_nanf("") : k_scale * a.scale, vs = bad ? __builtin_nanf("") : v_scale;
        if (more) {
            id_k = next_k;
            id_v = next_v;
        }
        next_k = page_at(tile + 2 * step, n >> 2);
        next_v = page_at(tile + 2 * step, grp);
        __builtin_amdgcn_sched_barrier(0);

        f32x4 sc[kScores][NT];
#pragma unroll
        for (int t = 0; t < kScores; ++t) {
#pragma unroll
            for (int u = 0; u < NT; ++u) sc[t][u] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const bf16x8 k0 = widen(kf[t][c][0], kf[t][c][1]), k1 = widen(kf[t][c][2], kf[t][c][3]);
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int s2 = QP - 1; s2 >= 0; --s2) {
                        sc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[u][2 * c][s2], sc[t][u], 0, 0, 0);
                        sc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[u][2 * c + 1][s2], sc[t][u], 0, 0, 0);
                    }
            }
        }

        __builtin_amdgcn_sched_barrier(0);
        load_scales(id_v);
        __builtin_amdgcn_sched_barrier(0);
        load_k(then, id_k);
        __builtin_amdgcn_sched_barrier(0);

        const bool masked = base + TILE > low_pos + 1;  // uniform: some row of the wave does not see them all
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
                            hits = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(one[2 * h], one[2 * h + 1]), see[h], hits, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (hits[i] > 0.0f) acc[d][u][i] = __builtin_nanf("");
                    }
                }
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int i = 0; i < kWords; ++i) vf[d][i] &= ~((nan_bytes(vf[d][i]) >> 7) * 0xffu);
            }
        }

#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float x[kBlock], top = -INFINITY;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                x[j] = sc[j >> 2][u][j & 3] * ks;
                if (masked) x[j] = base + kBlock * grp + j <= pos[u] ? x[j] : -INFINITY;
                top = fmaxf(top, x[j]);
            }
            const float m_new = fmaxf(m_run[u], rows_max(top));
            // Nothing seen so far (or only -inf): subtract 0, the weights are 0.
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;
            if (__ballot(m_new != m_run[u])) {
                const float keep = exp2_hw(m_run[u] - m_use);
                l_run[u] *= keep;
#pragma unroll
                for (int d = 0; d < kDims; ++d) acc[d][u] *= keep;
                m_run[u] = m_new;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                x[j] = exp2_hw(x[j] - m_use);
                sum += x[j];
                x[j] *= vs;
                if (masked) x[j] = base + kBlock * grp + j <= pos[u] ? x[j] : 0.0f;  // a scale that nobody sees may be anything
            }
            l_run[u] += sum;
            bf16x8 pf[kSteps][PP];
#pragma unroll
            for (int h = 0; h < kSteps; ++h) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = x[8 * h + j];
                split8<PP>(y, pf[h]);
            }
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
#pragma unroll
                for (int h = 0; h < kSteps; ++h) {
                    const bf16x8 v = widen(vf[d][2 * h], vf[d][2 * h + 1]);
#pragma unroll
                    for (int s2 = PP - 1; s2 >= 0; --s2)
                        acc[d][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[h][s2], acc[d][u], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(then, id_v);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) l_run[u] = rows_sum(l_run[u]);

    // The waves' shares of the same rows meet in LDS, in wave order.
    __shared__ float join_ml[SHARED ? 4 : 1][2][16 * NT];
    __shared__ f32x4 join_o[SHARED ? 3 : 1][SHARED ? kDims * NT : 1][kWave];
    if constexpr (SHARED) {
        if (grp == 0) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                join_ml[wave][0][16 * u + n] = m_run[u];
                join_ml[wave][1][16 * u + n] = l_run[u];
            }
        }
        if (wave > 0) {
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int u = 0; u < NT; ++u) join_o[wave - 1][d * NT + u][lane] = acc[d][u];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float m_all = m_run[u];
#pragma unroll
            for (int w = 1; w < 4; ++w) m_all = fmaxf(m_all, join_ml[w][0][16 * u + n]);
            const float m_use = m_all == -INFINITY ? 0.0f : m_all;
            float keep = exp2_hw(m_run[u] - m_use);
            l_run[u] *= keep;
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[d][u] *= keep;
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                keep = exp2_hw(join_ml[w][0][16 * u + n] - m_use);
                l_run[u] += keep * join_ml[w][1][16 * u + n];
#pragma unroll
                for (int d = 0; d < kDims; ++d) acc[d][u] += keep * join_o[w - 1][d * NT + u][lane];
            }
            m_run[u] = m_all;
        }
    }

#pragma unroll
    for (int u = 0; u < NT; ++u) {
        if (row[u] >= s.rows) continue;
        if (plan.active <= 1) {
            const float inv = 1.0f / l_run[u];
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = pos[u] < 0 ? 0.0f : acc[d][u][i] * inv;
                store4(a.out, a.out_dtype, out_at[u] + 16 * d + 4 * grp, v);
            }
        } else {
            const int64_t at = ((static_cast<int64_t>(slot) * a.splits + split) * p.kv_heads + g) * kRows + row[u];
            if (grp == 0) {
                a.partial[2 * at] = m_run[u];
                a.partial[2 * at + 1] = l_run[u];
            }
#pragma unroll
            for (int d = 0; d < kDims; ++d)
                *reinterpret_cast<f32x4*>(a.partial_o + at * D + 16 * d + 4 * grp) = acc[d][u];
        }
    }
}

// Host side: grid and rows of a slot for a call, and its launch.
struct AttnPlan {
    int rows, slots, splits, least;
    bool shared;
};

template <int D>
int launch_paged_attention(const AttnArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream);

template <int D, int QP, int PP>
int launch_attention_as(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream) {
    const int64_t blocks = static_cast<int64_t>(plan.slots) * plan.splits * a.p.kv_heads;
    if (blocks > 0x7fffffff) return NQ_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (plan.shared) {
        hipLaunchKernelGGL((k_paged_attention<D, QP, PP, 1, kTileFor<D>, true>), grid, dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((k_paged_attention<D, QP, PP, 1, kTileFor<D>, false>), grid, dim3(256), 0, stream, a);
    }
    return nq::launch_status();
}

template <int D>
int launch_attention_for(const AttnArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream) {
    const bool wide = a.out_dtype == NQ_DTYPE_F32;
    switch (q_dtype) {
        case NQ_DTYPE_F32:
            return wide ? launch_attention_as<D, 3, 3>(a, plan, stream) : launch_attention_as<D, 3, 2>(a, plan, stream);
        case NQ_DTYPE_F16:
            return wide ? launch_attention_as<D, 2, 3>(a, plan, stream) : launch_attention_as<D, 2, 2>(a, plan, stream);
        default:
            return wide ? launch_attention_as<D, 1, 3>(a, plan, stream) : launch_attention_as<D, 1, 2>(a, plan, stream);
    }
}

}  // namespace paged
}  // namespace nq
