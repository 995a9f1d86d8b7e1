// Log probability of given tokens, entropy of the distribution and its top
// alternatives from rows of logits, in one read of the logits.
//
// A workgroup of four waves takes a part of a row, all of it where there are rows
// enough. A lane keeps its own running maximum m and, relative to it, s = sum
// e^(x - m) and t = sum e^(x - m) (x - m); the next 64 x 16 values of its wave
// are on their way while these are worked on. With M the largest of the maxima,
//   lse = M + log S, S = sum s e^(m - M)
//   log p(x) = x - lse, entropy = log S - T / S, T = sum (t + s (m - M)) e^(m - M)
// m, s and t are fp32 up to a part's (a row's, where it has one part), the parts'
// sum, the logarithm and the differences fp64; results are rounded once from those.
// A row's parts meet in a second launch.
//
// Bound by the logits' bytes: 1531 rows of 151936 fp32 values (930 MB) are read at
// 6.4 TB/s (145 us; loads that leave the caches alone).
//
// For alternatives each lane also leaves the largest of its 16 values (a chunk) of
// every block of 1024. The k-th largest of a row's chunk maxima bounds the k-th
// largest value from below, fewer than k chunks lie above it, and only those
// chunks, and the first ones that touch the bound, are read again: selecting
// costs the first pass one 4-byte store for 16 values. The maxima of 16 chunks
// each are kept too, so that few chunk maxima have to be looked at. (48 rows of
// 50257 bf16, k = 20: 12.4 us; lists of k kept by each wave took 21.5, chunk maxima
// alone 15.8. One row of 151936 fp32, k = 5: 9.4 us, two launches and their waits. The
// join, 8 and 5.7 us of these, reads the groups' maxima twice, a bound between, and
// waits for the row's logarithm before it.)
#include <math.h>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;
constexpr int kJoinWaves = 8;
constexpr int kMostTop = 32;
constexpr int kValues = 16;   // of a lane at once
constexpr int kBlock = kWave * kValues;
constexpr int kGroup = 16;  // chunks whose largest value is kept too
constexpr int kMostParts = 64;  // of a row: one to a lane of the joining waves
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));

struct Args {
    const void* logits;
    const int64_t* tokens;
    int64_t row_stride;
    int32_t vocab, top, parts, blocks;  // blocks of a row; chunks = 64 blocks
    float* sums;       // [rows][parts][4]: M, S, T of a part (parts > 1)
    uint32_t* maxima;  // [rows][chunks]: the order of each chunk's largest value (top > 0)
    uint32_t* groups;  // [rows][chunks / 16]: of 16 chunks' largest value
    float *logprobs, *entropy, *top_logprobs;
    int64_t* top_ids;
};

// Orders as the values do, -0 as 0, NaN above all; 0 is below every value.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float value_of(uint32_t key) {
    if (key == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The largest value first, the lowest index first among equals; 0: no value.
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t index) {
    return order ? (static_cast<uint64_t>(order) << 32) | (0xffffffffu - index) : 0;
}

// Wave reductions with DPP row operations and four lane reads, in a fixed order.
template <int CTRL>
__device__ __forceinline__ float dpp(float x, float identity) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(identity), __float_as_int(x), CTRL, 0xf, 0xf, false));
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
}

__device__ __forceinline__ float lane_of(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0xB1>(v, -INFINITY));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp<0x4E>(v, -INFINITY));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp<0x141>(v, -INFINITY));  // row_half_mirror
    v = fmaxf(v, dpp<0x140>(v, -INFINITY));  // row_mirror
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0xB1>(v, 0.0f);
    v += dpp<0x4E>(v, 0.0f);
    v += dpp<0x141>(v, 0.0f);
    v += dpp<0x140>(v, 0.0f);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        const int2 w = __builtin_bit_cast(int2, v);
        v += __builtin_bit_cast(double, make_int2(__shfl_xor(w.x, m, kWave), __shfl_xor(w.y, m, kWave)));
    }
    return v;
}

__device__ __forceinline__ int count(bool on) { return __popcll(__ballot(on)); }

__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v += __shfl_xor(v, m, kWave);
    return v;
}

template <int DT>
struct Block {
    static constexpr int kVec = DT == NQ_DTYPE_F32 ? 4 : 8, kBytes = DT == NQ_DTYPE_F32 ? 4 : 2;
    u32x4 w[kValues / kVec];
};

// One lane's values of a block, 16 bytes at a time (rows may begin anywhere: such
// loads need no alignment); at a row's end, where 16 bytes would leave it, each
// value by itself and -inf outside.
template <int DT>
__device__ __forceinline__ void load_block(Block<DT>& b, const char* row, int64_t first, int vocab) {
    using B = Block<DT>;
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int c = 0; c < kValues / B::kVec; ++c) {
        const int64_t i = first + (c * kWave + lane) * B::kVec;
        if (i + B::kVec <= vocab) {
            b.w[c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_at2*>(row + i * B::kBytes));
        } else {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == NQ_DTYPE_F32) {
                    w[e] = i + e < vocab ? reinterpret_cast<const uint32_t*>(row)[i + e] : 0xff800000u;
                } else {
                    constexpr uint32_t low = DT == NQ_DTYPE_BF16 ? 0xff80u : 0xfc00u;
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
                    const int64_t j = i + 2 * e;
                    const uint32_t h0 = j < vocab ? h[j] : low, h1 = j + 1 < vocab ? h[j + 1] : low;
                    w[e] = h0 | (h1 << 16);
                }
            }
            b.w[c] = w;
        }
    }
}

template <int DT>
__device__ __forceinline__ void unpack(const Block<DT>& b, float (&x)[kValues]) {
    constexpr int VEC = Block<DT>::kVec;
#pragma unroll
    for (int e = 0; e < kValues; ++e) {
        if constexpr (DT == NQ_DTYPE_F32) {
            x[e] = __uint_as_float(b.w[e / VEC][e % VEC]);
        } else {
            const uint32_t w = b.w[e / VEC][(e % VEC) / 2];
            if constexpr (DT == NQ_DTYPE_BF16) {
                x[e] = __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
            } else {
                x[e] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(e & 1 ? w >> 16 : w & 0xffffu)));
            }
        }
    }
}

constexpr float kLog2e = 1.4426950408889634f;

// Sums s and t relative to m, and to a larger maximum (0 -inf is not meant; an
// infinite or NaN sum stays one).
struct Sums {
    float m, s, t;
};

__device__ __forceinline__ Sums moved(const Sums& a, float to) {
    const float d = a.m == -INFINITY ? -INFINITY : a.m - to;
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    return {to, a.s * f, (a.t + a.s * fmaxf(d, -1000.0f)) * f};
}

// A row's log of its sum and entropy; NaN where there is no distribution
// (nothing above -inf, an infinity, a NaN).
__device__ __forceinline__ double finish(const Args& a, int64_t row, float m, double s, double t, float x, bool writes) {
    const double log_s = log(s);
    const double lse = static_cast<double>(m) + log_s;
    if (writes) {
        a.logprobs[row] = static_cast<float>(static_cast<double>(x) - lse);
        a.entropy[row] = static_cast<float>(log_s - t / s);
    }
    return lse;
}

__device__ __forceinline__ void put_top(const Args& a, int64_t row, uint64_t key, int rank, double lse) {
    if (!key || rank >= a.top) return;
    a.top_ids[row * a.top + rank] = 0xffffffffu - static_cast<uint32_t>(key & 0xffffffffu);
    a.top_logprobs[row * a.top + rank] =
        static_cast<float>(static_cast<double>(value_of(static_cast<uint32_t>(key >> 32))) - lse);
}

__device__ __forceinline__ float logit_of(const Args& a, int dtype, int64_t row) {
    const int64_t token = a.tokens[row];
    return token >= 0 && token < a.vocab ? nq::load_f32(a.logits, dtype, row * a.row_stride + token) : __builtin_nanf("");
}

template <int DT>
__global__ __launch_bounds__(kWaves* kWave) void k_token_logprobs(const Args a) {
    constexpr int VEC = Block<DT>::kVec, kBytes = Block<DT>::kBytes;
    __shared__ Sums sums[kWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x - static_cast<int>(row) * a.parts;
    const char* base = static_cast<const char*>(a.logits) + row * a.row_stride * kBytes;
    const int each = (a.blocks + a.parts - 1) / a.parts;
    const int begin = part * each + wave, end = min(a.blocks, (part + 1) * each);

    float m = -INFINITY, s = 0.0f, t = 0.0f;
    Block<DT> next;
    if (begin < end) load_block<DT>(next, base, static_cast<int64_t>(begin) * kBlock, a.vocab);
    for (int block = begin; block < end; block += kWaves) {
        float x[kValues];
        unpack<DT>(next, x);
        if (block + kWaves < end) load_block<DT>(next, base, static_cast<int64_t>(block + kWaves) * kBlock, a.vocab);
        float high = x[0];
#pragma unroll
        for (int e = 1; e < kValues; ++e) high = fmaxf(high, x[e]);
        const float m_new = fmaxf(m, high);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        // What was summed so far moves to the new maximum.
        const float keep = __builtin_amdgcn_exp2f((m - m_use) * kLog2e);
        t = keep * fmaf(s, fmaxf(m - m_use, -1000.0f), t);
        s *= keep;
        float bs = 0.0f, bt = 0.0f;
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
            const float d = x[e] - m_use;
            const float w = __builtin_amdgcn_exp2f(d * kLog2e);
            bs += w;
            bt = fmaf(w, fmaxf(d, -1000.0f), bt);  // w is 0 there: 0 * -inf is not meant
        }
        if (a.top) {
            bool nan = false;
#pragma unroll
            for (int e = 0; e < kValues; ++e) nan |= x[e] != x[e];
            const bool any = static_cast<int64_t>(block) * kBlock + lane * VEC < a.vocab;  // the chunk's first value is in the row
            const int64_t chunk = (row * a.blocks + block) * kWave + lane;
            const uint32_t order = !any ? 0 : (nan ? 0xffffffffu : ordered(high));
            a.maxima[chunk] = order;
            uint32_t most = max(order, dpp<0xB1>(order));
            most = max(most, dpp<0x4E>(most));
            most = max(most, dpp<0x141>(most));
            most = max(most, dpp<0x140>(most));
            if (lane % kGroup == 0) a.groups[chunk / kGroup] = most;
        }
        s += bs;
        t += bt;
        m = m_new;
    }

    const float wave_m = wave_max(m);
    const Sums mine = moved({m, s, t}, wave_m);
    const Sums joined{wave_m, wave_sum(mine.s), wave_sum(mine.t)};
    if (lane == 0) sums[wave] = joined;
    __syncthreads();
    if (wave > 0) return;
    float high = sums[0].m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) high = fmaxf(high, sums[w].m);
    Sums all{high, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const Sums b = moved(sums[w], high);
        all.s += b.s;
        all.t += b.t;
    }
    if (a.sums) {
        if (lane == 0) {
            float* at = a.sums + 4 * (row * a.parts + part);
            at[0] = all.m;
            at[1] = all.s;
            at[2] = all.t;
        }
    } else {
        finish(a, row, all.m, all.s, all.t, logit_of(a, DT, row), lane == 0);
    }
}

// A row's parts and its alternatives.
__global__ __launch_bounds__(kJoinWaves* kWave) void k_token_logprobs_join(const Args a, int dtype) {
    constexpr int kThreads = kJoinWaves * kWave;
    constexpr int kList = 1024;  // chunks that may hold alternatives
    // Keys: of fewer than kMostTop chunks above the bound, fewer than kMostTop that
    // touch it in blocks before the last one taken, and 64 of that block.
    constexpr int kKeys = (2 * kMostTop + kWave) * kValues;
    __shared__ uint32_t bests[kThreads], list_id[kList], list_max[kList], bound_at;
    __shared__ uint64_t keys[kKeys];
    __shared__ uint32_t group_id[kList];
    __shared__ int grouped, listed, taken;
    __shared__ double lse_at;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = blockIdx.x;
    const int chunks = a.blocks * kWave;
    const uint32_t* maxima = a.maxima + (a.top ? row * chunks : 0);
    if (threadIdx.x == 0) {
        grouped = listed = taken = 0;
        bound_at = 0;
    }
    const int groups = chunks / kGroup;
    const uint32_t* group_max = a.groups + (a.top ? row * groups : 0);
    uint32_t best = 0;
    if (a.top)
#pragma unroll 4
        for (int i = threadIdx.x; i < groups; i += kThreads) best = max(best, group_max[i]);
    bests[threadIdx.x] = best;
    if (wave == 0) {
        const float* at = a.sums + 4 * (row * a.parts + (lane < a.parts ? lane : 0));
        Sums mine{at[0], at[1], at[2]};
        const float x = logit_of(a, dtype, row);
        if (lane >= a.parts) mine = {-INFINITY, 0.0f, 0.0f};
        const float high = wave_max(mine.m);
        const double d = mine.m == -INFINITY ? -INFINITY : static_cast<double>(mine.m) - static_cast<double>(high);
        const double f = exp(d);
        const double s = wave_sum(mine.s * f), t = wave_sum((mine.t + mine.s * fmax(d, -1000.0)) * f);
        const double of_row = finish(a, row, high, s, t, x, lane == 0);
        if (lane == 0) lse_at = of_row;
    }
    if (a.top == 0) return;
    __syncthreads();

    // The k-th largest of 64 maxima over a 64th of the groups each: a first bound,
    // usually little below the chunks' own k-th largest. (Its last bits are left 0.)
    best = 0;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) best = max(best, bests[w * kWave + lane]);
    uint32_t first = 0;
    for (int bit = 31; bit >= 8; --bit) {
        const uint32_t next = first | (1u << bit);
        if (count(best >= next) >= a.top) first = next;
    }
    first = max(first, 1u);
#pragma unroll 4
    for (int i = threadIdx.x; i < groups; i += kThreads)
        if (group_max[i] >= first) {
            const int place = atomicAdd(&grouped, 1);
            if (place < kList) group_id[place] = i;
        }
    __syncthreads();
    const int near = min(grouped, kList);
    for (int i = threadIdx.x / kGroup; i < near; i += kThreads / kGroup) {
        const int chunk = group_id[i] * kGroup + lane % kGroup;
        const uint32_t value = maxima[chunk];
        if (value >= first) {
            const int place = atomicAdd(&listed, 1);
            if (place < kList) {
                list_id[place] = chunk;
                list_max[place] = value;
            }
        }
    }
    __syncthreads();
    const int found = listed;
    const bool fits = found <= kList && grouped <= kList;
    const int n = min(found, kList);

    // The chunks' k-th largest, exactly; 1 (every value) where there are fewer.
    uint32_t bound = 1;
    if (fits) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t value = list_max[i];
            int above = 0, same = 0;
#pragma unroll 4
            for (int c = 0; c < n; ++c) {
                above += list_max[c] > value;
                same += list_max[c] == value;
            }
            if (above < a.top && above + same >= a.top) bound_at = value;  // all that write, write the same
        }
        __syncthreads();
        bound = max(bound_at, 1u);
    } else {  // many chunks near the top, such as equal ones
        uint32_t value = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = value | (1u << bit);
            int more = 0;
            for (int i = threadIdx.x; i < chunks; i += kThreads) more += maxima[i] >= next;
            more = wave_total(more);
            __syncthreads();
            if (lane == 0) bests[wave] = more;
            __syncthreads();
            more = 0;
#pragma unroll
            for (int w = 0; w < kJoinWaves; ++w) more += bests[w];
            if (more >= a.top) value = next;
        }
        bound = max(value, 1u);
    }

    // Values at or above the bound, of the chunks above it and of those that touch
    // it, block by block (a block's values follow the ones of the blocks before)
    // until there are k of those. Any order: a rank is a count of larger keys.
    const auto take = [&](int chunk) {  // the chunk's values by 16 lanes
        const int c = lane & (kValues - 1), vec = dtype == NQ_DTYPE_F32 ? 4 : 8;
        const int64_t i = static_cast<int64_t>(chunk / kWave) * kBlock + (c / vec) * (kWave * vec) + (chunk % kWave) * vec + c % vec;
        if (i >= a.vocab) return;
        const uint32_t order = ordered(nq::load_f32(a.logits, dtype, row * a.row_stride + i));
        if (order < bound) return;
        const int place = atomicAdd(&taken, 1);
        if (place < kKeys) keys[place] = key_of(order, static_cast<uint32_t>(i));
    };
    if (fits) {
        for (int i = threadIdx.x / kValues; i < n; i += kThreads / kValues) {
            const int chunk = list_id[i];
            const uint32_t value = list_max[i];
            if (value < bound) continue;
            int before = 0;  // chunks that touch the bound, of the blocks before
            if (value == bound)
#pragma unroll 4
                for (int c = 0; c < n; ++c) before += list_max[c] == bound && list_id[c] / kWave < chunk / kWave;
            if (before < a.top) take(chunk);
        }
    } else {
        int touching = 0;
        for (int block = 0; block < a.blocks; ++block) {
            const uint32_t value = maxima[block * kWave + lane];
            const uint64_t touch = __ballot(value == bound);
            const uint64_t in = __ballot(value > bound) | (touching < a.top ? touch : 0);
            touching += __popcll(touch);
            int c = 0;  // the in-th chunks, 16 lanes each
            for (uint64_t rest = in; rest; rest &= rest - 1, ++c)
                if (c % (kThreads / kValues) == threadIdx.x / kValues) take(block * kWave + __builtin_ctzll(rest));
        }
    }
    __syncthreads();
    const int reached = min(taken, kKeys);
    const double lse = lse_at;
    for (int i = threadIdx.x; i < reached; i += kThreads) {
        const uint64_t key = keys[i];
        int rank = 0;
#pragma unroll 8
        for (int c = 0; c < reached; ++c) rank += keys[c] > key;
        put_top(a, row, key, rank, lse);
    }
}

int64_t blocks_for(int64_t vocab) { return (vocab + kBlock - 1) / kBlock; }

// Parts of a row: enough workgroups for the chip, but a block for each wave.
int parts_for(int64_t rows, int64_t vocab) {
    constexpr int64_t kWorkgroups = 1024;
    const int64_t blocks = blocks_for(vocab);
    int64_t parts = (kWorkgroups + rows - 1) / rows;
    const int64_t most = (blocks + kWaves - 1) / kWaves;
    parts = parts < most ? parts : most;
    return static_cast<int>(parts < kMostParts ? parts : kMostParts);
}

}  // namespace

extern "C" int64_t nq_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) {
    if (rows <= 0 || rows > 0xffffff || vocab <= 0 || vocab > 0x7fffff00 || top < 0 || top > kMostTop || top > vocab)
        return -1;
    const int parts = parts_for(rows, vocab);
    if (!nq::launchable(rows * parts, kWaves * kWave) || (top && !nq::launchable(rows, kJoinWaves * kWave))) return -1;
    return parts == 1 && top == 0 ? 0 : rows * (parts * int64_t{16} + (top ? blocks_for(vocab) * (kWave + kWave / kGroup) * int64_t{4} : 0));
}

extern "C" int nq_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                 const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                 int64_t* top_ids, float* top_logprobs, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_ids || !top_logprobs)))
        return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(dtype)) return NQ_ERR_DTYPE;
    const int64_t need = nq_token_logprobs_workspace_bytes(rows, vocab, top);
    if (need < 0 || row_stride < vocab || row_stride > (int64_t{1} << 40)) return NQ_ERR_SHAPE;
    if (need > 0 && !workspace) return NQ_ERR_ARGUMENT;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(logits) % nq::dtype_bytes(dtype) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return NQ_ERR_ALIGNMENT;
    const int parts = parts_for(rows, vocab);
    const bool joins = parts > 1 || top > 0;
    float* sums = joins ? static_cast<float*>(workspace) : nullptr;
    uint32_t* maxima = top ? reinterpret_cast<uint32_t*>(sums + 4 * rows * parts) : nullptr;
    const Args a = {logits, tokens, row_stride, static_cast<int32_t>(vocab), top, parts,
                    static_cast<int32_t>(blocks_for(vocab)), sums, maxima,
                    top ? maxima + rows * blocks_for(vocab) * kWave : nullptr, logprobs, entropy, top_logprobs, top_ids};
    const dim3 grid(static_cast<unsigned>(rows * parts)), block(kWaves * kWave);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case NQ_DTYPE_F32: hipLaunchKernelGGL(k_token_logprobs<NQ_DTYPE_F32>, grid, block, 0, st, a); break;
        case NQ_DTYPE_F16: hipLaunchKernelGGL(k_token_logprobs<NQ_DTYPE_F16>, grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL(k_token_logprobs<NQ_DTYPE_BF16>, grid, block, 0, st, a); break;
    }
    if (const int status = nq::launch_status(); status != NQ_OK || !joins) return status;
    hipLaunchKernelGGL(k_token_logprobs_join, dim3(static_cast<unsigned>(rows)), dim3(kJoinWaves * kWave), 0, st, a, dtype);
    return nq::launch_status();
}
