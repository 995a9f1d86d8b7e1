// Log probability of given tokens, entropy of the distribution and its top
// alternatives from rows of logits, in one read.
//
// A workgroup of four waves takes a part of a row, all of it where there are rows
// enough. A lane keeps its own running maximum m and, relative to it, s = sum
// e^(x - m) and t = sum e^(x - m) (x - m); the next 64 x 16 values of its wave
// are on their way while these are worked on. With M the largest of the maxima,
//   lse = M + log S, S = sum s e^(m - M)
//   log p(x) = x - lse, entropy = log S - T / S, T = sum (t + s (m - M)) e^(m - M)
// rounded once from fp64; a row's parts meet in a second launch. Each wave keeps its k largest values in LDS; a block of values costs one
// comparison unless some value is above the smallest of them.
#include <math.h>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;
constexpr int kMostTop = 32;
constexpr int kRoom = kWave;  // values that a list takes in at once
constexpr int kValues = 16;   // of a lane at once
constexpr int kMostParts = 64;  // of a row: one to a lane of the joining wave
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));

struct Args {
    const void* logits;
    const int64_t* tokens;
    int64_t row_stride;
    int32_t vocab, top, parts;
    float* sums;       // [rows][parts][4]: M, S, T of a part (parts > 1)
    uint64_t* lists;   // [rows][parts][top]: its keys, largest first, 0 where there is none
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

__device__ __forceinline__ int lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

template <int DT>
__device__ __forceinline__ float element(const void* p, int64_t i) { return nq::load_f32(p, DT, i); }

// A wave's LDS operations stay in order; this keeps the compiler to it.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ uint64_t lane_key(uint64_t key, int lane) {
    return (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key >> 32), lane))) << 32) |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key & 0xffffffffu), lane));
}

// How many of the k keys of a list, largest first, are above `key`.
__device__ __forceinline__ int above_in(const uint64_t* list, int k, uint64_t key) {
    int low = 0;
#pragma unroll
    for (int step = kMostTop; step >= 1; step /= 2)
        if (low + step <= k && list[low + step - 1] > key) low += step;
    return low;
}

// The wave's list of its k largest keys so far, largest first (0 where there is
// none), and the order of the smallest of them.
struct Best {
    uint64_t* list;  // LDS, [kMostTop + kRoom]: the list, then room for what comes in
    uint32_t last;
};

// Takes a block of values into the list: key[e] is the order of the value with
// index first + (e / VEC) 64 VEC + lane VEC + e % VEC, 0 for none. Blocks come in
// index order, so a value equal to the last one stays out. When more than
// kRoom values are above it, the k-th largest of the lanes' maxima bounds
// from below what can get in; when that leaves too many, the block's own k-th
// largest value is found bit by bit, and of those equal to it the lowest
// indexes are taken.
template <int VEC>
__device__ __forceinline__ void take(Best& best, const uint32_t (&key)[kValues], int k, int64_t first) {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t bound = best.last + 1;
    int chosen = 0;
#pragma unroll
    for (int e = 0; e < kValues; ++e) chosen += count(key[e] >= bound);
    if (chosen > kRoom) {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < kValues; ++e) most = max(most, key[e]);
        uint32_t least = 0;
        for (int bit = 31; bit >= 8; --bit) {  // a bound from below need not be exact
            const uint32_t next = least | (1u << bit);
            if (count(most >= next) >= k) least = next;
        }
        bound = max(bound, least);
        chosen = 0;
#pragma unroll
        for (int e = 0; e < kValues; ++e) chosen += count(key[e] >= bound);
    }
    int at = 0;
    const auto put = [&](int e, bool in) {
        const uint64_t mask = __ballot(in);
        if (!mask) return;
        if (in)
            best.list[kMostTop + at + lanes_before(mask)] =
                key_of(key[e], static_cast<uint32_t>(first + (e / VEC) * (kWave * VEC) + lane * VEC + e % VEC));
        at += __popcll(mask);
    };
    if (chosen <= kRoom) {
#pragma unroll
        for (int e = 0; e < kValues; ++e) put(e, key[e] >= bound);
    } else {
        // More than k values are at or above the last bound, so the k-th largest is no less.
        bound = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = bound | (1u << bit);
            int n = 0;
#pragma unroll
            for (int e = 0; e < kValues; ++e) n += count(key[e] >= next);
            if (n >= k) bound = next;
        }
        int ties = k, tied = 0;  // of the values equal to it: taken, seen so far
#pragma unroll
        for (int e = 0; e < kValues; ++e) ties -= count(key[e] > bound);
#pragma unroll
        for (int c = 0; c < kValues / VEC; ++c) {
            // Places in index order: lanes before this one, then its own values.
            int tie_rank = tied;
#pragma unroll
            for (int e = c * VEC; e < (c + 1) * VEC; ++e) {
                const uint64_t mask = __ballot(key[e] == bound);
                tie_rank += lanes_before(mask);
                tied += __popcll(mask);
            }
#pragma unroll
            for (int e = c * VEC; e < (c + 1) * VEC; ++e) {
                const bool tie = key[e] == bound;
                put(e, key[e] > bound || (tie && tie_rank < ties));
                tie_rank += tie;
            }
        }
    }
    wave_lds_sync();
    // Lane i holds the list's i-th key and the i-th that came in: their ranks.
    const uint64_t had = lane < k ? best.list[lane] : 0, came = lane < at ? best.list[kMostTop + lane] : 0;
    const int held = count(had != 0);
    int had_rank = lane, came_rank = 0;
    for (int i = 0; i < held; ++i) came_rank += lane_key(had, i) > came;
    for (int i = 0; i < at; ++i) {
        const uint64_t key = lane_key(came, i);
        had_rank += key > had;
        came_rank += key > came;
    }
    wave_lds_sync();
    if (had && had_rank < k) best.list[had_rank] = had;
    if (came && came_rank < k) best.list[came_rank] = came;
    wave_lds_sync();
    best.last = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(best.list[k - 1] >> 32));
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

template <int DT, bool TOP>
__global__ __launch_bounds__(kWaves* kWave) void k_token_logprobs(const Args a) {
    constexpr int VEC = Block<DT>::kVec, kBytes = Block<DT>::kBytes;
    constexpr int kBlock = kWave * kValues;
    __shared__ uint64_t lists[TOP ? kWaves : 1][kMostTop + kRoom];
    __shared__ Sums sums[kWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x - static_cast<int>(row) * a.parts;
    const char* base = static_cast<const char*>(a.logits) + row * a.row_stride * kBytes;
    const int blocks = (a.vocab + kBlock - 1) / kBlock, each = (blocks + a.parts - 1) / a.parts;
    const int begin = part * each + wave, end = min(blocks, (part + 1) * each);
    const auto first_of = [&](int block) { return static_cast<int64_t>(block) * kBlock; };
    Best best{lists[TOP ? wave : 0], 0};
    if (TOP) {
        if (lane < kMostTop) best.list[lane] = 0;
        wave_lds_sync();
    }

    float m = -INFINITY, s = 0.0f, t = 0.0f;
    Block<DT> next;
    if (begin < end) load_block<DT>(next, base, first_of(begin), a.vocab);
    for (int block = begin; block < end; block += kWaves) {
        float x[kValues];
        unpack<DT>(next, x);
        if (block + kWaves < end) load_block<DT>(next, base, first_of(block + kWaves), a.vocab);
        float high = x[0];
        bool nan = x[0] != x[0];
#pragma unroll
        for (int e = 1; e < kValues; ++e) {
            high = fmaxf(high, x[e]);
            if (TOP) nan |= x[e] != x[e];
        }
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
        s += bs;
        t += bt;
        m = m_new;
        if (TOP && __ballot(nan || ordered(high) > best.last)) {
            const int64_t first = first_of(block);
            uint32_t key[kValues];
#pragma unroll
            for (int e = 0; e < kValues; ++e) {
                const int64_t i = first + (e / VEC) * (kWave * VEC) + lane * VEC + e % VEC;
                key[e] = i < a.vocab ? ordered(x[e]) : 0;  // outside the row: -inf for the sums, nothing here
            }
            take<VEC>(best, key, a.top, first);
        }
    }

    const float wave_m = wave_max(m);
    const Sums mine = moved({m, s, t}, wave_m);
    const Sums joined{wave_m, wave_sum(mine.s), wave_sum(mine.t)};
    if (lane == 0) sums[wave] = joined;
    const float x = wave == 0 && a.parts == 1 ? logit_of(a, DT, row) : 0.0f;
    __syncthreads();
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
    const int64_t at = row * a.parts + part;
    double lse = 0.0;
    if (a.parts == 1) {
        lse = finish(a, row, all.m, all.s, all.t, x, threadIdx.x == 0);
    } else if (threadIdx.x == 0) {
        a.sums[4 * at] = all.m;
        a.sums[4 * at + 1] = all.s;
        a.sums[4 * at + 2] = all.t;
    }
    if (!TOP) return;
    // The waves' lists as one: a key's rank is its place in its own and what the others have above it.
    for (int i = threadIdx.x; i < kWaves * kMostTop; i += kWaves * kWave) {
        const int w0 = i / kMostTop, j = i % kMostTop;
        if (j >= a.top) continue;
        const uint64_t key = lists[w0][j];
        int rank = j;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            if (w != w0) rank += above_in(lists[w], a.top, key);
        if (a.parts == 1) {
            put_top(a, row, key, rank, lse);
        } else if (key) {
            if (rank < a.top) a.lists[at * a.top + rank] = key;
        } else {
            // Empty places follow all lists' keys (rank counts the others' and j its
            // own): those of the lists before this one come first.
            for (int w = 0; w < w0; ++w) rank += a.top - above_in(lists[w], a.top, 0);
            if (rank < a.top) a.lists[at * a.top + rank] = 0;
        }
    }
}

// A row's parts: one to a lane for the sums; the lists in LDS.
__global__ __launch_bounds__(kWaves* kWave) void k_token_logprobs_join(const Args a, int dtype) {
    __shared__ uint64_t lists[kMostParts * kMostTop], reach[kMostParts * kMostTop];
    __shared__ int reached;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t row = blockIdx.x;
    const int keys = a.parts * a.top;
    for (int i = threadIdx.x; i < keys; i += kWaves * kWave) lists[i] = a.lists[row * keys + i];
    if (threadIdx.x == 0) reached = 0;
    const float* at = a.sums + 4 * (row * a.parts + (lane < a.parts ? lane : 0));
    Sums mine{at[0], at[1], at[2]};
    const float x = logit_of(a, dtype, row);
    if (lane >= a.parts) mine = {-INFINITY, 0.0f, 0.0f};
    const float high = wave_max(mine.m);
    const double d = mine.m == -INFINITY ? -INFINITY : static_cast<double>(mine.m) - static_cast<double>(high);
    const double f = exp(d);
    const double s = wave_sum(mine.s * f), t = wave_sum((mine.t + mine.s * fmax(d, -1000.0)) * f);
    const double lse = finish(a, row, high, s, t, x, threadIdx.x == 0);
    if (a.top == 0) return;
    __syncthreads();
    // The r-th largest of the lists' j-th keys, with r lists of j keys each at
    // least top together, bounds the top-th largest key from below.
    const int j = (a.top + a.parts - 1) / a.parts, r = (a.top + j - 1) / j;
    const uint32_t best = lane < a.parts ? static_cast<uint32_t>(lists[lane * a.top + j - 1] >> 32) : 0;
    uint32_t bound = 0;
    for (int bit = 31; bit >= 8; --bit) {
        const uint32_t next = bound | (1u << bit);
        if (count(best >= next) >= r) bound = next;
    }
    // The keys that reach it, in any order: a rank is a count of larger keys.
    for (int i = threadIdx.x; i < keys; i += kWaves * kWave) {
        const uint64_t key = lists[i];
        if (key && static_cast<uint32_t>(key >> 32) >= bound) reach[atomicAdd(&reached, 1)] = key;
    }
    __syncthreads();
    const int n = reached;
    for (int i = threadIdx.x; i < n; i += kWaves * kWave) {
        const uint64_t key = reach[i];
        int rank = 0;
#pragma unroll 8
        for (int c = 0; c < n; ++c) rank += reach[c] > key;
        put_top(a, row, key, rank, lse);
    }
}

// Parts of a row: enough workgroups for the chip, but a block for each wave.
int parts_for(int64_t rows, int64_t vocab) {
    constexpr int64_t kWorkgroups = 1024;
    const int64_t blocks = (vocab + kWave * kValues - 1) / (kWave * kValues);
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
    return parts == 1 ? 0 : rows * parts * (16 + 8 * static_cast<int64_t>(top));
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
    float* sums = static_cast<float*>(workspace);
    const Args a = {logits, tokens, row_stride, static_cast<int32_t>(vocab), top, parts, sums,
                    reinterpret_cast<uint64_t*>(sums + 4 * rows * parts), logprobs, entropy, top_logprobs, top_ids};
    const dim3 grid(static_cast<unsigned>(rows * parts)), block(kWaves * kWave);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NQ_LOGPROBS(DT)                                                                  \
    if (top) hipLaunchKernelGGL((k_token_logprobs<DT, true>), grid, block, 0, st, a);    \
    else hipLaunchKernelGGL((k_token_logprobs<DT, false>), grid, block, 0, st, a)
    switch (dtype) {
        case NQ_DTYPE_F32: NQ_LOGPROBS(NQ_DTYPE_F32); break;
        case NQ_DTYPE_F16: NQ_LOGPROBS(NQ_DTYPE_F16); break;
        default: NQ_LOGPROBS(NQ_DTYPE_BF16); break;
    }
#undef NQ_LOGPROBS
    if (const int status = nq::launch_status(); status != NQ_OK || parts == 1) return status;
    hipLaunchKernelGGL(k_token_logprobs_join, dim3(static_cast<unsigned>(rows)), block, 0, st, a, dtype);
    return nq::launch_status();
}
