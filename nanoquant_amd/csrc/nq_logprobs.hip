// Log probability of given tokens, entropy of the distribution and its top
// alternatives from rows of logits.
//
// One read of the logits. A workgroup takes a part of a row: each of its four
// waves keeps 64 V values in registers, with m their maximum sums e^(x - m) and
// e^(x - m) (x - m), and picks its top k from the registers; the four lists meet
// in LDS. A second launch, one wave to a row, joins the parts: with M the
// largest m,
//   lse = M + log S, S = sum of S_p e^(m_p - M)
//   log p(t) = x_t - lse, entropy = log S - T / S, T = sum of (T_p + S_p (m_p - M)) e^(m_p - M)
// in fp64, rounded once.
#include <math.h>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;
constexpr int kMostTop = 32;
constexpr int kMostParts = 128;  // of a row: two to a lane of the joining wave
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const void* logits;
    const int64_t* tokens;
    int64_t row_stride;
    int32_t vocab, top, parts;
    float* sums;      // [rows][parts][4]: m, S, T
    uint64_t* lists;  // [rows][parts][top]: keys, largest first, 0 where there is none
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v = fmaxf(v, __shfl_xor(v, m, kWave));
    return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v += __shfl_xor(v, m, kWave);
    return v;
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

// The wave's top k of its values key[V] (0: none) into list[0, k), largest
// first. Element e of lane l has index first + (e / VEC) 64 VEC + l VEC + e % VEC.
// The k-th largest of the lanes' maxima bounds the k-th largest value from
// below: what reaches it is usually little more than k values. When it is more
// than a wave can rank at once, the bound is made exact, and of the values
// equal to it the lowest indexes are taken.
template <int V, int VEC>
__device__ __forceinline__ void wave_top(const uint32_t (&key)[V], int k, int64_t first, uint64_t* scratch,
                                         uint64_t* list) {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t best = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) best = max(best, key[e]);
    uint32_t bound = 0;
    for (int bit = 31; bit >= 8; --bit) {  // a bound from below need not be exact
        const uint32_t next = bound | (1u << bit);
        if (count(best >= next) >= k) bound = next;
    }
    if (bound == 0) bound = 1;
    int chosen = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) chosen += count(key[e] >= bound);
    int ties = 1 << 30;  // how many of the values equal to the bound are taken
    if (chosen > kWave) {
        bound = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = bound | (1u << bit);
            int n = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) n += count(key[e] >= next);
            if (n >= k) bound = next;
        }
        if (bound == 0) bound = 1;
        int above = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) above += count(key[e] > bound);
        ties = k - above;
    }
    int at = 0, tied = 0;
#pragma unroll
    for (int c = 0; c < V / VEC; ++c) {
        // Places in index order: lanes before this one, then its own elements.
        int tie_rank = tied;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const uint64_t mask = __ballot(key[c * VEC + e] == bound);
            tie_rank += lanes_before(mask);
            tied += __popcll(mask);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const uint32_t x = key[c * VEC + e];
            const bool tie = x == bound;
            const bool take = x > bound || (tie && tie_rank < ties);
            tie_rank += tie;
            const uint64_t mask = __ballot(take);
            if (take)
                scratch[at + lanes_before(mask)] =
                    key_of(x, static_cast<uint32_t>(first + c * (kWave * VEC) + lane * VEC + e));
            at += __popcll(mask);
        }
    }
    // A wave's LDS operations stay in order; the fence keeps the compiler to it.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uint64_t mine = lane < at ? scratch[lane] : 0;
    int rank = 0;
    for (int i = 0; i < at; ++i) rank += scratch[i] > mine;
    if (lane < at && rank < k) list[rank] = mine;
    if (lane >= at && lane < k) list[lane] = 0;
}

template <int DT, int V>
__global__ __launch_bounds__(kWaves* kWave) void k_logprob_parts(const Args a) {
    constexpr int VEC = DT == NQ_DTYPE_F32 ? 4 : 8;
    constexpr int kPart = kWaves * kWave * V;
    __shared__ uint64_t scratch[kWaves][kWave];
    __shared__ uint64_t lists[kWaves][kMostTop];
    __shared__ float part_sums[kWaves][3];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x - static_cast<int>(row) * a.parts;
    constexpr int kBytes = DT == NQ_DTYPE_F32 ? 4 : 2;
    const char* base = static_cast<const char*>(a.logits) + row * a.row_stride * kBytes;
    // Places count from the 16-byte boundary at or before the row's start.
    const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15) / kBytes;
    const int64_t first = static_cast<int64_t>(part) * kPart + wave * (kWave * V) - lead;

    float x[V];
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < V / VEC; ++c) {
        const int64_t i = first + c * (kWave * VEC) + lane * VEC;
        if (i >= 0 && i + VEC <= a.vocab) {
            const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + i * kBytes));
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if constexpr (DT == NQ_DTYPE_F32) {
                    x[c * VEC + e] = __uint_as_float(w[e]);
                } else {
                    const uint32_t h = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
                    x[c * VEC + e] = DT == NQ_DTYPE_BF16
                                         ? __uint_as_float(h << 16)
                                         : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                x[c * VEC + e] = i + e >= 0 && i + e < a.vocab ? element<DT>(base, i + e) : -INFINITY;
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) m = fmaxf(m, x[e]);
    m = wave_max(m);
    const float m_use = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float d = x[e] - m_use;
        const float w = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
        s += w;
        t = fmaf(w, fmaxf(d, -1000.0f), t);  // w is 0 there: 0 * -inf is not meant
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) {
        part_sums[wave][0] = m;
        part_sums[wave][1] = s;
        part_sums[wave][2] = t;
    }
    if (a.top > 0) {
        uint32_t key[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int64_t i = first + (e / VEC) * (kWave * VEC) + lane * VEC + e % VEC;
            key[e] = i >= 0 && i < a.vocab ? ordered(x[e]) : 0;
        }
        wave_top<V, VEC>(key, a.top, first, scratch[wave], lists[wave]);
    }
    __syncthreads();
    const int64_t at = row * a.parts + part;
    if (threadIdx.x == 0) {
        float mm = part_sums[0][0];
        for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, part_sums[w][0]);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float ss = 0.0f, tt = 0.0f;
        for (int w = 0; w < kWaves; ++w) {
            const float d = fmaxf(part_sums[w][0] - mu, -1000.0f);
            const float f = __builtin_amdgcn_exp2f((part_sums[w][0] - mu) * 1.4426950408889634f);
            ss += f * part_sums[w][1];
            tt += f * (part_sums[w][2] + d * part_sums[w][1]);
        }
        a.sums[4 * at] = mm;
        a.sums[4 * at + 1] = ss;
        a.sums[4 * at + 2] = tt;
    }
    // The four lists' keys, ranked against each other.
    const int n = kWaves * a.top;
    for (int i = threadIdx.x; i < n; i += kWaves * kWave) {
        const uint64_t mine = lists[i / a.top][i % a.top];
        int rank = 0;
        for (int w = 0; w < kWaves; ++w)
            for (int j = 0; j < a.top; ++j) {
                const uint64_t other = lists[w][j];
                rank += other > mine || (other == 0 && mine == 0 && w * a.top + j < i);
            }
        if (rank < a.top) a.lists[at * a.top + rank] = mine;
    }
}

// One wave per row.
__global__ __launch_bounds__(kWave) void k_logprob_join(const Args a, int dtype) {
    // Keys that reach the k-th largest of the lanes' best: at most k lanes with
    // two parts of k keys each.
    __shared__ uint64_t keys[2 * kMostTop * kMostTop];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    float m = -INFINITY;
    for (int p = lane; p < a.parts; p += kWave) m = fmaxf(m, a.sums[4 * (row * a.parts + p)]);
    m = wave_max(m);
    double s = 0.0, t = 0.0;
    for (int p = lane; p < a.parts; p += kWave) {
        const float* sums = a.sums + 4 * (row * a.parts + p);
        const double d = static_cast<double>(sums[0]) - (m == -INFINITY ? 0.0 : static_cast<double>(m));
        const double f = exp(d);
        s += f * static_cast<double>(sums[1]);
        t += f * (static_cast<double>(sums[2]) + fmax(d, -1000.0) * static_cast<double>(sums[1]));
    }
    s = wave_sum(s);
    t = wave_sum(t);
    const double log_s = log(s);
    const double lse = static_cast<double>(m) + log_s;
    if (lane == 0) {
        const int64_t token = a.tokens[row];
        const bool ok = token >= 0 && token < a.vocab;
        const float x = ok ? nq::load_f32(a.logits, dtype, row * a.row_stride + token) : __builtin_nanf("");
        a.logprobs[row] = static_cast<float>(static_cast<double>(x) - lse);
        // Nothing to weigh (m -inf), an infinity or a NaN: no distribution, NaN.
        a.entropy[row] = static_cast<float>(log_s - t / s);
    }
    if (a.top == 0) return;
    const uint64_t* lists = a.lists + row * a.parts * a.top;
    uint64_t best = 0;
    for (int p = lane; p < a.parts; p += kWave) {
        const uint64_t head = lists[p * a.top];
        best = head > best ? head : best;
    }
    uint64_t bound = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t next = bound | (uint64_t{1} << bit);
        if (count(best >= next) >= a.top) bound = next;
    }
    if (bound == 0) bound = 1;
    int at = 0;
    for (int p0 = 0; p0 < a.parts; p0 += kWave) {
        for (int j = 0; j < a.top; ++j) {
            const uint64_t key = p0 + lane < a.parts ? lists[(p0 + lane) * a.top + j] : 0;
            const uint64_t mask = __ballot(key >= bound);
            if (!mask) break;  // each list falls
            if (key >= bound) keys[at + lanes_before(mask)] = key;
            at += __popcll(mask);
        }
    }
    __syncthreads();
    for (int i = lane; i < at; i += kWave) {
        const uint64_t mine = keys[i];
        int rank = 0;
        for (int j = 0; j < at; ++j) rank += keys[j] > mine;
        if (rank < a.top) {
            a.top_ids[row * a.top + rank] = 0xffffffffu - static_cast<uint32_t>(mine & 0xffffffffu);
            a.top_logprobs[row * a.top + rank] =
                static_cast<float>(static_cast<double>(value_of(static_cast<uint32_t>(mine >> 32))) - lse);
        }
    }
}

struct Plan {
    int values, parts;  // values to a lane, parts of a row
};

// 8 values to a lane where 32 would leave CUs without work, unless a row then
// has more parts than the joining wave holds.
Plan plan_for(int64_t rows, int64_t vocab) {
    const int64_t lead = 7;  // places before a row's start, at most
    const auto parts = [&](int v) { return (vocab + lead + kWaves * kWave * v - 1) / (kWaves * kWave * v); };
    const int v = rows * parts(32) < 1024 && parts(8) <= kMostParts ? 8 : 32;
    return {v, static_cast<int>(parts(v) < (1 << 20) ? parts(v) : (1 << 20))};
}

int64_t bytes_for(int64_t rows, int64_t parts, int64_t top) { return rows * parts * (16 + 8 * top); }

}  // namespace

extern "C" int64_t nq_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) {
    if (rows <= 0 || rows > 0xffffff || vocab <= 0 || top < 0 || top > kMostTop || top > vocab) return -1;
    const Plan plan = plan_for(rows, vocab);
    if (plan.parts > kMostParts || rows * plan.parts > 0x7fffffff) return -1;
    return bytes_for(rows, plan.parts, top);
}

extern "C" int nq_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                 const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                 int64_t* top_ids, float* top_logprobs, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    if (!logits || !tokens || !logprobs || !entropy || !workspace || (top > 0 && (!top_ids || !top_logprobs)))
        return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(dtype)) return NQ_ERR_DTYPE;
    const int64_t need = nq_token_logprobs_workspace_bytes(rows, vocab, top);
    if (need < 0 || row_stride < vocab || row_stride > (int64_t{1} << 40)) return NQ_ERR_SHAPE;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(logits) % nq::dtype_bytes(dtype) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return NQ_ERR_ALIGNMENT;
    const Plan plan = plan_for(rows, vocab);
    Args a{};
    a.logits = logits;
    a.tokens = tokens;
    a.row_stride = row_stride;
    a.vocab = static_cast<int32_t>(vocab);
    a.top = top;
    a.parts = plan.parts;
    a.sums = static_cast<float*>(workspace);
    a.lists = reinterpret_cast<uint64_t*>(a.sums + 4 * rows * plan.parts);
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(rows * plan.parts)), block(kWaves * kWave);
#define NQ_PARTS(DT)                                                                        \
    if (plan.values == 8) hipLaunchKernelGGL((k_logprob_parts<DT, 8>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((k_logprob_parts<DT, 32>), grid, block, 0, st, a)
    switch (dtype) {
        case NQ_DTYPE_F32: NQ_PARTS(NQ_DTYPE_F32); break;
        case NQ_DTYPE_F16: NQ_PARTS(NQ_DTYPE_F16); break;
        default: NQ_PARTS(NQ_DTYPE_BF16); break;
    }
#undef NQ_PARTS
    if (const int status = nq::launch_status(); status != NQ_OK) return status;
    hipLaunchKernelGGL(k_logprob_join, dim3(static_cast<unsigned>(rows)), dim3(kWave), 0, st, a, dtype);
    return nq::launch_status();
}
