// How much attention each row of an 8-bit paged cache receives from a call's
// tokens, added to what it received before:
//   W[j, g] (+)= sum over tokens t that see j, q heads h of kv head g
//                of e^(scaling q[t, h] . K_j - lse[t, h])
// The attention's log-sum-exps make the weights final at once: one pass over K,
// no maximum, no second pass. A wave holds 64 cache rows of one kv head and forms
// S^T = K Q^T as the attention does (nq_paged_attention.h): a lane has 16 rows of
// one query row, whose exponentials it adds up over the query rows, 16 at a time;
// the 16 lanes of a row are added once, at the end. Each cache row belongs to one
// wave (or, joined in LDS in wave order, to one workgroup), so there are no
// atomics and the result does not hang on an order.
#include <algorithm>

#include "nq_paged_attention.h"

namespace {

using namespace nq::paged;

constexpr int kWaves = 4;

struct WeightArgs {
    Pages p;
    const void* q;
    const float* lse;        // [tokens][q_heads]
    const float* before;     // [pages][kv_heads][page]
    float* out;              // the same; may be `before`
    float scale;             // scaling * log2(e)
    int32_t q_heads, group, first, slots;  // slots: workgroups of a sequence and kv head
};

// 16 values of each lane summed over the 16 lanes of a row: lane n of a row gets the sum of value n.
__device__ __forceinline__ float sum_rows(float (&w)[16], int n) {
#pragma unroll
    for (int half = 8; half > 0; half /= 2) {
        const bool upper = n & half;
#pragma unroll
        for (int j = 0; j < half; ++j) {
            const float mine = upper ? w[j + half] : w[j], other = upper ? w[j] : w[j + half];
            w[j] = mine + __shfl_xor(other, half, kWave);
        }
    }
    return w[0];
}

// TURNS: the waves of a workgroup hold the same cache rows and take the query rows in
// turn; otherwise each wave has cache rows of its own and takes all query rows.
template <int D, int QT, bool TURNS>
__global__ __launch_bounds__(kWaves* kWave) void k_attention_weights(const WeightArgs a) {
    constexpr int kChunks = D / 64, kQSteps = 2 * kChunks, QP = Query<QT>::kParts, kBlock = 16;
    __shared__ float join[TURNS ? kWaves : 1][kTile];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1), n = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int g = blockIdx.x % p.kv_heads, unit = blockIdx.x / p.kv_heads;
    const int b = unit / a.slots, slot = unit - b * a.slots;
    const int start = p.starts[b], stop = p.starts[b + 1], context = p.contexts[b];
    const int begin = min(max(start, 0), p.tokens), end = min(max(stop, begin), p.tokens);
    const int page = 1 << p.page_shift, cache_rows = p.table_pages << p.page_shift;
    // Cache rows [0, rows) are the sequence's; query rows [0, all) are its tokens' heads.
    const int rows = static_cast<int>(min(max(static_cast<int64_t>(context) + (end - begin), int64_t{0}), static_cast<int64_t>(cache_rows)));
    const int all = (end - begin) * a.group;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_pages;
    if (end <= begin || rows <= a.first) return;
    const int tiles = (rows + kTile - 1) / kTile, per = TURNS ? 1 : kWaves;
    for (int at = a.first / kTile + slot * per; at < tiles; at += a.slots * per) {
        const int tile = at + (TURNS ? 0 : wave), base = tile * kTile;
        float w[kBlock];
#pragma unroll
        for (int j = 0; j < kBlock; ++j) w[j] = 0.0f;
        // Block n / 4 of 16 rows for K, block grp for the scores; blocks behind the last row read the last row's page.
        const auto entry = [&](int block) { return table[min(base + kBlock * block, rows - 1) >> p.page_shift]; };
        const int id_k = entry(n >> 2), id = entry(grp);
        const auto base_of = [&](int i) {
            return static_cast<int64_t>(static_cast<uint32_t>(i) < static_cast<uint32_t>(p.pages) ? i : 0) * p.kv_heads + g;
        };
        const float k_scale = p.k_scales[base_of(id)];
        u32x4 kf[4][kChunks];
        const uint8_t* k_at = p.k + (base_of(id_k) * page + ((base + kBlock * (n >> 2)) & (page - 1)) + (n & 3)) * D + 16 * grp;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < kChunks; ++c) kf[t][c] = *reinterpret_cast<const u32x4*>(k_at + 4 * t * D + 64 * c);
        // Query rows before this see none of the tile's rows.
        const int64_t blind = static_cast<int64_t>(base) - context;
        const int from = blind > 0 ? static_cast<int>(min(blind * a.group, static_cast<int64_t>(all))) & ~15 : 0;
        if (tile < tiles) {
            for (int r0 = from + (TURNS ? 16 * wave : 0); r0 < all; r0 += TURNS ? 16 * kWaves : 16) {
                const int r = r0 + n;
                const bool on = r < all;
                const int place = on ? r / a.group : 0, head = on ? g * a.group + r - place * a.group : 0;
                const int pos = on ? row_of(context, place, cache_rows) : -1;
                const int64_t row = static_cast<int64_t>(begin + place) * a.q_heads + head;
                u32x4 part[kQSteps][QP];
                const float f = k_scale * a.scale * load_query<QT, kQSteps>(a.q, row * D + 16 * grp, on, part);
                const float lse = on ? a.lse[row] * 1.4426950408889634f : 0.0f;
                f32x4 sc[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < kQSteps; ++c) {
                        const u32x4 k = widen_k<QT>(kf[t][c / 2][2 * (c & 1)], kf[t][c / 2][2 * (c & 1) + 1]);
                        if constexpr (QP == 2) sc[t] = mfma_k<QT>(lowered(k), part[c][1], sc[t]);
                        sc[t] = mfma_k<QT>(k, part[c][0], sc[t]);
                    }
                }
                const int seen = pos + 1 - (base + kBlock * grp);
#pragma unroll
                for (int j = 0; j < kBlock; ++j) {
                    float x = fmaf(sc[j >> 2][j & 3], f, -lse);
                    x = x > 0.0f ? 0.0f : x;  // what rounding leaves above 0; NaN stays
                    w[j] += j < seen ? exp2_hw(x) : 0.0f;
                }
            }
        }
        float total = sum_rows(w, n);
        const int row = base + kBlock * grp + n;
        if constexpr (TURNS) {
            join[wave][lane] = total;
            __syncthreads();
            if (wave == 0) total = (join[0][lane] + join[1][lane]) + (join[2][lane] + join[3][lane]);
        }
        if ((!TURNS || wave == 0) && row >= a.first && row < rows && static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pages)) {
            const int64_t i = base_of(id) * page + (row & (page - 1));
            a.out[i] = row < context ? a.before[i] + total : total;
        }
        if constexpr (TURNS) __syncthreads();  // join is read
    }
}

template <int D, int QT>
int launch_as(WeightArgs& a, bool turns, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.p.batch) * a.slots * a.p.kv_heads)), block(kWaves * kWave);
    if (turns) hipLaunchKernelGGL((k_attention_weights<D, QT, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_attention_weights<D, QT, false>), grid, block, 0, stream, a);
    return nq::launch_status();
}

template <int D>
int launch_for(WeightArgs& a, int q_dtype, bool turns, hipStream_t stream) {
    switch (q_dtype) {
        case NQ_DTYPE_F32: return launch_as<D, NQ_DTYPE_F32>(a, turns, stream);
        case NQ_DTYPE_F16: return launch_as<D, NQ_DTYPE_F16>(a, turns, stream);
        default: return launch_as<D, NQ_DTYPE_BF16>(a, turns, stream);
    }
}

}  // namespace

extern "C" int nq_attention_weights(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads, const nq_paged_kv* kv,
                                    float scaling, const float* lse, int64_t first, const float* weights, float* out,
                                    void* stream) {
    if (!q || !lse || !weights || !out) return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(q_dtype)) return NQ_ERR_DTYPE;
    WeightArgs a{};
    if (const int st = check_pages(kv, tokens, a.p); st != NQ_OK) return st;
    if (q_heads <= 0 || q_heads > 65535 || q_heads % kv->kv_heads || tokens * q_heads > 0x3fffffff || first < 0)
        return NQ_ERR_SHAPE;
    if (!(scaling > 0.0f) || !(scaling < INFINITY)) return NQ_ERR_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(q) & 15) return NQ_ERR_ALIGNMENT;
    const int64_t cache_rows = kv->table_pages * kv->page_size;
    if (first >= cache_rows) return NQ_OK;
    a.q = q;
    a.lse = lse;
    a.before = weights;
    a.out = out;
    a.scale = scaling * 1.4426950408889634f;
    a.q_heads = q_heads;
    a.group = q_heads / kv->kv_heads;
    a.first = static_cast<int32_t>(first);
    const bool turns = tokens * a.group > 64 * kv->batch;
    const int64_t tiles = (cache_rows + kTile - 1) / kTile - first / kTile, units = kv->batch * kv->kv_heads;
    const int64_t most = turns ? tiles : (tiles + kWaves - 1) / kWaves;
    a.slots = static_cast<int32_t>(std::max(int64_t{1}, std::min(most, (4096 + units - 1) / units)));
    if (!nq::launchable(units * a.slots, kWaves * kWave)) return NQ_ERR_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (kv->head_dim) {
        case 64: return launch_for<64>(a, q_dtype, turns, st);
        case 128: return launch_for<128>(a, q_dtype, turns, st);
        default: return launch_for<256>(a, q_dtype, turns, st);
    }
}
