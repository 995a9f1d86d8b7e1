// How much attention each row of an 8-bit paged cache receives from a call's
// tokens, added to what it received before:
//   W[j, g] (+)= sum over tokens t that see j, q heads h of kv head g
//                of e^(scaling q[t, h] . K_j - lse[t, h])
// The attention's log-sum-exps make the weights final at once: one pass over K,
// no maximum, no second pass. A wave holds 16, 32 or 64 cache rows of one kv head
// and forms S^T = K Q^T as the attention does (nq_paged_attention.h): a lane has a quarter of them for
// one query row, whose exponentials it adds up over the query rows, 16 at a time;
// the 16 lanes of a row are added once, at the end. Each cache row belongs to one
// wave (or, joined in LDS in wave order, to one workgroup), so there are no
// atomics and the result does not hang on an order.
#include <algorithm>

#include "nq_paged_attention.h"

namespace {

using namespace nq::paged;

constexpr float kLarge = 1024.0f;  // log-sum-exps beyond this have weights held to 1

struct WeightArgs {
    Pages p;
    const void* q;
    const float* lse;        // [tokens][q_heads]
    const float* before;     // [pages][kv_heads][page]
    float* out;              // the same; may be `before`
    float scale;             // scaling * log2(e)
    int32_t q_heads, group, first, slots;  // slots: workgroups of a sequence and kv head
};

// N values of each lane summed over the 16 lanes of a row: lane n of a row gets the sum of value n % N.
template <int N>
__device__ __forceinline__ float sum_rows(float (&w)[N], int n) {
#pragma unroll
    for (int half = 8; half >= N; half /= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] += __shfl_xor(w[j], half, kWave);
#pragma unroll
    for (int half = N / 2; half > 0; half /= 2) {
        const bool upper = n & half;
#pragma unroll
        for (int j = 0; j < half; ++j) {
            const float mine = upper ? w[j + half] : w[j], other = upper ? w[j] : w[j + half];
            w[j] = mine + __shfl_xor(other, half, kWave);
        }
    }
    return w[0];
}

template <bool TURNS>
constexpr int kWavesOf = TURNS ? 8 : 4;

// Single tokens are bound by the wait for the table's entries and then for K and q (56% of a wave's cycles), and
// by the vector unit, which works in 66% of the SIMDs' (32 sequences of up to 4000 rows: 81 MB in 26.5 us; pages of 16
// rows are 2 KB of K each). Prompts: 16 exponentials, 16 fused and 16 plain additions a product of 16 rows take 52% of the
// SIMDs' cycles, the matrix unit 18%, and two waves to a SIMD wait in 56% of theirs (1531 tokens
// after 517: 8e9 products and sums in 53 us, the first rows' workgroups the last to end).
// TURNS: the waves of a workgroup hold the same cache rows and take the query rows in
// turn; otherwise each wave has cache rows of its own and takes all query rows.
// ROWS: cache rows of a tile.
template <int D, int QT, bool TURNS, int ROWS>
__global__ __launch_bounds__(kWavesOf<TURNS>* kWave) void k_attention_weights(const WeightArgs a) {
    constexpr int kWaves = kWavesOf<TURNS>;
    constexpr int kChunks = D / 64, kQSteps = 2 * kChunks, QP = Query<QT>::kParts;
    constexpr int kBlock = ROWS / 4, kScores = ROWS / 16;  // rows of a lane; products of 16 rows
    // Many query rows: K is widened once, and the next rows of q are on their way, where there are registers for it.
    constexpr bool kHeld = TURNS && QT != NQ_DTYPE_F32 && D <= 128;
    __shared__ float join[TURNS ? kWaves : 1][kWave];
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
    const int tiles = (rows + ROWS - 1) / ROWS, per = TURNS ? 1 : kWaves;
    for (int at = a.first / ROWS + slot * per; at < tiles; at += a.slots * per) {
        const int tile = at + (TURNS ? 0 : wave), base = tile * ROWS;
        float w[kBlock];
#pragma unroll
        for (int j = 0; j < kBlock; ++j) w[j] = 0.0f;
        // Block n / 4 of kBlock rows for K, block grp for the scores; blocks behind the last row read the last row's page.
        const auto entry = [&](int block) { return table[min(base + kBlock * block, rows - 1) >> p.page_shift]; };
        const int id_k = entry(n >> 2), id = entry(grp);
        const auto base_of = [&](int i) {
            return static_cast<int64_t>(static_cast<uint32_t>(i) < static_cast<uint32_t>(p.pages) ? i : 0) * p.kv_heads + g;
        };
        const float k_scale = p.k_scales[base_of(id)];
        u32x4 kf[kScores][kChunks];
        const uint8_t* k_at = p.k + (base_of(id_k) * page + ((base + kBlock * (n >> 2)) & (page - 1)) + (n & 3)) * D + 16 * grp;
#pragma unroll
        for (int t = 0; t < kScores; ++t)
#pragma unroll
            for (int c = 0; c < kChunks; ++c) kf[t][c] = *reinterpret_cast<const u32x4*>(k_at + 4 * t * D + 64 * c);
        // Query rows before this see none of the tile's rows.
        const int64_t blind = static_cast<int64_t>(base) - context;
        const int from = blind > 0 ? static_cast<int>(min(blind * a.group, static_cast<int64_t>(all))) & ~15 : 0;
        const int row = base + kBlock * grp + (n & (kBlock - 1));
        const bool mine = n < kBlock && row >= a.first && row < rows && static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pages);
        const int64_t place_of_row = base_of(id) * page + (row & (page - 1));
        float old = 0.0f;
        if (!TURNS || wave == 0) old = a.before[place_of_row];  // a page's row, whatever it is
        u32x4 wide[kHeld ? kScores : 1][kHeld ? kQSteps : 1];
        if constexpr (kHeld) {
#pragma unroll
            for (int t = 0; t < kScores; ++t)
#pragma unroll
                for (int c = 0; c < kQSteps; ++c) wide[t][c] = widen_k<QT>(kf[t][c / 2][2 * (c & 1)], kf[t][c / 2][2 * (c & 1) + 1]);
        }
        // 16 query rows: this lane's one, as the products take it.
        struct Rows {
            u32x4 part[kQSteps][QP];
            float up, lse;
            int pos;
        };
        // The lane's next row, its token's place and its head in the group: stepped, not divided.
        constexpr int kStep = TURNS ? 16 * kWaves : 16;
        const int step_places = kStep / a.group, step_heads = kStep - step_places * a.group;
        int r0 = from + (TURNS ? 16 * wave : 0);
        int r = r0 + n, place = r / a.group, sub = r - place * a.group;
        const auto load = [&] {
            Rows x;
            const bool on = r < all;
            x.pos = on ? row_of(context, place, cache_rows) : -1;
            const int64_t at = on ? static_cast<int64_t>(begin + place) * a.q_heads + g * a.group + sub : 0;
            x.lse = on ? a.lse[at] : 0.0f;
            x.up = load_query<QT, kQSteps>(a.q, at * D + 16 * grp, on, x.part);
            r += kStep;
            place += step_places;
            sub += step_heads;
            if (sub >= a.group) {
                sub -= a.group;
                ++place;
            }
            return x;
        };
        if (tile < tiles) {
            Rows x;
            if (r0 < all) x = load();
            for (; r0 < all; r0 += kStep) {
                Rows next;
                if constexpr (kHeld) {
                    next = load();  // behind the last one: nothing
                } else {
                    // K's bytes as the compiler may not know them: it would widen them all ahead of the
                    // loop and take the registers of other waves (32 sequences, tiles of 64 rows: 33.6 us, 42.5 so).
#pragma unroll
                    for (int t = 0; t < kScores; ++t)
#pragma unroll
                        for (int c = 0; c < kChunks; ++c) asm volatile("" : "+v"(kf[t][c]));
                }
                f32x4 sc[kScores];
#pragma unroll
                for (int t = 0; t < kScores; ++t) {
                    sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < kQSteps; ++c) {
                        u32x4 k;
                        if constexpr (kHeld) k = wide[t][c];
                        else k = widen_k<QT>(kf[t][c / 2][2 * (c & 1)], kf[t][c / 2][2 * (c & 1) + 1]);
                        if constexpr (QP == 2) sc[t] = mfma_k<QT>(lowered(k), x.part[c][1], sc[t]);
                        sc[t] = mfma_k<QT>(k, x.part[c][0], sc[t]);
                    }
                }
                const float f = k_scale * a.scale * x.up, lse = x.lse * 1.4426950408889634f;
                const int seen = x.pos + 1 - (base + kBlock * grp);
                const bool large = fabsf(lse) > kLarge;  // of this lane's query row alone
                if (__ballot(seen < kBlock || large)) {
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) {
                        float y = fmaf(sc[j >> 2][j & 3], f, -lse);
                        if (large) y = y > 0.0f ? 0.0f : y;  // what rounding leaves above 0; NaN stays
                        w[j] += j < seen ? exp2_hw(y) : 0.0f;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) w[j] += exp2_hw(fmaf(sc[j >> 2][j & 3], f, -lse));
                }
                if constexpr (kHeld) x = next;
                else if (r0 + kStep < all) x = load();
            }
        }
        float total = sum_rows(w, n);
        if constexpr (TURNS) {
            join[wave][lane] = total;
            __syncthreads();
            total = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) total += join[i][lane];
        }
        if ((!TURNS || wave == 0) && mine) a.out[place_of_row] = row < context ? old + total : total;
        if constexpr (TURNS) __syncthreads();  // join is read
    }
}

// Whether the waves of a workgroup take the query rows of one tile in turn (`rows` of
// a sequence, `waves` tiles of all): where tiles are too few for the chip, or there are so many rows
// that the last tiles' would keep it waiting. bf16, 32/8 heads of 128, tiles of 64 rows, in turn and not:
// one sequence after 512 rows, 32 tokens (128 rows) 9.0 and 13.6 us, 128 tokens 13 and 33, 1531
// tokens 53 and 269; four of 512 tokens (512 tiles) 45 and 100; eight after 1000 (1088 tiles), 64 tokens (256 rows) 47
// and 27, 128 tokens 56 and 43, 512 tokens (2048 rows) 129 and 141; 32 of 64 tokens 95 and 38. Up to 64
// rows a wave has four products' worth: never.
bool takes_turns(int64_t rows, int64_t waves) { return rows > 64 && (waves < 768 || rows > 1024); }

// Cache rows of a tile, by a sequence's mean query rows and the number of tiles of 64. A wave's steps wait for one
// another (table, K, q, products, exponentials, sums), and all but the wait are shorter for fewer rows: with 16, 32 and
// 64 rows one token after 700 takes 4.1, 5.1 and 8.4 us, eight after 1000 5.3, 6.1 and 8.9, 32 after 1000 (4352 tiles)
// 12.6, 12.8 and 17.6, 32 of up to 4000 25.3, 26.5 and 33.7, one after 131000 71, 56 and 72. With more query rows
// reading q for every tile weighs more: eight sequences of 64 tokens, 256 query rows, 42, 28 and 26.
// In turn, 32 and 64 rows: one sequence after 512, 32 tokens (72 tiles) 5.6 and 9.1, 512 tokens (128 tiles) 19.4 and
// 23.1, two of 512 (256 tiles) 38 and 24.
int tile_rows(bool turns, int64_t rows, int64_t tiles) {
    if (turns) return tiles < 192 ? 32 : 64;
    if (rows > 64) return 64;
    return rows <= 16 && tiles < 4096 ? 16 : 32;
}

template <int D, int QT>
int launch_as(WeightArgs& a, bool turns, int rows, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.p.batch) * a.slots * a.p.kv_heads));
    const dim3 block(static_cast<unsigned>((turns ? kWavesOf<true> : kWavesOf<false>) * kWave));
    if (turns && rows == 32) hipLaunchKernelGGL((k_attention_weights<D, QT, true, 32>), grid, block, 0, stream, a);
    else if (turns) hipLaunchKernelGGL((k_attention_weights<D, QT, true, 64>), grid, block, 0, stream, a);
    else if (rows == 16) hipLaunchKernelGGL((k_attention_weights<D, QT, false, 16>), grid, block, 0, stream, a);
    else if (rows == 32) hipLaunchKernelGGL((k_attention_weights<D, QT, false, 32>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_attention_weights<D, QT, false, 64>), grid, block, 0, stream, a);
    return nq::launch_status();
}

template <int D>
int launch_for(WeightArgs& a, int q_dtype, bool turns, int rows, hipStream_t stream) {
    switch (q_dtype) {
        case NQ_DTYPE_F32: return launch_as<D, NQ_DTYPE_F32>(a, turns, rows, stream);
        case NQ_DTYPE_F16: return launch_as<D, NQ_DTYPE_F16>(a, turns, rows, stream);
        default: return launch_as<D, NQ_DTYPE_BF16>(a, turns, rows, stream);
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
    const int64_t units = kv->batch * kv->kv_heads;
    int64_t tiles = (cache_rows + kTile - 1) / kTile - first / kTile;
    const int64_t mean = (tokens * a.group + kv->batch - 1) / kv->batch;
    const bool turns = takes_turns(mean, units * tiles);
    const int rows = tile_rows(turns, mean, units * tiles);
    tiles = (cache_rows + rows - 1) / rows - first / rows;
    const int64_t most = turns ? tiles : (tiles + kWavesOf<false> - 1) / kWavesOf<false>;
    // (32 sequences of one token after up to 4000 rows, 8 heads, tiles of 64 rows: 33.7 us with 4096 or 8192 workgroups, 36.3 with
    // 2048, 39.8 with 1024.)
    a.slots = static_cast<int32_t>(std::max(int64_t{1}, std::min(most, (4096 + units - 1) / units)));
    if (!nq::launchable(units * a.slots, kWavesOf<true> * kWave)) return NQ_ERR_SHAPE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (kv->head_dim) {
        case 64: return launch_for<64>(a, q_dtype, turns, rows, st);
        case 128: return launch_for<128>(a, q_dtype, turns, rows, st);
        default: return launch_for<256>(a, q_dtype, turns, rows, st);
    }
}
