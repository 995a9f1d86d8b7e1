// Eviction from an 8-bit paged cache by accumulated attention weight.
//
// Of a sequence with more than `budget` rows stay, for each kv head, the first
// ones, the newest ones, and of those between the heaviest:
//   the budget - first - recent largest by (weight, -row), NaN above all.
// The first launch finds these rows (a radix selection over the weights' ordered
// bits, then the places of the chosen rows in their order), the second moves them
// to fresh pages, whose scales are the append's: the least power of two that
// brings the page's rows within 448. Sources are read alone, so nothing has to
// wait for anything, and pages that others share stay whole.
#include <algorithm>

#include "nq_paged.h"

namespace {

using namespace nq::paged;

struct EvictArgs {
    Pages p;
    float* weights;        // [pages][kv_heads][page]
    const int32_t* into;   // [batch][slots]
    int32_t *table, *lens, *rows;  // [batch][entries], [batch], [batch][kv_heads][budget]
    uint32_t* bins;
    int32_t budget, first, recent, entries, kept, slots, parts;  // kept: pages in front that stay; slots = entries - kept
};

// The weights in an order of whole numbers: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kBins = 2048, kLevels = 3;  // of 11, 11 and 10 bits of a key, the highest first

__host__ __device__ constexpr int shift_of(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t bin_of(uint32_t key, int level) { return key >> shift_of(level) & (level == 2 ? 1023u : 2047u); }
// Whether a key has the threshold's bits above a level's.
__device__ __forceinline__ bool in_reach(uint32_t key, uint32_t prefix, int level) {
    return level == 0 || key >> shift_of(level - 1) == prefix >> shift_of(level - 1);
}

// What all workgroups of a sequence and kv head know.
struct Sequence {
    const int32_t* table;
    int32_t* rows;
    int g, n, end, keep;  // of rows [first, end) the `keep` heaviest
    bool longer;
};

__device__ __forceinline__ Sequence sequence_of(const EvictArgs& a, int unit) {
    const Pages& p = a.p;
    const int b = unit / p.kv_heads;
    Sequence s;
    s.g = unit - b * p.kv_heads;
    s.table = p.table + static_cast<int64_t>(b) * p.table_pages;
    s.rows = a.rows + static_cast<int64_t>(unit) * a.budget;
    s.n = min(max(p.contexts[b], 0), p.table_pages << p.page_shift);
    s.longer = s.n > a.budget;
    s.end = s.n - a.recent;
    s.keep = a.budget - a.first - a.recent;
    return s;
}

// The rows that stay whatever their weight, the new table and length.
__device__ __forceinline__ void write_frame(const EvictArgs& a, const Sequence& s, int unit) {
    const Pages& p = a.p;
    const int b = unit / p.kv_heads;
    if (s.g == 0) {
        for (int i = threadIdx.x; i < a.entries; i += kSelectThreads)
            a.table[static_cast<int64_t>(b) * a.entries + i] =
                s.longer && i >= a.kept ? a.into[static_cast<int64_t>(b) * a.slots + i - a.kept] : i < p.table_pages ? s.table[i] : -1;
        if (threadIdx.x == 0) a.lens[b] = s.longer ? a.budget : p.contexts[b];
    }
    if (!s.longer) {
        for (int i = threadIdx.x; i < a.budget; i += kSelectThreads) s.rows[i] = i < s.n ? i : -1;
        return;
    }
    for (int i = threadIdx.x; i < a.first; i += kSelectThreads) s.rows[i] = i;
    for (int i = threadIdx.x; i < a.recent; i += kSelectThreads) s.rows[a.budget - a.recent + i] = s.end + i;
}

__device__ __forceinline__ uint32_t key_at(const EvictArgs& a, const Sequence& s, int row) {
    const Pages& p = a.p;
    const int32_t id = s.table[row >> p.page_shift];
    const bool on = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pages);
    const int64_t at = (static_cast<int64_t>(on ? id : 0) * p.kv_heads + s.g << p.page_shift) + (row & ((1 << p.page_shift) - 1));
    const uint32_t key = key_of(a.weights[at]);
    return on ? key : 0xffffffffu;
}

// The sum of the values of the waves before this one.
__device__ __forceinline__ uint32_t waves_before(const uint32_t (&of)[kSelectWaves]) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t v = lane < wave ? of[lane] : 0u;
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(running_sum(v)), kWave - 1));
}

// The bin of a level that the keep-th greatest key lies in, and how many keys are
// greater than all of it: `above` of higher levels and those of this level's higher
// bins. Thread t has bins kBins - 1 - 2 t and the one below. All threads get the answer.
struct Bin {
    uint32_t bin, above;
};

__device__ __forceinline__ Bin find_bin(const uint32_t (&c)[2], uint32_t keep, uint32_t above, uint32_t (&waves)[kSelectWaves],
                                        uint32_t (&found)[2]) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t mine = c[0] + c[1], upto = running_sum(mine);
    if (lane == kWave - 1) waves[wave] = upto;
    __syncthreads();
    uint32_t before = above + upto - mine + waves_before(waves);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (before < keep && before + c[j] >= keep) {
            found[0] = kBins - 1 - 2 * threadIdx.x - j;
            found[1] = before;
        }
        before += c[j];
    }
    __syncthreads();
    const Bin b = {found[0], found[1]};
    __syncthreads();  // found and waves are read
    return b;
}

// Writes the rows of a wave, 64 at a time from `begin` on, whose keys are above the threshold, and
// the first `ties` of those that equal it; `more` and `same` of these lie before it.
struct Writer {
    uint32_t threshold, ties, more, same;

    __device__ __forceinline__ void operator()(const EvictArgs& a, const Sequence& s, int row, bool on, uint32_t key) {
        const int lane = threadIdx.x & (kWave - 1);
        const uint64_t greater = __ballot(on && key > threshold), equal = __ballot(on && key == threshold);
        const uint64_t before = (uint64_t{1} << lane) - 1;
        const uint32_t my_same = same + __popcll(equal & before), my_more = more + __popcll(greater & before);
        if ((greater >> lane & 1) || ((equal >> lane & 1) && my_same < ties)) s.rows[a.first + my_more + min(my_same, ties)] = row;
        more += __popcll(greater);
        same += __popcll(equal);
    }
};

// One workgroup per sequence and kv head. Up to 1024 R rows wait in registers as
// their keys; more are read again for each level. Bound by its rounds: table, weights,
// three levels of counting in LDS (24 sequences of up to 6001 rows, 4 heads: 8.8 us).
template <int R>
__global__ __launch_bounds__(kSelectThreads) void k_evict_select(const EvictArgs a) {
    __shared__ uint32_t bins[kBins], counts[2][kSelectWaves], found[2];
    const Sequence s = sequence_of(a, blockIdx.x);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int all = s.end - a.first;
    const bool held = s.longer && s.keep > 0 && all <= kSelectThreads * R;
    const int per = ((all + kSelectWaves - 1) / kSelectWaves + kWave - 1) & ~(kWave - 1);
    const int begin = a.first + wave * per, stop = min(s.end, begin + per);
    uint32_t keys[R];
    if (held) {
#pragma unroll
        for (int j = 0; j < R; ++j) keys[j] = key_at(a, s, min(begin + kWave * j + lane, s.end - 1));
    }
    write_frame(a, s, blockIdx.x);
    if (!s.longer || s.keep == 0) return;
    const auto for_each = [&](auto&& f) {
        if (held) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (begin + kWave * j >= stop) break;
                f(begin + kWave * j + lane, keys[j]);
            }
        } else {
            for (int row = begin + lane; row - lane < stop; row += kWave) f(row, key_at(a, s, min(row, s.end - 1)));
        }
    };
    uint32_t prefix = 0, above = 0;
    for (int level = 0; level < kLevels; ++level) {
        for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
        __syncthreads();
        for_each([&](int row, uint32_t key) {
            if (row < stop && in_reach(key, prefix, level)) atomicAdd(&bins[bin_of(key, level)], 1u);
        });
        __syncthreads();
        const uint32_t c[2] = {bins[kBins - 1 - 2 * threadIdx.x], bins[kBins - 2 - 2 * threadIdx.x]};
        const Bin b = find_bin(c, s.keep, above, counts[0], found);
        prefix |= b.bin << shift_of(level);
        above = b.above;
    }
    uint32_t more = 0, same = 0;
    for_each([&](int row, uint32_t key) {
        more += __popcll(__ballot(row < stop && key > prefix));
        same += __popcll(__ballot(row < stop && key == prefix));
    });
    if (lane == 0) {
        counts[0][wave] = more;
        counts[1][wave] = same;
    }
    __syncthreads();
    Writer write = {prefix, static_cast<uint32_t>(s.keep) - above, waves_before(counts[0]), waves_before(counts[1])};
    for_each([&](int row, uint32_t key) { write(a, s, row, row < stop, key); });
}

// The same with a long sequence's rows in parts of kPart, a workgroup each: a launch
// counts each level's bins (a.bins: [sequence and head][level][part][kBins]), the last
// one writes. Every workgroup adds the parts' counts up for itself.
constexpr int kPartsAtOnce = 8;  // counts of parts that a thread loads at once
constexpr int kPartKeys = 8, kPart = kSelectThreads * kPartKeys;

template <int LEVEL>
__global__ __launch_bounds__(kSelectThreads) void k_evict_part(const EvictArgs a) {
    __shared__ uint32_t bins[kBins], counts[2][kSelectWaves], found[2], passed[2];
    const int unit = blockIdx.x / a.parts, part = blockIdx.x - unit * a.parts;
    const Sequence s = sequence_of(a, unit);
    if (LEVEL == 0 && part == 0) write_frame(a, s, unit);
    if (!s.longer || s.keep == 0) return;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int from = a.first + part * kPart, parts = (s.end - a.first + kPart - 1) / kPart;
    if (part >= parts) return;
    const int begin = from + wave * (kPart / kSelectWaves), stop = min(s.end, begin + kPart / kSelectWaves);
    uint32_t keys[kPartKeys];
#pragma unroll
    for (int j = 0; j < kPartKeys; ++j) keys[j] = key_at(a, s, min(begin + kWave * j + lane, s.end - 1));
    uint32_t* mine = a.bins + static_cast<int64_t>(unit) * kLevels * a.parts * kBins;
    // All parts' counts, and those of the parts before this one.
    uint32_t c[LEVEL + 1][2] = {}, before[LEVEL + 1][2] = {};
    const uint32_t* at = mine + kBins - 2 - 2 * threadIdx.x;
    for (int i0 = 0; i0 < parts; i0 += kPartsAtOnce) {
        uint2 v[LEVEL + 1][kPartsAtOnce];
#pragma unroll
        for (int level = 0; level < LEVEL; ++level)
#pragma unroll
            for (int i = 0; i < kPartsAtOnce; ++i)
                v[level][i] = *reinterpret_cast<const uint2*>(at + (static_cast<int64_t>(level) * a.parts + min(i0 + i, parts - 1)) * kBins);
#pragma unroll
        for (int level = 0; level < LEVEL; ++level)
#pragma unroll
            for (int i = 0; i < kPartsAtOnce; ++i) {
                const uint32_t on = i0 + i < parts, ahead = i0 + i < part;
                c[level][0] += on ? v[level][i].y : 0u;
                c[level][1] += on ? v[level][i].x : 0u;
                before[level][0] += ahead ? v[level][i].y : 0u;
                before[level][1] += ahead ? v[level][i].x : 0u;
            }
    }
    uint32_t prefix = 0, above = 0;
    if (threadIdx.x < 2) passed[threadIdx.x] = 0;
#pragma unroll
    for (int level = 0; level < LEVEL; ++level) {
        const Bin b = find_bin(c[level], s.keep, above, counts[0], found);
        prefix |= b.bin << shift_of(level);
        above = b.above;
        if constexpr (LEVEL == kLevels) {
            uint32_t more = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t bin = kBins - 1 - 2 * threadIdx.x - j;
                if (bin > b.bin) more += before[level][j];
                if (level == kLevels - 1 && bin == b.bin) passed[1] = before[level][j];
            }
            more = running_sum(more);
            if (lane == kWave - 1 && more) atomicAdd(&passed[0], more);
        }
    }
    if constexpr (LEVEL < kLevels) {
        for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPartKeys; ++j)
            if (begin + kWave * j + lane < stop && in_reach(keys[j], prefix, LEVEL)) atomicAdd(&bins[bin_of(keys[j], LEVEL)], 1u);
        __syncthreads();
        uint32_t* to = mine + (static_cast<int64_t>(LEVEL) * a.parts + part) * kBins;
        for (int i = threadIdx.x; i < kBins; i += kSelectThreads) to[i] = bins[i];
    } else {
        uint32_t more = 0, same = 0;
#pragma unroll
        for (int j = 0; j < kPartKeys; ++j) {
            const bool on = begin + kWave * j + lane < stop;
            more += __popcll(__ballot(on && keys[j] > prefix));
            same += __popcll(__ballot(on && keys[j] == prefix));
        }
        if (lane == 0) {
            counts[0][wave] = more;
            counts[1][wave] = same;
        }
        __syncthreads();
        Writer write = {prefix, static_cast<uint32_t>(s.keep) - above, passed[0] + waves_before(counts[0]),
                        passed[1] + waves_before(counts[1])};
#pragma unroll
        for (int j = 0; j < kPartKeys; ++j) {
            const int row = begin + kWave * j + lane;
            write(a, s, row, row < stop, keys[j]);
        }
    }
}

// Threads that move a page: 64 bytes to each, or as many as a workgroup should have.
template <int D, int SHIFT>
constexpr int kMoveThreads = (D << SHIFT) <= 4096 ? 64 : (D << SHIFT) <= 8192 ? 128 : 256;

// Source pages that V's rows of a fresh page come from, first to last, up to which they
// are read whole, in 16-byte pieces, and their bytes picked from LDS: scattered bytes go
// to the memory pipe one lane at a time. 131000 rows, pages of 128, cut to a half (2 or 3 pages each) 115 us,
// 163 gathered; to a quarter 94 and 108; to an eighth (8 or 9) 85 and 86; to a thirty-second 87 and 82. Pages
// of 16: to a half 121 and 159, to an eighth 84 and 78, to a thirty-second 82 and 47.
constexpr int kMostSpan = 8;

// One workgroup per sequence, fresh page, kv head and K or V. A thread holds its
// share of the page's bytes in registers until the page's scale is known: 16-byte
// pieces of K's rows, words of four rows of V's lines, whose bytes it gathers. A page
// waits for its rows' numbers, their pages and their bytes one after the other and
// does little in between, so small pages take one wave: as many of them as possible wait
// at once (24 sequences to 2000 rows, pages of 32 rows of 64: 23.0 us the call, 34.3 with 256 threads each).
template <int D, int SHIFT, bool IS_V>
__device__ __forceinline__ void move_page(const EvictArgs& a, int64_t to, const int64_t* source, const float* scales,
                                          const uint32_t* keep, uint32_t& top, int count, const int* place,
                                          const int32_t* table, int span, int g, u32x4* block) {
    constexpr int kThreads = kMoveThreads<D, SHIFT>, kPage = 1 << SHIFT, kBytes = D << SHIFT;
    constexpr int kUnits = kBytes / (IS_V ? 4 : 16) / kThreads, kWords = IS_V ? 1 : 4;
    constexpr int kAtOnce = IS_V && kUnits > 16 ? 16 : kUnits;
    // Unit i is line i / (page / 4), rows 4 (i % (page / 4)) of V (a thread has the same rows of every
    // line); row i / (D / 16) of K.
    const Pages& p = a.p;
    const int quad = threadIdx.x & (kPage / 4 - 1);
    const auto row_of_unit = [&](int i) { return IS_V ? 4 * quad : i / (D / 16); };
    uint32_t w[kUnits][kWords];
    if constexpr (IS_V) {
        const uint32_t kept = keep[quad];
        if (span <= kMostSpan) {
            // Whole source pages through LDS, the next one on its way while bytes are picked.
            constexpr int kPieces = kBytes / 16 / kThreads;
            static_assert(kPieces * 16 * kThreads == kBytes, "a page is whole rounds of 16-byte pieces");
            u32x4 piece[kPieces];
            const auto load = [&](int i) {
                const int32_t id = table[i];
                const int64_t at = (static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pages) ? static_cast<int64_t>(id) : 0) * p.kv_heads + g;
#pragma unroll
                for (int k = 0; k < kPieces; ++k)
                    piece[k] = reinterpret_cast<const u32x4*>(p.v + at * kBytes)[threadIdx.x + k * kThreads];
            };
            int mine[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[j] = place[4 * quad + j];
#pragma unroll
            for (int k = 0; k < kUnits; ++k) w[k][0] = 0;
            load(0);
            for (int i = 0; i < span; ++i) {
                if (i) __syncthreads();  // the page before is read
#pragma unroll
                for (int k = 0; k < kPieces; ++k) block[threadIdx.x + k * kThreads] = piece[k];
                __syncthreads();
                load(min(i + 1, span - 1));
                const uint8_t* bytes = reinterpret_cast<const uint8_t*>(block) + threadIdx.x / (kPage / 4) * kPage;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (mine[j] >> SHIFT != i) continue;
#pragma unroll
                    for (int k = 0; k < kUnits; ++k)
                        w[k][0] |= static_cast<uint32_t>(bytes[k * (kThreads / (kPage / 4)) * kPage + (mine[j] & (kPage - 1))]) << (8 * j);
                }
            }
#pragma unroll
            for (int k = 0; k < kUnits; ++k) w[k][0] = (w[k][0] & kept) | (~kept & 0x7f7f7f7fu);
        } else {
            const uint8_t* from[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) from[j] = p.v + source[4 * quad + j];
#pragma unroll
            for (int k0 = 0; k0 < kUnits; k0 += kAtOnce) {
                uint32_t bytes[kAtOnce][4];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) bytes[k][j] = from[j][((threadIdx.x + (k0 + k) * kThreads) / (kPage / 4)) * kPage];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k)
                    w[k0 + k][0] = ((bytes[k][0] | bytes[k][1] << 8 | bytes[k][2] << 16 | bytes[k][3] << 24) & kept) | (~kept & 0x7f7f7f7fu);
            }
        }
    } else {
        u32x4 v[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int i = threadIdx.x + k * kThreads;
            v[k] = *reinterpret_cast<const u32x4*>(p.k + source[row_of_unit(i)] + 16 * (i % (D / 16)));
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int row = row_of_unit(threadIdx.x + k * kThreads);
            const bool on = keep[row / 4] >> (8 * (row & 3)) & 1u;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[k][j] = on ? v[k][j] : 0x7f7f7f7fu;
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const int row = row_of_unit(threadIdx.x + k * kThreads);
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            const float x[4] = {__builtin_amdgcn_cvt_f32_fp8(w[k][j], 0), __builtin_amdgcn_cvt_f32_fp8(w[k][j], 1),
                                __builtin_amdgcn_cvt_f32_fp8(w[k][j], 2), __builtin_amdgcn_cvt_f32_fp8(w[k][j], 3)};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float y = fabsf(x[m] * scales[IS_V ? row + m : row]);
                most = fmaxf(most, y < INFINITY ? y : 0.0f);
            }
        }
    }
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) most = fmaxf(most, __shfl_xor(most, m, kWave));
    if ((threadIdx.x & (kWave - 1)) == 0) atomicMax(&top, __float_as_uint(most));  // values >= 0: ordered as their bits
    __syncthreads();
    const float scale = scale_for(__uint_as_float(top));
    if (threadIdx.x == 0) (IS_V ? p.v_scales : p.k_scales)[to] = scale;
    uint8_t* out = (IS_V ? p.v : p.k) + to * kBytes;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const int i = threadIdx.x + k * kThreads, row = row_of_unit(i);
        if (row >= count) continue;
        if constexpr (IS_V) {
            const float from[4] = {scales[row], scales[row + 1], scales[row + 2], scales[row + 3]};
            const uint32_t v = rescaled4(w[k][0], from, scale);
            uint8_t* at = out + i / (kPage / 4) * kPage + row;
            if (row + 4 <= count) {
                *reinterpret_cast<uint32_t*>(at) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (row + j < count) at[j] = static_cast<uint8_t>(v >> (8 * j));
            }
        } else {
            const float from[4] = {scales[row], scales[row], scales[row], scales[row]};
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = rescaled4(w[k][j], from, scale);
            *reinterpret_cast<u32x4*>(out + row * D + 16 * (i % (D / 16))) = v;
        }
    }
}

template <int D, int SHIFT>
__global__ __launch_bounds__((kMoveThreads<D, SHIFT>)) void k_evict_move(const EvictArgs a) {
    constexpr int kPage = 1 << SHIFT;
    __shared__ int64_t source[kPage];    // each row's offset in K, or in line 0 of V; any page's where there is none
    __shared__ float scales[kPage];      // 0 behind the last row
    __shared__ uint32_t keep[kPage / 4];  // a byte for each row, 0 where its page is none
    __shared__ int place[kPage];         // each row's place behind the first one's page; negative behind the last row
    __shared__ u32x4 block[(D << SHIFT) / 16];
    __shared__ uint32_t top;
    const Pages& p = a.p;
    const int g = blockIdx.x % p.kv_heads;
    int unit = blockIdx.x / p.kv_heads;
    const bool is_v = unit & 1;
    unit >>= 1;
    const int b = unit / a.slots, slot = unit - b * a.slots;
    const int first = (a.kept + slot) << SHIFT, count = min(kPage, a.budget - first);
    const bool there = static_cast<int>(threadIdx.x) < count;
    // What does not wait for anything is loaded together.
    const int context = p.contexts[b];
    const int32_t id = a.into[static_cast<int64_t>(b) * a.slots + slot];
    const int32_t* rows = a.rows + (static_cast<int64_t>(b) * p.kv_heads + g) * a.budget + first;
    const int row = rows[min(static_cast<int>(threadIdx.x), count - 1)];
    const int lowest = rows[0] >> SHIFT, span = (rows[count - 1] >> SHIFT) - lowest + 1;
    if (min(max(context, 0), p.table_pages << SHIFT) <= a.budget) return;
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.pages)) return;
    const int64_t to = static_cast<int64_t>(id) * p.kv_heads + g;
    if (threadIdx.x == 0) top = 0;
    if (threadIdx.x < kPage) {
        const int32_t from = p.table[static_cast<int64_t>(b) * p.table_pages + (row >> SHIFT)];
        const bool on = static_cast<uint32_t>(from) < static_cast<uint32_t>(p.pages);
        const int64_t at = static_cast<int64_t>(on ? from : 0) * p.kv_heads + g;
        const int offset = row & (kPage - 1);
        place[threadIdx.x] = there ? row - (lowest << SHIFT) : -1;
        source[threadIdx.x] = is_v ? at * (D << SHIFT) + offset : ((at << SHIFT) + offset) * D;
        reinterpret_cast<uint8_t*>(keep)[threadIdx.x] = on ? 0xff : 0;
        scales[threadIdx.x] = !there ? 0.0f : on ? (is_v ? p.v_scales : p.k_scales)[at] : 1.0f;
        if (!is_v && there) a.weights[(to << SHIFT) + threadIdx.x] = on ? a.weights[(at << SHIFT) + offset] : __builtin_nanf("");
    }
    __syncthreads();
    const int32_t* from = p.table + static_cast<int64_t>(b) * p.table_pages + lowest;
    if (is_v) move_page<D, SHIFT, true>(a, to, source, scales, keep, top, count, place, from, span, g, block);
    else move_page<D, SHIFT, false>(a, to, source, scales, keep, top, count, place, from, span, g, block);
}

template <int D, int SHIFT>
int launch_move_as(const EvictArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(2 * static_cast<int64_t>(a.p.batch) * a.slots * a.p.kv_heads));
    hipLaunchKernelGGL((k_evict_move<D, SHIFT>), grid, dim3(kMoveThreads<D, SHIFT>), 0, stream, a);
    return nq::launch_status();
}

template <int D>
int launch_move(const EvictArgs& a, hipStream_t stream) {
    switch (a.p.page_shift) {
        case 4: return launch_move_as<D, 4>(a, stream);
        case 5: return launch_move_as<D, 5>(a, stream);
        case 6: return launch_move_as<D, 6>(a, stream);
        default: return launch_move_as<D, 7>(a, stream);
    }
}

constexpr int kFewKeys = 8, kManyKeys = 32;

// Parts of a sequence's rows, or 0 where a workgroup takes a sequence and head alone: where its
// registers hold the keys parts gain nothing (2, 4 and 8 sequences of 20000 rows, 8 heads: 55, 78 and 116 us
// either way), and where there are workgroups for half of the chip they cost (16: 193 us, 208 in parts). One sequence of
// 131000 rows takes 33 us in parts, 356 by a workgroup that reads them again and again.
int64_t parts_of(int64_t units, int64_t rows) {
    if (rows <= kSelectThreads * kManyKeys || units >= 128) return 0;
    return (rows + kPart - 1) / kPart;
}

}  // namespace

extern "C" int64_t nq_paged_evict_workspace_bytes(int64_t batch, int32_t kv_heads, int32_t page_size, int64_t table_pages,
                                                  int64_t budget) {
    if (batch <= 0 || batch > 0xffffff || kv_heads <= 0 || kv_heads > 65535 || page_size <= 0 || page_size > 128 ||
        table_pages <= 0 || table_pages > 0x3fffffff / page_size || budget <= 0 || budget > 0x3fffffff)
        return -1;
    const int64_t parts = parts_of(batch * kv_heads, table_pages * page_size);
    if (!nq::launchable(batch * kv_heads * std::max<int64_t>(parts, 1), kSelectThreads)) return -1;
    if (!nq::launchable(2 * batch * kv_heads * ((budget + page_size - 1) / page_size), 256)) return -1;
    return batch * kv_heads * parts * kLevels * kBins * static_cast<int64_t>(sizeof(uint32_t));
}

extern "C" int nq_paged_evict(const nq_paged_kv* kv, float* weights, const int32_t* into, int64_t budget, int64_t first,
                              int64_t recent, int32_t* page_table_out, int32_t* context_lens_out, int32_t* rows_out,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    if (!kv || !weights || !page_table_out || !context_lens_out || !rows_out) return NQ_ERR_ARGUMENT;
    EvictArgs a{};
    nq_paged_kv cache = *kv;
    cache.query_starts = cache.context_lens;  // not read
    if (const int st = check_pages(&cache, 1, a.p); st != NQ_OK) return st;
    const int64_t need = nq_paged_evict_workspace_bytes(kv->batch, kv->kv_heads, kv->page_size, kv->table_pages, budget);
    if (need < 0 || first < 0 || recent < 0 || first > budget || recent > budget - first) return NQ_ERR_SHAPE;
    if (need > 0 && !workspace) return NQ_ERR_ARGUMENT;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return NQ_ERR_ALIGNMENT;
    a.weights = weights;
    a.into = into;
    a.table = page_table_out;
    a.lens = context_lens_out;
    a.rows = rows_out;
    a.budget = static_cast<int32_t>(budget);
    a.first = static_cast<int32_t>(first);
    a.recent = static_cast<int32_t>(recent);
    a.entries = static_cast<int32_t>((budget + kv->page_size - 1) / kv->page_size);
    a.kept = static_cast<int32_t>(first / kv->page_size);
    a.slots = a.entries - a.kept;
    if (a.slots > 0 && !into) return NQ_ERR_ARGUMENT;
    // Other workgroups still read what one would write there.
    if (page_table_out == kv->page_table || context_lens_out == kv->context_lens) return NQ_ERR_ARGUMENT;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t units = kv->batch * kv->kv_heads;
    a.parts = static_cast<int32_t>(parts_of(units, kv->table_pages * kv->page_size));
    a.bins = static_cast<uint32_t*>(workspace);
    const dim3 block(kSelectThreads), grid(static_cast<unsigned>(units * std::max(a.parts, 1)));
    if (a.parts > 0) {
        hipLaunchKernelGGL(k_evict_part<0>, grid, block, 0, st, a);
        hipLaunchKernelGGL(k_evict_part<1>, grid, block, 0, st, a);
        hipLaunchKernelGGL(k_evict_part<2>, grid, block, 0, st, a);
        hipLaunchKernelGGL(k_evict_part<3>, grid, block, 0, st, a);
    } else if (kv->table_pages * kv->page_size <= kSelectThreads * kFewKeys) {
        hipLaunchKernelGGL(k_evict_select<kFewKeys>, grid, block, 0, st, a);
    } else {
        hipLaunchKernelGGL(k_evict_select<kManyKeys>, grid, block, 0, st, a);
    }
    if (const int status = nq::launch_status(); status != NQ_OK || a.slots == 0) return status;
    switch (kv->head_dim) {
        case 64: return launch_move<64>(a, st);
        case 128: return launch_move<128>(a, st);
        default: return launch_move<256>(a, st);
    }
}
