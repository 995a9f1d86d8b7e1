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
    int32_t budget, first, recent, entries, kept, slots;  // kept: pages in front that stay; slots = entries - kept
};

// The weights in an order of whole numbers: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;

// One workgroup per sequence and kv head.
__global__ __launch_bounds__(kSelectThreads) void k_evict_select(const EvictArgs a) {
    __shared__ uint32_t bins[256], counts[2][kSelectWaves], found[2];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int b = blockIdx.x / p.kv_heads, g = blockIdx.x - b * p.kv_heads;
    const int page = 1 << p.page_shift, held = p.table_pages << p.page_shift;
    const int context = p.contexts[b], n = min(max(context, 0), held);
    const bool longer = n > a.budget;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_pages;
    int32_t* rows = a.rows + static_cast<int64_t>(blockIdx.x) * a.budget;
    if (g == 0) {
        for (int i = threadIdx.x; i < a.entries; i += kSelectThreads)
            a.table[static_cast<int64_t>(b) * a.entries + i] =
                longer && i >= a.kept ? a.into[static_cast<int64_t>(b) * a.slots + i - a.kept] : i < p.table_pages ? table[i] : -1;
        if (threadIdx.x == 0) a.lens[b] = longer ? a.budget : context;
    }
    if (!longer) {
        for (int i = threadIdx.x; i < a.budget; i += kSelectThreads) rows[i] = i < n ? i : -1;
        return;
    }
    for (int i = threadIdx.x; i < a.first; i += kSelectThreads) rows[i] = i;
    for (int i = threadIdx.x; i < a.recent; i += kSelectThreads) rows[a.budget - a.recent + i] = n - a.recent + i;
    // Of rows [a.first, end) the `keep` heaviest.
    const int end = n - a.recent, keep = a.budget - a.first - a.recent;
    if (keep == 0) return;
    const auto key_at = [&](int row) {
        const int32_t id = table[row >> p.page_shift];
        if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.pages)) return 0xffffffffu;
        return key_of(a.weights[(static_cast<int64_t>(id) * p.kv_heads + g) * page + (row & (page - 1))]);
    };
    // The keep-th greatest key, 8 bits at a time: `above` keys have a greater prefix.
    uint32_t prefix = 0, above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) bins[threadIdx.x] = 0;
        __syncthreads();
        for (int row = a.first + static_cast<int>(threadIdx.x); row < end; row += kSelectThreads) {
            const uint32_t key = key_at(row);
            if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&bins[key >> shift & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // Lane l has bins 255 - 4 l down to 252 - 4 l.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += c[j] = bins[255 - 4 * lane - j];
            const uint32_t upto = running_sum(sum);
            uint32_t before = above + upto - sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < static_cast<uint32_t>(keep) && before + c[j] >= static_cast<uint32_t>(keep)) {
                    found[0] = prefix | static_cast<uint32_t>(255 - 4 * lane - j) << shift;
                    found[1] = before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        prefix = found[0];
        above = found[1];
        __syncthreads();
    }
    // Keys above `prefix` are chosen, and the first keep - above of those that equal it.
    const uint32_t ties = static_cast<uint32_t>(keep) - above;
    const int per = ((end - a.first + kSelectWaves - 1) / kSelectWaves + kWave - 1) & ~(kWave - 1);
    const int begin = a.first + wave * per, stop = min(end, begin + per);
    uint32_t more = 0, same = 0;
    for (int row = begin + lane; row - lane < stop; row += kWave) {
        const uint32_t key = row < stop ? key_at(row) : 0u;
        more += __popcll(__ballot(row < stop && key > prefix));
        same += __popcll(__ballot(row < stop && key == prefix));
    }
    if (lane == 0) {
        counts[0][wave] = more;
        counts[1][wave] = same;
    }
    __syncthreads();
    more = same = 0;
    for (int w = 0; w < wave; ++w) {
        more += counts[0][w];
        same += counts[1][w];
    }
    for (int row = begin + lane; row - lane < stop; row += kWave) {
        const uint32_t key = row < stop ? key_at(row) : 0u;
        const uint64_t greater = __ballot(row < stop && key > prefix), equal = __ballot(row < stop && key == prefix);
        const uint64_t before = (uint64_t{1} << lane) - 1;
        const uint32_t my_same = same + __popcll(equal & before), my_more = more + __popcll(greater & before);
        const bool mine = (greater >> lane & 1) || ((equal >> lane & 1) && my_same < ties);
        if (mine) rows[a.first + my_more + min(my_same, ties)] = row;
        more += __popcll(greater);
        same += __popcll(equal);
    }
}

constexpr int kMoveThreads = 256;

// One workgroup per sequence, fresh page, kv head and K or V: the rows' bytes wait
// in LDS until the page's scale is known.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(const EvictArgs a) {
    constexpr int kWords = D / 4, kLine = kWords + 1, kMost = 128;
    __shared__ int64_t source[kMost];  // each row's page and head, or -1
    __shared__ float scales[kMost];
    __shared__ int offset[kMost];      // the row in its page
    __shared__ uint32_t top;
    extern __shared__ uint32_t bytes[];
    const Pages& p = a.p;
    const int page = 1 << p.page_shift, held = p.table_pages << p.page_shift;
    const int g = blockIdx.x % p.kv_heads;
    int unit = blockIdx.x / p.kv_heads;
    const bool is_v = unit & 1;
    unit >>= 1;
    const int b = unit / a.slots, slot = unit - b * a.slots;
    if (min(max(p.contexts[b], 0), held) <= a.budget) return;
    const int32_t id = a.into[static_cast<int64_t>(b) * a.slots + slot];
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.pages)) return;
    const int first = (a.kept + slot) << p.page_shift, count = min(page, a.budget - first);
    const int32_t* rows = a.rows + (static_cast<int64_t>(b) * p.kv_heads + g) * a.budget + first;
    const int64_t to = static_cast<int64_t>(id) * p.kv_heads + g;
    if (threadIdx.x == 0) top = 0;
    if (static_cast<int>(threadIdx.x) < count) {
        const int row = rows[threadIdx.x];
        const int32_t from = p.table[static_cast<int64_t>(b) * p.table_pages + (row >> p.page_shift)];
        const bool on = static_cast<uint32_t>(from) < static_cast<uint32_t>(p.pages);
        const int64_t at = on ? static_cast<int64_t>(from) * p.kv_heads + g : -1;
        source[threadIdx.x] = at;
        offset[threadIdx.x] = row & (page - 1);
        scales[threadIdx.x] = on ? (is_v ? p.v_scales : p.k_scales)[at] : 1.0f;
        if (!is_v) a.weights[to * page + threadIdx.x] = on ? a.weights[at * page + (row & (page - 1))] : __builtin_nanf("");
    }
    __syncthreads();
    float most = 0.0f;
    const auto hold = [&](int row, int c, uint32_t w) {
        bytes[row * kLine + c] = w;
        const float scale = scales[row];
        const float x[4] = {__builtin_amdgcn_cvt_f32_fp8(w, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale,
                            __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale};
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(x[j]) < INFINITY ? fabsf(x[j]) : 0.0f);
    };
    if (!is_v) {
        for (int i = threadIdx.x; i < count * kWords; i += kMoveThreads) {
            const int row = i / kWords, c = i - row * kWords;
            const int64_t at = source[row];
            hold(row, c, at < 0 ? 0x7f7f7f7fu : *reinterpret_cast<const uint32_t*>(p.k + (at * page + offset[row]) * D + 4 * c));
        }
    } else {
        for (int i = threadIdx.x; i < count * kWords; i += kMoveThreads) {
            const int c = i / count, row = i - c * count;  // neighbours read neighbouring bytes of V's lines
            const int64_t at = source[row];
            uint32_t w = 0x7f7f7f7fu;
            if (at >= 0) {
                w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= static_cast<uint32_t>(p.v[(at * D + 4 * c + j) * page + offset[row]]) << (8 * j);
            }
            hold(row, c, w);
        }
    }
    atomicMax(&top, __float_as_uint(most));  // values >= 0: ordered as their bits
    __syncthreads();
    const float scale = scale_for(__uint_as_float(top));
    if (threadIdx.x == 0) (is_v ? p.v_scales : p.k_scales)[to] = scale;
    for (int i = threadIdx.x; i < count * kWords; i += kMoveThreads) {
        const int row = is_v ? i % count : i / kWords, c = is_v ? i / count : i - row * kWords;
        const uint32_t w = rescaled4(bytes[row * kLine + c], scales[row], scale);
        if (!is_v) {
            *reinterpret_cast<uint32_t*>(p.k + (to * page + row) * D + 4 * c) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) p.v[(to * D + 4 * c + j) * page + row] = static_cast<uint8_t>(w >> (8 * j));
        }
    }
}

template <int D>
int launch_move(const EvictArgs& a, hipStream_t stream) {
    const size_t bytes = static_cast<size_t>(D + 4) << a.p.page_shift;  // 33 KB at most
    const dim3 grid(static_cast<unsigned>(2 * static_cast<int64_t>(a.p.batch) * a.slots * a.p.kv_heads)), block(kMoveThreads);
    hipLaunchKernelGGL(k_evict_move<D>, grid, block, bytes, stream, a);
    return nq::launch_status();
}

}  // namespace

extern "C" int64_t nq_paged_evict_workspace_bytes(int64_t batch, int32_t kv_heads, int32_t page_size, int64_t table_pages,
                                                  int64_t budget) {
    if (batch <= 0 || batch > 0xffffff || kv_heads <= 0 || kv_heads > 65535 || page_size <= 0 || page_size > 128 ||
        table_pages <= 0 || table_pages > 0x3fffffff / page_size || budget <= 0 || budget > 0x3fffffff)
        return -1;
    if (!nq::launchable(batch * kv_heads, kSelectThreads)) return -1;
    if (!nq::launchable(2 * batch * kv_heads * ((budget + page_size - 1) / page_size), kMoveThreads)) return -1;
    return 0;
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(kv->batch * kv->kv_heads));
    hipLaunchKernelGGL(k_evict_select, grid, dim3(kSelectThreads), 0, st, a);
    if (const int status = nq::launch_status(); status != NQ_OK || a.slots == 0) return status;
    switch (kv->head_dim) {
        case 64: return launch_move<64>(a, st);
        case 128: return launch_move<128>(a, st);
        default: return launch_move<256>(a, st);
    }
}
