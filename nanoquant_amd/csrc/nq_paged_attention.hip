// Attention over the 8-bit paged cache: plan, merge of the splits, entry points.
#include <algorithm>

#include "nq_paged_attention.h"

namespace nq {
namespace paged {

template <> int launch_paged_attention<64>(const AttnArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_paged_attention<128>(const AttnArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_paged_attention<256>(const AttnArgs&, const AttnPlan&, int, hipStream_t);

// How a call is laid out. All rules go by sizes that the host knows: the page
// table's width stands for the cache's length, the mean for the query rows of a
// sequence (its tokens times the q heads of a kv head). Times: 32/8 heads of 128,
// after that many cached rows.
//
// Usually a slot's waves share its rows and take the cache's tiles in turn; slots
// have 32 rows, which read the cache half as often as 16 (16 sequences of 12 tokens
// after 3000 rows: 40 us, 50 with 16), but 16
//  - up to a mean of 16 (4 tokens after 3000: 12 us, 15 with 32);
//  - where those do not fill the chip and the cache is short (4 sequences of 12
//    tokens after 500: 11 us, 17 with 32; 256-wide heads, 40 tokens after 30: 10 us,
//    16 with 32, but 16 sequences of 6 after 3000: 38, 43 with 16).
// Slots of 128 rows, a quarter to each wave, read the cache still less, but leave a
// chip that they do not fill to one after the other: they are taken from a number
// of such slots and heads on (work_of), and after very long caches. One bf16 prompt,
// own rows and shared: 2816 tokens (704 of them) 122 and 148 us, 2048 (512) 81 and 87,
// 1792 (448) 71 and 71, 1536 (384) 61 and 57, 1280 (320) 52 and 46, 1024 (256) 93
// and 36; 1531 after 517 (384) 84 and 87. Between 256 and 448 the two are within 13%,
// which of them is ahead depends on the rows cached before. Heads of 64: one prompt of
// 4096 (1024) 145 and 162, 2560 (640) 71 and 75, 2048 (512) 55 and 52; prompts of 2048
// of 14/2 heads, 5 (1120) 112 and 110, 4 (896) 97 and 89, 2 (448) 67 and 48: one long
// prompt would go over sooner, several later. Very long caches: 512 tokens after
// 20000 rows 289 and 313, 64 after 30000 74 and 79, but 512 after 8000 148 and 142.
// 256-wide heads have them never (4096 tokens of 16/4: 366 us shared, 508 in slots
// of 64, before a step that made both faster).
//
// Splits of the cache, joined in a second launch:
//  - Short caches (up to 12 tiles of 64 rows) and few 16-row slots have none: eight
//    waves (one sequence of 700 rows: 10.5 us, as with splits, but a launch less).
//  - Slots and heads that fill the chip have none (32 sequences of up to 4000 rows:
//    37.5 us, 44 split), unless the table has room for long sequences: then a split
//    for each 96 tiles, up to 16, so that a long sequence among short ones does not
//    keep one workgroup (one of 131000 rows and 31 of 500: 71 us, 718 without; 32
//    of 32000: 372, 363 without). It costs calls whose sequences are all short,
//    most of all more than 64, whose empty splits are workgroups too (one token each
//    after 500 rows, tables of 8192, 32768 and 131072 rows: 32 sequences 9.5, 12 and
//    16 us, 128 sequences 31, 47 and 124). Not more than a sequence of the mean length
//    needs to fill the chip by itself, and none for one sequence: long prompts have
//    slots enough (16/4 heads of 256 under a table of 131072 rows, one prompt of 4096
//    tokens: 345 us, 1273 in 16 splits; two of 2048, table 32768: 235 us, 670 in 5;
//    8 of 100 after 500 rows: 101 us, 103 in 16, and with one of them after 130000:
//    534 and 609).
//  - Otherwise as many as make the workgroups that the chip holds at once (8
//    sequences of 5000 rows: 22.4 us with 512 workgroups, 25.9 with 1024; one of
//    131000: 60.3, 66.0; 32-row slots of 256-wide heads have a compute unit each:
//    38 us for 16 sequences of 6 tokens with 256, 52 with 384), of at least 8
//    tiles, or 4 where the chip would stay empty.
//  - Never more than 1 GiB of partial results holds (256 sequences of 16 tokens
//    after 300 rows, table 131072: 462 us in 10 splits, 693 in 16 and 1.7 GB).
AttnPlan plan_attention(int64_t tokens, int64_t batch, int q_heads, int kv_heads, int head_dim, int64_t cache_rows) {
    constexpr int64_t kMostNarrow = 16, kMostShared = 64, kFull = 256, kShort = 12, kMedium = 64, kVeryLong = 256;
    constexpr int64_t kMostSplits = 128, kSkew = 96, kMostPartials = int64_t{1} << 30;
    AttnPlan plan;
    const int64_t rows = tokens * (q_heads / kv_heads), mean = (rows + batch - 1) / batch;
    const int64_t tiles = (cache_rows + kTile - 1) / kTile;
    const bool narrow = head_dim < 256;
    // Slots in use, if all sequences have the mean.
    const auto work_of = [&](int64_t of) { return batch * ((mean + of - 1) / of) * kv_heads; };
    plan.shared = !narrow || rows <= kMostShared * batch ||
                  (work_of(kOwnRows) < (head_dim == 64 ? 1024 : 352) && (mean <= kOwnRows || tiles < kVeryLong));
    plan.rows = !plan.shared ? kOwnRows
                : rows <= kMostNarrow * batch || (work_of(16) < kFull && tiles <= (narrow ? kMedium : kShort)) ? 16 : 32;
    plan.slots = static_cast<int>(rows / plan.rows + batch);
    const int64_t units = static_cast<int64_t>(plan.slots) * kv_heads;
    const int64_t work = work_of(plan.rows);
    const bool full = units >= kFull;
    plan.least = plan.shared && units * ((tiles + 7) / 8) < 512 ? 4 : 8;
    plan.waves = 4;
    int64_t target = !narrow && plan.rows == 32 ? 256 : 512;  // workgroups that the chip holds at once
    if (plan.shared) {
        if (narrow && plan.rows == 16 && !full && tiles <= kShort) plan.waves = 8;
        if (plan.waves == 8 || (full && narrow)) target = 0;
    }
    int64_t splits = target / work;
    // Workgroups of one sequence: from kFull on it fills the chip by itself.
    const int64_t alone = (mean + plan.rows - 1) / plan.rows * kv_heads;
    if (full && plan.shared && batch > 1 && alone < kFull) {
        const int64_t skew = std::min({tiles / kSkew, int64_t{16}, 512 / alone});
        splits = std::max(splits, skew);
    }
    const int64_t each = units * plan.rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
    splits = std::min({splits, (tiles + plan.least - 1) / plan.least, kMostSplits, kMostPartials / each});
    plan.splits = static_cast<int>(std::max(splits, int64_t{1}));
    return plan;
}

}  // namespace paged
}  // namespace nq

namespace {

using namespace nq::paged;

// One workgroup per token and q head: its waves take the splits in turn, eight
// loads in flight, and meet in LDS:
//   out = sum_i w_i o_i / sum_i w_i l_i, w_i = 2^(m_i - max m)
// Bound by the wait for a launch and two rounds of loads: 3.5 to 5 us.
template <int D>
__global__ __launch_bounds__(256) void k_paged_merge(const AttnArgs a, int rows) {
    constexpr int E = D / kWave, kWaves = 4, kMost = 2;  // kMost: 64 splits each
    __shared__ float join[kWaves][D], weights[kMost * kWave];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int token = blockIdx.x / a.q_heads, head = blockIdx.x - token * a.q_heads;
    const int g = head / a.group;
    const Work work = find<true>(p, token, head - g * a.group, a.group, rows, a.splits, a.least);
    const Found& f = work.f;
    if (token < f.span.begin || token >= f.span.end) return;
    const SplitPlan plan = work.plan;
    if (plan.active <= 1) return;  // the attention wrote the output itself
    const int64_t item = work.first + work.local;
    if (item < 0 || item + plan.active > static_cast<int64_t>(a.slots) * a.splits) return;  // query_starts out of order
    const uint32_t r = static_cast<uint32_t>(token - f.span.begin) * a.group + head - g * a.group;
    const int64_t first = (item * p.kv_heads + g) * rows + r % static_cast<uint32_t>(rows);
    const int64_t next = static_cast<int64_t>(p.kv_heads) * rows;  // from one split's row to the next split's
    float w[kMost], l[kMost], m = -INFINITY;
#pragma unroll
    for (int c = 0; c < kMost; ++c) {
        const int i = lane + kWave * c;
        const bool on = i < plan.active;
        w[c] = on ? a.partial[2 * (first + i * next)] : -INFINITY;
        l[c] = on ? a.partial[2 * (first + i * next) + 1] : 0.0f;
        m = fmaxf(m, w[c]);
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) m = fmaxf(m, __shfl_xor(m, k, kWave));
    const float m_use = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, o[E];
#pragma unroll
    for (int c = 0; c < kMost; ++c) {
        w[c] = exp2_hw(w[c] - m_use);
        if (wave == 0) weights[lane + kWave * c] = w[c];
        sum += w[c] * l[c];
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) sum += __shfl_xor(sum, k, kWave);
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = 0.0f;
    __syncthreads();
#pragma unroll 8
    for (int i = wave; i < plan.active; i += kWaves) {
        const float weight = weights[i];
        const float* at = a.partial_o + (first + i * next) * D + lane;
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] += weight * at[kWave * j];
    }
#pragma unroll
    for (int j = 0; j < E; ++j) join[wave][lane + kWave * j] = o[j];
    __syncthreads();
    const bool off = row_of(f.context, token - f.span.begin, p.table_pages << p.page_shift) < 0;
    for (int d = threadIdx.x; d < D; d += kWaves * kWave) {
        const float all = (join[0][d] + join[1][d]) + (join[2][d] + join[3][d]);
        nq::store_f32_as(a.out, a.out_dtype, static_cast<int64_t>(blockIdx.x) * D + d, off ? 0.0f : all / sum);
    }
}

int64_t partial_rows(const AttnPlan& plan, int kv_heads) {
    return plan.splits <= 1 ? 0 : static_cast<int64_t>(plan.slots) * plan.splits * kv_heads * plan.rows;
}

}  // namespace

extern "C" int64_t nq_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int32_t q_heads, int32_t kv_heads,
                                                      int32_t head_dim, int32_t page_size, int64_t table_pages) {
    if (tokens <= 0 || tokens > 0xffffff || batch <= 0 || batch > 0xffffff || kv_heads <= 0 || q_heads <= 0 ||
        q_heads > 65535 || q_heads % kv_heads || page_size <= 0 || page_size > 128 || table_pages <= 0 ||
        table_pages > 0x3fffffff / page_size || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return -1;
    if (tokens * q_heads > 0x3fffffff) return -1;
    const AttnPlan plan = plan_attention(tokens, batch, q_heads, kv_heads, head_dim, table_pages * page_size);
    // (The merge has a workgroup for each partial row of a split at most: 1 GiB holds 2^22.)
    if (!nq::launchable(static_cast<int64_t>(plan.slots) * plan.splits * kv_heads, plan.waves * kWave)) return -1;
    return partial_rows(plan, kv_heads) * (2 + head_dim) * static_cast<int64_t>(sizeof(float));
}

extern "C" int nq_paged_attention(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads,
                                  const nq_paged_kv* kv, float scaling, void* out, int32_t out_dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    if (!q || !out) return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(q_dtype) || !nq::is_float_dtype(out_dtype)) return NQ_ERR_DTYPE;
    AttnArgs a{};
    if (const int st = check_pages(kv, tokens, a.p); st != NQ_OK) return st;
    const int64_t need = nq_paged_attention_workspace_bytes(tokens, kv->batch, q_heads, kv->kv_heads, kv->head_dim,
                                                            kv->page_size, kv->table_pages);
    if (need < 0) return NQ_ERR_SHAPE;
    if (!(scaling > 0.0f) || !(scaling < INFINITY)) return NQ_ERR_ARGUMENT;
    if (need > 0 && !workspace) return NQ_ERR_ARGUMENT;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return NQ_ERR_ALIGNMENT;
    const AttnPlan plan = plan_attention(tokens, kv->batch, q_heads, kv->kv_heads, kv->head_dim, kv->table_pages * kv->page_size);
    a.q = q;
    a.out = out;
    a.partial_o = static_cast<float*>(workspace);
    a.partial = a.partial_o ? a.partial_o + partial_rows(plan, kv->kv_heads) * kv->head_dim : nullptr;
    a.scale = scaling * 1.4426950408889634f;
    a.out_dtype = out_dtype;
    a.q_heads = q_heads;
    a.group = q_heads / kv->kv_heads;
    a.slots = plan.slots;
    a.splits = plan.splits;
    a.least = plan.least;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int status;
    switch (kv->head_dim) {
        case 64: status = launch_paged_attention<64>(a, plan, q_dtype, st); break;
        case 128: status = launch_paged_attention<128>(a, plan, q_dtype, st); break;
        default: status = launch_paged_attention<256>(a, plan, q_dtype, st); break;
    }
    if (status != NQ_OK || plan.splits <= 1) return status;
    const dim3 grid(static_cast<unsigned>(tokens * q_heads));
    switch (kv->head_dim) {
        case 64: hipLaunchKernelGGL(k_paged_merge<64>, grid, dim3(256), 0, st, a, plan.rows); break;
        case 128: hipLaunchKernelGGL(k_paged_merge<128>, grid, dim3(256), 0, st, a, plan.rows); break;
        default: hipLaunchKernelGGL(k_paged_merge<256>, grid, dim3(256), 0, st, a, plan.rows); break;
    }
    return nq::launch_status();
}
