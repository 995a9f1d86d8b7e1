// Attention over the 8-bit paged cache: plan, merge of the splits, entry points.
#include "nq_paged_attention.h"

namespace nq {
namespace paged {

template <> int launch_paged_attention<64>(const AttnArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_paged_attention<128>(const AttnArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_paged_attention<256>(const AttnArgs&, const AttnPlan&, int, hipStream_t);

}  // namespace paged
}  // namespace nq

namespace {

using namespace nq::paged;

// One workgroup per token and q head: its waves take the splits in turn, eight
// loads in flight, and meet in LDS.
template <int D>
__global__ __launch_bounds__(256) void k_paged_merge(const AttnArgs a, int rows) {
    constexpr int E = D / kWave, kWaves = 4, kMost = 2;  // kMost: 64 splits each
    __shared__ float join[kWaves][D], weights[kMost * kWave];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int token = blockIdx.x / a.q_heads, head = blockIdx.x - token * a.q_heads;
    const Found f = sequence_at(p, token, [](int, int begin) { return static_cast<int64_t>(begin); });
    if (token < f.span.begin || token >= f.span.end) return;
    const int g = head / a.group;
    const int64_t r = static_cast<int64_t>(token - f.span.begin) * a.group + head - g * a.group;
    const int64_t slot = first_slot_of(f.b, f.span.begin, a.group, rows) + r / rows;
    const SlotSpan s = slot_span(p, f, slot, a.group, rows);
    const SplitPlan plan = split_plan(s.visible, a.splits, a.least);
    if (plan.active <= 1) return;  // the attention wrote the output itself
    const int64_t first = (slot * a.splits * p.kv_heads + g) * rows + r % rows;
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
    const bool off = row_of(s.context, token - s.begin, p.table_pages << p.page_shift) < 0;
    for (int d = threadIdx.x; d < D; d += kWaves * kWave) {
        const float all = (join[0][d] + join[1][d]) + (join[2][d] + join[3][d]);
        nq::store_f32_as(a.out, a.out_dtype, static_cast<int64_t>(blockIdx.x) * D + d, off ? 0.0f : all / sum);
    }
}

// How a call is laid out. All rules go by sizes that the host knows: the page
// table's width stands for the cache's length, the mean for the query rows of a
// sequence (its tokens times the q heads of a kv head). Times: 32/8 heads of 128.
//
// Up to 64 query rows: a slot's waves share its rows and take the cache's tiles in
// turn. Slots of 16 rows up to a mean of 16 (4 tokens after 3000 rows: 12 us, 18 in
// a slot of 32), otherwise of 32, which read the cache half as often (16 sequences
// of 12 tokens: 56 us, 100 with rows of their own; 16 sequences of 6 tokens of 16/4
// heads of 256: 52 us, 76 in slots of 16).
//  - Short caches (up to 12 tiles of 64 rows) of 16-row slots are not split: eight
//    waves, one launch (700 rows of one sequence: 10.5 us against 7.7 + 3 with a
//    merge; 17 tiles: 13.9 against 11.3).
//  - Slots and heads that fill the chip by themselves are not split either, and
//    16-row ones take eight waves from 32 tiles on (32 sequences of up to 4000
//    rows: 39.2 us, four waves and three splits 45.7; 64 sequences of 1000 rows:
//    33.9 against 29.7 of four waves), unless the table has room for long
//    sequences: then a split for each 96 tiles, up to 16, so that a long sequence
//    among short ones does not keep one workgroup (one of 131000 rows and 31 of
//    500: 86 us, 718 without; 32 of 32000: 356 to 375, 370 without).
//  - Otherwise the cache is split until there are about 1024 workgroups, for one
//    sequence 512 (131000 rows: 60.5 us against 73.8 with 1024), of at least 8
//    tiles, or 4 where the chip would stay empty.
// 256-wide heads take four waves: their registers leave one to a SIMD.
// More rows: slots of 128 rows (64 of 256-wide heads), a quarter to each wave. Every
// split's share of every row goes through memory, so the cache is split (to 512
// workgroups) only into as many parts as it has rows for each query row (256
// tokens after 8000 rows: 97 us, 150 with two splits; 2048 tokens of two sequences,
// 14/2 heads of 64, not split: 69 us, 165 with two).
AttnPlan plan_attention(int64_t tokens, int64_t batch, int q_heads, int kv_heads, int head_dim, int64_t cache_rows) {
    constexpr int64_t kMostNarrow = 16, kMostShared = 64, kFull = 256, kShort = 12, kLong = 32, kMostSplits = 128, kSkew = 96;
    AttnPlan plan;
    const int64_t rows = tokens * (q_heads / kv_heads);
    plan.shared = rows <= kMostShared * batch;
    plan.rows = !plan.shared ? own_rows(head_dim) : rows <= kMostNarrow * batch ? 16 : 32;
    plan.slots = static_cast<int>(rows / plan.rows + batch);
    const int64_t tiles = (cache_rows + kTile - 1) / kTile, units = static_cast<int64_t>(plan.slots) * kv_heads;
    const bool full = units >= kFull, narrow = head_dim < 256;
    plan.least = plan.shared && units * ((tiles + 7) / 8) < 512 ? 4 : 8;
    plan.waves = 4;
    int64_t target = 0;
    if (plan.shared) {
        target = batch > 1 ? 1024 : 512;
        if (narrow && plan.rows == 16 && ((full && tiles >= kLong) || (!full && tiles <= kShort))) plan.waves = 8;
        if (plan.waves == 8 || (full && narrow)) target = 0;
    } else {
        const int64_t worth = batch * cache_rows / rows;
        target = worth < 2 ? 0 : 512;
        if (target / units > worth) target = worth * units;
    }
    int64_t splits = target / units;
    if (full && plan.shared && tiles / kSkew > splits) splits = tiles / kSkew < 16 ? tiles / kSkew : 16;
    const int64_t most = (tiles + plan.least - 1) / plan.least;
    splits = splits < most ? splits : most;
    plan.splits = static_cast<int>(splits < 1 ? 1 : (splits > kMostSplits ? kMostSplits : splits));
    return plan;
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
