// Attention over the 8-bit paged cache for sequences that hold the same first
// rows, with each query row's log-sum-exp: plan, join of the shares, entry points.
//
// Where many sequences have few query rows each, a tile of the shared rows serves
// 16 or 32 query rows of different sequences at once, and the rows' bytes are read
// once for each such slot, not once for each sequence. What a row gets from the
// shared rows and from its own sequence's meets in the join, as splits of a cache do:
//   m = max m_i,  out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,
//   lse = log 2 (m + log2 sum_i 2^(m_i - m) l_i)
#include <algorithm>

#include "nq_paged_attention.h"

namespace nq {
namespace paged {

template <> int launch_shared_attention<64>(const SharedArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_shared_attention<128>(const SharedArgs&, const AttnPlan&, int, hipStream_t);
template <> int launch_shared_attention<256>(const SharedArgs&, const AttnPlan&, int, hipStream_t);

}  // namespace paged
}  // namespace nq

namespace {

using namespace nq::paged;

constexpr int kMostShares = kWave;  // splits of the shared rows, and of a sequence's own, that the join takes

// One workgroup per token and q head: its waves take the shares in turn and meet in
// LDS. Bound by the wait for a launch and two rounds of loads: 2.9 to 4.9 us.
template <int D>
__global__ __launch_bounds__(256) void k_shared_merge(const SharedArgs a, int rows) {
    constexpr int E = D / kWave, kWaves = 4;
    __shared__ float join[kWaves][D], weights[2 * kMostShares];
    __shared__ int64_t at[2 * kMostShares];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int token = blockIdx.x / a.q_heads, head = blockIdx.x - token * a.q_heads;
    const int g = head / a.group;
    const Work work = find<true>(p, token, head - g * a.group, a.group, rows, a.splits, a.least, a.skip);
    const Found& f = work.f;
    if (token < f.span.begin || token >= f.span.end) return;
    const int shared = a.blocks ? a.shared_splits : 0, own = work.plan.active;
    if (shared == 0 && own <= 1) return;  // the attention wrote the output itself
    const int64_t items = static_cast<int64_t>(a.slots) * a.splits, item = work.first + work.local;
    if (item < 0 || item + own > items || own > kMostShares) return;  // query_starts out of order
    const uint32_t r = static_cast<uint32_t>(token - f.span.begin) * a.group + head - g * a.group;
    const uint32_t r_all = static_cast<uint32_t>(token) * a.group + head - g * a.group, nth = r_all / static_cast<uint32_t>(rows);
    const int64_t next = static_cast<int64_t>(p.kv_heads) * rows;  // from one split's row to the next split's
    // The row's share in split `lane` of its own sequence's rows and of the shared rows.
    const int64_t from[2] = {(item * p.kv_heads + g) * rows + r % static_cast<uint32_t>(rows) + lane * next,
                             ((items + static_cast<int64_t>(nth) * shared) * p.kv_heads + g) * rows +
                                 (r_all - nth * rows) + lane * next};
    float w[2], l[2], m = -INFINITY;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const bool on = lane < (c ? shared : own);
        w[c] = on ? a.partial[2 * from[c]] : -INFINITY;
        l[c] = on ? a.partial[2 * from[c] + 1] : 0.0f;
        m = fmaxf(m, w[c]);
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) m = fmaxf(m, __shfl_xor(m, k, kWave));
    const float m_use = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, o[E];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        w[c] = exp2_hw(w[c] - m_use);
        if (wave == 0 && lane < (c ? shared : own)) {
            weights[c * own + lane] = w[c];
            at[c * own + lane] = from[c];
        }
        sum += w[c] * l[c];
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) sum += __shfl_xor(sum, k, kWave);
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = 0.0f;
    __syncthreads();
#pragma unroll 8
    for (int i = wave; i < own + shared; i += kWaves) {
        const float weight = weights[i];
        const float* o_at = a.partial_o + at[i] * D + lane;
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] += weight * o_at[kWave * j];
    }
#pragma unroll
    for (int j = 0; j < E; ++j) join[wave][lane + kWave * j] = o[j];
    __syncthreads();
    const bool off = row_of(f.context, token - f.span.begin, p.table_pages << p.page_shift) < 0;
    if (a.lse && threadIdx.x == 0) a.lse[blockIdx.x] = off ? -INFINITY : log_of_sum(m_use, sum);
    for (int d = threadIdx.x; d < D; d += kWaves * kWave) {
        const float all = (join[0][d] + join[1][d]) + (join[2][d] + join[3][d]);
        nq::store_f32_as(a.out, a.out_dtype, static_cast<int64_t>(blockIdx.x) * D + d, off ? 0.0f : all / sum);
    }
}

// How a call is laid out: the plan of the rows behind the shared ones, and the
// splits of the shared ones (0: every sequence reads them itself).
struct SharedPlan {
    AttnPlan own;
    int skip, splits, per;
};

int64_t share_bytes(const SharedPlan& plan, int64_t rows, int kv_heads, int head_dim) {
    if (plan.splits == 0 && plan.own.splits <= 1) return 0;
    const int64_t slots = (rows + plan.own.rows - 1) / plan.own.rows;
    const int64_t items = static_cast<int64_t>(plan.own.slots) * plan.own.splits + slots * plan.splits;
    return items * kv_heads * plan.own.rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

// The shared rows get as many splits as make 256 workgroups, one for a compute unit (they hold
// 64 KB of LDS), so that the sequences' own rows run beside them: 32 sequences of one token over 16000
// shared rows and up to 700 of their own, 32/8 heads of 128, 34 us; with 128 workgroups 50, 192 38, 384
// 39, 512 39, 1024 48. Slots of 16 rows read the shared rows twice as often: 36 at their best. Above 64
// query rows to a sequence its own rows fill the slots, and nothing is gained by sharing.
// Where the table has room for long histories behind the shared rows, a split for each 96 tiles of them, up to
// 16, of at least 8 tiles, as plan_attention has: one long conversation among short ones does not keep one
// workgroup (4096 shared rows, 32 sequences of one token, one with 100000 rows of its own: 115 us, 879 without, 118
// in nq_paged_attention; 16 sequences, the others 300 rows: 73 us, 117 in splits of at least 4 tiles, 305
// without). It costs batches of more than 64 short sequences under such a table their empty splits (128 of
// them: 126 us, 51 without, 227 in nq_paged_attention); 32 take 27 us either way.
// (32 KB of shared K and V of one head meet 32 query rows at a time: the vector unit widens them and takes
// the exponentials, about as long as the bytes take.)
SharedPlan plan_shared(int64_t tokens, int64_t batch, int q_heads, int kv_heads, int head_dim, int page, int64_t cache_rows,
                       int64_t shared_rows) {
    constexpr int64_t kMostMean = 64, kMostBytes = int64_t{1} << 30, kTarget = 512, kShared = 256, kSkew = 96;
    const int64_t rows = tokens * (q_heads / kv_heads), mean = (rows + batch - 1) / batch;
    const int grain = std::max(page, kTile);
    SharedPlan plan{};
    plan.skip = static_cast<int>(shared_rows / grain * grain);
    const int64_t tiles = plan.skip / kTile, own_tiles = (cache_rows - plan.skip + kTile - 1) / kTile;
    if (tiles > 0 && mean <= kMostMean && batch > 1) {
        plan.own = AttnPlan{};
        plan.own.shared = true;
        plan.own.waves = 4;
        plan.own.rows = rows <= 16 ? 16 : 32;
        plan.own.slots = static_cast<int>(rows / plan.own.rows + batch);
        const int64_t slots = (rows + plan.own.rows - 1) / plan.own.rows;
        const int64_t splits = std::max(int64_t{1}, std::min({kShared / (slots * kv_heads), (tiles + 3) / 4, int64_t{kMostShares}}));
        plan.per = static_cast<int>((tiles + splits - 1) / splits);
        plan.splits = static_cast<int>((tiles + plan.per - 1) / plan.per);
        const int64_t units = static_cast<int64_t>(plan.own.slots) * kv_heads;
        const int64_t alone = (mean + plan.own.rows - 1) / plan.own.rows * kv_heads;
        const int64_t skew = std::min({own_tiles / kSkew, int64_t{16}, kTarget / alone});
        plan.own.least = skew > kTarget / units ? 8 : 4;
        const int64_t each = kv_heads * plan.own.rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
        const int64_t room = (kMostBytes / each - slots * plan.splits) / plan.own.slots;
        plan.own.splits = static_cast<int>(std::max(int64_t{1}, std::min({std::max(kTarget / units, skew), (own_tiles + 3) / 4,
                                                                         int64_t{kMostShares}, room})));
        if (share_bytes(plan, rows, kv_heads, head_dim) <= kMostBytes) return plan;
    }
    // Each sequence's slots are full of its own rows, or there is nothing to share.
    plan.skip = plan.splits = plan.per = 0;
    plan.own = plan_attention(tokens, batch, q_heads, kv_heads, head_dim, cache_rows);
    plan.own.waves = 4;
    plan.own.splits = std::min(plan.own.splits, kMostShares);
    return plan;
}

}  // namespace

extern "C" int64_t nq_shared_attention_workspace_bytes(int64_t tokens, int64_t batch, int32_t q_heads, int32_t kv_heads,
                                                       int32_t head_dim, int32_t page_size, int64_t table_pages,
                                                       int64_t shared_rows) {
    if (nq_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, head_dim, page_size, table_pages) < 0) return -1;
    if (shared_rows < 0 || shared_rows > table_pages * page_size) return -1;
    const SharedPlan plan = plan_shared(tokens, batch, q_heads, kv_heads, head_dim, page_size, table_pages * page_size, shared_rows);
    const int64_t rows = tokens * (q_heads / kv_heads), slots = (rows + plan.own.rows - 1) / plan.own.rows;
    const int64_t items = static_cast<int64_t>(plan.own.slots) * plan.own.splits + slots * plan.splits;
    if (!nq::launchable(items * kv_heads, 4 * kWave)) return -1;
    const int64_t bytes = share_bytes(plan, rows, kv_heads, head_dim);
    if (bytes > 0 && !nq::launchable(tokens * q_heads, 256)) return -1;
    return bytes;
}

extern "C" int nq_shared_attention(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads, const nq_paged_kv* kv,
                                   int64_t shared_rows, float scaling, void* out, int32_t out_dtype, float* lse,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    if (!q || !out) return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(q_dtype) || !nq::is_float_dtype(out_dtype)) return NQ_ERR_DTYPE;
    SharedArgs a{};
    if (const int st = check_pages(kv, tokens, a.p); st != NQ_OK) return st;
    const int64_t need = nq_shared_attention_workspace_bytes(tokens, kv->batch, q_heads, kv->kv_heads, kv->head_dim,
                                                             kv->page_size, kv->table_pages, shared_rows);
    if (need < 0) return NQ_ERR_SHAPE;
    if (!(scaling > 0.0f) || !(scaling < INFINITY)) return NQ_ERR_ARGUMENT;
    if (need > 0 && !workspace) return NQ_ERR_ARGUMENT;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return NQ_ERR_ALIGNMENT;
    const SharedPlan plan = plan_shared(tokens, kv->batch, q_heads, kv->kv_heads, kv->head_dim, kv->page_size,
                                        kv->table_pages * kv->page_size, shared_rows);
    a.group = q_heads / kv->kv_heads;
    const int64_t rows = tokens * a.group, slots = (rows + plan.own.rows - 1) / plan.own.rows;
    const int64_t shares = need / ((kv->head_dim + 2) * static_cast<int64_t>(sizeof(float)));
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.partial_o = static_cast<float*>(workspace);
    a.partial = a.partial_o ? a.partial_o + shares * kv->head_dim : nullptr;
    a.scale = scaling * 1.4426950408889634f;
    a.out_dtype = out_dtype;
    a.q_heads = q_heads;
    a.slots = plan.own.slots;
    a.splits = plan.own.splits;
    a.least = plan.own.least;
    a.skip = plan.skip;
    a.shared_splits = plan.splits;
    a.shared_per = plan.per;
    a.blocks = static_cast<int32_t>(slots * plan.splits * kv->kv_heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int status;
    switch (kv->head_dim) {
        case 64: status = launch_shared_attention<64>(a, plan.own, q_dtype, st); break;
        case 128: status = launch_shared_attention<128>(a, plan.own, q_dtype, st); break;
        default: status = launch_shared_attention<256>(a, plan.own, q_dtype, st); break;
    }
    if (status != NQ_OK || need == 0) return status;
    const dim3 grid(static_cast<unsigned>(tokens * q_heads));
    switch (kv->head_dim) {
        case 64: hipLaunchKernelGGL(k_shared_merge<64>, grid, dim3(256), 0, st, a, plan.own.rows); break;
        case 128: hipLaunchKernelGGL(k_shared_merge<128>, grid, dim3(256), 0, st, a, plan.own.rows); break;
        default: hipLaunchKernelGGL(k_shared_merge<256>, grid, dim3(256), 0, st, a, plan.own.rows); break;
    }
    return nq::launch_status();
}
