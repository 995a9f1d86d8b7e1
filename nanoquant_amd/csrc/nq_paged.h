// The 8-bit paged KV cache: what its append and its attention share.
#pragma once

#include <math.h>

#include <type_traits>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace nq {
namespace paged {

constexpr int kWave = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A checked nq_paged_kv as the kernels take it: rows of the cache and token
// counts fit 32 bits, page offsets are formed in 64.
struct Pages {
    uint8_t* k;               // [pages][kv_heads][page][head_dim]
    uint8_t* v;               // [pages][kv_heads][head_dim][page]
    float* k_scales;          // [pages][kv_heads]
    float* v_scales;
    const int32_t* table;     // [batch][table_pages]
    const int32_t* starts;    // [batch + 1]
    const int32_t* contexts;  // [batch]
    int64_t pages;
    int32_t kv_heads, page_shift, table_pages, batch, tokens;
};

int check_pages(const nq_paged_kv* kv, int64_t tokens, Pages& out);

// Tokens [begin, end) of sequence b, forced into [0, tokens] and into order:
// whatever the caller's array holds, no token outside the buffers is named.
struct Span {
    int begin, end;
};

// A sequence with its span and the rows it had cached before the call.
struct Found {
    int b, context;
    Span span;
};

// The last sequence b with first(b, its first token) <= slot, for a `first` that
// does not decrease (sequence 0 when there is none). All lanes of a wave search
// together, 64 ways a round; in the last round they load the sequences' ends
// and contexts too, so up to 64 sequences take one round trip. With starts that
// are not in order some sequence comes out; its span decides whether the slot
// names anything.
template <class First>
__device__ __forceinline__ Found sequence_at(const Pages& p, int64_t slot, const First& first) {
    const int lane = threadIdx.x & (kWave - 1);
    int low = 0, count = p.batch;
    while (count > kWave) {
        const int step = (count + kWave - 1) / kWave;
        const int at = lane * step, b = low + (at < count ? at : 0);
        const uint64_t below = __ballot(at < count && first(b, min(max(p.starts[b], 0), p.tokens)) <= slot);
        const int hit = below ? 63 - __builtin_clzll(below) : 0;
        low += hit * step;
        count = min(step, count - hit * step);
    }
    const int b = low + (lane < count ? lane : 0);
    const int start = p.starts[b], stop = p.starts[b + 1], context = p.contexts[b];
    const int begin = min(max(start, 0), p.tokens), end = min(max(stop, begin), p.tokens);
    const uint64_t below = __ballot(lane < count && first(b, begin) <= slot);
    const int hit = below ? 63 - __builtin_clzll(below) : 0;
    return {__builtin_amdgcn_readfirstlane(low + hit), __builtin_amdgcn_readlane(context, hit),
            {__builtin_amdgcn_readlane(begin, hit), __builtin_amdgcn_readlane(end, hit)}};
}

// Sum of a lane's value and those of the lanes before it (DPP).
__device__ __forceinline__ uint32_t running_sum(uint32_t v) {
    const auto add = [&](auto ctrl, auto rows) {
        v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value,
                                                               decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr:1
    add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15 to rows 1 and 3
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31 to rows 2 and 3
    return v;
}

// A token's cache row: its sequence's context plus its place, or -1 outside
// the rows [0, rows) that the page table holds.
__device__ __forceinline__ int row_of(int context, int place, int rows) {
    const int64_t row = static_cast<int64_t>(context) + place;
    return row >= 0 && row < rows ? static_cast<int>(row) : -1;
}

}  // namespace paged
}  // namespace nq
