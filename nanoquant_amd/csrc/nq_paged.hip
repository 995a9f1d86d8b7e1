// q/k norm, RoPE and the append of a ragged batch's new keys and values to an
// 8-bit paged cache.
//
// A page holds `page` consecutive rows of one sequence, for each kv head K as
// [page][head_dim] and V transposed as [head_dim][page], e4m3 bytes that stand
// for byte * scale with one power-of-two scale per page, head and K or V. The
// scale is the least power of two, from 2^-126 on, that brings every row of the
// page within e4m3's 448 (0.875 * 2^9), so it only grows while a page fills. A
// power of two costs e4m3 no precision (its significand has 4 bits at every
// exponent), makes x / scale exact, and moves older rows of the page to a grown
// scale without a second rounding, but for values that leave e4m3's normal
// range (below 2^-6 of the scale).
#include "nq_paged.h"

namespace nq {
namespace paged {

// Cache rows of a sequence at most: row numbers a few tiles further fit 32 bits.
constexpr int64_t kMostRows = 0x3fffffff;

int check_pages(const nq_paged_kv* kv, int64_t tokens, Pages& out) {
    if (!kv || !kv->k_pages || !kv->v_pages || !kv->k_scales || !kv->v_scales || !kv->page_table ||
        !kv->query_starts || !kv->context_lens)
        return NQ_ERR_ARGUMENT;
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return NQ_ERR_SHAPE;
    int shift = 4;
    while (shift < 7 && (1 << shift) != kv->page_size) ++shift;
    if ((1 << shift) != kv->page_size) return NQ_ERR_SHAPE;
    if (kv->num_pages <= 0 || kv->num_pages > 0x7fffffff || kv->kv_heads <= 0 || kv->kv_heads > 65535 ||
        kv->batch <= 0 || kv->batch > 0xffffff || kv->table_pages <= 0 || kv->table_pages > (kMostRows >> shift) ||
        tokens <= 0 || tokens > 0xffffff)
        return NQ_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(kv->k_pages) | reinterpret_cast<uintptr_t>(kv->v_pages)) & 15)
        return NQ_ERR_ALIGNMENT;
    out = {static_cast<uint8_t*>(kv->k_pages), static_cast<uint8_t*>(kv->v_pages), kv->k_scales, kv->v_scales,
           kv->page_table, kv->query_starts, kv->context_lens, kv->num_pages, kv->kv_heads, shift,
           static_cast<int32_t>(kv->table_pages), static_cast<int32_t>(kv->batch), static_cast<int32_t>(tokens)};
    return NQ_OK;
}

}  // namespace paged
}  // namespace nq

namespace {

using namespace nq::paged;

struct AppendArgs {
    Pages p;
    const void *q, *k, *v, *q_norm, *k_norm;
    const float *cos_table, *sin_table;
    const int32_t* rope_starts;  // [batch] position of each sequence's first token; null: its cache row
    void* q_out;
    float eps;
    int32_t norm_dtype, q_dtype, q_heads, q_groups, rope_rows, kv_blocks;
};

constexpr int kPageTokens = 8;  // new rows of a page that a wave holds in registers
constexpr int kQHeads = 8;      // q heads of a token that a wave takes
constexpr int E = 4;            // adjacent values of a head vector that a lane holds

// A head vector takes D / 4 lanes: a wave works on this many at once.
template <int D>
constexpr int kHeads = kWave * E / D;

// Lane values permuted within rows of 16 (DPP).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
}

// The value of lane l ^ 8, l ^ 16 or l ^ 32: half a head vector away.
template <int D>
__device__ __forceinline__ uint32_t partner_of(uint32_t v) {
    if constexpr (D == 64) return dpp<0x128>(v);  // row_ror:8
    if constexpr (D == 128) {
        const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // both rows' lower and upper values
        return (threadIdx.x & 16) ? rows[0] : rows[1];
    }
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? halves[0] : halves[1];
}

template <int D>
__device__ __forceinline__ float partner_of(float v) { return __uint_as_float(partner_of<D>(__float_as_uint(v))); }

template <int D>
__device__ __forceinline__ double partner_of(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2(partner_of<D>(w.x), partner_of<D>(w.y)));
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __uint_as_float(dpp<CTRL>(__float_as_uint(v))); }

template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2(dpp<CTRL>(w.x), dpp<CTRL>(w.y)));
}

// Sum over a head vector's lanes, in a fixed order.
template <int D, class T>
__device__ __forceinline__ T head_sum(T v) {
    v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp<0x141>(v);  // row_half_mirror
    v += dpp<0x140>(v);  // row_mirror
    if constexpr (D >= 128) v += partner_of<128>(v);
    if constexpr (D >= 256) v += partner_of<256>(v);
    return v;
}

// Maximum of values >= 0 over the wave.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    v = fmaxf(v, dpp<0x140>(v));
    v = fmaxf(v, partner_of<128>(v));
    return fmaxf(v, partner_of<256>(v));
}

// The hardware's estimate (1 ulp) does for q.
__device__ __forceinline__ float inverse_root(float x) { return __builtin_amdgcn_rsqf(x); }

// The hardware's estimate is good to 2^-24; each step y (3 - x y^2) / 2 squares
// the error. 0 and infinity (of an infinite or a zero mean) are kept.
__device__ __forceinline__ double inverse_root(double x) {
    const double y0 = __builtin_amdgcn_rsq(x);
    double y = y0;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = y * fma(-0.5 * x * y, y, 1.5);
    return y0 > 0.0 && y0 < INFINITY ? y : y0;
}

// x as fp32 for an e4m3 rounding: the nearest fp32 value does, unless it lies
// where e4m3 rounds to even or where a scale ends. All of those have 0 in their
// last 19 bits, but for subnormal ones (at the smallest scales).
__device__ __forceinline__ float for_e4m3(double x) {
    float f = static_cast<float>(x);
    const uint32_t u = __float_as_uint(f);
    if (__ballot(f != 0.0f && ((u & 0x7ffffu) == 0 || (u & 0x7f800000u) == 0))) f = round_to_odd(x);
    return f;
}

// E adjacent values, at any address that fits the value's type.
template <int DT>
__device__ __forceinline__ void load_values(const void* p, int64_t i, float (&v)[E]) {
    if constexpr (DT == NQ_DTYPE_F32) {
        typedef float vec __attribute__((ext_vector_type(E), aligned(4)));
        const vec x = *reinterpret_cast<const vec*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = x[j];
    } else {
        typedef uint16_t vec __attribute__((ext_vector_type(E), aligned(2)));
        const vec x = *reinterpret_cast<const vec*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if constexpr (DT == NQ_DTYPE_BF16) v[j] = __uint_as_float(static_cast<uint32_t>(x[j]) << 16);
            else v[j] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x[j])));
        }
    }
}

__device__ __forceinline__ void store_values(void* p, int dtype, int64_t i, const float (&v)[E]) {
    if (dtype == NQ_DTYPE_F32) {
        typedef float vec __attribute__((ext_vector_type(E), aligned(4)));
        vec x;
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = v[j];
        *reinterpret_cast<vec*>(static_cast<float*>(p) + i) = x;
        return;
    }
    typedef uint16_t vec __attribute__((ext_vector_type(E), aligned(2)));
    vec x;
#pragma unroll
    for (int j = 0; j < E; ++j)
        x[j] = dtype == NQ_DTYPE_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(v[j]))
                                      : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[j]));
    *reinterpret_cast<vec*>(static_cast<uint16_t*>(p) + i) = x;
}

// Head vectors, lane l of one holding the values from d = 4 l on: RMSNorm with
// weight w (has_w), then rotate-half RoPE, in place; sn is negative in the first
// half. In T = double the result is correct to far below an e4m3 rounding's
// border.
template <int D, class T>
__device__ __forceinline__ void norm_rope(T (&v)[E], const float (&w)[E], bool has_w, float eps, const float (&cs)[E],
                                          const float (&sn)[E]) {
    if (has_w) {
        T ss = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) ss += v[j] * v[j];
        const T inv = inverse_root(head_sum<D>(ss) * static_cast<T>(1.0 / D) + static_cast<T>(eps));
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = static_cast<T>(w[j]) * (v[j] * inv);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = v[j] * static_cast<T>(cs[j]) + partner_of<D>(v[j]) * static_cast<T>(sn[j]);
}

template <int D>
__device__ __forceinline__ void load_rope_row(const AppendArgs& a, int row, int place, float (&cs)[E], float (&sn)[E]) {
    const int64_t i = static_cast<int64_t>(row) * (D / 2) + (place & (D / 2 - 1));
    load_values<NQ_DTYPE_F32>(a.cos_table, i, cs);
    load_values<NQ_DTYPE_F32>(a.sin_table, i, sn);
    if (place < D / 2)
#pragma unroll
        for (int j = 0; j < E; ++j) sn[j] = -sn[j];
}

__device__ __forceinline__ void load_weight(const void* w, int dtype, int place, float (&out)[E]) {
    if (!w) return;
    if (dtype == NQ_DTYPE_F32) load_values<NQ_DTYPE_F32>(w, place, out);
    else if (dtype == NQ_DTYPE_F16) load_values<NQ_DTYPE_F16>(w, place, out);
    else load_values<NQ_DTYPE_BF16>(w, place, out);
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }

// e4m3 bytes of x inv (at most 448), NaN for what is not finite.
__device__ __forceinline__ uint32_t e4m3x4(const float (&x)[E], float inv) {
    float y[E];
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = fabsf(x[j]) < INFINITY ? x[j] * inv : __builtin_nanf("");
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
    return static_cast<uint32_t>(r);
}

__device__ __forceinline__ uint32_t moved4(uint32_t w, float ratio) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(w, 0) * ratio,
                                        __builtin_amdgcn_cvt_f32_fp8(w, 1) * ratio, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(w, 2) * ratio,
                                        __builtin_amdgcn_cvt_f32_fp8(w, 3) * ratio, r, true);
    return static_cast<uint32_t>(r);
}

// Workgroups [0, kv_blocks): the new rows of one page and kv head, kPageTokens
// to a wave, which holds them in registers until the page's scale is known;
// V's bytes are transposed in LDS. Sequence b has at most (its tokens)
// / page + 2 pages with new rows, and its slots begin at starts[b] / page + 2 b:
// the grid follows from the host's counts alone. The rest: q, one wave per token
// and kQHeads of its heads.
//
// Long prompts are bound by bytes (8192 fp32 tokens of 32/8 heads of 128: 356 MB in
// 74 us, 4.8 TB/s, where a copy reaches 5.04; q with 4 heads a wave took 82, with
// 16 75.5), decode steps by the chain of dependent loads (starts, table, row,
// scale: one token 4.6 us, one of 48 sequences each 5.0).
template <int D, int DT, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void k_paged_append(const AppendArgs a) {
    constexpr int kPage = WAVES * kPageTokens, kThreads = WAVES * kWave, H = kHeads<D>;
    // V's bytes: a line of kPage for each of D, padded by a word against bank conflicts.
    constexpr int kLine = kPage + 4;
    __shared__ float red[2][WAVES];
    __shared__ uint32_t tile[D * kLine / 4];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int rows = p.table_pages << p.page_shift;
    const int sub = lane / (kWave / H), place = (lane & (kWave / H - 1)) * E;  // head vector of the wave, place in it
    float w[E] = {};

    if (static_cast<int>(blockIdx.x) >= a.kv_blocks) {
        const int64_t item = static_cast<int64_t>(blockIdx.x - a.kv_blocks) * WAVES + wave;
        const int token = static_cast<int>(item / a.q_groups);
        const int head = static_cast<int>(item - static_cast<int64_t>(token) * a.q_groups) * kQHeads;
        if (token >= p.tokens) return;
        const Found f = sequence_at(p, token, [](int, int begin) { return static_cast<int64_t>(begin); });
        const Span s = f.span;
        const int row = token >= s.begin && token < s.end ? row_of(f.context, token - s.begin, rows) : -1;
        const int64_t position = a.rope_starts ? static_cast<int64_t>(a.rope_starts[f.b]) + (token - s.begin) : row;
        if (row < 0 || position < 0 || position >= a.rope_rows) return;
        float cs[E], sn[E], x[kQHeads / H][E];
        const int64_t at = (static_cast<int64_t>(token) * a.q_heads + head) * D + place;
        const int last = a.q_heads - 1 - head;
#pragma unroll
        for (int i = 0; i < kQHeads / H; ++i) load_values<DT>(a.q, at + min(i * H + sub, last) * D, x[i]);
        load_weight(a.q_norm, a.norm_dtype, place, w);
        load_rope_row<D>(a, static_cast<int>(position), place, cs, sn);
#pragma unroll
        for (int i = 0; i < kQHeads / H; ++i) {
            norm_rope<D>(x[i], w, a.q_norm != nullptr, a.eps, cs, sn);
            if (i * H + sub <= last) store_values(a.q_out, a.q_dtype, at + (i * H + sub) * D, x[i]);
        }
        return;
    }

    const int slot = blockIdx.x / p.kv_heads, g = blockIdx.x - slot * p.kv_heads;
    const auto first_slot = [&](int i, int begin) {
        return static_cast<int64_t>(begin / kPage) + 2 * static_cast<int64_t>(i);
    };
    const Found f = sequence_at(p, slot, first_slot);
    const Span s = f.span;
    const int b = f.b, context = f.context;
    const int64_t slot0 = first_slot(b, s.begin);
    // New rows of the sequence that have a place and, `turned` further, a row of the RoPE tables: [low, high).
    const int64_t turned = a.rope_starts ? static_cast<int64_t>(a.rope_starts[b]) - context : 0;
    const int64_t low = max(max(static_cast<int64_t>(context), int64_t{0}), -turned);
    const int64_t high = min(static_cast<int64_t>(context) + (s.end - s.begin),
                             min(static_cast<int64_t>(rows), a.rope_rows - turned));
    const int64_t nth = low / kPage + (slot - slot0);
    const int64_t begin = max(low, nth * kPage), end = min(high, (nth + 1) * kPage);
    if (slot < slot0 || begin >= end) return;
    const int32_t id = p.table[static_cast<int64_t>(b) * p.table_pages + nth];
    const int r0 = static_cast<int>(begin) & (kPage - 1), n = static_cast<int>(end - begin);
    const int64_t token0 = s.begin + (begin - context);

    // Row wave H + i WAVES H + sub of the new ones; the last one again behind it,
    // which changes no maximum and is not stored.
    float kf[kPageTokens / H][E], vf[kPageTokens / H][E];
    const auto row_at = [&](int i) { return (wave + i * WAVES) * H + sub; };
    const auto any_at = [&](int i) { return (wave + i * WAVES) * H < n; };  // the same for the wave
    load_weight(a.k_norm, a.norm_dtype, place, w);
    float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int i = 0; i < kPageTokens / H; ++i) {
        if (!any_at(i)) break;
        const int64_t at = ((token0 + min(row_at(i), n - 1)) * p.kv_heads + g) * D + place;
        load_values<DT>(a.k, at, kf[i]);
        load_values<DT>(a.v, at, vf[i]);
    }
#pragma unroll
    for (int i = 0; i < kPageTokens / H; ++i) {
        if (!any_at(i)) break;
        float cs[E], sn[E];
        load_rope_row<D>(a, static_cast<int>(begin + turned) + min(row_at(i), n - 1), place, cs, sn);
        double y[E];
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = static_cast<double>(kf[i][j]);
        norm_rope<D>(y, w, a.k_norm != nullptr, a.eps, cs, sn);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            kf[i][j] = for_e4m3(y[j]);
            kmax = fmaxf(kmax, finite_or_zero(kf[i][j]));
            vmax = fmaxf(vmax, finite_or_zero(vf[i][j]));
        }
    }
    if (id < 0 || id >= p.pages) return;  // the same for all waves
    const int64_t base = static_cast<int64_t>(id) * p.kv_heads + g;
    uint8_t* kp = p.k + base * kPage * D;
    uint8_t* vp = p.v + base * kPage * D;
    kmax = wave_max(kmax);
    vmax = wave_max(vmax);
    if (lane == 0) {
        red[0][wave] = kmax;
        red[1][wave] = vmax;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        kmax = fmaxf(kmax, red[0][i]);
        vmax = fmaxf(vmax, red[1][i]);
    }
    float ks = scale_for(kmax), vs = scale_for(vmax);
    if (r0) {
        // Rows [0, r0) stay; their scale may have to grow, and they with it.
        const float ko = p.k_scales[base], vo = p.v_scales[base];
        ks = fmaxf(ks, ko);
        vs = fmaxf(vs, vo);
        if (ks != ko) {
            const float ratio = ko / ks;
            for (int i = threadIdx.x * 4; i < r0 * D; i += kThreads * 4) {
                uint32_t* at = reinterpret_cast<uint32_t*>(kp + i);
                *at = moved4(*at, ratio);
            }
        }
        if (vs != vo) {
            const float ratio = vo / vs;
            for (int i = threadIdx.x; i < r0 * D; i += kThreads) {
                uint8_t* at = vp + (i / r0) * kPage + i % r0;
                *at = static_cast<uint8_t>(moved4(*at, ratio) & 0xff);
            }
        }
        __syncthreads();  // every wave has read the old scales
    }
    if (threadIdx.x == 0) {
        p.k_scales[base] = ks;
        p.v_scales[base] = vs;
    }
    // Exact for the powers of two that this kernel writes.
    const float ki = 1.0f / ks, vi = 1.0f / vs;
    if (n == 1) {  // one row: nothing to gain from LDS
        if (wave == 0 && sub == 0) {
            *reinterpret_cast<uint32_t*>(kp + r0 * D + place) = e4m3x4(kf[0], ki);
            const uint32_t w4 = e4m3x4(vf[0], vi);
#pragma unroll
            for (int j = 0; j < E; ++j) vp[(place + j) * kPage + r0] = static_cast<uint8_t>(w4 >> (8 * j));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kPageTokens / H; ++i)
        if (any_at(i) && row_at(i) < n)
            *reinterpret_cast<uint32_t*>(kp + (r0 + row_at(i)) * D + place) = e4m3x4(kf[i], ki);
    uint8_t* bytes = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
    for (int i = 0; i < kPageTokens / H; ++i)
        if (any_at(i) && row_at(i) < n) {
            const uint32_t w4 = e4m3x4(vf[i], vi);
#pragma unroll
            for (int j = 0; j < E; ++j) bytes[(place + j) * kLine + r0 + row_at(i)] = static_cast<uint8_t>(w4 >> (8 * j));
        }
    __syncthreads();
    // Whole words of V's lines where they are new, single bytes at the ends.
    constexpr int kWords = kPage / 4;
    for (int i = threadIdx.x; i < D * kWords; i += kThreads) {
        const int line = i / kWords, c = (i - line * kWords) * 4;
        if (c + 4 <= r0 || c >= r0 + n) continue;
        const uint32_t w4 = tile[line * (kLine / 4) + c / 4];
        uint8_t* at = vp + line * kPage + c;
        if (c >= r0 && c + 4 <= r0 + n) {
            *reinterpret_cast<uint32_t*>(at) = w4;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k >= r0 && c + k < r0 + n) at[k] = static_cast<uint8_t>(w4 >> (8 * k));
        }
    }
}

template <int D, int DT>
int launch_append(AppendArgs& a, int64_t tokens, int kv_heads, int64_t batch, hipStream_t stream) {
    const int waves = (1 << a.p.page_shift) / kPageTokens;
    const int64_t kv_blocks = ((tokens >> a.p.page_shift) + 2 * batch) * kv_heads;
    const int64_t blocks = kv_blocks + (tokens * a.q_groups + waves - 1) / waves;
    if (!nq::launchable(blocks, waves * kWave)) return NQ_ERR_SHAPE;
    a.kv_blocks = static_cast<int32_t>(kv_blocks);
    const dim3 grid(static_cast<unsigned>(blocks)), block(static_cast<unsigned>(waves * kWave));
    switch (waves) {
        case 2: hipLaunchKernelGGL((k_paged_append<D, DT, 2>), grid, block, 0, stream, a); break;
        case 4: hipLaunchKernelGGL((k_paged_append<D, DT, 4>), grid, block, 0, stream, a); break;
        case 8: hipLaunchKernelGGL((k_paged_append<D, DT, 8>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((k_paged_append<D, DT, 16>), grid, block, 0, stream, a); break;
    }
    return nq::launch_status();
}

template <int D>
int launch_append(AppendArgs& a, int dtype, int64_t tokens, int kv_heads, int64_t batch, hipStream_t stream) {
    switch (dtype) {
        case NQ_DTYPE_F32: return launch_append<D, NQ_DTYPE_F32>(a, tokens, kv_heads, batch, stream);
        case NQ_DTYPE_F16: return launch_append<D, NQ_DTYPE_F16>(a, tokens, kv_heads, batch, stream);
        default: return launch_append<D, NQ_DTYPE_BF16>(a, tokens, kv_heads, batch, stream);
    }
}

bool float_code(int d) { return nq::is_float_dtype(d); }

}  // namespace

extern "C" int nq_paged_append_at(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens,
                                  int32_t q_heads, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                                  const float* cos_table, const float* sin_table, int64_t rope_positions,
                                  const nq_paged_kv* kv, const int32_t* rope_starts, void* q_out, int32_t q_out_dtype,
                                  void* stream) {
    if (!q || !k || !v || !cos_table || !sin_table || !q_out || (q_norm == nullptr) != (k_norm == nullptr))
        return NQ_ERR_ARGUMENT;
    if (!float_code(dtype) || !float_code(q_out_dtype) || (q_norm && !float_code(norm_dtype))) return NQ_ERR_DTYPE;
    AppendArgs a{};
    if (const int st = check_pages(kv, tokens, a.p); st != NQ_OK) return st;
    if (q_heads <= 0 || q_heads > 65535 || q_heads % kv->kv_heads || rope_positions <= 0) return NQ_ERR_SHAPE;
    if (!(eps >= 0.0f)) return NQ_ERR_ARGUMENT;
    a.q = q; a.k = k; a.v = v; a.q_norm = q_norm; a.k_norm = k_norm;
    a.cos_table = cos_table; a.sin_table = sin_table; a.rope_starts = rope_starts; a.q_out = q_out;
    a.eps = eps; a.norm_dtype = norm_dtype; a.q_dtype = q_out_dtype; a.q_heads = q_heads;
    a.rope_rows = static_cast<int32_t>(rope_positions < 0x7fffffff ? rope_positions : 0x7fffffff);
    a.q_groups = (q_heads + kQHeads - 1) / kQHeads;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (kv->head_dim) {
        case 64: return launch_append<64>(a, dtype, tokens, kv->kv_heads, kv->batch, st);
        case 128: return launch_append<128>(a, dtype, tokens, kv->kv_heads, kv->batch, st);
        default: return launch_append<256>(a, dtype, tokens, kv->kv_heads, kv->batch, st);
    }
}

extern "C" int nq_paged_append(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens,
                               int32_t q_heads, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                               const float* cos_table, const float* sin_table, int64_t rope_positions,
                               const nq_paged_kv* kv, void* q_out, int32_t q_out_dtype, void* stream) {
    return nq_paged_append_at(q, k, v, dtype, tokens, q_heads, q_norm, k_norm, norm_dtype, eps, cos_table, sin_table,
                              rope_positions, kv, nullptr, q_out, q_out_dtype, stream);
}
