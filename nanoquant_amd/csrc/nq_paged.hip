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

int check_pages(const nq_paged_kv* kv, int64_t tokens, Pages& out) {
    if (!kv || !kv->k_pages || !kv->v_pages || !kv->k_scales || !kv->v_scales || !kv->page_table ||
        !kv->query_starts || !kv->context_lens)
        return NQ_ERR_ARGUMENT;
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return NQ_ERR_SHAPE;
    int shift = 4;
    while (shift < 7 && (1 << shift) != kv->page_size) ++shift;
    if ((1 << shift) != kv->page_size) return NQ_ERR_SHAPE;
    if (kv->num_pages <= 0 || kv->num_pages > 0x7fffffff || kv->kv_heads <= 0 || kv->kv_heads > 65535 ||
        kv->batch <= 0 || kv->batch > 0xffffff || kv->table_pages <= 0 || kv->table_pages > (0x7fffff00 >> shift) ||
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
    void* q_out;
    float eps;
    int32_t dtype, norm_dtype, q_dtype, q_heads, q_groups, rope_rows, kv_blocks;
};

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__shfl_xor(w.x, mask, kWave), __shfl_xor(w.y, mask, kWave)));
}

// Sum over the wave, in a fixed order.
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v += shfl_xor_f64(v, m);
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v = fmaxf(v, __shfl_xor(v, m, kWave));
    return v;
}

// fp64 -> fp32 towards zero with the last bit set where that drops something:
// a later rounding to fewer bits (e4m3 keeps 4) then rounds the fp64 value.
__device__ __forceinline__ float round_to_odd(double x) {
    float f = static_cast<float>(x);
    if (!(fabsf(f) < INFINITY)) return f;  // beyond fp32, or not finite
    if (static_cast<double>(f) != x) {
        uint32_t u = __float_as_uint(f);
        if (fabs(static_cast<double>(f)) > fabs(x)) u -= 1;
        f = __uint_as_float(u | 1u);
    }
    return f;
}

// One wave's head vector, lane l holding d = l + 64 j: RMSNorm with weight nw
// when it is not NULL, then rotate-half RoPE. In T = double the result is
// correct to far below an e4m3 rounding's border.
template <int D, class T>
__device__ __forceinline__ void norm_rope(const void* x, int dtype, int64_t at, const float (&w)[D / kWave], bool has_w,
                                          float eps, const float (&cs)[D / kWave], const float (&sn)[D / kWave],
                                          int lane, T (&y)[D / kWave]) {
    constexpr int E = D / kWave;
    T v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = static_cast<T>(nq::load_f32(x, dtype, at + lane + kWave * j));
    if (has_w) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < E; ++j) ss += static_cast<double>(v[j]) * static_cast<double>(v[j]);
        const double mean = wave_sum_f64(ss) / D + static_cast<double>(eps);
        const T inv = static_cast<T>(1.0 / sqrt(mean));
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = static_cast<T>(w[j]) * (v[j] * inv);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const bool first = lane + kWave * j < D / 2;
        T partner;
        if constexpr (E == 1) {
            if constexpr (sizeof(T) == 8) partner = shfl_xor_f64(v[0], 32);
            else partner = __shfl_xor(v[0], 32, kWave);
        } else {
            partner = first ? v[j + E / 2] : v[j - E / 2];
        }
        if (first) partner = -partner;
        y[j] = v[j] * static_cast<T>(cs[j]) + partner * static_cast<T>(sn[j]);
    }
}

template <int D>
__device__ __forceinline__ void load_rope_row(const AppendArgs& a, int row, int lane, float (&cs)[D / kWave],
                                              float (&sn)[D / kWave]) {
#pragma unroll
    for (int j = 0; j < D / kWave; ++j) {
        const int64_t i = static_cast<int64_t>(row) * (D / 2) + ((lane + kWave * j) & (D / 2 - 1));
        cs[j] = a.cos_table[i];
        sn[j] = a.sin_table[i];
    }
}

template <int D>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int lane, float (&out)[D / kWave]) {
#pragma unroll
    for (int j = 0; j < D / kWave; ++j) out[j] = w ? nq::load_f32(w, dtype, lane + kWave * j) : 1.0f;
}

// The least power of two 2^e, e >= -126, with amax <= 448 * 2^e = 1.75 * 2^(8 + e).
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, -126) + 127) << 23);
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }

// e4m3 byte of x (|x| <= 448), NaN for what is not finite.
__device__ __forceinline__ uint8_t e4m3(float x) {
    const float y = fabsf(x) < INFINITY ? x : __builtin_nanf("");
    return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xff);
}

__device__ __forceinline__ uint32_t moved4(uint32_t w, float ratio) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(w, 0) * ratio,
                                        __builtin_amdgcn_cvt_f32_fp8(w, 1) * ratio, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_cvt_f32_fp8(w, 2) * ratio,
                                        __builtin_amdgcn_cvt_f32_fp8(w, 3) * ratio, r, true);
    return static_cast<uint32_t>(r);
}

// Workgroups [0, kv_blocks): the new rows of one page and kv head. Sequence b
// has at most (its tokens) / page + 2 pages with new rows, and its slots begin
// at starts[b] / page + 2 b: the grid follows from the host's counts alone.
// The rest: q, one wave per token and two of its heads.
template <int D, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void k_paged_append(const AppendArgs a) {
    constexpr int E = D / kWave;
    __shared__ float red[2][WAVES];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int rows = p.table_pages << p.page_shift;
    float w[E], cs[E], sn[E];

    if (static_cast<int>(blockIdx.x) >= a.kv_blocks) {
        const int item = blockIdx.x - a.kv_blocks, token = item / a.q_groups;
        const int head = ((item - token * a.q_groups) * WAVES + wave) * 2;
        if (head >= a.q_heads) return;
        const Found f = sequence_at(p, token, [](int, int begin) { return static_cast<int64_t>(begin); });
        const Span s = f.span;
        const int row = token >= s.begin && token < s.end ? row_of(f.context, token - s.begin, rows) : -1;
        if (row < 0 || row >= a.rope_rows) return;
        load_weight<D>(a.q_norm, a.norm_dtype, lane, w);
        load_rope_row<D>(a, row, lane, cs, sn);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (head + i >= a.q_heads) break;
            const int64_t at = (static_cast<int64_t>(token) * a.q_heads + head + i) * D;
            float y[E];
            norm_rope<D, float>(a.q, a.dtype, at, w, a.q_norm != nullptr, a.eps, cs, sn, lane, y);
#pragma unroll
            for (int j = 0; j < E; ++j) nq::store_f32_as(a.q_out, a.q_dtype, at + lane + kWave * j, y[j]);
        }
        return;
    }

    const int slot = blockIdx.x / p.kv_heads, g = blockIdx.x - slot * p.kv_heads, page = 1 << p.page_shift;
    const auto first_slot = [&](int i, int begin) {
        return static_cast<int64_t>(begin >> p.page_shift) + 2 * static_cast<int64_t>(i);
    };
    const Found f = sequence_at(p, slot, first_slot);
    const Span s = f.span;
    const int b = f.b, context = f.context;
    const int64_t slot0 = first_slot(b, s.begin);
    // New rows of the sequence that have a place: positions [low, high).
    const int64_t low = max(static_cast<int64_t>(context), int64_t{0});
    const int64_t high = min(static_cast<int64_t>(context) + (s.end - s.begin), static_cast<int64_t>(min(rows, a.rope_rows)));
    const int64_t nth = (low >> p.page_shift) + (slot - slot0);
    const int64_t begin = max(low, nth << p.page_shift), end = min(high, (nth + 1) << p.page_shift);
    if (slot < slot0 || begin >= end) return;
    const int32_t id = p.table[static_cast<int64_t>(b) * p.table_pages + nth];
    if (id < 0 || id >= p.pages) return;
    const int r0 = static_cast<int>(begin) & (page - 1), n = static_cast<int>(end - begin);
    const int64_t token0 = s.begin + (begin - context);
    const int64_t base = static_cast<int64_t>(id) * p.kv_heads + g;
    uint8_t* kp = p.k + base * page * D;
    uint8_t* vp = p.v + base * page * D;
    load_weight<D>(a.k_norm, a.norm_dtype, lane, w);

    float kmax = 0.0f, vmax = 0.0f;
    for (int i = wave; i < n; i += WAVES) {
        const int64_t at = ((token0 + i) * p.kv_heads + g) * D;
        double y[E];
        load_rope_row<D>(a, static_cast<int>(begin) + i, lane, cs, sn);
        norm_rope<D, double>(a.k, a.dtype, at, w, a.k_norm != nullptr, a.eps, cs, sn, lane, y);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            kmax = fmaxf(kmax, finite_or_zero(round_to_odd(y[j])));
            vmax = fmaxf(vmax, finite_or_zero(nq::load_f32(a.v, a.dtype, at + lane + kWave * j)));
        }
    }
    kmax = wave_max(kmax);
    vmax = wave_max(vmax);
    if (WAVES > 1) {
        if (lane == 0) {
            red[0][wave] = kmax;
            red[1][wave] = vmax;
        }
        __syncthreads();
        for (int i = 0; i < WAVES; ++i) {
            kmax = fmaxf(kmax, red[0][i]);
            vmax = fmaxf(vmax, red[1][i]);
        }
    }
    float ks = scale_for(kmax), vs = scale_for(vmax);
    if (r0) {
        // Rows [0, r0) stay; their scale may have to grow, and they with it.
        const float ko = p.k_scales[base], vo = p.v_scales[base];
        ks = fmaxf(ks, ko);
        vs = fmaxf(vs, vo);
        if (ks != ko) {
            const float ratio = ko / ks;
            for (int i = threadIdx.x * 4; i < r0 * D; i += WAVES * kWave * 4) {
                uint32_t* at = reinterpret_cast<uint32_t*>(kp + i);
                *at = moved4(*at, ratio);
            }
        }
        if (vs != vo) {
            const float ratio = vo / vs;
            for (int i = threadIdx.x; i < r0 * D; i += WAVES * kWave) {
                uint8_t* at = vp + (i / r0) * page + i % r0;
                *at = static_cast<uint8_t>(moved4(*at, ratio) & 0xff);
            }
        }
    }
    if (WAVES > 1) __syncthreads();  // every wave has read the old scales
    if (threadIdx.x == 0) {
        p.k_scales[base] = ks;
        p.v_scales[base] = vs;
    }
    // 1 / scale as a power of two; the old scale of a page may be any value.
    const float ki = 1.0f / ks, vi = 1.0f / vs;
    for (int i = wave; i < n; i += WAVES) {
        const int64_t at = ((token0 + i) * p.kv_heads + g) * D;
        double y[E];
        load_rope_row<D>(a, static_cast<int>(begin) + i, lane, cs, sn);
        norm_rope<D, double>(a.k, a.dtype, at, w, a.k_norm != nullptr, a.eps, cs, sn, lane, y);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int d = lane + kWave * j;
            kp[(r0 + i) * D + d] = e4m3(round_to_odd(y[j]) * ki);
            vp[d * page + r0 + i] = e4m3(nq::load_f32(a.v, a.dtype, at + d) * vi);
        }
    }
}

bool float_code(int d) { return nq::is_float_dtype(d); }

}  // namespace

extern "C" int nq_paged_append(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens,
                               int32_t q_heads, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                               const float* cos_table, const float* sin_table, int64_t rope_positions,
                               const nq_paged_kv* kv, void* q_out, int32_t q_out_dtype, void* stream) {
    if (!q || !k || !v || !cos_table || !sin_table || !q_out || (q_norm == nullptr) != (k_norm == nullptr))
        return NQ_ERR_ARGUMENT;
    if (!float_code(dtype) || !float_code(q_out_dtype) || (q_norm && !float_code(norm_dtype))) return NQ_ERR_DTYPE;
    AppendArgs a{};
    if (const int st = check_pages(kv, tokens, a.p); st != NQ_OK) return st;
    if (q_heads <= 0 || q_heads > 65535 || q_heads % kv->kv_heads || rope_positions <= 0) return NQ_ERR_SHAPE;
    if (!(eps >= 0.0f)) return NQ_ERR_ARGUMENT;
    a.q = q; a.k = k; a.v = v; a.q_norm = q_norm; a.k_norm = k_norm;
    a.cos_table = cos_table; a.sin_table = sin_table; a.q_out = q_out;
    a.eps = eps; a.dtype = dtype; a.norm_dtype = norm_dtype; a.q_dtype = q_out_dtype; a.q_heads = q_heads;
    a.rope_rows = static_cast<int32_t>(rope_positions < 0x7fffffff ? rope_positions : 0x7fffffff);
    constexpr int kWaves = 4;
    a.q_groups = (q_heads + 2 * kWaves - 1) / (2 * kWaves);
    const int64_t kv_blocks = ((tokens >> a.p.page_shift) + 2 * kv->batch) * kv->kv_heads;
    const int64_t blocks = kv_blocks + tokens * a.q_groups;
    if (blocks > 0x7fffffff) return NQ_ERR_SHAPE;
    a.kv_blocks = static_cast<int32_t>(kv_blocks);
    const dim3 grid(static_cast<unsigned>(blocks));
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (kv->head_dim) {
        case 64: hipLaunchKernelGGL((k_paged_append<64, 4>), grid, dim3(256), 0, st, a); break;
        case 128: hipLaunchKernelGGL((k_paged_append<128, 4>), grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL((k_paged_append<256, 4>), grid, dim3(256), 0, st, a); break;
    }
    return nq::launch_status();
}
