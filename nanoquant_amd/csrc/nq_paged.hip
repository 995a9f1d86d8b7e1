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

constexpr int kPageTokens = 8;  // new rows of a page that a wave holds in registers
constexpr int kQHeads = 4;      // q heads of a token that a wave takes

// Lane values permuted within rows of 16 (DPP), 0 where a source lane is off.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const int2 w = __builtin_bit_cast(int2, x);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, w.x, CTRL, 0xf, 0xf, false),
                                                __builtin_amdgcn_update_dpp(0, w.y, CTRL, 0xf, 0xf, false)));
}

__device__ __forceinline__ float lane_of(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

__device__ __forceinline__ double lane_of(double v, int lane) {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(w.x, lane), __builtin_amdgcn_readlane(w.y, lane)));
}

// Sum over the wave, in a fixed order.
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp<0x141>(v);  // row_half_mirror
    v += dpp<0x140>(v);  // row_mirror
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// Maximum of values >= 0 over the wave.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    v = fmaxf(v, dpp<0x140>(v));
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

__device__ __forceinline__ float partner_of(float v) { return __shfl_xor(v, 32, kWave); }

__device__ __forceinline__ double partner_of(double v) {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__shfl_xor(w.x, 32, kWave), __shfl_xor(w.y, 32, kWave)));
}

__device__ __forceinline__ float inverse_root(float x) { return 1.0f / sqrtf(x); }

// The hardware's estimate is good to 2^-24; each step y (3 - x y^2) / 2 squares
// the error. 0 and infinity (of an infinite or a zero mean) are kept.
__device__ __forceinline__ double inverse_root(double x) {
    const double y0 = __builtin_amdgcn_rsq(x);
    double y = y0;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = y * fma(-0.5 * x * y, y, 1.5);
    return y0 > 0.0 && y0 < INFINITY ? y : y0;
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

// x as fp32 for an e4m3 rounding: the nearest fp32 value does, unless it lies
// where e4m3 rounds to even or where a scale ends. All of those have 0 in their
// last 19 bits.
__device__ __forceinline__ float for_e4m3(double x) {
    float f = static_cast<float>(x);
    if (__ballot((__float_as_uint(f) & 0x7ffffu) == 0 && f != 0.0f)) f = round_to_odd(x);
    return f;
}

// One wave's head vector, lane l holding d = l + 64 j: RMSNorm with weight w
// (has_w), then rotate-half RoPE, in place. In T = double the result is correct
// to far below an e4m3 rounding's border.
template <int D, class T>
__device__ __forceinline__ void norm_rope(T (&v)[D / kWave], const float (&w)[D / kWave], bool has_w, float eps,
                                          const float (&cs)[D / kWave], const float (&sn)[D / kWave], int lane) {
    constexpr int E = D / kWave;
    if (has_w) {
        T ss = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) ss += v[j] * v[j];
        const T inv = inverse_root(wave_sum(ss) * static_cast<T>(1.0 / D) + static_cast<T>(eps));
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = static_cast<T>(w[j]) * (v[j] * inv);
    }
    T y[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const bool first = lane + kWave * j < D / 2;
        T partner;
        if constexpr (E == 1) partner = partner_of(v[0]);
        else partner = first ? v[j + E / 2] : v[j - E / 2];
        y[j] = v[j] * static_cast<T>(cs[j]) + (first ? -partner : partner) * static_cast<T>(sn[j]);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = y[j];
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

template <int D>
__device__ __forceinline__ void load_head(const void* x, int dtype, int64_t at, int lane, float (&v)[D / kWave]) {
#pragma unroll
    for (int j = 0; j < D / kWave; ++j) v[j] = nq::load_f32(x, dtype, at + lane + kWave * j);
}

// A tile of bytes in LDS, [lines][width] with each line's bytes [first, first +
// n) new, to memory: whole words where they are new, single bytes at the ends.
__device__ __forceinline__ void store_lines(const uint8_t* tile, int stride, uint8_t* out, int lines, int width, int first, int n,
                                            int threads) {
    const int words = width / 4;
    for (int i = threadIdx.x; i < lines * words; i += threads) {
        const int line = i / words, c = (i - line * words) * 4;
        if (c + 4 <= first || c >= first + n) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + line * stride + c);
        uint8_t* at = out + line * width + c;
        if (c >= first && c + 4 <= first + n) {
            *reinterpret_cast<uint32_t*>(at) = w;
        } else {
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (c + b >= first && c + b < first + n) at[b] = static_cast<uint8_t>(w >> (8 * b));
        }
    }
}

// Workgroups [0, kv_blocks): the new rows of one page and kv head, kPageTokens
// to a wave, which holds them in registers until the page's scale is known; the
// bytes go out through LDS, V's transposed. Sequence b has at most (its tokens)
// / page + 2 pages with new rows, and its slots begin at starts[b] / page + 2 b:
// the grid follows from the host's counts alone. The rest: q, one wave per token
// and kQHeads of its heads.
template <int D, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void k_paged_append(const AppendArgs a) {
    constexpr int E = D / kWave, kPage = WAVES * kPageTokens, kThreads = WAVES * kWave;
    // K: a row of D bytes after the other; V: a line of kPage bytes, padded by a
    // word against bank conflicts, for each of D.
    constexpr int kLine = kPage + 4;
    __shared__ float red[2][WAVES];
    __shared__ uint32_t tile[D * kLine / 4];
    const Pages& p = a.p;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int rows = p.table_pages << p.page_shift;
    float w[E];

    if (static_cast<int>(blockIdx.x) >= a.kv_blocks) {
        const int64_t item = static_cast<int64_t>(blockIdx.x - a.kv_blocks) * WAVES + wave;
        const int token = static_cast<int>(item / a.q_groups);
        const int head = static_cast<int>(item - static_cast<int64_t>(token) * a.q_groups) * kQHeads;
        if (token >= p.tokens) return;
        const Found f = sequence_at(p, token, [](int, int begin) { return static_cast<int64_t>(begin); });
        const Span s = f.span;
        const int row = token >= s.begin && token < s.end ? row_of(f.context, token - s.begin, rows) : -1;
        if (row < 0 || row >= a.rope_rows) return;
        float cs[E], sn[E], x[kQHeads][E];
        const int64_t at = (static_cast<int64_t>(token) * a.q_heads + head) * D;
#pragma unroll
        for (int i = 0; i < kQHeads; ++i) load_head<D>(a.q, a.dtype, at + min(i, a.q_heads - 1 - head) * D, lane, x[i]);
        load_weight<D>(a.q_norm, a.norm_dtype, lane, w);
        load_rope_row<D>(a, row, lane, cs, sn);
#pragma unroll
        for (int i = 0; i < kQHeads; ++i) {
            norm_rope<D, float>(x[i], w, a.q_norm != nullptr, a.eps, cs, sn, lane);
            if (head + i >= a.q_heads) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) nq::store_f32_as(a.q_out, a.q_dtype, at + i * D + lane + kWave * j, x[i][j]);
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
    // New rows of the sequence that have a place: positions [low, high).
    const int64_t low = max(static_cast<int64_t>(context), int64_t{0});
    const int64_t high = min(static_cast<int64_t>(context) + (s.end - s.begin), static_cast<int64_t>(min(rows, a.rope_rows)));
    const int64_t nth = low / kPage + (slot - slot0);
    const int64_t begin = max(low, nth * kPage), end = min(high, (nth + 1) * kPage);
    if (slot < slot0 || begin >= end) return;
    const int32_t id = p.table[static_cast<int64_t>(b) * p.table_pages + nth];
    const int r0 = static_cast<int>(begin) & (kPage - 1), n = static_cast<int>(end - begin);
    const int64_t token0 = s.begin + (begin - context);

    // Loads first, of the wave's last row again where it has fewer.
    float kf[kPageTokens][E], vf[kPageTokens][E];
    const int mine = wave < n ? (n - wave + WAVES - 1) / WAVES : 0;  // rows wave, wave + WAVES, ...
    load_weight<D>(a.k_norm, a.norm_dtype, lane, w);
    float kmax = 0.0f, vmax = 0.0f;
    const auto load_row = [&](int i) {
        const int64_t at = ((token0 + wave + i * WAVES) * p.kv_heads + g) * D;
        load_head<D>(a.k, a.dtype, at, lane, kf[i]);
        load_head<D>(a.v, a.dtype, at, lane, vf[i]);
    };
    const auto turn_row = [&](int i, const float (&cs)[E], const float (&sn)[E]) {
        double y[E];
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = static_cast<double>(kf[i][j]);
        norm_rope<D, double>(y, w, a.k_norm != nullptr, a.eps, cs, sn, lane);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            kf[i][j] = for_e4m3(y[j]);
            kmax = fmaxf(kmax, finite_or_zero(kf[i][j]));
            vmax = fmaxf(vmax, finite_or_zero(vf[i][j]));
        }
    };
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i)
        if (i < mine) load_row(i);
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i) {
        if (i >= mine) break;
        float cs[E], sn[E];
        load_rope_row<D>(a, static_cast<int>(begin) + wave + i * WAVES, lane, cs, sn);
        turn_row(i, cs, sn);
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
        if (wave == 0)
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int d = lane + kWave * j;
                kp[r0 * D + d] = e4m3(kf[0][j] * ki);
                vp[d * kPage + r0] = e4m3(vf[0][j] * vi);
            }
        return;
    }
    uint8_t* bytes = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i) {
        if (i >= mine) break;
#pragma unroll
        for (int j = 0; j < E; ++j) bytes[(wave + i * WAVES) * D + lane + kWave * j] = e4m3(kf[i][j] * ki);
    }
    __syncthreads();
    store_lines(bytes, D, kp + r0 * D, n, D, 0, D, kThreads);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPageTokens; ++i) {
        if (i >= mine) break;
#pragma unroll
        for (int j = 0; j < E; ++j) bytes[(lane + kWave * j) * kLine + r0 + wave + i * WAVES] = e4m3(vf[i][j] * vi);
    }
    __syncthreads();
    store_lines(bytes, kLine, vp, D, kPage, r0, n, kThreads);
}

template <int D>
int launch_append(AppendArgs& a, int64_t tokens, int kv_heads, int64_t batch, hipStream_t stream) {
    const int waves = (1 << a.p.page_shift) / kPageTokens;
    const int64_t kv_blocks = ((tokens >> a.p.page_shift) + 2 * batch) * kv_heads;
    const int64_t blocks = kv_blocks + (tokens * a.q_groups + waves - 1) / waves;
    if (blocks > 0x7fffffff) return NQ_ERR_SHAPE;
    a.kv_blocks = static_cast<int32_t>(kv_blocks);
    const dim3 grid(static_cast<unsigned>(blocks)), block(static_cast<unsigned>(waves * kWave));
    switch (waves) {
        case 2: hipLaunchKernelGGL((k_paged_append<D, 2>), grid, block, 0, stream, a); break;
        case 4: hipLaunchKernelGGL((k_paged_append<D, 4>), grid, block, 0, stream, a); break;
        case 8: hipLaunchKernelGGL((k_paged_append<D, 8>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((k_paged_append<D, 16>), grid, block, 0, stream, a); break;
    }
    return nq::launch_status();
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
    a.q_groups = (q_heads + kQHeads - 1) / kQHeads;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (kv->head_dim) {
        case 64: return launch_append<64>(a, tokens, kv->kv_heads, kv->batch, st);
        case 128: return launch_append<128>(a, tokens, kv->kv_heads, kv->batch, st);
        default: return launch_append<256>(a, tokens, kv->kv_heads, kv->batch, st);
    }
}
