// Products of a few tokens with 4-bit weights and group scales:
//   y[t, o] = sum_i s[o, i / G] (w[o, i] - z[o, i / G]) x[t, i]
//
// Exact integer arithmetic inside a group: x is held as three int8 digits of base
// 256 and one exponent for each token and group (within 2^-23 of the group's
// largest value), the nibbles are int8 operands as they are, and
// v_mfma_i32_16x16x64_i8 sums them. Per group and row
//   y += s 2^e 256^d (sum_i w_i x_id - z sum_i x_id), d = 0, 1, 2,
// in fp32, the digits' sums sum_i x_id known beforehand.
//
// A chunk is 128 columns: lane 16 q + r of a wave holds 16 bytes of row r, columns 32 q
// to 32 q + 31, whose low nibbles (even columns) are the A operand of one product and
// whose high ones that of another. B's 16 columns are divided among the chunk's
// 128 / G groups; a group's columns are a few tokens' digits, and zero in the lanes of
// other groups, so that one product keeps the groups apart.
#include <algorithm>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace {

constexpr int kWave = 64, kChunk = 128, kDigits = 3;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct Int4Args {
    const void* x;
    const uint8_t* packed;   // [outs][ins / 2]
    const void* scales;      // [outs][groups]
    const uint8_t* zeros;    // the same, or null: 8
    void* y;
    uint64_t* best;          // [tiles] largest value and its row, of one token; may be null
    // The tokens' digits: bytes [tokens][3][chunks][2][64], for each token, chunk and group of it 2^e
    // ([tokens][chunks][4]), and the digits' sums ([tokens][3][chunks][4]).
    uint8_t* digits;
    float* units;
    int32_t* sums;
    int64_t outs, ins;
    int32_t tokens, chunks, groups, x_dtype, scale_dtype, y_dtype;
};

// Groups of a chunk, columns of B that one of them has, and tokens of these.
template <int G>
struct Shape {
    static constexpr int kGroups = kChunk / G, kColumns = 16 / kGroups, kTokens = kColumns / kDigits;
};

// One thread per 8 columns of a token.
template <int G>
__global__ __launch_bounds__(256) void k_int4_digits(const Int4Args a) {
    constexpr int kGroup = G / 8;  // threads of a group
    const int token = blockIdx.y, at = blockIdx.x * 256 + threadIdx.x, chunk = at / 16, t = at & 15;
    if (chunk >= a.chunks) return;  // whole groups of lanes
    float x[8], most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = static_cast<int64_t>(at) * 8 + j;
        x[j] = i < a.ins ? nq::load_f32(a.x, a.x_dtype, token * a.ins + i) : 0.0f;
        finite = finite && fabsf(x[j]) < INFINITY;
        most = fmaxf(most, fabsf(x[j]));
    }
    if (!finite) most = INFINITY;
#pragma unroll
    for (int k = 1; k < kGroup; k *= 2) most = fmaxf(most, __shfl_xor(most, k, kWave));
    finite = most < INFINITY;
    // The largest value is below 2^(k + 1), or so near it that a rounding reaches it: 2^(k + 2).
    const uint32_t bits = __float_as_uint(most);
    const int k = max(static_cast<int>(bits >> 23) - 127 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0), -100);
    const float up = finite ? __uint_as_float(static_cast<uint32_t>(22 - k + 127) << 23) : 0.0f;
    uint32_t even[kDigits] = {}, odd[kDigits] = {};
    int sum[kDigits] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int n = finite ? static_cast<int>(rintf(x[j] * up)) : 0;
#pragma unroll
        for (int d = 0; d < kDigits; ++d) {
            const int digit = static_cast<int8_t>(n);
            n = (n - digit) >> 8;
            sum[d] += digit;
            (j & 1 ? odd : even)[d] |= static_cast<uint32_t>(digit & 255) << (8 * (j / 2));
        }
    }
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
        uint32_t* to = reinterpret_cast<uint32_t*>(a.digits + ((static_cast<int64_t>(token) * kDigits + d) * a.chunks + chunk) * kChunk);
        to[t] = even[d];
        to[16 + t] = odd[d];
#pragma unroll
        for (int m = 1; m < kGroup; m *= 2) sum[d] += __shfl_xor(sum[d], m, kWave);
        if (t % kGroup == 0) a.sums[((static_cast<int64_t>(token) * kDigits + d) * a.chunks + chunk) * 4 + t / kGroup] = sum[d];
    }
    if (t % kGroup == 0)
        a.units[(static_cast<int64_t>(token) * a.chunks + chunk) * 4 + t / kGroup] =
            finite ? __uint_as_float(static_cast<uint32_t>(k - 22 + 127) << 23) : __builtin_nanf("");
}

__device__ __forceinline__ uint64_t order_of(float v, uint32_t row) {
    const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
    return static_cast<uint64_t>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - row);
}

constexpr int kWaves = 4;

// A workgroup has 16 rows; its waves take the chunks in turn.
template <int G>
__global__ __launch_bounds__(kWaves* kWave) void k_int4_product(const Int4Args a) {
    using S = Shape<G>;
    __shared__ float join[kWaves][16][17];
    __shared__ uint64_t keys[16];
    const int lane = threadIdx.x & (kWave - 1), c = lane & 15, q = lane >> 4, wave = threadIdx.x / kWave;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 16;
    const int64_t half = a.ins / 2;
    const uint8_t* row = a.packed + min(row0 + c, a.outs - 1) * half;
    // This lane's column of B.
    const int group = c / S::kColumns, in_group = c % S::kColumns, local = in_group / kDigits, digit = in_group % kDigits;
    const float power = digit == 0 ? 1.0f : digit == 1 ? 256.0f : 65536.0f;
    const bool mine = q * S::kGroups / 4 == group;
    for (int first = 0; first < a.tokens; first += S::kTokens) {
        const int token = first + local;
        const bool on = local < S::kTokens && token < a.tokens;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int chunk = wave; chunk < a.chunks; chunk += kWaves) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(row + min(static_cast<int64_t>(chunk) * 64 + 16 * q, half - 16));
            const int64_t at = (static_cast<int64_t>(on ? token : 0) * kDigits + (on ? digit : 0)) * a.chunks + chunk;
            u32x4 b[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (on && mine) {
                const u32x4* from = reinterpret_cast<const u32x4*>(a.digits + at * kChunk);
                b[0] = from[q];
                b[1] = from[4 + q];
            }
            const u32x4 low = w & 0x0f0f0f0fu, high = (w >> 4) & 0x0f0f0f0fu;
            i32x4 dot = {0, 0, 0, 0};
            dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, low), __builtin_bit_cast(i32x4, b[0]), dot, 0, 0, 0);
            dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, high), __builtin_bit_cast(i32x4, b[1]), dot, 0, 0, 0);
            if (on) {
                const float unit = power * a.units[(static_cast<int64_t>(token) * a.chunks + chunk) * 4 + group];
                const int sum = a.sums[at * 4 + group];
                const int64_t g = min(chunk * S::kGroups + group, a.groups - 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t s = min(row0 + 4 * q + i, a.outs - 1) * a.groups + g;
                    const int zero = a.zeros ? a.zeros[s] : 8;
                    acc[i] += nq::load_f32(a.scales, a.scale_dtype, s) * unit * static_cast<float>(dot[i] - zero * sum);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) join[wave][4 * q + i][c] = on ? acc[i] : 0.0f;
        __syncthreads();
        // Thread 16 t + r: token first + t, row r.
        const int r = threadIdx.x & 15, t = threadIdx.x >> 4;
        if (t < S::kTokens && first + t < a.tokens) {
            float y = 0.0f;
#pragma unroll
            for (int d = kDigits - 1; d >= 0; --d)
#pragma unroll
                for (int s = 0; s < S::kGroups; ++s)
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) y += join[w][r][s * S::kColumns + t * kDigits + d];
            const bool there = row0 + r < a.outs;
            if (there) nq::store_f32_as(a.y, a.y_dtype, static_cast<int64_t>(first + t) * a.outs + row0 + r, y);
            if (a.best && t == 0) keys[r] = there ? order_of(y, static_cast<uint32_t>(row0 + r)) : 0;
        }
        __syncthreads();
    }
    if (a.best && threadIdx.x == 0) {
        uint64_t top = keys[0];
        for (int r = 1; r < 16; ++r) top = keys[r] > top ? keys[r] : top;
        a.best[blockIdx.x] = top;
    }
}

int64_t chunks_of(int64_t ins) { return (ins + kChunk - 1) / kChunk; }

template <int G>
int launch_for(const Int4Args& a, hipStream_t stream) {
    const dim3 pre(static_cast<unsigned>((a.chunks + 15) / 16), static_cast<unsigned>(a.tokens));
    hipLaunchKernelGGL(k_int4_digits<G>, pre, dim3(256), 0, stream, a);
    if (const int st = nq::launch_status(); st != NQ_OK) return st;
    hipLaunchKernelGGL(k_int4_product<G>, dim3(static_cast<unsigned>((a.outs + 15) / 16)), dim3(kWaves * kWave), 0, stream, a);
    return nq::launch_status();
}

}  // namespace

extern "C" int64_t nq_int4_projection_workspace_bytes(int64_t tokens, int64_t out_features, int64_t in_features, int32_t group) {
    if (tokens <= 0 || tokens > 65535 || out_features <= 0 || out_features > 0x7fffffff || in_features <= 0 || in_features % 32 ||
        in_features > (1 << 24) || (group != 32 && group != 64 && group != 128))
        return -1;
    if (!nq::launchable((out_features + 15) / 16, kWaves * kWave)) return -1;
    if (!nq::launchable((chunks_of(in_features) + 15) / 16 * tokens, 256)) return -1;
    // Digits, their sums, and an exponent for each token and group.
    return tokens * chunks_of(in_features) * (kDigits * kChunk + (kDigits + 1) * 4 * 4);
}

extern "C" int64_t nq_int4_projection_partials(int64_t out_features) { return out_features <= 0 ? -1 : (out_features + 15) / 16; }

extern "C" int nq_int4_projection(const void* x, int32_t x_dtype, int64_t tokens, const void* packed, const void* scales,
                                  int32_t scale_dtype, const uint8_t* zeros, int64_t out_features, int64_t in_features,
                                  int32_t group, void* y, int32_t y_dtype, void* partials, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    if (!x || !packed || !scales || !y || !workspace) return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(x_dtype) || !nq::is_float_dtype(scale_dtype) || !nq::is_float_dtype(y_dtype)) return NQ_ERR_DTYPE;
    const int64_t need = nq_int4_projection_workspace_bytes(tokens, out_features, in_features, group);
    if (need < 0 || (partials && tokens != 1)) return NQ_ERR_SHAPE;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(workspace)) & 15) return NQ_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(partials) & 7) return NQ_ERR_ALIGNMENT;
    Int4Args a{};
    a.x = x;
    a.packed = static_cast<const uint8_t*>(packed);
    a.scales = scales;
    a.zeros = zeros;
    a.y = y;
    a.best = static_cast<uint64_t*>(partials);
    a.outs = out_features;
    a.ins = in_features;
    a.tokens = static_cast<int32_t>(tokens);
    a.chunks = static_cast<int32_t>(chunks_of(in_features));
    a.groups = static_cast<int32_t>((in_features + group - 1) / group);
    a.x_dtype = x_dtype;
    a.scale_dtype = scale_dtype;
    a.y_dtype = y_dtype;
    a.digits = static_cast<uint8_t*>(workspace);
    a.units = reinterpret_cast<float*>(a.digits + tokens * a.chunks * kDigits * kChunk);
    a.sums = reinterpret_cast<int32_t*>(a.units + tokens * a.chunks * 4);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (group) {
        case 32: return launch_for<32>(a, st);
        case 64: return launch_for<64>(a, st);
        default: return launch_for<128>(a, st);
    }
}
