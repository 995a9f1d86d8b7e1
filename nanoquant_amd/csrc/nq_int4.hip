// Products of a few tokens with 4-bit weights and group scales:
//   y[t, o] = sum_i s[o, i / G] (w[o, i] - z[o, i / G]) x[t, i]
//
// Exact integer arithmetic inside a group: x is held as int8 digits of base 256 and
// one exponent for each token and group, the nibbles are int8 operands as they are, and
// v_mfma_i32_16x16x64_i8 sums them. Per group and row
//   y += s 2^e 256^d (sum_i w_i x_id - z sum_i x_id), d = 0, 1, 2 (and 3 for fp32 x),
// in fp32, the digits' sums sum_i x_id known beforehand.
//
// Digits: a 16-bit x has three, within 2^-23 of its group's largest value, so that bf16 values
// are exact down to 2^-15 of it and fp16 values down to 2^-12 (what is lost below is less than their own
// rounding down to 2^-14 and 2^-11); fp32 x has four, within 2^-31, exact down to 2^-7 of it. With three, an
// fp32 value far below another one of its group whose weights are at the zero point (so that nothing hides the
// loss) would keep few bits of its own. Four cost one token of a large matrix nothing (151936 x 4096: 55.9
// us, 56.0 with three), 11 tokens of 2560 x 10240, groups of 64, 17.8 us for 17.2, and with groups of 128 what reading the
// weights for 4 tokens to a block and 24 at once does, not 5 and 30 (4096 x 4096: 5 tokens 11.7 us for 9.9, 30 24.4 for 21.3).
//
// A chunk is 128 columns: lane 16 q + r of a wave holds 16 bytes of row r, columns 32 q
// to 32 q + 31, whose low nibbles (even columns) are the A operand of one product and
// whose high ones that of another. B's 16 columns are divided among the chunk's
// 128 / G groups; a group's columns are a few tokens' digits, and zero in the lanes of
// other groups, so that one product keeps the groups apart.
#include <algorithm>
#include <type_traits>

#include "nq_common.h"
#include "../../include/nqamd_shell.h"

namespace {

constexpr int kWave = 64, kChunk = 128;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// How a call is laid out: `blocks` blocks of tokens at once, of each row's chunks a
// `slice` for a workgroup, in stages of `stage` that LDS holds the digits of.
struct Int4Plan {
    int waves, blocks, passes, share, slices, slice, stage;
    int64_t groups;  // workgroups of a pass and slice
};

struct Int4Args {
    const void* x;
    const uint8_t* packed;   // [outs][ins / 2]
    const void* scales;      // [outs][groups]
    const uint8_t* zeros;    // the same, or null: 8
    void* y;
    float* partial;          // [slices][tokens][outs] where the slices are joined in a second launch
    uint64_t* best;          // [tiles] largest value and its row, of one token; may be null
    int64_t outs, ins, tiles, step;  // step: tiles from one of a wave's to its next
    int32_t tokens, chunks, groups, x_dtype, y_dtype;
    int32_t share, slice, stage;
};

// Digits of x by its type.
constexpr int digits_for(int x_dtype) { return x_dtype == NQ_DTYPE_F32 ? 4 : 3; }

// Groups of a chunk, columns of B that one of them has, and tokens of these.
template <int G, int DG>
struct Shape {
    static constexpr int kGroups = kChunk / G, kColumns = 16 / kGroups, kTokens = kColumns / DG;
};

__device__ __forceinline__ uint64_t order_of(float v, uint32_t row) {
    const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
    return static_cast<uint64_t>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - row);
}

// The largest (value, row) of a tile's 16 rows, which 16 lanes hold.
__device__ __forceinline__ uint64_t best_of_tile(uint64_t key) {
#pragma unroll
    for (int m = 1; m < 16; m *= 2) {
        const uint32_t low = __shfl_xor(static_cast<uint32_t>(key), m, kWave);
        const uint32_t high = __shfl_xor(static_cast<uint32_t>(key >> 32), m, kWave);
        const uint64_t other = static_cast<uint64_t>(high) << 32 | low;
        key = other > key ? other : key;
    }
    return key;
}

// What a wave's lanes wrote to LDS is what its lanes read after this.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kAhead = 2;   // rounds of x
constexpr int kAtOnce = 4;  // chunks whose weights a wave loads at once: 256 bytes of each of 16 rows

// Digits in LDS: a line of `stage` chunks, [2][64] bytes each (even and odd columns), for each token and
// digit; 64 bytes more a line, so that a product's columns lie in different banks.
__host__ __device__ constexpr int line_bytes(int stage) { return stage * kChunk + 64; }

// Words of LDS that each wave has for itself.
template <int GROUPS>
constexpr int kEachWave = 16 * 16 * 4 + 16 * 17 + kAtOnce * GROUPS * (16 + 4);

// A column of B in a chunk: what a product with it is multiplied by, but for the
// row's scale, and the sum of its digits.
struct Column {
    float unit, sum;
};

// A 16-bit value's bits as fp32.
__device__ __forceinline__ float from_half(uint32_t bits, int dtype) {
    return dtype == NQ_DTYPE_BF16 ? __uint_as_float(bits << 16)
                                  : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}

// Eight adjacent values' bits, at any address that fits their type.
struct Eight {
    uint32_t w[8];
};

__device__ __forceinline__ Eight load8(const void* p, int dtype, int64_t i) {
    Eight v;
    if (dtype == NQ_DTYPE_F32) {
        typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(4)));
        const vec* from = reinterpret_cast<const vec*>(static_cast<const uint32_t*>(p) + i);
        const vec x0 = from[0], x1 = from[1];
#pragma unroll
        for (int j = 0; j < 8; ++j) v.w[j] = j < 4 ? x0[j & 3] : x1[j & 3];
    } else {
        typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
        const vec x = *reinterpret_cast<const vec*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v.w[j] = x[j & 3];
    }
    return v;
}

__device__ __forceinline__ void widen8(const Eight& v, int dtype, float (&x)[8]) {
    if (dtype == NQ_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(v.w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = from_half(v.w[j / 2] >> (16 * (j & 1)) & 0xffffu, dtype);
    }
}

// Eight adjacent columns of a token as DG digits.
template <int G, int DG>
__device__ __forceinline__ void digits_of(const float (&x)[8], uint32_t (&even)[DG], uint32_t (&odd)[DG], int (&sum)[DG],
                                          float& unit) {
    constexpr int kGroup = G / 8;  // lanes of a group
    constexpr int kBits = 8 * DG - 2, kLowest = DG == 4 ? -96 : -100;  // 2^(kBits - kLowest) is a number
    constexpr uint32_t kBias = 0x80808080u >> (32 - 8 * DG);
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        finite = finite && fabsf(x[j]) < INFINITY;
        most = fmaxf(most, fabsf(x[j]));
    }
    if (!finite) most = INFINITY;
#pragma unroll
    for (int k = 1; k < kGroup; k *= 2) most = fmaxf(most, __shfl_xor(most, k, kWave));
    finite = most < INFINITY;
    // The largest value is below 2^(k + 1), or so near it that a rounding reaches it: 2^(k + 2).
    const uint32_t bits = __float_as_uint(most);
    const int k = max(static_cast<int>(bits >> 23) - 127 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0), kLowest);
    const float up = finite ? __uint_as_float(static_cast<uint32_t>(kBits - k + 127) << 23) : 0.0f;
    // n + 0x808080 (or 0x80808080) has the digits plus 128 each as its bytes: n is at most
    // 2^22 * 1.984375 = 0x7f0000 (2^30 * 1.984375 = 0x7f000000) either way.
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = static_cast<uint32_t>(finite ? static_cast<int>(rintf(x[j] * up)) : 0) + kBias;
#pragma unroll
    for (int d = 0; d < DG; ++d) {
        // Byte d of four values in a word.
        const uint32_t pair = 0x0c0c0400u + 0x0101u * d;
        const auto four = [&](uint32_t a, uint32_t b, uint32_t e, uint32_t f) {
            return (__builtin_amdgcn_perm(b, a, pair) | __builtin_amdgcn_perm(f, e, pair) << 16) ^ 0x80808080u;
        };
        even[d] = four(u[0], u[2], u[4], u[6]);
        odd[d] = four(u[1], u[3], u[5], u[7]);
        sum[d] = __builtin_amdgcn_sdot4(static_cast<int>(even[d]), 0x01010101,
                                        __builtin_amdgcn_sdot4(static_cast<int>(odd[d]), 0x01010101, 0, false), false);
    }
#pragma unroll
    for (int d = 0; d < DG; ++d)
#pragma unroll
        for (int m = 1; m < kGroup; m *= 2) sum[d] += __shfl_xor(sum[d], m, kWave);
    unit = finite ? __uint_as_float(static_cast<uint32_t>(k - kBits + 127) << 23) : __builtin_nanf("");
}

// Large matrices of one token are bound by their bytes (151936 x 4096: 321 MB in 54.9 us, 5.9
// TB/s, where a copy reaches 5.04): every load takes 256 bytes of a row (64 of each of 16
// rows, as the products want them, took 70.7 us), LDS turns them. Small ones wait for x, then
// for the digits and the weights (6912 x 1152: 5.9 us, a launch 1.65). With more tokens than a
// block has the products' operands come from LDS, 2 KB a chunk and block, and bound it.
// A workgroup has a slice of the chunks and, share waves to a tile of 16 rows, kWaves / share tiles
// at a time; the waves of a tile each take a part of a stage's chunks. NB blocks of tokens.
template <int G, int NB, int ST, int kWaves, int DG>
__global__ __launch_bounds__(kWaves* kWave, kWaves == 8 ? 1 : NB <= 3 ? 3 : 2) void k_int4_product(const Int4Args a) {
    constexpr int kThreads = kWaves * kWave;
    using S = Shape<G, DG>;
    constexpr int kTogether = NB <= 2 ? 2 : 1;
    constexpr int kMost = kAtOnce * S::kGroups;  // groups whose scales a wave holds in LDS
    extern __shared__ u32x4 lds[];
    // Zeros, digits, columns; for each wave 16 rows' units, sums [16][17], scales [kMost][16] and zeros [kMost][16].
    uint8_t* digits = reinterpret_cast<uint8_t*>(lds) + 64;
    const int first = blockIdx.z * NB * S::kTokens, tokens = min(NB * S::kTokens, a.tokens - first);
    const int line = line_bytes(a.stage);
    Column* columns = reinterpret_cast<Column*>(digits + tokens * DG * line);  // [stage][NB][16]
    float* mine_f = reinterpret_cast<float*>(columns + a.stage * NB * 16);
    const int lane = threadIdx.x & (kWave - 1), c = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    constexpr int kRow = S::kColumns + 1;  // a row's sums, in another bank than the next one's
    constexpr int kEach = kEachWave<S::kGroups>;
    u32x4* units = reinterpret_cast<u32x4*>(mine_f + wave * kEach);
    float* sums = reinterpret_cast<float*>(units + 16 * 16);
    float* scales = sums + 16 * 17;
    uint8_t* zeros = reinterpret_cast<uint8_t*>(scales + kMost * 16);
    if (threadIdx.x < 16) reinterpret_cast<uint32_t*>(lds)[threadIdx.x] = 0;

    const int chunk0 = blockIdx.y * a.slice, chunk1 = min(chunk0 + a.slice, a.chunks);
    const int part = wave % a.share;
    const int64_t half = a.ins / 2;
    const int group = c / S::kColumns, in_group = c % S::kColumns, local = in_group / DG, digit = in_group % DG;
    const bool mine = q * S::kGroups / 4 == group && local < S::kTokens;
    // Where this lane's operand of a block begins in LDS, and its odd columns' behind; 0: zeros.
    int from_at[NB], odd_at[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int token = b * S::kTokens + local;
        const bool on = mine && token < tokens;
        from_at[b] = on ? 64 + (token * DG + digit) * line + 16 * q : 0;
        odd_at[b] = on ? 64 : 0;
    }

    // The digits of chunks [begin, begin + n), eight columns of a token to a thread and round. The
    // first rounds' columns are loaded before the weights, which take longer.
    Eight ahead[kAhead];
    const auto bits_at = [&](int begin, int n, int i) {
        const int token = tokens == 1 ? 0 : i / (16 * n);
        const int64_t at = static_cast<int64_t>(begin + (i >> 4) - token * n) * kChunk + 8 * (i & 15);
        Eight v = {};
        if (i < tokens * n * 16 && at < a.ins) v = load8(a.x, a.x_dtype, (first + token) * a.ins + at);  // ins is a multiple of 32
        return v;
    };
    const auto fill = [&](int begin, int n) {
        const auto round = [&](int i, const Eight& bits) {
            const int t = i & 15, token = tokens == 1 ? 0 : i / (16 * n), at = (i >> 4) - token * n;
            float x[8];
            uint32_t even[DG], odd[DG];
            int sum[DG];
            float unit;
            widen8(bits, a.x_dtype, x);
            digits_of<G, DG>(x, even, odd, sum, unit);
            const int block = token / S::kTokens, in_block = token - block * S::kTokens;
            float power = 1.0f;
#pragma unroll
            for (int d = 0; d < DG; ++d) {
                uint32_t* to = reinterpret_cast<uint32_t*>(digits + (token * DG + d) * line + at * kChunk);
                to[t] = even[d];
                to[16 + t] = odd[d];
                if (t % (G / 8) == 0)
                    columns[(at * NB + block) * 16 + t / (G / 8) * S::kColumns + in_block * DG + d] =
                        Column{unit * power, static_cast<float>(sum[d])};
                power *= 256.0f;
            }
        };
        const int all = tokens * n * 16;  // whole rows of 16 lanes
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = threadIdx.x + j * kThreads;
            if (i < all) round(i, ahead[j]);
        }
        for (int i = threadIdx.x + kAhead * kThreads; i < all; i += kThreads) round(i, bits_at(begin, n, i));
    };
    // Columns that no token has.
    for (int i = threadIdx.x; i < a.stage * NB * 16; i += kThreads) {
        const int at = i & 15, t = at % S::kColumns / DG;
        if (t >= S::kTokens || (i >> 4) % NB * S::kTokens + t >= tokens) columns[i] = Column{0.0f, 0.0f};
    }

    for (int64_t tile0 = static_cast<int64_t>(blockIdx.x) * (kWaves / a.share); tile0 < a.tiles; tile0 += a.step) {
        const int64_t tile = tile0 + wave / a.share, row0 = min(tile, a.tiles - 1) * 16;
        const uint8_t* row[4];  // lane 16 g + u loads 16-byte unit u of rows g, 4 + g, 8 + g and 12 + g
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = a.packed + min(row0 + 4 * j + q, a.outs - 1) * half;
        const int64_t scale_row = min(row0 + c, a.outs - 1) * a.groups;
        float acc[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[b][i] = 0.0f;
        for (int begin = chunk0; begin < chunk1; begin += a.stage) {
            const int n = min(a.stage, chunk1 - begin);
            // This wave's chunks [at, end) of the stage. Weights, scales and zeros (lane 16 q + r
            // loads a quarter of row r's) are on their way while those before are worked on.
            const int per = (n + a.share - 1) / a.share, end = min(n, (part + 1) * per);
            u32x4 w[4];
            std::conditional_t<ST == NQ_DTYPE_F32, uint32_t, uint16_t> s_next[kMost / 4];
            uint8_t z_next[kMost / 4] = {};
            const auto load = [&](int at) {
                const auto g = [&](int j) { return scale_row + min((begin + at) * S::kGroups + q * (kMost / 4) + j, a.groups - 1); };
                if constexpr (ST == NQ_DTYPE_F32) {
#pragma unroll
                    for (int j = 0; j < kMost / 4; ++j) s_next[j] = static_cast<const uint32_t*>(a.scales)[g(j)];
                } else {
#pragma unroll
                    for (int j = 0; j < kMost / 4; ++j) s_next[j] = static_cast<const uint16_t*>(a.scales)[g(j)];
                }
                if (a.zeros) {
#pragma unroll
                    for (int j = 0; j < kMost / 4; ++j) z_next[j] = a.zeros[g(j)];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
                        row[j] + min(static_cast<int64_t>(begin + at) * 64 + 16 * c, half - 16)));
            };
            const bool fills = tile0 == static_cast<int64_t>(blockIdx.x) * (kWaves / a.share) || a.stage < a.slice;
            if (fills) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) ahead[j] = bits_at(begin, n, threadIdx.x + j * kThreads);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (part * per < end) load(part * per);
            if (fills) {
                if (begin != chunk0 || a.stage < a.slice) __syncthreads();  // the stage before is read
                fill(begin, n);
                __syncthreads();
            }
            for (int at = part * per; at < end; at += kAtOnce) {
#pragma unroll
                for (int j = 0; j < kMost / 4; ++j) {
                    scales[(q * (kMost / 4) + j) * 16 + c] =
                        ST == NQ_DTYPE_F32 ? __uint_as_float(s_next[j]) : from_half(s_next[j], ST);
                    zeros[(q * (kMost / 4) + j) * 16 + c] = a.zeros ? z_next[j] : 8;
                }
                // Unit u of row r lies at r's place u ^ r: the products' lanes read 16 rows from 16 places.
#pragma unroll
                for (int j = 0; j < 4; ++j) units[(4 * j + q) * 16 + (c ^ (4 * j + q))] = w[j];
                if (at + kAtOnce < end) load(at + kAtOnce);
                wave_sync();
                // Everything that LDS has for a few chunks, then their products: what waits in between
                // waits once for all.
#pragma unroll
                for (int j0 = 0; j0 < kAtOnce; j0 += kTogether) {
                    if (at + j0 >= end) break;
                    u32x4 now[kTogether];
                    f32x4 s[kTogether];
                    uint32_t z[kTogether];
                    i32x4 x[kTogether][NB][2];
                    Column col[kTogether][NB];
#pragma unroll
                    for (int k = 0; k < kTogether; ++k) {
                        const int j = j0 + k, chunk = min(at + j, end - 1);
                        now[k] = units[c * 16 + ((4 * j + q) ^ c)];
                        s[k] = *reinterpret_cast<const f32x4*>(scales + (j * S::kGroups + group) * 16 + 4 * q);
                        z[k] = *reinterpret_cast<const uint32_t*>(zeros + (j * S::kGroups + group) * 16 + 4 * q);
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const uint8_t* from = reinterpret_cast<const uint8_t*>(lds) + (from_at[b] ? from_at[b] + chunk * kChunk : 0);
                            x[k][b][0] = *reinterpret_cast<const i32x4*>(from);
                            x[k][b][1] = *reinterpret_cast<const i32x4*>(from + odd_at[b]);
                            col[k][b] = columns[(chunk * NB + b) * 16 + c];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < kTogether; ++k) {
                        if (at + j0 + k >= end) break;
                        const u32x4 low = now[k] & 0x0f0f0f0fu, high = (now[k] >> 4) & 0x0f0f0f0fu;
                        i32x4 dot[NB];
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            dot[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, low), x[k][b][0],
                                                                          i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            dot[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, high), x[k][b][1], dot[b], 0, 0, 0);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // Whole numbers below 2^24: exact.
                                const float zero = static_cast<float>(z[k] >> (8 * i) & 255u);
                                const float t = fmaf(-zero, col[k][b].sum, static_cast<float>(dot[b][i]));
                                acc[b][i] = fmaf(s[k][i] * col[k][b].unit, t, acc[b][i]);
                            }
                    }
                }
                wave_sync();
            }
        }
        // The groups' columns are added in registers, a token's digits and the waves of a tile in
        // LDS: lane 16 t + r has token t's of row r.
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = S::kColumns; m < 16; m *= 2) acc[b][i] += __shfl_xor(acc[b][i], m, kWave);
            if (a.share > 1) __syncthreads();
            if (c < S::kColumns) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[(4 * q + i) * kRow + c] = acc[b][i];
            }
            if (a.share > 1) __syncthreads();
            else wave_sync();
            if (part == 0) {
#pragma unroll
                for (int t0 = 0; t0 < S::kTokens; t0 += 4) {
                    const int t = t0 + q, token = b * S::kTokens + t;
                    if (t >= S::kTokens || token >= tokens) break;
                    float y = 0.0f;
#pragma unroll
                    for (int o = 0; o < kWaves; ++o) {
                        if (o >= a.share) break;
#pragma unroll
                        for (int d = DG - 1; d >= 0; --d) y += sums[o * kEach + c * kRow + t * DG + d];
                    }
                    const bool there = tile < a.tiles && row0 + c < a.outs;
                    if (a.partial) {
                        if (there) a.partial[(static_cast<int64_t>(blockIdx.y) * a.tokens + first + token) * a.outs + row0 + c] = y;
                    } else {
                        if (there) nq::store_f32_as(a.y, a.y_dtype, static_cast<int64_t>(first + token) * a.outs + row0 + c, y);
                        if (a.best) {
                            const uint64_t top = best_of_tile(there ? order_of(y, static_cast<uint32_t>(row0 + c)) : 0);
                            if (c == 0 && tile < a.tiles) a.best[tile] = top;
                        }
                    }
                }
            }
            wave_sync();
        }
    }
}

// The slices' sums, in order; 16 lanes have a tile.
__global__ __launch_bounds__(256) void k_int4_join(const Int4Args a, int slices) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int token = blockIdx.y;
    float y = 0.0f;
    if (row < a.outs) {
        constexpr int kMost = 16;
        float part[kMost];
#pragma unroll
        for (int i = 0; i < kMost; ++i) part[i] = i < slices ? a.partial[(static_cast<int64_t>(i) * a.tokens + token) * a.outs + row] : 0.0f;
#pragma unroll
        for (int i = 0; i < kMost; ++i) y += part[i];
        nq::store_f32_as(a.y, a.y_dtype, token * a.outs + row, y);
    }
    if (a.best) {
        const uint64_t top = best_of_tile(row < a.outs ? order_of(y, static_cast<uint32_t>(row)) : 0);
        if ((threadIdx.x & 15) == 0 && row < a.outs) a.best[row / 16] = top;
    }
}

int64_t chunks_of(int64_t ins) { return (ins + kChunk - 1) / kChunk; }

size_t lds_bytes(int waves, int tokens, int digits, int blocks, int groups, int stage) {
    const int wave = groups == 1 ? kEachWave<1> : groups == 2 ? kEachWave<2> : kEachWave<4>;
    return 64 + static_cast<size_t>(tokens) * digits * line_bytes(stage) + static_cast<size_t>(stage) * blocks * 16 * sizeof(Column) +
           static_cast<size_t>(waves) * wave * sizeof(float);
}

// How a call is laid out. A workgroup makes the digits of its tokens and slice itself, in
// LDS, from x (2 to 4 bytes a value from the L2; a launch of its own for them took 4 us).
//  - One token's digits fit LDS for the whole row (12 KB at 4096 columns, 16 of fp32). Waves have tiles of
//    their own from 2048 tiles on, fewer tiles are shared by four waves (4096 columns, one token:
//    4096 rows 6.5 us shared and 10.2 not, 14336 rows 10.8 and 11.4, 24576 13.6 and 13.7, 32768 16.6 and 15.2).
//    768 workgroups walk over the tiles of a large matrix (151936 rows 59.4 us; with 512 65.7, 1024
//    64.6, all at once 64.7, before what LDS has was read ahead: 54.9 since).
//  - Digits of many tokens that LDS does not hold and few tiles: slices of the row, as many as make 2048 waves,
//    eight waves of one slice around the same digits, joined in a second launch (11 tokens, 2560 x
//    10240, groups of 64: 18.3 us; four waves 21.2, 1280 waves 25.3, 2560 waves 28.8).
//  - Otherwise the row in stages, whose digits are made one after the other.
// Blocks: more of them read the weights once for more tokens, and hold more registers.
Int4Plan plan_int4(int64_t tokens, int64_t outs, int64_t ins, int group, int digits) {
    // As many chunks as three digits of them fit 60 KB, and two workgroups a compute unit either way (fp32, 11 tokens of
    // 2560 x 10240, groups of 64: 17.8 us, 19.0 with 60 KB; 16 of 6912 x 4096, groups of 128: 23.4 and 26.0; 6 of 14336
    // x 4096, groups of 32: 33.7 and 36.8; but 8 of it, groups of 128: 30.5 and 23.2, whose slices do better).
    const size_t budget = (digits == 4 ? 78 : 60) * 1024;
    const int groups = kChunk / group, each = 16 / groups / digits;
    const int64_t blocks = (tokens + each - 1) / each, chunks = chunks_of(ins), tiles = (outs + 15) / 16;
    Int4Plan p{};
    p.passes = static_cast<int>((blocks + 5) / 6);
    const int64_t at_once = (blocks + p.passes - 1) / p.passes;
    p.blocks = at_once <= 3 ? static_cast<int>(at_once) : 6;
    p.passes = static_cast<int>((blocks + p.blocks - 1) / p.blocks);
    const int held = static_cast<int>(std::min<int64_t>(tokens, int64_t{p.blocks} * each));
    // Chunks whose digits LDS holds at once. (Four more waves of the slices' form bring their own 5.5 to 6.5 KB each on
    // top: at most 87 KB of a workgroup, 103 with four digits, of 160.)
    const size_t fixed = lds_bytes(4, held, digits, p.blocks, groups, 0), each_chunk = lds_bytes(4, held, digits, p.blocks, groups, 1) - fixed;
    const int most = static_cast<int>(std::min<int64_t>(chunks, std::max<int64_t>(1, static_cast<int64_t>((budget - std::min(fixed, budget)) / each_chunk))));
    p.slices = 1;
    p.waves = 4;
    p.share = tiles * p.passes >= 2048 ? 1 : 4;
    if (most < chunks && tiles * p.passes < 2048) {
        // Digits that LDS does not hold at once, and few tiles: slices.
        p.share = 1;
        p.waves = p.blocks == 6 ? 8 : 4;
        const int64_t want = (2048 + tiles * p.passes - 1) / (tiles * p.passes);
        p.slices = static_cast<int>(std::min<int64_t>({16, chunks, std::max<int64_t>(want, 1)}));
    }
    p.slice = static_cast<int>((chunks + p.slices - 1) / p.slices);
    p.slices = static_cast<int>((chunks + p.slice - 1) / p.slice);
    const int stages = (p.slice + most - 1) / most;
    p.stage = (p.slice + stages - 1) / stages;
    const int64_t per = p.waves / p.share, all = (tiles + per - 1) / per;
    // Digits made once serve several tiles.
    p.groups = stages == 1 ? std::min<int64_t>(all, std::max<int64_t>(1, 768 / (int64_t{p.passes} * p.slices))) : all;
    return p;
}

template <int G, int NB, int ST, int DG, int WV>
int launch_on(const Int4Args& a, const Int4Plan& p, hipStream_t stream) {
    using S = Shape<G, DG>;
    const int held = std::min(a.tokens, NB * S::kTokens);
    const dim3 grid(static_cast<unsigned>(p.groups), static_cast<unsigned>(p.slices), static_cast<unsigned>(p.passes));
    hipLaunchKernelGGL((k_int4_product<G, NB, ST, WV, DG>), grid, dim3(WV * kWave), lds_bytes(WV, held, DG, NB, S::kGroups, a.stage),
                       stream, a);
    return nq::launch_status();
}

template <int G, int NB, int ST, int DG>
int launch_as(const Int4Args& a, const Int4Plan& p, hipStream_t stream) {
    if constexpr (NB == 6) {
        if (p.waves == 8) return launch_on<G, NB, ST, DG, 8>(a, p, stream);
    }
    return launch_on<G, NB, ST, DG, 4>(a, p, stream);
}

template <int G, int NB, int DG>
int launch_with(const Int4Args& a, const Int4Plan& p, int scale_dtype, hipStream_t stream) {
    switch (scale_dtype) {
        case NQ_DTYPE_F32: return launch_as<G, NB, NQ_DTYPE_F32, DG>(a, p, stream);
        case NQ_DTYPE_F16: return launch_as<G, NB, NQ_DTYPE_F16, DG>(a, p, stream);
        default: return launch_as<G, NB, NQ_DTYPE_BF16, DG>(a, p, stream);
    }
}

template <int G, int DG>
int launch_blocks(const Int4Args& a, const Int4Plan& p, int scale_dtype, hipStream_t stream) {
    switch (p.blocks) {
        case 1: return launch_with<G, 1, DG>(a, p, scale_dtype, stream);
        case 2: return launch_with<G, 2, DG>(a, p, scale_dtype, stream);
        case 3: return launch_with<G, 3, DG>(a, p, scale_dtype, stream);
        default: return launch_with<G, 6, DG>(a, p, scale_dtype, stream);
    }
}

template <int G>
int launch_for(const Int4Args& a, const Int4Plan& p, int scale_dtype, hipStream_t stream) {
    return digits_for(a.x_dtype) == 4 ? launch_blocks<G, 4>(a, p, scale_dtype, stream)
                                      : launch_blocks<G, 3>(a, p, scale_dtype, stream);
}

}  // namespace

extern "C" int64_t nq_int4_projection_workspace_bytes(int64_t tokens, int64_t out_features, int64_t in_features, int32_t group) {
    if (tokens <= 0 || tokens > 65535 || out_features <= 0 || out_features > 0x7fffffff || in_features <= 0 || in_features % 32 ||
        in_features > (1 << 24) || (group != 32 && group != 64 && group != 128))
        return -1;
    int64_t most = 0;
    for (const int digits : {3, 4}) {  // whatever the type of x
        const Int4Plan p = plan_int4(tokens, out_features, in_features, group, digits);
        if (!nq::launchable(p.groups * p.slices * p.passes, p.waves * kWave)) return -1;
        if (p.slices > 1) most = std::max(most, p.slices * tokens * out_features * static_cast<int64_t>(sizeof(float)));
    }
    return most;
}

extern "C" int64_t nq_int4_projection_partials(int64_t out_features) {
    return out_features <= 0 || out_features > 0x7fffffff ? -1 : (out_features + 15) / 16;
}

extern "C" int nq_int4_projection(const void* x, int32_t x_dtype, int64_t tokens, const void* packed, const void* scales,
                                  int32_t scale_dtype, const uint8_t* zeros, int64_t out_features, int64_t in_features,
                                  int32_t group, void* y, int32_t y_dtype, void* partials, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    if (!x || !packed || !scales || !y) return NQ_ERR_ARGUMENT;
    if (!nq::is_float_dtype(x_dtype) || !nq::is_float_dtype(scale_dtype) || !nq::is_float_dtype(y_dtype)) return NQ_ERR_DTYPE;
    const int64_t need = nq_int4_projection_workspace_bytes(tokens, out_features, in_features, group);
    if (need < 0 || (partials && tokens != 1)) return NQ_ERR_SHAPE;
    if (need > 0 && !workspace) return NQ_ERR_ARGUMENT;
    if (workspace_bytes < need) return NQ_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(workspace)) & 15) return NQ_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(partials) & 7) return NQ_ERR_ALIGNMENT;
    const Int4Plan p = plan_int4(tokens, out_features, in_features, group, digits_for(x_dtype));
    Int4Args a{};
    a.x = x;
    a.packed = static_cast<const uint8_t*>(packed);
    a.scales = scales;
    a.zeros = zeros;
    a.y = y;
    a.partial = p.slices > 1 ? static_cast<float*>(workspace) : nullptr;
    a.best = static_cast<uint64_t*>(partials);
    a.outs = out_features;
    a.ins = in_features;
    a.tiles = (out_features + 15) / 16;
    a.step = p.groups * (p.waves / p.share);
    a.tokens = static_cast<int32_t>(tokens);
    a.chunks = static_cast<int32_t>(chunks_of(in_features));
    a.groups = static_cast<int32_t>((in_features + group - 1) / group);
    a.x_dtype = x_dtype;
    a.y_dtype = y_dtype;
    a.share = p.share;
    a.slice = p.slice;
    a.stage = p.stage;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int status;
    switch (group) {
        case 32: status = launch_for<32>(a, p, scale_dtype, st); break;
        case 64: status = launch_for<64>(a, p, scale_dtype, st); break;
        default: status = launch_for<128>(a, p, scale_dtype, st); break;
    }
    if (status != NQ_OK || p.slices == 1) return status;
    const dim3 grid(static_cast<unsigned>((out_features + 255) / 256), static_cast<unsigned>(tokens));
    hipLaunchKernelGGL(k_int4_join, grid, dim3(256), 0, st, a, p.slices);
    return nq::launch_status();
}
