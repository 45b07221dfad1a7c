// Linear layers on a few rows with the weight in 4 bits, for gfx950:
//   w[n, k] = (code[n, k] - 8) scale[n, k / group],  y[m, n] = act_out(act_in(x)[m, k] . w[n, k]^T + bias[n]),  m <= 8
// two codes to a byte (even k in the low half), one scale in the storage type per group of 32, 64 or 128 of them.
#include "msd_device.h"
#include "msd_internal.h"

#include <algorithm>
#include <type_traits>

namespace msd {
namespace {

// ---------------------------------------------------------------------------
// Codes and scales of a weight: a = the largest finite |w| of a group, scale = a / 7 in the storage type,
// code = round(w / scale) clamped to +-7, plus 8.  A lane per byte, the lanes of a group beside each other: once for a weight, 16384 x
// 8192 float16 in 149 us, float32 in 154 (4.0 TB/s).
// ---------------------------------------------------------------------------
constexpr uint32_t kPackThreads = 256;
constexpr float kPackTiny = 1e-30f;  // groups below this are zeros (1 / scale would not be finite)

template <typename T, int GROUP>
__global__ __launch_bounds__(kPackThreads) void q4_pack_kernel(const T *w, uint8_t *packed, T *scales, size_t bytes) {
    constexpr int kLanes = GROUP / 2;
    const size_t step = (size_t)gridDim.x * kPackThreads;
    for (size_t i = (size_t)blockIdx.x * kPackThreads + threadIdx.x; i < bytes; i += step) {
        const float a = Store<T>::load1(w + 2 * i), b = Store<T>::load1(w + 2 * i + 1);  // (groups are whole: all of a team's lanes are here)
        const float fa = fabsf(a), fb = fabsf(b), inf = __builtin_huge_valf();
        const float most = team_max<kLanes>(fmaxf(fa < inf ? fa : 0.0f, fb < inf ? fb : 0.0f));
        const float scale = most < kPackTiny ? 0.0f : round_to_storage<T>(most / 7.0f);
        const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
        auto code = [inv](float v) {  // (a scale of 0: 8, of infinities and NaN too)
            return inv > 0.0f ? (uint32_t)((int)fminf(fmaxf(__builtin_rintf(v * inv), -7.0f), 7.0f) + 8) : 8u;
        };
        packed[i] = (uint8_t)(code(a) | code(b) << 4);
        if (threadIdx.x % kLanes == 0) Store<T>::store1(scales + i / kLanes, scale);
    }
}

// ---------------------------------------------------------------------------
// Any alignment: a wavefront per column, a lane per byte of its codes.  25 times the time of the kernel below (16384 x 8192, 8 rows
// float16: 539 us), for views that begin in the middle of 16 bytes and for k below 128 or above 2^22.
// ---------------------------------------------------------------------------
constexpr uint32_t kQ4Threads = 256;
constexpr size_t kQ4MaxBlocks = 0xFFFFFFFFu / 512;  // (a grid holds less than 2^32 lanes)

template <typename T>
__global__ __launch_bounds__(kQ4Threads) void linear_q4_generic_kernel(const T *x, const uint8_t *packed, const T *scales,
                                                                       const float *bias, T *y, uint32_t m, uint32_t n,
                                                                       uint32_t k, uint32_t group, int act_in, int act_out) {
    const uint32_t lane = threadIdx.x % kWave, step = gridDim.x * (kQ4Threads / kWave);
    for (uint32_t col = blockIdx.x * (kQ4Threads / kWave) + threadIdx.x / kWave; col < n; col += step) {
        const uint8_t *row = packed + (size_t)col * (k / 2);
        for (uint32_t i = 0; i < m; i++) {
            const T *xr = x + (size_t)i * k;
            float acc = 0.0f;
            for (uint32_t j = lane; j < k / 2; j += kWave) {
                float a = Store<T>::load1(xr + 2 * j), b = Store<T>::load1(xr + 2 * j + 1);
                if (act_in) {
                    a = silu_f(a);
                    b = silu_f(b);
                }
                const uint32_t codes = row[j];
                const float s = Store<T>::load1(scales + (size_t)col * (k / group) + 2 * j / group);
                acc = fmaf(a, (float)((int)(codes & 15) - 8) * s, acc);  // (a code times x could be infinite)
                acc = fmaf(b, (float)((int)(codes >> 4) - 8) * s, acc);
            }
            acc = wave_sum(acc);
            if (lane == 0) {
                float r = acc + (bias != nullptr ? bias[col] : 0.0f);
                if (act_out) r = silu_f(r);
                Store<T>::store1(y + (size_t)i * n + col, r);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// On the matrix cores.  A workgroup owns 16 CT columns, each of its wavefronts every W-th step of 128 of k; their sums meet in
// LDS at the end.  A wavefront brings its part of x to LDS itself and for itself: no barrier before that.
//
// v_mfma_f32_16x16x32_f16 multiplies 16 rows of x with 16 columns of weights, 32 of k at a time.  A code minus 8 is exact in
// float16, and so are the products and, to float32, their sums; the scale of a group multiplies the sum of its products, not
// the weights.  Of the 16 rows 8 are those of x; where x is float32, or activated, they hold its upper 11 bits and the other
// 8 rows, which would stand empty, the next 11, the 128 values of a row and step being brought to the range of float16 by a
// power of two.  What is left out of a value is at most 2^-23 of it, as two roundings of float32 would leave out, down to 2^-26 of the
// largest of the 128 (Q4Scale); what the float16 of smaller ones lack is found again behind the steps and summed up in float32.  The sums
// are closer than a float32 sum of k products (against 64 bits, k = 2048: 1.3e-7, torch's float32 product 4e-7).
//
// Weights: a lane loads 16 bytes, 32 of its column's weights; the four lanes of a column then swap 4-byte pieces so that each
// instruction gets 32 neighbouring ones, which never mix two scales.  Within a piece, codes come out in pairs (0, 4), (1, 5),
// (2, 6), (3, 7) by masks alone; x is laid out in LDS in that order.
//
// How k is dealt depends on k alone, so a row has the same bits for any CT, number of rows and company.
//
// What bounds it: codes and scales are read once, 69 MB at 16384 x 8192 in 21.7 us, 3.2 TB/s (half of what memory gives).  A
// wavefront there (two to a SIMD) issues an instruction in 23 % of its cycles, 40 % it waits for its requests, which are one step
// ahead, 37 % for the instruction before (each eight codes are nine instructions and an MFMA that wait for one another).  Neither
// side alone gives: sixteen wavefronts a workgroup 25.4 us against 23.1 (passes in a graph), workgroups that begin at different
// steps, so that not all are at the same channels of memory, 23.9.  Small calls are latency: 1280 x 1280, 1 row float16 3.6 us of
// 0.9 MB, 22 projections of 20160 x 1280, 2 rows float16 8.5, 8 rows float32 12.3.
// ---------------------------------------------------------------------------
constexpr int kMmMaxWaves = 8;
constexpr int kMmTile = 16;                   // columns of a tile
constexpr int kMmStep = 128;                  // of k
constexpr int kMmRows = 8;                    // most rows of x
constexpr int kMmEntries = kMmStep / 8;       // 16-byte pieces of a row and step in LDS
constexpr uint32_t kEights = 0x88888888u;     // codes of zeros

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Eight codes minus 8, as float16, in the order 0 4 1 5 2 6 3 7.  k1024: 0x64006400 in a vector register, so that each mask and
// the or behind it are one instruction (two constants of which one is in a scalar register).
__device__ __forceinline__ f16x8 q4_values(uint32_t w, uint32_t k1024) {
    const uint32_t v = w >> 8;
    auto low = [k1024](uint32_t u) {  // 1024 + code - 1032
        return __builtin_bit_cast(f16x2, (u & 0x000F000Fu) | k1024) - f16x2{1032.0f, 1032.0f};
    };
    auto high = [k1024](uint32_t u) {  // (1024 + 16 code) / 16 - 72
        return __builtin_bit_cast(f16x2, (u & 0x00F000F0u) | k1024) * f16x2{0.0625f, 0.0625f} - f16x2{72.0f, 72.0f};
    };
    const f16x2 a = low(w), b = high(w), c = low(v), d = high(v);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Piece j of row q of lanes <-> piece q of row j.
__device__ __forceinline__ void q4_transpose(u32x4 &v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    v = u32x4{c[0], c[1], d[0], d[1]};
}

// Two neighbouring values of a row of x, as they are in memory.
template <typename T>
struct XPair;
template <>
struct XPair<float> {
    float2 v = make_float2(0.0f, 0.0f);
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const float2 *>(p); }
    __device__ __forceinline__ float2 floats() const { return v; }
};
template <>
struct XPair<__half> {
    uint32_t v = 0;
    __device__ __forceinline__ void load(const __half *p) { v = *reinterpret_cast<const uint32_t *>(p); }
    __device__ __forceinline__ float2 floats() const {
        const f16x2 h = __builtin_bit_cast(f16x2, v);
        return make_float2(h[0], h[1]);
    }
};

// Between LDS accesses of some lanes of a wavefront and those of others to the same place: the hardware keeps their order, this
// makes the compiler keep it.  (Fences of the wavefront's scope and its barrier cost 3 % at 16384 x 8192, 8 rows float16: they end what
// can be scheduled together.)
__device__ __forceinline__ void lanes_in_step() { asm volatile("" ::: "memory"); }

struct Q4Layer {
    const uint8_t *packed;
    const void *scales;
    const float *bias;
    void *y;
    uint32_t n;
};

// What a wavefront requests for a step: the codes and scales of CT tiles, and PAIRS pairs of rows of x, 32 lanes a row, the values
// 0 1 4 5 (even lanes) or 2 3 6 7 of eight.  Everything stays as it came until it is used: a conversion would wait for it.
template <typename T, int NS, int CT, int PAIRS>
struct Q4Stage {
    u32x4 codes[CT];
    T scale[CT][NS];
    XPair<T> raw[PAIRS][2];
};

// Maximum over 32 lanes of values that are not less than zero, whose order is that of their bits: as floats, the compiler makes each of
// them canonical before it compares (22 instructions in place of 9).
__device__ __forceinline__ float half_wave_max(float v) {
    uint32_t u = __float_as_uint(v);
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, kDppXor1, 0xF, 0xF, true));
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, kDppXor2, 0xF, 0xF, true));
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, kDppHalfMirror, 0xF, 0xF, true));
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, kDppRowMirror, 0xF, 0xF, true));
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(max(r[0], r[1]));
}

// How a row's 128 values of a step become two float16 each, from the largest of them: times 2^(141 - exponent), which brings that to
// 2^14 ... 2^15.  From 2^26 times less on a value is off by 2^-23 of itself at most; below `smallest` the float16 run out of digits.
struct Q4Scale {
    float up, factor, smallest;  // factor: 1 / up, of which the products are multiples
    __device__ __forceinline__ explicit Q4Scale(float most) {
        constexpr uint32_t kBand = 26;
        const uint32_t exponent = max(__float_as_uint(most) >> 23, 20u);
        up = __uint_as_float((268u - exponent) << 23);
        factor = __uint_as_float((exponent - 14u) << 23);
        smallest = __uint_as_float((max(exponent, kBand) - kBand) << 23);
    }
    // of two values; lo times 2048
    __device__ __forceinline__ void split(float f, float g, f16x2 &hi, f16x2 &lo) const {
        hi = f16x2{(_Float16)(f * up), (_Float16)(g * up)};
        const float r = fmaf(f, up, -(float)hi[0]), s = fmaf(g, up, -(float)hi[1]);
        lo = f16x2{(_Float16)(r * 2048.0f), (_Float16)(s * 2048.0f)};
        lo = __builtin_elementwise_max(lo, f16x2{-16384.0f, -16384.0f});  // (never less than that; of an infinity: not NaN)
    }
    // what the two float16 of values below `smallest` lack of them (exactly: they have the upper digits), else 0
    __device__ __forceinline__ void lacks(float &f, float &g) const {
        f16x2 hi, lo;
        split(f, g, hi, lo);
        f = fabsf(f) < smallest ? f - fmaf((float)lo[0], 1.0f / 2048.0f, (float)hi[0]) * factor : 0.0f;
        g = fabsf(g) < smallest ? g - fmaf((float)lo[1], 1.0f / 2048.0f, (float)hi[1]) * factor : 0.0f;
    }
};

// What the two float16 of the smaller ones of a row's 128 values of a step lack, times a column's weights, in float32; x: the lane's 32 of
// them (`none`: of none).
template <typename T, int NS, int CT>
__device__ __forceinline__ void q4_small_values(const T *x, bool none, int act_in, const Q4Scale &to_halves, const uint8_t *packed,
                                                const uint32_t *code_at, const char *scales, const uint32_t *scale_at, float *sum) {
    auto value = [&](uint32_t e) {
        const float v = none ? 0.0f : Store<T>::load1(x + e);
        return act_in ? silu_f(v) : v;
    };
#pragma unroll
    for (int c = 0; c < CT; c++) sum[c] = 0.0f;
#pragma unroll 1
    for (uint32_t e0 = 0; e0 < 32; e0 += 8) {
        float f[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; e += 2) {
            f[e] = value(e0 + e);
            f[e + 1] = value(e0 + e + 1);
            to_halves.lacks(f[e], f[e + 1]);
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t codes = *reinterpret_cast<const uint32_t *>(packed + code_at[c] + e0 / 2);
            const float scale = Store<T>::load1(reinterpret_cast<const T *>(scales + scale_at[c]));
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) sum[c] = fmaf(f[e], (float)((int)((codes >> (4 * e)) & 15u) - 8) * scale, sum[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {  // of the four lanes of the column
        sum[c] += __shfl_xor(sum[c], 16);
        sum[c] += __shfl_xor(sum[c], 32);
    }
}

// SPLIT: two float16 for a value of x.  NS: scales per step (128 / group).  PAIRS: of rows of x that there is room for.
template <typename T, bool SPLIT, int NS, int CT, int PAIRS>
__device__ __forceinline__ void linear_q4_body(const T *x, const Q4Layer &layer, uint32_t col0, uint32_t m, uint32_t k, int act_in,
                                               int act_out) {
    extern __shared__ u32x4 lds[];  // per wavefront [kMmEntries][slots] of x and [kMmRows] factors
    constexpr int kGroup = kMmStep / NS, kAhead = CT == 4 || (NS == 4 && CT * PAIRS >= 4) ? 1 : 2;
    const uint32_t n = layer.n, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t waves = blockDim.x / kWave, i = lane % kMmTile, q = lane / kMmTile;
    const uint32_t groups = k / kGroup, steps = (k + kMmStep - 1) / kMmStep;
    const uint8_t *packed = layer.packed + (size_t)col0 * (k / 2);
    const char *scales = static_cast<const char *>(layer.scales) + (size_t)col0 * groups * sizeof(T);
    // offsets in bytes, of 32 bits from addresses that a wavefront shares: k is at most 2^22
    uint32_t code_at[CT], scale_at[CT];  // (columns past the last repeat it and are not stored)
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const uint32_t col = min(col0 + c * kMmTile + i, n - 1) - col0;
        code_at[c] = col * (k / 2) + q * 16;
        scale_at[c] = col * groups * sizeof(T);
    }
    const uint32_t half = lane / 32, tl = lane % 32;
    const uint32_t slots = SPLIT ? 2 * m : m;
    u32x4 *mine = lds + wave * (kMmEntries * slots + 2);
    float *factors = reinterpret_cast<float *>(mine + kMmEntries * slots);
    const uint32_t slot = SPLIT && i >= kMmRows ? m + min(i - kMmRows, m - 1) : min(i, m - 1);  // (rows past the last repeat it)

    const char *xs = reinterpret_cast<const char *>(x);
    uint32_t x_at[PAIRS];  // (rows past the last repeat it)
#pragma unroll
    for (int u = 0; u < PAIRS; u++) x_at[u] = (min(2 * u + half, m - 1) * k + tl / 2 * 8 + tl % 2 * 2) * (uint32_t)sizeof(T);
    typedef Q4Stage<T, NS, CT, PAIRS> Stage;
    // The last step begins where a whole one fits; what the step before it has had then counts as zeros.  Requests are made
    // without a branch and stay in this order: a value that is loaded on one path and not on another is copied where they meet,
    // which waits for the load, and a load that overtakes the next step's makes its use wait for those.
    auto start = [&](uint32_t step) { return min(step * kMmStep, k - kMmStep); };
    auto request = [&](Stage &to, uint32_t step) {
        const uint32_t at = start(step);
        __builtin_amdgcn_sched_barrier(0);
        const char *from = xs + (size_t)at * sizeof(T);
#pragma unroll
        for (int u = 0; u < PAIRS; u++) {
            to.raw[u][0].load(reinterpret_cast<const T *>(from + x_at[u]));
            to.raw[u][1].load(reinterpret_cast<const T *>(from + x_at[u]) + 4);
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            to.codes[c] = *reinterpret_cast<const u32x4 *>(packed + at / 2 + code_at[c]);
            const T *scale = reinterpret_cast<const T *>(scales + (size_t)(at / kGroup) * sizeof(T) + scale_at[c]);
#pragma unroll
            for (int j = 0; j < NS; j++) to.scale[c][j] = scale[j];
        }
        __builtin_amdgcn_sched_barrier(0);
        lanes_in_step();  // (what the step before left has been read)
    };
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    f32x4 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) acc[c] = f32x4{0, 0, 0, 0};
    uint64_t lost = 0;  // bit i: in the wavefront's steps i, i + 64, ... are values whose float16 lack digits
    uint32_t turn = 0;
    auto multiply = [&](Stage &from, uint32_t step) {
        const uint32_t had = step * kMmStep - start(step);  // values of the step that count as zeros
        uint2 *to = reinterpret_cast<uint2 *>(mine);
        uint64_t met = 0;  // lanes that have met such values
#pragma unroll
        for (int u = 0; u < PAIRS; u++) {
            if (2 * u >= (int)m) break;
            const uint32_t row = min(2 * u + half, m - 1), at = (tl / 2 * slots + row) * 2 + tl % 2;  // (an odd last row twice)
            const bool none = had != 0 && tl / 2 * 8 < had;
            if constexpr (SPLIT) {
                const float2 first = from.raw[u][0].floats(), second = from.raw[u][1].floats();
                float f[4] = {first.x, first.y, second.x, second.y};
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = none ? 0.0f : f[e];
                if (act_in) {
#pragma unroll
                    for (int e = 0; e < 4; e++) f[e] = silu_f(f[e]);
                }
                // (an infinity here leaves nothing but infinities and NaN of its row, which it gives whatever the others are)
                const float most = half_wave_max(fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3]))));
                const Q4Scale scale(most);
                uint32_t least = ~0u;  // of twice the bits less one, of which zeros have the largest
#pragma unroll
                for (int e = 0; e < 4; e++) least = min(least, (__float_as_uint(f[e]) << 1) - 1);
                f16x2 hi[2], lo[2];  // (0, 2) and (1, 3): the order of the codes
                scale.split(f[0], f[2], hi[0], lo[0]);
                scale.split(f[1], f[3], hi[1], lo[1]);
                met |= __ballot(least < __float_as_uint(scale.smallest) << 1);
                to[at] = make_uint2(__builtin_bit_cast(uint32_t, hi[0]), __builtin_bit_cast(uint32_t, hi[1]));
                to[at + 2 * m] = make_uint2(__builtin_bit_cast(uint32_t, lo[0]), __builtin_bit_cast(uint32_t, lo[1]));
                if (tl == 0) factors[row] = scale.factor;
            } else {
                const uint32_t v = __builtin_amdgcn_perm(from.raw[u][1].v, from.raw[u][0].v, 0x05040100u);
                const uint32_t w = __builtin_amdgcn_perm(from.raw[u][1].v, from.raw[u][0].v, 0x07060302u);
                to[at] = none ? make_uint2(0, 0) : make_uint2(v, w);
            }
        }
        lost |= (uint64_t)(met != 0) << (turn++ % 64);
        lanes_in_step();
        f16x8 a[4];
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = __builtin_bit_cast(f16x8, mine[(j * 4 + q) * slots + slot]);
        f32x4 factor = {1, 1, 1, 1};
        if (SPLIT) {
            factor = *reinterpret_cast<const f32x4 *>(factors + 4 * (q & 1));
            factor *= q < 2 ? 1.0f : 1.0f / 2048.0f;
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            if (had != 0) from.codes[c] = q * 32 < had ? u32x4{kEights, kEights, kEights, kEights} : from.codes[c];
            q4_transpose(from.codes[c]);
            f32x4 sum = SPLIT ? f32x4{0, 0, 0, 0} : acc[c];
#pragma unroll
            for (int s = 0; s < NS; s++) {
                f32x4 d = {0, 0, 0, 0};
#pragma unroll
                for (int j = s * (4 / NS); j < (s + 1) * (4 / NS); j++)
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], q4_values(from.codes[c][j], k1024), d, 0, 0, 0);
                const float scale = Store<T>::load1(&from.scale[c][s]);
#pragma unroll
                for (int r = 0; r < 4; r++) sum[r] = fmaf(d[r], scale, sum[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) acc[c][r] = SPLIT ? fmaf(sum[r], factor[r], acc[c][r]) : sum[r];
        }
    };

    Stage stage[kAhead];
    const uint32_t last = steps - 1;
#pragma unroll
    for (int d = 0; d < kAhead; d++) request(stage[d], min(wave + d * waves, last));
    for (uint32_t first = wave; first < steps; first += kAhead * waves) {
#pragma unroll
        for (int d = 0; d < kAhead; d++) {
            const uint32_t step = first + d * waves;
            if (step < steps) multiply(stage[d], step);
            request(stage[d], min(step + kAhead * waves, last));  // (past the end: what is in the cache)
        }
    }

    if constexpr (SPLIT) {
        // Rarely: steps once more, for the rows that have such values there (16384 x 8192, 8 rows float32: 2.7 us more for one value, and
        // 379 in place of 28 where every row has them in every step).
        turn = 0;
        for (uint32_t step = wave; lost != 0 && step < steps; step += waves) {
            if ((lost >> (turn++ % 64) & 1) == 0) continue;
            const uint32_t at = start(step), had = step * kMmStep - at;
            for (uint32_t row = 0; row < m; row++) {
                XPair<T> raw;
                raw.load(x + (size_t)row * k + at + 2 * lane);
                float2 f = 2 * lane < had ? make_float2(0.0f, 0.0f) : raw.floats();
                if (act_in) f = make_float2(silu_f(f.x), silu_f(f.y));
                const float most = half_wave_max(fmaxf(fabsf(f.x), fabsf(f.y)));
                const Q4Scale to_halves(fmaxf(most, __shfl_xor(most, 32)));
                auto small = [&](float v) { return v != 0.0f && fabsf(v) < to_halves.smallest; };
                if (__ballot(small(f.x) || small(f.y)) == 0) continue;
                float sum[CT];
                q4_small_values<T, NS, CT>(x + (size_t)row * k + at + q * 32, q * 32 < had, act_in, to_halves, packed + at / 2, code_at,
                                           scales + (size_t)(at / kGroup + q * 32 / kGroup) * sizeof(T), scale_at, sum);
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) acc[c][r] += row == 4 * q + r ? sum[c] : 0.0f;
            }
        }
    }

    // the wavefronts' sums; a lane has column i of rows 4 q ... 4 q + 3, of the upper (q < 2) or the lower parts
    f32x4 *parts = reinterpret_cast<f32x4 *>(lds);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; c++) parts[(wave * CT + c) * kWave + lane] = acc[c];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < kMmTile * CT * m; o += blockDim.x) {
        const uint32_t tile = o % (kMmTile * CT), row = o / (kMmTile * CT), col = col0 + tile;
        if (col >= n) continue;
        const float *at = reinterpret_cast<const float *>(parts + tile / kMmTile * kWave + row / 4 * kMmTile + tile % kMmTile) + row % 4;
        float sum = 0.0f;
#pragma unroll 4
        for (uint32_t w = 0; w < waves; w++) {
            sum += at[w * CT * kWave * 4];
            if (SPLIT) sum += at[(w * CT * kWave + 2 * kMmTile) * 4];
        }
        sum += layer.bias != nullptr ? layer.bias[col] : 0.0f;
        if (act_out) sum = silu_f(sum);
        Store<T>::store1(static_cast<T *>(layer.y) + (size_t)row * n + col, sum);
    }
}

template <typename T, bool SPLIT, int NS, int CT, int PAIRS>
__global__ __launch_bounds__(kMmMaxWaves *kWave, 4) void linear_q4_kernel(const T *x, const uint8_t *packed, const T *scales, uint32_t k,
                                                                       uint32_t n, uint32_t m, int act_in, int act_out,
                                                                       const float *bias, T *y) {
    linear_q4_body<T, SPLIT, NS, CT, PAIRS>(x, Q4Layer{packed, scales, bias, y, n}, blockIdx.x * (kMmTile * CT), m, k, act_in, act_out);
}

// Several layers in one launch: the workgroups are laid end to end, and a wavefront finds its layer with one load of all
// layers' first workgroups, a lane each.
constexpr int kQ4GroupMax = 32;  // layers per launch
struct Q4Layers {
    uint32_t first_block[kQ4GroupMax + 1];  // first_block[count ...] = number of workgroups
    Q4Layer layer[kQ4GroupMax];
};

template <typename T, bool SPLIT, int NS, int CT, int PAIRS>
__global__ __launch_bounds__(kMmMaxWaves *kWave, 4) void linear_q4_grouped_kernel(const T *x, uint32_t k, uint32_t m, int act_in,
                                                                               int act_out, Q4Layers layers) {
    const uint32_t next = layers.first_block[min(threadIdx.x % kWave + 1, (uint32_t)kQ4GroupMax)];
    const uint32_t p = min((uint32_t)__popcll(__ballot(blockIdx.x >= next)), (uint32_t)kQ4GroupMax - 1);
    const uint32_t at = __builtin_amdgcn_readfirstlane(p);
    linear_q4_body<T, SPLIT, NS, CT, PAIRS>(x, layers.layer[at], (blockIdx.x - layers.first_block[at]) * (kMmTile * CT), m, k, act_in, act_out);
}

struct Q4Launch {
    uint32_t m, k, waves;
    int act_in, act_out;
    hipStream_t stream;
};

template <typename T, bool SPLIT, int NS, int CT, int PAIRS>
void launch_q4(const T *x, const Q4Layers &layers, uint32_t count, const Q4Launch &a) {
    const size_t rows = (kMmEntries * (SPLIT ? 2 : 1) * a.m + 2) * sizeof(u32x4);
    const size_t lds = a.waves * std::max<size_t>(rows, CT * kWave * sizeof(f32x4));
    const dim3 grid(layers.first_block[kQ4GroupMax]), block(a.waves * kWave);
    const Q4Layer &l = layers.layer[0];
    if (count == 1)
        launch(linear_q4_kernel<T, SPLIT, NS, CT, PAIRS>, grid, block, lds, a.stream, x, l.packed, static_cast<const T *>(l.scales), a.k, l.n,
               a.m, a.act_in, a.act_out, l.bias, static_cast<T *>(l.y));
    else
        launch(linear_q4_grouped_kernel<T, SPLIT, NS, CT, PAIRS>, grid, block, lds, a.stream, x, a.k, a.m, a.act_in, a.act_out, layers);
}

template <typename T, bool SPLIT>
void launch_q4_group(const T *x, const Q4Layers &layers, uint32_t count, uint32_t group, int ct, const Q4Launch &a) {
    auto with_pairs = [&](auto ns, auto tiles) {
        if (a.m <= 2) launch_q4<T, SPLIT, ns.value, tiles.value, 1>(x, layers, count, a);
        else launch_q4<T, SPLIT, ns.value, tiles.value, kMmRows / 2>(x, layers, count, a);
    };
    auto with_tiles = [&](auto ns) {
        if (ct == 1) with_pairs(ns, std::integral_constant<int, 1>{});
        else if (ct == 2) with_pairs(ns, std::integral_constant<int, 2>{});
        else with_pairs(ns, std::integral_constant<int, 4>{});
    };
    if (group == 32) with_tiles(std::integral_constant<int, 4>{});
    else if (group == 64) with_tiles(std::integral_constant<int, 2>{});
    else with_tiles(std::integral_constant<int, 1>{});
}

}  // namespace

template <typename T>
int q4_pack_dispatch(const void *w, uint8_t *packed, void *scales, size_t n, size_t k, size_t group, hipStream_t stream) {
    const size_t bytes = n * (k / 2);
    if (bytes == 0) return MSD_OK;
    const dim3 grid((uint32_t)std::min<size_t>(16384, (bytes + kPackThreads - 1) / kPackThreads));
    const T *in = static_cast<const T *>(w);
    T *s = static_cast<T *>(scales);
    if (group == 32) launch(q4_pack_kernel<T, 32>, grid, dim3(kPackThreads), 0, stream, in, packed, s, bytes);
    else if (group == 64) launch(q4_pack_kernel<T, 64>, grid, dim3(kPackThreads), 0, stream, in, packed, s, bytes);
    else launch(q4_pack_kernel<T, 128>, grid, dim3(kPackThreads), 0, stream, in, packed, s, bytes);
    return launch_status();
}
template int q4_pack_dispatch<float>(const void *, uint8_t *, void *, size_t, size_t, size_t, hipStream_t);
template int q4_pack_dispatch<__half>(const void *, uint8_t *, void *, size_t, size_t, size_t, hipStream_t);

template <typename T>
int linear_q4_dispatch(const void *x, const uint8_t *const *packed, const void *const *scales, const float *const *biases,
                       void *const *ys, const size_t *ns, size_t count, size_t m, size_t k, size_t group, int act_in, int act_out,
                       hipStream_t stream) {
    if (m == 0) return MSD_OK;
    const T *rows = static_cast<const T *>(x);
    auto bias_of = [&](size_t i) { return biases != nullptr ? biases[i] : nullptr; };
    // Each layer by its own alignment, so that its bits and its time are the same whatever layers come with it.
    const bool fast_rows = aligned16(x) && k >= kMmStep && k <= (size_t)1 << 22;  // (offsets within a workgroup's columns: 32 bits)
    auto fast = [&](size_t i) { return ns[i] != 0 && fast_rows && aligned16(packed[i]); };
    size_t tiles = 0;
    for (size_t i = 0; i < count; i++) tiles += fast(i) ? (ns[i] + kMmTile - 1) / kMmTile : 0;
    // Wavefronts: as many as share the steps evenly, eight at most, so that several workgroups share a CU.  Tiles per workgroup: more
    // of them share the work on x, as long as 160 workgroups are left; of one or two rows that work is little.  us, one tile / two /
    // four, fp16, k = 1280: 2560 columns, 1 row 2.5 3.0 3.9, 8 rows 3.2 3.8 4.6; 5120, 8 rows 3.9 3.5 4.8; 10240, 1 row 3.8 4.1 4.0,
    // 8 rows 6.0 5.7 4.8; 20160, 2 rows 6.4 6.2 6.5, 8 rows 9.1 7.9 7.3; 8192 x 8192, 1 row 11.0 9.9 14.9; 16384 x 512 3.9 3.6 2.9.
    const size_t steps = (k + kMmStep - 1) / kMmStep, rounds = (steps + kMmMaxWaves - 1) / kMmMaxWaves, waves = (steps + rounds - 1) / rounds;
    const int ct = tiles < 320 ? 1 : (m > 2 ? tiles >= 640 : tiles >= 1024 && waves <= 4) ? 4 : 2;
    const Q4Launch a = {(uint32_t)m, (uint32_t)k, (uint32_t)waves, act_in, act_out, stream};
    const size_t columns = (size_t)kMmTile * ct;
    auto blocks_of = [&](size_t i) { return (ns[i] + columns - 1) / columns; };
    for (size_t i = 0; i < count; i++)
        if (fast(i) && blocks_of(i) > kQ4MaxBlocks) return MSD_ERR_INVALID_VALUE;
    Q4Layers layers{};
    uint32_t held = 0;
    auto send = [&] {
        if (held == 0) return;
        if (sizeof(T) == 4 || act_in) launch_q4_group<T, true>(rows, layers, held, (uint32_t)group, ct, a);
        else if constexpr (sizeof(T) == 2) launch_q4_group<T, false>(rows, layers, held, (uint32_t)group, ct, a);
        layers = Q4Layers{};
        held = 0;
    };
    for (size_t i = 0; i < count; i++) {
        if (ns[i] == 0) continue;
        if (!fast(i)) {
            launch(linear_q4_generic_kernel<T>, dim3((uint32_t)std::min<size_t>(kQ4MaxBlocks, (ns[i] + kQ4Threads / kWave - 1) / (kQ4Threads / kWave))),
                   dim3(kQ4Threads), 0, stream, rows, packed[i], static_cast<const T *>(scales[i]), bias_of(i),
                   static_cast<T *>(ys[i]), (uint32_t)m, (uint32_t)ns[i], (uint32_t)k, (uint32_t)group, act_in, act_out);
            continue;
        }
        if (held == kQ4GroupMax || layers.first_block[held] + blocks_of(i) > kQ4MaxBlocks) send();
        const uint32_t blocks = layers.first_block[held] + (uint32_t)blocks_of(i);
        layers.layer[held++] = {packed[i], scales[i], bias_of(i), ys[i], (uint32_t)ns[i]};
        for (uint32_t j = held; j <= kQ4GroupMax; j++) layers.first_block[j] = blocks;
    }
    send();
    return launch_status();
}
template int linear_q4_dispatch<float>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                       const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);
template int linear_q4_dispatch<__half>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                        const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);

}  // namespace msd
