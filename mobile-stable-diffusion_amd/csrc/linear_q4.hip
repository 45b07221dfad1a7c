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
// code = round(w / scale) clamped to +-7, plus 8.  A lane per byte, the lanes of a group beside each other.
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
        auto code = [inv](float v) { return (uint32_t)((int)fminf(fmaxf(__builtin_rintf(v * inv), -7.0f), 7.0f) + 8); };
        packed[i] = (uint8_t)(code(a) | code(b) << 4);
        if (threadIdx.x % kLanes == 0) Store<T>::store1(scales + i / kLanes, scale);
    }
}

// ---------------------------------------------------------------------------
// Any alignment: a wavefront per column, a lane per byte of its codes.
// ---------------------------------------------------------------------------
constexpr uint32_t kQ4Threads = 256;

template <typename T>
__global__ __launch_bounds__(kQ4Threads) void linear_q4_generic_kernel(const T *x, const uint8_t *packed, const T *scales,
                                                                       const float *bias, T *y, uint32_t m, uint32_t n,
                                                                       uint32_t k, uint32_t group, int act_in, int act_out) {
    const uint32_t lane = threadIdx.x % kWave, col = blockIdx.x * (kQ4Threads / kWave) + threadIdx.x / kWave;
    if (col >= n) return;
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

// ---------------------------------------------------------------------------
// On the matrix cores.  A workgroup of eight wavefronts owns 16 CT columns and walks k in chunks of eight steps of 128, a step
// per wavefront, so that the weights of a chunk are in flight together and a row of x is read once per workgroup.
//
// v_mfma_f32_16x16x32_f16 multiplies 16 rows of x with 16 columns of weights, 32 of k at a time.  A code minus 8 is exact in
// float16, and so are the products and, to float32, their sums; the scale of a group multiplies the sum of its products, not
// the weights.  Of the 16 rows 8 are those of x; where x is float32, or activated, they hold its upper 11 bits and the other
// 8 rows, which would stand empty, the next 11: with the 128 values of a row and step brought to the same range by a power
// of two, no bit of float32 that matters is lost, at the price of the same instructions.
//
// Weights: a lane loads 16 bytes, 32 of its column's weights; the four lanes of a column then swap 4-byte pieces so that each
// instruction gets 32 neighbouring ones, which never mix two scales.  Within a piece, codes come out in pairs (0, 4), (1, 5),
// (2, 6), (3, 7) by masks alone; x is laid out in LDS in that order.
// ---------------------------------------------------------------------------
constexpr int kMmWaves = 8;
constexpr int kMmThreads = kMmWaves * kWave;
constexpr int kMmTile = 16;                   // columns of a tile
constexpr int kMmStep = 128;                  // of k, per wavefront and chunk
constexpr int kMmRows = 8;                    // most rows of x
constexpr int kMmUnits = kMmRows * kMmWaves / (kMmThreads / 32);  // (row, step) pairs a team of 32 lanes brings to LDS
constexpr int kMmEntries = kMmStep / 8;       // 16-byte pieces of a row and step in LDS
constexpr uint32_t kEights = 0x88888888u;     // codes of zeros

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kQ4GroupMax = 32;  // layers per launch
template <int N>
struct Q4Layers {
    const uint8_t *packed[N];
    const void *scales[N];
    const float *bias[N];
    void *y[N];
    uint32_t n[N];
    uint32_t first_block[N + 1];  // first_block[count] = number of workgroups
    uint32_t count;
};

// Eight codes minus 8, as float16, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ f16x8 q4_values(uint32_t w) {
    const uint32_t v = w >> 8;
    auto low = [](uint32_t u) {  // 1024 + code - 1032
        return __builtin_bit_cast(f16x2, (u & 0x000F000Fu) | 0x64006400u) - f16x2{1032.0f, 1032.0f};
    };
    auto high = [](uint32_t u) {  // (1024 + 16 code) / 16 - 72
        return __builtin_bit_cast(f16x2, (u & 0x00F000F0u) | 0x64006400u) * f16x2{0.0625f, 0.0625f} - f16x2{72.0f, 72.0f};
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

template <typename T>
struct XPiece;  // four neighbouring values of a row of x
template <>
struct XPiece<float> {
    u32x4 v;
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const u32x4 *>(p); }
    __device__ __forceinline__ void floats(float *f) const { Store<float>::unpack(v, f); }
};
template <>
struct XPiece<__half> {
    uint2 v;
    __device__ __forceinline__ void load(const __half *p) { v = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void floats(float *f) const {
        const f16x2 a = __builtin_bit_cast(f16x2, v.x), b = __builtin_bit_cast(f16x2, v.y);
        f[0] = a[0];
        f[1] = a[1];
        f[2] = b[0];
        f[3] = b[1];
    }
};

__device__ __forceinline__ uint32_t half_bits(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ uint32_t dpp_xor1(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor1, 0xF, 0xF, true);
}

// SPLIT: two float16 for a value of x.  NS: scales per step (128 / group).
template <typename T, bool SPLIT, int NS, int CT, int N>
__global__ __launch_bounds__(kMmThreads) void linear_q4_kernel(const T *x, Q4Layers<N> layers, uint32_t m, uint32_t k, int act_in,
                                                               int act_out) {
    extern __shared__ u32x4 lds[];  // [2][kMmWaves][kMmEntries][slots] of x, then [2][kMmWaves][kMmRows] factors
    uint32_t p = 0;
    while (N > 1 && p + 1 < layers.count && blockIdx.x >= layers.first_block[p + 1]) p++;  // uniform: scalar loop
    const uint8_t *packed = layers.packed[p];
    const T *scales = static_cast<const T *>(layers.scales[p]);
    const uint32_t n = layers.n[p], col0 = (blockIdx.x - (N > 1 ? layers.first_block[p] : 0)) * (kMmTile * CT);
    const uint32_t lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t i = lane % kMmTile, q = lane / kMmTile;
    const uint32_t groups = k / (kMmStep / NS), chunks = (k + kMmWaves * kMmStep - 1) / (kMmWaves * kMmStep);
    const uint32_t slots = SPLIT ? 2 * m : m, buffer = kMmWaves * kMmEntries * slots;
    float *factors = reinterpret_cast<float *>(lds + 2 * buffer);

    u32x4 codes[CT], next[CT];
    float scale[CT][NS], next_scale[CT][NS];
    auto request = [&](uint32_t chunk, u32x4 *to, float (*s)[NS]) {
        const uint32_t step = chunk * kMmWaves + wave, at = step * kMmStep + q * 32;
#pragma unroll
        for (int c = 0; c < CT; c++) {  // (columns past the last repeat it and are not stored)
            const uint32_t col = min(col0 + c * kMmTile + i, n - 1);
            to[c] = u32x4{kEights, kEights, kEights, kEights};
            if (at < k) to[c] = load_stream(reinterpret_cast<const u32x4 *>(packed + (size_t)col * (k / 2) + at / 2));
#pragma unroll
            for (int j = 0; j < NS; j++) s[c][j] = Store<T>::load1(scales + (size_t)col * groups + min(step * NS + j, groups - 1));
        }
    };
    // x: a team of 32 lanes per (row, step), four values a lane
    const uint32_t team = threadIdx.x / 32, tl = threadIdx.x % 32;
    XPiece<T> raw[kMmUnits];
    auto request_x = [&](uint32_t chunk) {
#pragma unroll
        for (int u = 0; u < kMmUnits; u++) {
            const uint32_t unit = u * (kMmThreads / 32) + team, row = unit / kMmWaves, step = chunk * kMmWaves + unit % kMmWaves;
            const uint32_t at = step * kMmStep + tl * 4;
            raw[u] = XPiece<T>{};
            if (row < m && at < k) raw[u].load(x + (size_t)row * k + at);
        }
    };
    auto place_x = [&](uint32_t chunk) {
        uint2 *to = reinterpret_cast<uint2 *>(lds + (chunk & 1) * buffer);
#pragma unroll
        for (int u = 0; u < kMmUnits; u++) {
            const uint32_t unit = u * (kMmThreads / 32) + team, row = unit / kMmWaves, step = unit % kMmWaves;
            if (row >= m) continue;  // (the same for a team, whose lanes alone meet below)
            float f[4];
            raw[u].floats(f);
            uint32_t v[4];  // the upper float16 in the low half
            if (SPLIT) {
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (act_in) f[e] = silu_f(f[e]);
                    const float a = fabsf(f[e]);
                    most = fmaxf(most, a < __builtin_huge_valf() ? a : 0.0f);
                }
                most = team_max<32>(most);
                const uint32_t exponent = max(__float_as_uint(most) >> 23, 20u);  // most * 2^(141 - exponent) < 2^15
                const float up = __uint_as_float((268u - exponent) << 23);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float s = f[e] * up;
                    const _Float16 hi = (_Float16)s;
                    const float rest = (s - (float)hi) * 2048.0f;
                    v[e] = half_bits(s) | (fabsf(s) < __builtin_huge_valf() ? half_bits(rest) << 16 : 0u);
                }
                if (tl == 0) factors[((chunk & 1) * kMmWaves + step) * kMmRows + row] = __uint_as_float((exponent - 14u) << 23);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = half_bits(f[e]);
            }
            // values 0 - 3 of eight are in the even lane, 4 - 7 in the odd one; each stores two of the four pairs
            const bool odd = tl & 1;
            const uint32_t r0 = dpp_xor1(odd ? v[0] : v[2]), r1 = dpp_xor1(odd ? v[1] : v[3]);
            const uint32_t a0 = odd ? r0 : v[0], b0 = odd ? v[2] : r0, a1 = odd ? r1 : v[1], b1 = odd ? v[3] : r1;
            const uint32_t entry = step * kMmEntries + tl / 2;
            to[(entry * slots + row) * 2 + odd] = make_uint2((a0 & 0xFFFFu) | b0 << 16, (a1 & 0xFFFFu) | b1 << 16);
            if (SPLIT) to[(entry * slots + m + row) * 2 + odd] = make_uint2(a0 >> 16 | (b0 & 0xFFFF0000u), a1 >> 16 | (b1 & 0xFFFF0000u));
        }
    };

    f32x4 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) acc[c] = f32x4{0, 0, 0, 0};
    const bool has_row = i % kMmRows < m && (SPLIT || i < kMmRows);
    const uint32_t slot = i < kMmRows ? i : m + i - kMmRows;
    request(0, codes, scale);
    request_x(0);
    place_x(0);
    __syncthreads();
    for (uint32_t chunk = 0; chunk < chunks; chunk++) {
        const bool more = chunk + 1 < chunks;
        if (more) {
            request(chunk + 1, next, next_scale);
            request_x(chunk + 1);
        }
        if ((chunk * kMmWaves + wave) * kMmStep < k) {
            f16x8 a[4];
            const u32x4 *from = lds + (chunk & 1) * buffer + wave * kMmEntries * slots;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u32x4 zero = {0, 0, 0, 0};
                a[j] = __builtin_bit_cast(f16x8, has_row ? from[(j * 4 + q) * slots + slot] : zero);
            }
            f32x4 factor = {1, 1, 1, 1};
            if (SPLIT) {
                factor = *reinterpret_cast<const f32x4 *>(factors + ((chunk & 1) * kMmWaves + wave) * kMmRows + 4 * (q & 1));
                factor *= q < 2 ? 1.0f : 1.0f / 2048.0f;
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                q4_transpose(codes[c]);
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    f32x4 d = {0, 0, 0, 0};
#pragma unroll
                    for (int j = s * (4 / NS); j < (s + 1) * (4 / NS); j++)
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], q4_values(codes[c][j]), d, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        acc[c][r] = SPLIT ? fmaf(d[r] * scale[c][s], factor[r], acc[c][r]) : fmaf(d[r], scale[c][s], acc[c][r]);
                }
            }
        }
        if (more) {
            place_x(chunk + 1);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                codes[c] = next[c];
#pragma unroll
                for (int s = 0; s < NS; s++) scale[c][s] = next_scale[c][s];
            }
        }
        __syncthreads();
    }

    // the wavefronts' sums meet in LDS; a lane has column i of rows 4 q ... 4 q + 3, of the upper (q < 2) or the lower parts
    f32x4 *parts = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int c = 0; c < CT; c++) parts[(wave * CT + c) * kWave + lane] = acc[c];
    __syncthreads();
    const uint32_t tile = threadIdx.x % (kMmTile * CT), row = threadIdx.x / (kMmTile * CT), col = col0 + tile;
    if (row >= m || col >= n) return;
    const float *at = reinterpret_cast<const float *>(parts + tile / kMmTile * kWave + row / 4 * kMmTile + tile % kMmTile) + row % 4;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kMmWaves; w++) {
        sum += at[w * CT * kWave * 4];
        if (SPLIT) sum += at[(w * CT * kWave + 2 * kMmTile) * 4];
    }
    const float *bias = layers.bias[p];
    sum += bias != nullptr ? bias[col] : 0.0f;
    if (act_out) sum = silu_f(sum);
    Store<T>::store1(static_cast<T *>(layers.y[p]) + (size_t)row * n + col, sum);
}

// One launch for at most N layers.
template <typename T, bool SPLIT, int NS, int CT, int N>
void launch_q4(const T *x, const Q4Layers<N> &layers, uint32_t m, uint32_t k, int act_in, int act_out, hipStream_t stream) {
    const uint32_t slots = SPLIT ? 2 * m : m;
    const size_t rows = 2 * kMmWaves * (kMmEntries * slots * sizeof(u32x4) + kMmRows * sizeof(float));
    launch(linear_q4_kernel<T, SPLIT, NS, CT, N>, dim3(layers.first_block[layers.count]), dim3(kMmThreads),
           std::max<size_t>(rows, kMmWaves * CT * kWave * sizeof(f32x4)), stream, x, layers, m, k, act_in, act_out);
}

template <typename T, bool SPLIT, int N>
void launch_q4_group(const T *x, const Q4Layers<N> &layers, uint32_t m, uint32_t k, uint32_t group, int ct, int act_in, int act_out,
                     hipStream_t stream) {
    auto with_ns = [&](auto ns) {
        if (ct == 1) launch_q4<T, SPLIT, ns.value, 1, N>(x, layers, m, k, act_in, act_out, stream);
        else if (ct == 2) launch_q4<T, SPLIT, ns.value, 2, N>(x, layers, m, k, act_in, act_out, stream);
        else launch_q4<T, SPLIT, ns.value, 4, N>(x, layers, m, k, act_in, act_out, stream);
    };
    if (group == 32) with_ns(std::integral_constant<int, 4>{});
    else if (group == 64) with_ns(std::integral_constant<int, 2>{});
    else with_ns(std::integral_constant<int, 1>{});
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
    size_t tiles = 0;
    bool aligned = aligned16(x) && k != 0;
    for (size_t i = 0; i < count; i++) {
        if (ns[i] == 0) continue;
        tiles += (ns[i] + kMmTile - 1) / kMmTile;
        aligned = aligned && aligned16(packed[i]);
    }
    if (!aligned) {
        for (size_t i = 0; i < count; i++)
            if (ns[i] != 0)
                launch(linear_q4_generic_kernel<T>, dim3((uint32_t)((ns[i] + kQ4Threads / kWave - 1) / (kQ4Threads / kWave))),
                       dim3(kQ4Threads), 0, stream, rows, packed[i], static_cast<const T *>(scales[i]), bias_of(i),
                       static_cast<T *>(ys[i]), (uint32_t)m, (uint32_t)ns[i], (uint32_t)k, (uint32_t)group, act_in, act_out);
        return launch_status();
    }
    const int ct = tiles >= 2048 ? 4 : tiles >= 1024 ? 2 : 1;
    auto run = [&](const auto &layers) {
        if constexpr (sizeof(T) == 4) {
            launch_q4_group<T, true>(rows, layers, (uint32_t)m, (uint32_t)k, (uint32_t)group, ct, act_in, act_out, stream);
        } else {
            if (act_in) launch_q4_group<T, true>(rows, layers, (uint32_t)m, (uint32_t)k, (uint32_t)group, ct, act_in, act_out, stream);
            else launch_q4_group<T, false>(rows, layers, (uint32_t)m, (uint32_t)k, (uint32_t)group, ct, act_in, act_out, stream);
        }
    };
    auto add = [&](auto &layers, size_t i) {
        const uint32_t at = layers.count++, columns = kMmTile * ct;
        layers.packed[at] = packed[i];
        layers.scales[at] = scales[i];
        layers.bias[at] = bias_of(i);
        layers.y[at] = ys[i];
        layers.n[at] = (uint32_t)ns[i];
        layers.first_block[at + 1] = layers.first_block[at] + ((uint32_t)ns[i] + columns - 1) / columns;
    };
    if (count == 1) {
        Q4Layers<1> one{};
        if (ns[0] != 0) {
            add(one, 0);
            run(one);
        }
        return launch_status();
    }
    Q4Layers<kQ4GroupMax> many{};
    for (size_t i = 0; i < count; i++) {
        if (ns[i] != 0) add(many, i);
        if (many.count == kQ4GroupMax || (i + 1 == count && many.count != 0)) {
            run(many);
            many = Q4Layers<kQ4GroupMax>{};
        }
    }
    return launch_status();
}
template int linear_q4_dispatch<float>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                       const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);
template int linear_q4_dispatch<__half>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                        const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);

}  // namespace msd
