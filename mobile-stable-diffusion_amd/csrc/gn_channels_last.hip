// GroupNorm over channels-last tensors for gfx950, its gradient, and the 8-bit copy of its input
// that the gradient can read instead of the input.
//
// x is [batch, P, C] with the channels next to each other (P positions), groups of C / G channels.
//   h = x (+ chunk[b, c], rounded to the storage type);  u = (h - mean) rstd;  z = gamma u + beta
//   y = z, or z / (1 + exp(-z))
// and with dz = dy (times the derivative of SiLU at z), S1[b, c] = sum_p dz, S2[b, c] = sum_p dz u,
// m1, m2 = the means over a group of gamma dz and gamma dz u:
//   dx = rstd (gamma dz - m1 - u m2);  dgamma = sum_b S2;  dbeta = sum_b S1
//   dchunk[b, c] = sum_p dx = rstd (gamma S1 - P m1 - m2 sum_p u)
//
// A group's statistics need all positions of a sample, so each direction is a pass of sums and a pass
// that applies them.  A workgroup owns `tx` columns (a column: VEC neighbouring channels, what a lane
// moves at once) of a slice of positions; its lanes lie along the columns first, so a wavefront reads
// whole rows one after the other, and a lane keeps its channels, whose constants stay in registers.
#include "msd_device.h"
#include "msd_internal.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <numeric>
#include <type_traits>

namespace msd {
namespace {

constexpr uint32_t kClThreads = 512;    // most lanes of a workgroup
constexpr uint32_t kClMaxTx = 320;      // most columns of a workgroup
constexpr uint32_t kClRows = 4;         // rows a lane requests before it uses the first
constexpr uint32_t kClMaxParts = 128;   // partial sums per group up to which every workgroup adds them up itself
constexpr uint32_t kClTeam = 16;        // lanes that add up a group
constexpr uint32_t kCodeBlock = 32;     // channels of one position that share a scale
constexpr float kCodeTiny = 1e-30f;     // blocks below this are kept as zeros (1 / a would not be finite)

struct ClPlan {
    uint32_t positions, channels, columns, groups;
    uint32_t tx, ty, chunks;            // columns and rows of a workgroup; workgroups along the columns
    uint32_t slices, rows;              // workgroups along the positions, positions of each (but the last)
    uint32_t spans;                     // most chunks that share one group
    FastDiv per_group, by_tx;
};

// What a workgroup is: sample, slice, chunk and its bounds.
struct ClTile {
    uint32_t b, slice, chunk, col0, cols, row0, rows, tx, ty;
    bool live;
    __device__ ClTile(const ClPlan &p, uint32_t block) {
        slice = block % p.slices;
        const uint32_t rest = block / p.slices;
        chunk = rest % p.chunks;
        b = rest / p.chunks;
        col0 = chunk * p.tx;
        cols = min(p.tx, p.columns - col0);
        row0 = slice * p.rows;
        rows = min(p.rows, p.positions - row0);
        ty = fast_div(threadIdx.x, p.by_tx);
        tx = threadIdx.x - ty * p.tx;
        live = ty < p.ty && tx < cols;
    }
};

// Groups that have channels in [c0, c1), and which of a group's chunks this is.
struct ClGroups {
    uint32_t first, count;
    __device__ ClGroups(const ClPlan &p, uint32_t c0, uint32_t c1) {
        first = fast_div(c0, p.per_group);
        count = fast_div(c1 - 1, p.per_group) + 1 - first;
    }
};

template <typename T, int VEC>
struct Row;  // VEC neighbouring elements
template <typename T>
struct Row<T, 16 / sizeof(T)> {
    u32x4 v;
    __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const u32x4 *>(p); }
    __device__ __forceinline__ void floats(float *f) const { Store<T>::unpack(v, f); }
    static __device__ __forceinline__ void store(T *p, const float *f) { *reinterpret_cast<u32x4 *>(p) = Store<T>::pack(f); }
};
template <typename T>
struct Row<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T *p) { v = *p; }
    __device__ __forceinline__ void floats(float *f) const { f[0] = Store<T>::load1(&v); }
    static __device__ __forceinline__ void store(T *p, const float *f) { Store<T>::store1(p, f[0]); }
};

// The codes of VEC neighbouring channels and their scale.
template <int VEC>
struct Codes {
    int8_t v[VEC];
    float scale;
    __device__ __forceinline__ void load(const int8_t *p, const float *s) {
        if constexpr (VEC == 8) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            *reinterpret_cast<uint2 *>(v) = w;
        } else if constexpr (VEC == 4) {
            *reinterpret_cast<uint32_t *>(v) = *reinterpret_cast<const uint32_t *>(p);
        } else {
            v[0] = *p;
        }
        scale = *s;
    }
    __device__ __forceinline__ void floats(float *f) const {
#pragma unroll
        for (int e = 0; e < VEC; e++) f[e] = (float)v[e] * scale;
    }
};

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;  // (false for NaN)
}
__device__ __forceinline__ float code_inverse(float most) { return most < kCodeTiny ? 0.0f : 127.0f * (1.0f / most); }
__device__ __forceinline__ float code_scale(float most) { return most < kCodeTiny ? 0.0f : most * (1.0f / 127.0f); }
__device__ __forceinline__ int code_of(float h, float inv) {
    return (int)fminf(fmaxf(__builtin_rintf(h * inv), -127.0f), 127.0f);
}

// h of a row: the input, plus the addend in the storage type.
template <typename T, int VEC, bool ADD>
__device__ __forceinline__ void add_chunk(float *f, const float *add) {
    if (ADD) {
#pragma unroll
        for (int e = 0; e < VEC; e++) f[e] = round_to_storage<T>(f[e] + add[e]);
    }
}

// Adds `count` floats per channel over the rows of the workgroup: red holds [ty][cols * VEC].
template <int VEC>
__device__ __forceinline__ void put_channels(float *red, const ClTile &t, const float *v) {
    if (t.live) {
#pragma unroll
        for (int e = 0; e < VEC; e++) red[(t.ty * t.cols + t.tx) * VEC + e] = v[e];
    }
}

// ---------------------------------------------------------------------------
// Statistics: mean and sum of squared deviations of a slice's part of every group.  Deviations are taken from the
// slice's first row, channel by channel, so that a mean far from zero costs no digits; channels are then joined by the
// formula for parts of equal size, M2 = sum M2_c + n sum (mean_c - mean)^2.
// ---------------------------------------------------------------------------
template <typename T, int VEC, bool ADD>
__global__ __launch_bounds__(kClThreads) void cl_stats_kernel(const T *x, const T *chunk, float2 *partials, ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t(p, blockIdx.x);
    const uint32_t cc = t.cols * VEC, c0 = t.col0 * VEC;
    float s1[VEC], s2[VEC], shift[VEC], add[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) s1[e] = s2[e] = 0.0f;
    if (t.live) {
        const uint32_t c = c0 + t.tx * VEC;
        const T *at = x + ((size_t)t.b * p.positions + t.row0) * p.channels + c;
        Row<T, VEC> r[kClRows], first;
        first.load(at);
        if (ADD) {
            Row<T, VEC> a;
            a.load(chunk + (size_t)t.b * p.channels + c);
            a.floats(add);
        }
        first.floats(shift);
        add_chunk<T, VEC, ADD>(shift, add);
        for (uint32_t row = t.ty; row < t.rows; row += p.ty * kClRows) {
#pragma unroll
            for (uint32_t i = 0; i < kClRows; i++) r[i].load(at + (size_t)min(row + i * p.ty, t.rows - 1) * p.channels);
#pragma unroll
            for (uint32_t i = 0; i < kClRows; i++) {
                if (row + i * p.ty < t.rows) {
                    float f[VEC];
                    r[i].floats(f);
                    add_chunk<T, VEC, ADD>(f, add);
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const float d = f[e] - shift[e];
                        s1[e] += d;
                        s2[e] = fmaf(d, d, s2[e]);
                    }
                }
            }
        }
    }
    float *red1 = lds, *red2 = lds + p.ty * cc, *first_row = red2 + p.ty * cc;
    put_channels<VEC>(red1, t, s1);
    put_channels<VEC>(red2, t, s2);
    if (t.ty == 0) put_channels<VEC>(first_row, t, shift);
    __syncthreads();
    const float n = (float)t.rows;
    for (uint32_t c = threadIdx.x; c < cc; c += blockDim.x) {
        float a = 0.0f, q = 0.0f;
        for (uint32_t j = 0; j < p.ty; j++) {
            a += red1[j * cc + c];
            q += red2[j * cc + c];
        }
        red1[c] = first_row[c] + a / n;                 // mean of the channel
        const float m2 = fmaf(-a / n, a, q);            // its squared deviations
        red2[c] = m2 < 0.0f ? 0.0f : m2;                // (NaN stays)
    }
    __syncthreads();
    const ClGroups groups(p, c0, c0 + cc);
    const uint32_t team = threadIdx.x / kClTeam, lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const uint32_t lo = max(g * p.per_group.d, c0) - c0, hi = min((g + 1) * p.per_group.d, c0 + cc) - c0;
        float sum = 0.0f;
        for (uint32_t c = lo + lane; c < hi; c += kClTeam) sum += red1[c];
        const float mean = team_sum<kClTeam>(sum) / (float)(hi - lo);
        float m2 = 0.0f;
        for (uint32_t c = lo + lane; c < hi; c += kClTeam) {
            const float d = red1[c] - mean;
            m2 += fmaf(n * d, d, red2[c]);
        }
        m2 = team_sum<kClTeam>(m2);
        const uint32_t span = t.chunk - g * p.per_group.d / VEC / p.tx;
        if (lane == 0)
            partials[(((size_t)t.b * p.slices + t.slice) * p.spans + span) * p.groups + g] = make_float2(mean, m2);
    }
}

// How many values partial (slice, span) of group g is of.
__device__ __forceinline__ float part_count(const ClPlan &p, uint32_t vec, uint32_t g, uint32_t slice, uint32_t span) {
    const uint32_t lo = g * p.per_group.d, hi = lo + p.per_group.d, chunk_channels = p.tx * vec;
    const uint32_t c0 = (lo / chunk_channels + span) * chunk_channels;
    const uint32_t a = max(lo, c0), b = min(hi, c0 + chunk_channels);
    return (float)min(p.rows, p.positions - slice * p.rows) * (float)(b - a);
}
__device__ __forceinline__ uint32_t group_spans(const ClPlan &p, uint32_t vec, uint32_t g) {
    const uint32_t lo = g * p.per_group.d, hi = lo + p.per_group.d, chunk_channels = p.tx * vec;
    return (hi - 1) / chunk_channels - lo / chunk_channels + 1;
}

template <int TEAM>
__device__ __forceinline__ float sum_over(float v) {
    if constexpr (TEAM > 1) v = team_sum<TEAM>(v);
    return v;
}

// Mean and 1 / sqrt(variance + eps) of group g of sample b, by a team of TEAM lanes; every lane gets them.
template <int TEAM>
__device__ __forceinline__ float2 join_stats(const ClPlan &p, uint32_t vec, const float2 *partials, uint32_t b, uint32_t g,
                                             float eps, uint32_t lane) {
    const uint32_t spans = group_spans(p, vec, g), parts = p.slices * spans;
    const float2 *at = partials + (size_t)b * p.slices * p.spans * p.groups + g;
    const float total = (float)p.positions * (float)p.per_group.d;
    float sum = 0.0f;
    for (uint32_t i = lane; i < parts; i += TEAM) {
        const uint32_t slice = i / spans, span = i % spans;
        sum = fmaf(at[((size_t)slice * p.spans + span) * p.groups].x, part_count(p, vec, g, slice, span) / total, sum);
    }
    const float mean = sum_over<TEAM>(sum);
    float m2 = 0.0f;
    for (uint32_t i = lane; i < parts; i += TEAM) {
        const uint32_t slice = i / spans, span = i % spans;
        const float2 v = at[((size_t)slice * p.spans + span) * p.groups];
        const float d = v.x - mean;
        m2 += fmaf(part_count(p, vec, g, slice, span) * d, d, v.y);
    }
    m2 = sum_over<TEAM>(m2);
    return make_float2(mean, 1.0f / sqrtf(m2 / total + eps));
}

// Means over group g of the two summands of the gradient.
template <int TEAM>
__device__ __forceinline__ float2 join_sums(const ClPlan &p, uint32_t vec, const float2 *partials, uint32_t b, uint32_t g,
                                            uint32_t lane) {
    const uint32_t spans = group_spans(p, vec, g), parts = p.slices * spans;
    const float2 *at = partials + (size_t)b * p.slices * p.spans * p.groups + g;
    float a = 0.0f, q = 0.0f;
    for (uint32_t i = lane; i < parts; i += TEAM) {
        const float2 v = at[((size_t)(i / spans) * p.spans + i % spans) * p.groups];
        a += v.x;
        q += v.y;
    }
    a = sum_over<TEAM>(a);
    q = sum_over<TEAM>(q);
    const float total = (float)p.positions * (float)p.per_group.d;
    return make_float2(a / total, q / total);
}

// One wavefront per (sample, group), for more parts than every workgroup should add up by itself.
template <bool STATS>
__global__ __launch_bounds__(kWave) void cl_join_kernel(const float2 *partials, float2 *joined, float eps, uint32_t vec, ClPlan p) {
    const uint32_t b = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
    const float2 v = STATS ? join_stats<kWave>(p, vec, partials, b, g, eps, threadIdx.x)
                           : join_sums<kWave>(p, vec, partials, b, g, threadIdx.x);
    if (threadIdx.x == 0) joined[blockIdx.x] = v;
}

// ---------------------------------------------------------------------------
// y = act(gamma (h - mean) rstd + beta), and with KEEP the 8-bit codes of h.
// `joined`: the statistics, where cl_join_kernel has been there.  `stats`: receives them, or null.
// ---------------------------------------------------------------------------
template <typename T, int VEC, bool ADD, bool SILU, bool KEEP>
__global__ __launch_bounds__(kClThreads) void cl_apply_kernel(const T *x, const T *chunk, T *y, const float *gamma,
                                                              const float *beta, const float2 *partials,
                                                              const float2 *joined, float2 *stats, int8_t *codes,
                                                              float *scales, float eps, ClPlan p) {
    extern __shared__ float2 of_group[];
    const ClTile t(p, blockIdx.x);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC;
    const ClGroups groups(p, c0, c0 + cc);
    const uint32_t team = threadIdx.x / kClTeam, team_lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const float2 v = joined != nullptr ? joined[(size_t)t.b * p.groups + g]
                                           : join_stats<kClTeam>(p, VEC, partials, t.b, g, eps, team_lane);
        if (team_lane == 0) {
            of_group[i] = v;
            if (stats != nullptr && t.slice == 0) stats[(size_t)t.b * p.groups + g] = v;  // (a group's chunks agree)
        }
    }
    __syncthreads();
    if (!t.live) return;
    const uint32_t c = c0 + t.tx * VEC;
    float mean[VEC], mul[VEC], off[VEC], add[VEC];
    if (ADD) {
        Row<T, VEC> a;
        a.load(chunk + (size_t)t.b * p.channels + c);
        a.floats(add);
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float2 s = of_group[fast_div(c + e, p.per_group) - groups.first];
        mean[e] = s.x;
        mul[e] = s.y * gamma[c + e];
        off[e] = beta[c + e];
    }
    const size_t base = ((size_t)t.b * p.positions + t.row0) * p.channels + c;
    const uint32_t blocks = (p.channels + kCodeBlock - 1) / kCodeBlock;
    for (uint32_t row = t.ty; row < t.rows; row += p.ty * kClRows) {
        Row<T, VEC> r[kClRows];
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++) r[i].load(x + base + (size_t)min(row + i * p.ty, t.rows - 1) * p.channels);
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++) {
            const uint32_t at = row + i * p.ty;
            if (at >= t.rows) break;
            float f[VEC];
            r[i].floats(f);
            add_chunk<T, VEC, ADD>(f, add);
            if (KEEP) {
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; e++) most = fmaxf(most, finite_abs(f[e]));
                most = team_max<kCodeBlock / VEC>(most);  // (the lanes of a block share a row: tx is a multiple of their number)
                const float inv = code_inverse(most);
                uint32_t packed[VEC / 4 + (VEC < 4)];
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    uint32_t w = 0;
#pragma unroll
                    for (int k = 0; k < 4 && e + k < VEC; k++) w |= (uint32_t)(code_of(f[e + k], inv) & 255) << (8 * k);
                    packed[e / 4] = w;
                }
                uint32_t *to = reinterpret_cast<uint32_t *>(codes + base + (size_t)at * p.channels);
                if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(packed[0], packed[1]);
                else *to = packed[0];
                if (t.tx % (kCodeBlock / VEC) == 0)
                    scales[((size_t)t.b * p.positions + t.row0 + at) * blocks + c / kCodeBlock] = code_scale(most);
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float z = fmaf(f[e] - mean[e], mul[e], off[e]);
                f[e] = SILU ? silu_f(z) : z;
            }
            Row<T, VEC>::store(y + base + (size_t)at * p.channels, f);
        }
    }
}

// The 8-bit codes where the lanes of cl_apply_kernel are not whole blocks: 32 lanes per block.
template <typename T>
__global__ __launch_bounds__(256) void cl_codes_kernel(const T *x, const T *chunk, int8_t *codes, float *scales,
                                                       size_t rows, uint32_t positions, uint32_t channels) {
    const uint32_t blocks = (channels + kCodeBlock - 1) / kCodeBlock, lane = threadIdx.x % kCodeBlock;
    const size_t total = rows * blocks, step = (size_t)gridDim.x * (blockDim.x / kCodeBlock);
    for (size_t i = (size_t)blockIdx.x * (blockDim.x / kCodeBlock) + threadIdx.x / kCodeBlock; i < total; i += step) {
        const size_t row = i / blocks;
        const uint32_t c = (uint32_t)(i % blocks) * kCodeBlock + lane;
        float h = 0.0f;
        if (c < channels) {
            h = Store<T>::load1(x + row * channels + c);
            if (chunk != nullptr) h = round_to_storage<T>(h + Store<T>::load1(chunk + row / positions * channels + c));
        }
        const float most = team_max<kCodeBlock>(finite_abs(h));
        if (c < channels) codes[row * channels + c] = (int8_t)code_of(h, code_inverse(most));
        if (lane == 0) scales[i] = code_scale(most);
    }
}

// ---------------------------------------------------------------------------
// Gradient.  What both of its passes read: h from the input, from input and addend, or from the codes.
// ---------------------------------------------------------------------------
enum { kFromX = 0, kFromXAdd = 1, kFromCodes = 2 };

template <typename T, int VEC, int FROM>
struct HRow {
    Row<T, VEC> x;
    __device__ __forceinline__ void load(const T *xp, const int8_t *, const float *, size_t at, size_t) { x.load(xp + at); }
    __device__ __forceinline__ void floats(float *f, const float *add) const {
        x.floats(f);
        add_chunk<T, VEC, FROM == kFromXAdd>(f, add);
    }
};
template <typename T, int VEC>
struct HRow<T, VEC, kFromCodes> {
    Codes<VEC> q;
    __device__ __forceinline__ void load(const T *, const int8_t *codes, const float *scales, size_t at, size_t scale_at) {
        q.load(codes + at, scales + scale_at);
    }
    __device__ __forceinline__ void floats(float *f, const float *) const { q.floats(f); }
};

// d silu(z) / dz = s (1 + z (1 - s))
__device__ __forceinline__ float silu_slope(float z) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    return s * fmaf(z, 1.0f - s, 1.0f);
}

// Sums over a slice of positions: per channel S1, S2 and sum_p u (channel_sums [batch][slices][3][channels]), per group
// sum gamma dz and sum gamma dz u (partials, as in cl_stats_kernel).
template <typename T, int VEC, int FROM, bool SILU>
__global__ __launch_bounds__(kClThreads) void cl_sums_kernel(const T *dy, const T *x, const T *chunk, const int8_t *codes,
                                                             const float *scales, const float2 *stats, const float *gamma,
                                                             const float *beta, float2 *partials, float *channel_sums,
                                                             ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t(p, blockIdx.x);
    const uint32_t cc = t.cols * VEC, c0 = t.col0 * VEC;
    float sums[3][VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[0][e] = sums[1][e] = sums[2][e] = 0.0f;
    if (t.live) {
        const uint32_t c = c0 + t.tx * VEC;
        float mean[VEC], rstd[VEC], g[VEC], off[VEC], add[VEC];
        if (FROM == kFromXAdd) {
            Row<T, VEC> a;
            a.load(chunk + (size_t)t.b * p.channels + c);
            a.floats(add);
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float2 s = stats[(size_t)t.b * p.groups + fast_div(c + e, p.per_group)];
            mean[e] = s.x;
            rstd[e] = s.y;
            g[e] = gamma[c + e];
            off[e] = beta[c + e];
        }
        const size_t first = (size_t)t.b * p.positions + t.row0, base = first * p.channels + c;
        const uint32_t blocks = (p.channels + kCodeBlock - 1) / kCodeBlock;
        for (uint32_t row = t.ty; row < t.rows; row += p.ty * kClRows) {
            HRow<T, VEC, FROM> hr[kClRows];
            Row<T, VEC> dr[kClRows];
#pragma unroll
            for (uint32_t i = 0; i < kClRows; i++) {
                const uint32_t at = min(row + i * p.ty, t.rows - 1);
                hr[i].load(x, codes, scales, base + (size_t)at * p.channels, (first + at) * blocks + c / kCodeBlock);
                dr[i].load(dy + base + (size_t)at * p.channels);
            }
#pragma unroll
            for (uint32_t i = 0; i < kClRows; i++) {
                if (row + i * p.ty < t.rows) {
                    float f[VEC], d[VEC];
                    hr[i].floats(f, add);
                    dr[i].floats(d);
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const float u = (f[e] - mean[e]) * rstd[e];
                        const float dz = SILU ? d[e] * silu_slope(fmaf(u, g[e], off[e])) : d[e];
                        sums[0][e] += dz;
                        sums[1][e] = fmaf(dz, u, sums[1][e]);
                        sums[2][e] += u;
                    }
                }
            }
        }
    }
    float *red = lds, *totals = lds + p.ty * cc;  // totals: gamma S1, gamma S2
    for (int q = 0; q < 3; q++) {
        if (q != 0) __syncthreads();
        put_channels<VEC>(red, t, sums[q]);
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < cc; c += blockDim.x) {
            float a = 0.0f;
            for (uint32_t j = 0; j < p.ty; j++) a += red[j * cc + c];
            channel_sums[(((size_t)t.b * p.slices + t.slice) * 3 + q) * p.channels + c0 + c] = a;
            if (q < 2) totals[q * cc + c] = gamma[c0 + c] * a;
        }
    }
    __syncthreads();
    const ClGroups groups(p, c0, c0 + cc);
    const uint32_t team = threadIdx.x / kClTeam, lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const uint32_t lo = max(g * p.per_group.d, c0) - c0, hi = min((g + 1) * p.per_group.d, c0 + cc) - c0;
        float a = 0.0f, q = 0.0f;
        for (uint32_t c = lo + lane; c < hi; c += kClTeam) {
            a += totals[c];
            q += totals[cc + c];
        }
        a = team_sum<kClTeam>(a);
        q = team_sum<kClTeam>(q);
        const uint32_t span = t.chunk - g * p.per_group.d / VEC / p.tx;
        if (lane == 0) partials[(((size_t)t.b * p.slices + t.slice) * p.spans + span) * p.groups + g] = make_float2(a, q);
    }
}

template <typename T, int VEC, int FROM, bool SILU>
__global__ __launch_bounds__(kClThreads) void cl_dx_kernel(const T *dy, const T *x, const T *chunk, const int8_t *codes,
                                                           const float *scales, const float2 *stats, const float *gamma,
                                                           const float *beta, T *dx, const float2 *partials,
                                                           const float2 *joined, ClPlan p) {
    extern __shared__ float2 of_group[];
    const ClTile t(p, blockIdx.x);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC;
    const ClGroups groups(p, c0, c0 + cc);
    const uint32_t team = threadIdx.x / kClTeam, team_lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const float2 v = joined != nullptr ? joined[(size_t)t.b * p.groups + g]
                                           : join_sums<kClTeam>(p, VEC, partials, t.b, g, team_lane);
        if (team_lane == 0) of_group[i] = v;
    }
    __syncthreads();
    if (!t.live) return;
    const uint32_t c = c0 + t.tx * VEC;
    // dx = mul dz - low - (h - mean) slope, with mul = rstd gamma, low = rstd m1, slope = rstd^2 m2
    float mean[VEC], mul[VEC], off[VEC], low[VEC], slope[VEC], add[VEC];
    if (FROM == kFromXAdd) {
        Row<T, VEC> a;
        a.load(chunk + (size_t)t.b * p.channels + c);
        a.floats(add);
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const uint32_t g = fast_div(c + e, p.per_group);
        const float2 s = stats[(size_t)t.b * p.groups + g], m = of_group[g - groups.first];
        mean[e] = s.x;
        mul[e] = s.y * gamma[c + e];
        off[e] = beta[c + e];
        low[e] = s.y * m.x;
        slope[e] = s.y * s.y * m.y;
    }
    const size_t first = (size_t)t.b * p.positions + t.row0, base = first * p.channels + c;
    const uint32_t blocks = (p.channels + kCodeBlock - 1) / kCodeBlock;
    for (uint32_t row = t.ty; row < t.rows; row += p.ty * kClRows) {
        HRow<T, VEC, FROM> hr[kClRows];
        Row<T, VEC> dr[kClRows];
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++) {
            const uint32_t at = min(row + i * p.ty, t.rows - 1);
            hr[i].load(x, codes, scales, base + (size_t)at * p.channels, (first + at) * blocks + c / kCodeBlock);
            dr[i].load(dy + base + (size_t)at * p.channels);
        }
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++) {
            const uint32_t at = row + i * p.ty;
            if (at >= t.rows) break;
            float f[VEC], d[VEC];
            hr[i].floats(f, add);
            dr[i].floats(d);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float hc = f[e] - mean[e];
                const float dz = SILU ? d[e] * silu_slope(fmaf(hc, mul[e], off[e])) : d[e];
                f[e] = fmaf(mul[e], dz, -low[e]) - hc * slope[e];
            }
            Row<T, VEC>::store(dx + base + (size_t)at * p.channels, f);
        }
    }
}

// Gradients of gamma and beta (the blocks of tile i < tiles) and of the addend (the others, one tile of one sample each)
// from the channels' sums: 64 channels a block, its wavefronts share the samples and slices.
template <typename T>
__global__ __launch_bounds__(kClThreads) void cl_channel_grads_kernel(const float *channel_sums, const float2 *stats,
                                                                      const float *gamma, const float2 *partials,
                                                                      const float2 *joined, float *dgamma, float *dbeta,
                                                                      T *dchunk, uint32_t affine_tiles, uint32_t vec,
                                                                      uint32_t batch, ClPlan p) {
    constexpr uint32_t kWaves = kClThreads / kWave;
    __shared__ float red[3][kWaves][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t tiles = (p.channels + kWave - 1) / kWave;
    const bool affine = blockIdx.x < affine_tiles;
    const uint32_t job = affine ? blockIdx.x : blockIdx.x - affine_tiles;
    const uint32_t c = job % tiles * kWave + lane, b = job / tiles;
    const uint32_t parts = affine ? batch * p.slices : p.slices;
    float a[3] = {0.0f, 0.0f, 0.0f};
    if (c < p.channels) {
        const float *at = channel_sums + (size_t)b * p.slices * 3 * p.channels + c;
        for (uint32_t i = wave; i < parts; i += kWaves) {
#pragma unroll
            for (int q = 0; q < 3; q++) a[q] += at[((size_t)i * 3 + q) * p.channels];
        }
    }
#pragma unroll
    for (int q = 0; q < 3; q++) red[q][wave][lane] = a[q];
    __syncthreads();
    if (wave != 0 || c >= p.channels) return;
#pragma unroll
    for (int q = 0; q < 3; q++) {
        a[q] = 0.0f;
        for (uint32_t w = 0; w < kWaves; w++) a[q] += red[q][w][lane];
    }
    if (affine) {
        dbeta[c] = a[0];
        dgamma[c] = a[1];
        return;
    }
    const uint32_t g = fast_div(c, p.per_group);
    const float2 s = stats[(size_t)b * p.groups + g];
    const float2 m = joined != nullptr ? joined[(size_t)b * p.groups + g] : join_sums<1>(p, vec, partials, b, g, 0);
    Store<T>::store1(dchunk + (size_t)b * p.channels + c,
                     s.y * (gamma[c] * a[0] - (float)p.positions * m.x - m.y * a[2]));
}

// ---- host ----
constexpr uint64_t kClMaxBlocks = 0x7FFFFFFFull;

// Plan of a shape; false where it is beyond what the kernels count in 32 bits.
bool cl_plan(size_t elt, size_t batch, size_t positions, size_t channels, size_t groups, bool vectors, ClPlan *p, uint32_t *vec) {
    if (positions > 0x7FFFFFFFull || channels > 0x3FFFFFFFull || batch > 0x7FFFFFFFull || batch * groups > 0x7FFFFFFFull)
        return false;
    const uint32_t epv = (uint32_t)(16 / elt);
    *vec = vectors && channels % epv == 0 ? epv : 1;
    const uint32_t per_group = (uint32_t)(channels / groups), columns = (uint32_t)(channels / *vec);
    p->positions = (uint32_t)positions;
    p->channels = (uint32_t)channels;
    p->columns = columns;
    p->groups = (uint32_t)groups;
    p->per_group = make_fast_div(per_group);
    // whole groups and whole code blocks in a chunk where that leaves it short enough, else whole code blocks
    const uint32_t block_columns = kCodeBlock / *vec;
    const uint64_t unit = std::lcm<uint64_t, uint64_t>(std::lcm<uint64_t, uint64_t>(per_group, *vec) / *vec, block_columns);
    const uint32_t n = (columns + kClMaxTx - 1) / kClMaxTx, even = (columns + n - 1) / n;
    const uint64_t whole = (even + unit - 1) / unit * unit;
    p->tx = n == 1 ? columns : whole <= kClThreads ? (uint32_t)whole : (even + block_columns - 1) / block_columns * block_columns;
    p->chunks = (columns + p->tx - 1) / p->tx;
    p->by_tx = make_fast_div(p->tx);
    p->ty = std::max<uint32_t>(1, std::min<uint32_t>(kClThreads / p->tx, p->positions));
    const uint64_t across = (uint64_t)batch * p->chunks;
    const uint64_t most = std::max<uint64_t>(1, 1024 / across);
    const uint64_t wanted = ((uint64_t)positions + (uint64_t)p->ty * kClRows - 1) / ((uint64_t)p->ty * kClRows);
    const uint64_t slices = std::max<uint64_t>(1, std::min(wanted, most));
    p->rows = (uint32_t)((positions + slices - 1) / slices);
    p->slices = (uint32_t)((positions + p->rows - 1) / p->rows);
    const uint32_t chunk_channels = p->tx * *vec;
    p->spans = p->chunks == 1 ? 1 : (uint32_t)std::min<uint64_t>(p->chunks, ((uint64_t)per_group + chunk_channels - 2) / chunk_channels + 1);
    return across * p->slices <= kClMaxBlocks;
}

size_t partial_floats(const ClPlan &p, size_t batch) { return 2 * batch * p.slices * p.spans * p.groups; }
size_t joined_floats(const ClPlan &p, size_t batch) { return 2 * batch * p.groups; }
size_t channel_floats(const ClPlan &p, size_t batch) { return 3 * batch * p.slices * (size_t)p.channels; }
bool joins(const ClPlan &p) { return p.slices * p.spans > kClMaxParts; }
uint32_t cl_lanes(const ClPlan &p) { return (p.tx * p.ty + kWave - 1) / kWave * kWave; }

// f(std::bool_constant) of a runtime flag
template <typename F>
void with_flag(bool flag, F f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

template <typename T, int VEC>
int cl_forward(const ClPlan &p, const ClForward &a, size_t batch, float eps, bool silu, hipStream_t stream) {
    const T *x = static_cast<const T *>(a.x), *chunk = static_cast<const T *>(a.chunk);
    float2 *partials = static_cast<float2 *>(a.workspace), *joined = nullptr, *stats = reinterpret_cast<float2 *>(a.stats);
    const dim3 grid((uint32_t)(batch * p.chunks * p.slices)), block(cl_lanes(p));
    const size_t cc = (size_t)std::min(p.tx, p.columns) * VEC;
    with_flag(chunk != nullptr, [&](auto add) {
        launch(cl_stats_kernel<T, VEC, add.value>, grid, block, (2 * p.ty + 1) * cc * sizeof(float), stream, x, chunk, partials, p);
    });
    if (joins(p)) {
        joined = stats != nullptr ? stats : partials + partial_floats(p, batch) / 2;
        launch(cl_join_kernel<true>, dim3((uint32_t)(batch * p.groups)), dim3(kWave), 0, stream, partials, joined, eps, VEC, p);
        stats = nullptr;
    }
    const bool keep_here = a.codes != nullptr && VEC > 1 && p.channels % kCodeBlock == 0;
    if (a.codes != nullptr && !keep_here) {
        const size_t rows = batch * p.positions, blocks = rows * ((p.channels + kCodeBlock - 1) / kCodeBlock);
        launch(cl_codes_kernel<T>, dim3((uint32_t)std::min<size_t>(8192, (blocks + 7) / 8)), dim3(256), 0, stream, x, chunk,
               a.codes, a.scales, rows, p.positions, p.channels);
    }
    with_flag(chunk != nullptr, [&](auto add) {
        with_flag(silu, [&](auto act) {
            with_flag(keep_here, [&](auto keep) {
                if constexpr (VEC > 1 || !keep.value)
                    launch(cl_apply_kernel<T, VEC, add.value, act.value, keep.value>, grid, block,
                           std::min<size_t>(p.groups, cc) * sizeof(float2), stream, x, chunk, static_cast<T *>(a.y), a.gamma, a.beta,
                           partials, joined, stats, a.codes, a.scales, eps, p);
            });
        });
    });
    return launch_status();
}

template <typename T, int VEC, int FROM>
void cl_backward_from(const ClPlan &p, const ClBackward &a, size_t batch, bool silu, hipStream_t stream) {
    const T *dy = static_cast<const T *>(a.dy), *x = static_cast<const T *>(a.x), *chunk = static_cast<const T *>(a.chunk);
    const float2 *stats = reinterpret_cast<const float2 *>(a.stats);
    float *channel_sums = static_cast<float *>(a.workspace);
    float2 *partials = reinterpret_cast<float2 *>(channel_sums + (channel_floats(p, batch) + 1) / 2 * 2), *joined = nullptr;
    const dim3 grid((uint32_t)(batch * p.chunks * p.slices)), block(cl_lanes(p));
    const size_t cc = (size_t)std::min(p.tx, p.columns) * VEC;
    with_flag(silu, [&](auto act) {
        launch(cl_sums_kernel<T, VEC, FROM, act.value>, grid, block, (p.ty + 2) * cc * sizeof(float), stream, dy, x, chunk, a.codes,
               a.scales, stats, a.gamma, a.beta, partials, channel_sums, p);
    });
    if (joins(p)) {
        joined = partials + partial_floats(p, batch) / 2;
        launch(cl_join_kernel<false>, dim3((uint32_t)(batch * p.groups)), dim3(kWave), 0, stream, partials, joined, 0.0f, VEC, p);
    }
    with_flag(silu, [&](auto act) {
        launch(cl_dx_kernel<T, VEC, FROM, act.value>, grid, block, std::min<size_t>(p.groups, cc) * sizeof(float2), stream, dy, x,
               chunk, a.codes, a.scales, stats, a.gamma, a.beta, static_cast<T *>(a.dx), partials, joined, p);
    });
    const uint32_t tiles = (p.channels + kWave - 1) / kWave;
    const size_t affine = a.dgamma != nullptr ? tiles : 0, added = a.dchunk != nullptr ? batch * tiles : 0;
    if (affine + added != 0)
        launch(cl_channel_grads_kernel<T>, dim3((uint32_t)(affine + added)), dim3(kClThreads), 0, stream, channel_sums, stats,
               a.gamma, partials, joined, a.dgamma, a.dbeta, static_cast<T *>(a.dchunk), (uint32_t)affine, VEC, (uint32_t)batch, p);
}

template <typename T, int VEC>
int cl_backward(const ClPlan &p, const ClBackward &a, size_t batch, bool silu, hipStream_t stream) {
    if (a.codes != nullptr) cl_backward_from<T, VEC, kFromCodes>(p, a, batch, silu, stream);
    else if (a.chunk != nullptr) cl_backward_from<T, VEC, kFromXAdd>(p, a, batch, silu, stream);
    else cl_backward_from<T, VEC, kFromX>(p, a, batch, silu, stream);
    return launch_status();
}

template <typename T>
__global__ __launch_bounds__(256) void cl_zero_kernel(float *dgamma, float *dbeta, T *dchunk, size_t channels, size_t added) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (dgamma != nullptr && i < channels) dgamma[i] = dbeta[i] = 0.0f;
    if (dchunk != nullptr && i < added) Store<T>::store1(dchunk + i, 0.0f);
}

bool all_aligned16(std::initializer_list<const void *> pointers) {
    return std::all_of(pointers.begin(), pointers.end(), [](const void *q) { return aligned16(q); });
}

}  // namespace

size_t cl_workspace_bytes(size_t elt, size_t batch, size_t positions, size_t channels, size_t groups, bool backward) {
    size_t most = 0;
    for (const bool vectors : {false, true}) {  // (what the operands' alignment allows is not known here)
        ClPlan p;
        uint32_t vec;
        if (!cl_plan(elt, batch, positions, channels, groups, vectors, &p, &vec)) return SIZE_MAX;
        size_t floats = partial_floats(p, batch) + (joins(p) ? joined_floats(p, batch) : 0);
        if (backward) floats += (channel_floats(p, batch) + 1) / 2 * 2;
        most = std::max(most, floats * sizeof(float));
    }
    return most;
}

template <typename T>
int cl_forward_dispatch(const ClForward &a, size_t batch, size_t positions, size_t channels, size_t groups, float eps, bool silu,
                        hipStream_t stream) {
    if (batch == 0 || positions == 0) return MSD_OK;
    ClPlan p;
    uint32_t vec;
    const bool vectors = all_aligned16({a.x, a.chunk, a.y, a.codes});
    if (!cl_plan(sizeof(T), batch, positions, channels, groups, vectors, &p, &vec)) return MSD_ERR_INVALID_VALUE;
    return vec == 1 ? cl_forward<T, 1>(p, a, batch, eps, silu, stream)
                    : cl_forward<T, 16 / sizeof(T)>(p, a, batch, eps, silu, stream);
}
template int cl_forward_dispatch<float>(const ClForward &, size_t, size_t, size_t, size_t, float, bool, hipStream_t);
template int cl_forward_dispatch<__half>(const ClForward &, size_t, size_t, size_t, size_t, float, bool, hipStream_t);

template <typename T>
int cl_backward_dispatch(const ClBackward &a, size_t batch, size_t positions, size_t channels, size_t groups, bool silu,
                         hipStream_t stream) {
    if (batch == 0 || positions == 0) {  // sums over nothing
        const size_t added = a.dchunk != nullptr ? batch * channels : 0, most = std::max(a.dgamma != nullptr ? channels : 0, added);
        if (most != 0)
            launch(cl_zero_kernel<T>, dim3((uint32_t)((most + 255) / 256)), dim3(256), 0, stream, a.dgamma, a.dbeta,
                   static_cast<T *>(a.dchunk), channels, added);
        return launch_status();
    }
    ClPlan p;
    uint32_t vec;
    const bool vectors = all_aligned16({a.dy, a.x, a.chunk, a.codes, a.dx});
    if (!cl_plan(sizeof(T), batch, positions, channels, groups, vectors, &p, &vec)) return MSD_ERR_INVALID_VALUE;
    return vec == 1 ? cl_backward<T, 1>(p, a, batch, silu, stream) : cl_backward<T, 16 / sizeof(T)>(p, a, batch, silu, stream);
}
template int cl_backward_dispatch<float>(const ClBackward &, size_t, size_t, size_t, size_t, bool, hipStream_t);
template int cl_backward_dispatch<__half>(const ClBackward &, size_t, size_t, size_t, size_t, bool, hipStream_t);

}  // namespace msd
