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
// A column is VEC neighbouring channels, what a lane moves at once.  A workgroup owns `tx` columns (a
// chunk) of some positions; its lanes lie along the columns first, so a wavefront reads whole rows one
// after the other, and a lane keeps its channels, whose constants stay in registers.
// A group's statistics need all positions of a sample.  Small samples: a workgroup has all positions of
// its chunk in registers, one launch (cl_unit_kernel, cl_unit_grads_kernel).  Others: a launch of sums
// over slices of the positions and a launch that joins them and applies them.
//
// What bounds it: the memory, whose copies reach 6.7 TB/s here (1 GiB), and for halves with SiLU the vector instructions.  Passes
// in a captured graph, us: 320 channels at 64 x 64 float16, 2 samples 11.5, 16 samples 27.0 (read twice, written once: 4.7 TB/s);
// 128 at 512 x 512 float32 67.7 (5.9 TB/s); forward and gradient of 320 at 64 x 64, 8 samples float16 43, 16 samples by way of the 8-bit
// codes 77; of 640 at 32 x 32, 4 samples float32, codes, 31.  No atomics: sums have one order.
#include "msd_device.h"
#include "msd_internal.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <numeric>
#include <type_traits>

namespace msd {
namespace {

// Slices, as passes in a graph, us: 320 channels at 64 x 64 float16, 2 samples / the same, forward and gradient, 8 samples / 128 at
// 512 x 512 float32 (when channels were joined in one sum).  512 lanes, 256 workgroups, 2 rows: 11.6, 43, 67.  512 workgroups 14.1, 50, 74; 1024 lanes 14.6, 51, 71: more
// of either pay for more sums to join and for rows in flight that the memory does not need.  1 row at a time 11.6, 43, 69; with
// codes 1 row is 4 % faster in float32 (29.3 against 30.6 at 640 channels) and 4 % slower in float16 (79.6 against 76.7).
constexpr uint32_t kClThreads = 512;    // most lanes of a workgroup that has a slice of the positions
constexpr uint32_t kClBlocks = 256;     // workgroups of a launch of slices: one per CU
constexpr uint32_t kClMaxTx = 320;      // columns of a workgroup (rounded up to whole groups, kClThreads at most)
constexpr uint32_t kClRows = 2;         // rows a lane uses while as many are on their way
constexpr uint32_t kClMaxParts = 256;   // parts of a group up to which every workgroup joins them itself (groups over more chunks have more)
constexpr uint32_t kClTeam = 16;        // lanes that add up a group's channels
constexpr uint32_t kClUnitThreads = 1024;
constexpr uint32_t kClUnitMaxK = 4;     // most rows a lane holds of a workgroup that has all positions
constexpr size_t kClMaxLds = 160 * 1024;  // of a workgroup
constexpr uint32_t kCodeBlock = 32;     // channels of one position that share a scale
constexpr float kCodeTiny = 1e-30f;     // blocks below this are kept as zeros (1 / a would not be finite)

struct ClPlan {
    uint32_t positions, channels, columns, groups;
    uint32_t tx, ty, chunks;            // columns and rows of a workgroup; workgroups along the columns
    uint32_t slices;                    // workgroups along the positions: each takes every slices-th block of ty of them
    uint32_t spans;                     // most chunks that share one group
    FastDiv per_group, by_tx, by_slices, by_chunks;
};

// What a wavefront needs to ask for its data comes as plain values in front of all else, which arrive in scalar registers with the
// launch (16 words of them); a plan as a structure is loaded from memory first.
#define CL_GEOMETRY                                                                                                       \
    uint32_t positions, uint32_t channels, uint32_t counts, uint32_t mul_tx, uint32_t mul_slices, uint32_t mul_chunks,   \
        uint32_t shifts, uint32_t ty
#define CL_TILE(VEC, block) ClTile(block, (VEC), positions, channels, counts, mul_tx, mul_slices, mul_chunks, shifts, ty)
#define CL_GEOMETRY_OF(p)                                                                                                 \
    (p).positions, (p).channels, (p).slices | (p).chunks << 16, (p).by_tx.mul, (p).by_slices.mul,               \
        (p).by_chunks.mul, (p).tx | (p).by_tx.shift << 16 | (p).by_slices.shift << 21 | (p).by_chunks.shift << 26, (p).ty
constexpr uint32_t kClMaxCount = 0xFFFF;  // slices, chunks

// What a workgroup is: sample, slice, chunk and its bounds; a lane's rows are first, first + step, ... below the positions.
// Blocks of neighbouring rows go to neighbouring workgroups: with a run of rows each, workgroups a power of two apart would all
// be at the same memory channels (128 channels at 512 x 512: 3.7 TB/s).
struct ClTile {
    uint32_t b, slice, chunk, col0, cols, tx, ty, first, step;
    bool live;
    __device__ __forceinline__ ClTile(uint32_t block, uint32_t vec, uint32_t positions, uint32_t channels, uint32_t counts, uint32_t mul_tx,
                                      uint32_t mul_slices, uint32_t mul_chunks, uint32_t shifts, uint32_t rows) {
        const uint32_t slices = counts & 0xFFFFu, chunks = counts >> 16, width = shifts & 0xFFFFu;
        const uint32_t rest = fast_div(block, FastDiv{mul_slices, (shifts >> 21) & 31u, 0});
        slice = block - rest * slices;
        b = fast_div(rest, FastDiv{mul_chunks, shifts >> 26, 0});
        chunk = rest - b * chunks;
        col0 = chunk * width;
        cols = min(width, channels / vec - col0);
        ty = fast_div(threadIdx.x, FastDiv{mul_tx, (shifts >> 16) & 31u, 0});
        tx = threadIdx.x - ty * width;
        first = slice * rows + ty;
        step = slices * rows;
        live = ty < rows && tx < cols;
    }
};
// Rows of the slices, which take turns with blocks of ty.
struct SliceRows {
    uint32_t each, rest, ty;
    __device__ __forceinline__ SliceRows(uint32_t positions, uint32_t slices, uint32_t ty) : ty(ty) {
        const uint32_t round = slices * ty;
        each = positions / round;
        rest = positions - each * round;
    }
    __device__ __forceinline__ uint32_t extra(uint32_t slice) const { return min(rest - min(rest, slice * ty), ty); }
    __device__ __forceinline__ uint32_t of(uint32_t slice) const { return each * ty + extra(slice); }
};
// Rows of the lanes of a column, the same for all columns of a workgroup: `each`, and one more in the first `extra` lanes.
struct LaneRows {
    uint32_t extra;
    float each, more, all;
    __device__ __forceinline__ LaneRows(uint32_t n, uint32_t extra, uint32_t ty)
        : extra(extra), each(uniform((float)n)), more(uniform((float)(n + 1))), all(uniform((float)(n * ty + extra))) {}
    __device__ __forceinline__ float of(uint32_t lane) const { return lane < extra ? more : each; }
    static __device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
};

// Groups that have channels in [c0, c1).
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
    static __device__ __forceinline__ void store(T *p, const float *f) { store_stream(reinterpret_cast<u32x4 *>(p), Store<T>::pack(f)); }
    // the sum, rounded to the storage type (of halves: once, as by way of float32, whose 24 bits are 2 * 11 + 2)
    __device__ __forceinline__ void add(const Row &o) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(o.v[i]));
            } else {
                const uint32_t a = v[i], b = o.v[i];
                const __half2 h = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
                v[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
    }
};
template <typename T>
struct Row<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T *p) { v = *p; }
    __device__ __forceinline__ void floats(float *f) const { f[0] = Store<T>::load1(&v); }
    static __device__ __forceinline__ void store(T *p, const float *f) { Store<T>::store1(p, f[0]); }
    __device__ __forceinline__ void add(const Row &o) { Store<T>::store1(&v, Store<T>::load1(&v) + Store<T>::load1(&o.v)); }
};

// The codes of VEC neighbouring channels and their scale.
template <int VEC>
struct Codes {
    uint32_t w[(VEC + 3) / 4];
    float scale;
    __device__ __forceinline__ void load(const int8_t *p, const float *s) {
        if constexpr (VEC == 8) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x;
            w[1] = v.y;
        } else if constexpr (VEC == 4) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            w[0] = *reinterpret_cast<const uint8_t *>(p);
        }
        scale = *s;
    }
    __device__ __forceinline__ void floats(float *f) const {
#pragma unroll
        for (int e = 0; e < VEC; e++) {  // (bytes become floats in one instruction: as code + 128)
            const uint32_t v = w[e / 4] ^ 0x80808080u;
            f[e] = ((float)((v >> (8 * (e % 4))) & 255u) - 128.0f) * scale;
        }
    }
};

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;  // (false for NaN)
}
__device__ __forceinline__ float code_inverse(float most) { return most < kCodeTiny ? 0.0f : 127.0f * (1.0f / most); }
__device__ __forceinline__ float code_scale(float most) { return most < kCodeTiny ? 0.0f : most * (1.0f / 127.0f); }
__device__ __forceinline__ int code_of(float h, float inv) {
    if (inv == 0.0f) return 0;  // (of infinities and NaN too)
    return (int)fminf(fmaxf(__builtin_rintf(h * inv), -127.0f), 127.0f);
}

// Stores the codes of a lane's VEC channels, and their scale from the first lane of the block.  The lanes of a block are
// neighbours of one row: chunks begin at whole blocks, and their columns are a multiple of a block's.
template <int VEC>
__device__ __forceinline__ void keep_codes(const float *f, int8_t *codes, float *scale, bool first) {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; e++) most = fmaxf(most, fabsf(f[e]));
    most = team_max<kCodeBlock / VEC>(most);
    const bool infinite = most > 3.402823466e38f;  // (the same for all lanes of the block; NaN are not seen here)
    if (infinite) {
        most = 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; e++) most = fmaxf(most, finite_abs(f[e]));
        most = team_max<kCodeBlock / VEC>(most);
    }
    const float inv = code_inverse(most);
    uint32_t c[VEC], seen = 0;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        // 1.5 * 2^23 leaves the whole part, rounded to even, in the low bits; products of finite values are within +-127
        float v = f[e] * inv;
        asm volatile("" : "+v"(v));  // (the product is rounded by itself)
        c[e] = __float_as_uint(v + 12582912.0f);
        seen |= c[e];
    }
    // the sums of finite values have the exponent 0x96, so that only a NaN sets bit 29; one test for all of them, where a choice for
    // each element made the kernel compute both sides (8 instructions an element in place of 2)
    if (infinite || (seen & 0x20000000u) != 0) {
        asm volatile("");  // (a branch: not to be computed beside the above)
#pragma unroll
        for (int e = 0; e < VEC; e++) c[e] = (uint32_t)code_of(f[e], inv);
    }
    uint32_t w[VEC / 4];
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
        w[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[e + 3], c[e + 2], 0x0C0C0400u), __builtin_amdgcn_perm(c[e + 1], c[e], 0x0C0C0400u), 0x05040100u);
    if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(codes) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(codes) = w[0];
    if (first) *scale = code_scale(most);
}

// ---------------------------------------------------------------------------
// Sums over the rows of a workgroup, through LDS: red holds [ty][cc], a lane has put its channels there.
// On return row 0 has the totals.
// ---------------------------------------------------------------------------
template <int VEC>
__device__ __forceinline__ void put_channels(float *red, const ClTile &t, const float *v) {
    if (t.live) {
#pragma unroll
        for (int e = 0; e < VEC; e++) red[(t.ty * t.cols + t.tx) * VEC + e] = v[e];
    }
}

// Sums of rows first, first + step, ... of a column; four reads under way at a time.
template <int N>
__device__ __forceinline__ void add_column(const float *red, uint32_t stride, uint32_t cc, uint32_t c, uint32_t first, uint32_t step,
                                           uint32_t ty, float *total) {
#pragma unroll
    for (int i = 0; i < N; i++) total[i] = 0.0f;
    for (uint32_t r = first; r < ty; r += 4 * step) {
        float v[N][4];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i][k] = red[i * stride + min(r + k * step, ty - 1) * cc + c];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < N; i++) total[i] += r + k * step < ty ? v[i][k] : 0.0f;
    }
}

template <int N>
__device__ __forceinline__ void add_rows(float *red, uint32_t stride, uint32_t ty, uint32_t cc) {
    const uint32_t lanes = min(blockDim.x / cc, ty / 4);  // lanes that share a channel
    float total[N];
    __syncthreads();
    if (lanes > 1) {
        const uint32_t j = threadIdx.x / cc, c = threadIdx.x - j * cc;
        if (j < lanes) {
            add_column<N>(red, stride, cc, c, j, lanes, ty, total);
#pragma unroll
            for (int i = 0; i < N; i++) red[i * stride + threadIdx.x] = total[i];  // (row j: no other lane reads this one's rows)
        }
        __syncthreads();
        ty = lanes;
    }
    for (uint32_t c = threadIdx.x; c < cc; c += blockDim.x) {
        add_column<N>(red, stride, cc, c, 0, 1, ty, total);
#pragma unroll
        for (int i = 0; i < N; i++) red[i * stride + c] = total[i];
    }
    __syncthreads();
}

// Mean and squared deviations of every channel from those of its lanes.  red: [2][ty][cc], the lanes' means and sums of squared
// deviations from them (SQUARES; otherwise every lane has one row, and there are none); on return row 0 has the channel's.  Two sums
// one after the other, of the means and of M2_lane + n_lane (mean_lane - mean)^2: nothing is subtracted from a sum, whatever the rows
// are.  parts: [2][blockDim].
//
// `lanes` (a power of two) share a channel: lane j sums rows j, j + lanes, ..., of which HELD stay in registers between the two
// sums.  As few instructions as that takes: with weights and bounds worked out for each row the sums of 320 channels' slices took 0.5 us
// more (16 samples of 64 x 64, float16).
constexpr uint32_t kMostLanes = 32;  // (8 channels at 64 x 64 float16 in 11.1 us, with 16 in 13.5)
template <bool SQUARES, uint32_t HELD>
struct ChannelLanes {
    const float *red;  // of the channel
    uint32_t stride, ty, cc, j, log_lanes, whole;
    const LaneRows &rows;
    float means[HELD], m2s[HELD];

    __device__ __forceinline__ ChannelLanes(const float *red, uint32_t stride, uint32_t ty, uint32_t cc, uint32_t j, uint32_t log_lanes, const LaneRows &rows)
        : red(red + j * cc), stride(stride), ty(ty), cc(cc), j(j), log_lanes(log_lanes), whole(ty >> log_lanes), rows(rows) {}
    // f(i, row, mean, M2) for this lane's rows, i = 0 ... 3 in turn; `held`: the first are in registers
    template <typename F>
    __device__ __forceinline__ void each_row(bool held, F f) {
        const uint32_t step = cc << log_lanes;
        const float *at = red;
#pragma unroll
        for (uint32_t k = 0; k < HELD; k++) {
            if (!held && k < whole) {
                means[k] = at[0];
                if (SQUARES) m2s[k] = at[stride];
                at += step;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < HELD; k++)
            if (k < whole) f(k % 4, j + (k << log_lanes), means[k], SQUARES ? m2s[k] : 0.0f);
        at = red + HELD * step;
        for (uint32_t k = HELD; k < whole; k += 4) {
            float mean[4], m2[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const float *from = at + min(i, whole - 1 - k) * step;
                mean[i] = from[0];
                m2[i] = SQUARES ? from[stride] : 0.0f;
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                if (k + i < whole) f(i, j + ((k + i) << log_lanes), mean[i], m2[i]);
            at += 4 * step;
        }
        const uint32_t last = j + (whole << log_lanes);
        if (last < ty) {
            const float *from = red + whole * step;
            f(0, last, from[0], SQUARES ? from[stride] : 0.0f);
        }
    }
    // (four sums: an addition in four waits for the one before, and has that much fewer roundings in front of it)
    __device__ __forceinline__ float offsets(float pivot) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        each_row(false, [&](uint32_t i, uint32_t row, float mean, float) { sum[i] = fmaf(rows.of(row), mean - pivot, sum[i]); });
        return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    __device__ __forceinline__ float squares(float whole_mean) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        each_row(true, [&](uint32_t i, uint32_t row, float mean, float m2) {
            const float d = mean - whole_mean;
            sum[i] = fmaf(rows.of(row) * d, d, sum[i]);
            if (SQUARES) sum[i] += m2;
        });
        return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
};

template <bool SQUARES, uint32_t HELD>
__device__ __forceinline__ void join_lanes(float *red, float *parts, uint32_t ty, uint32_t cc, const LaneRows &rows) {
    const uint32_t stride = ty * cc, log_lanes = 31 - __builtin_clz(max(min(min(blockDim.x / cc, ty / 4), kMostLanes), 1u)), lanes = 1u << log_lanes;
    const float one_nth = LaneRows::uniform(1.0f / rows.all);
    __syncthreads();
    if (lanes == 1) {
        for (uint32_t c = threadIdx.x; c < cc; c += blockDim.x) {
            ChannelLanes<SQUARES, HELD> channel(red + c, stride, ty, cc, 0, 0, rows);
            const float pivot = red[c], mean = fmaf(channel.offsets(pivot), one_nth, pivot), m2 = channel.squares(mean);
            red[c] = mean;
            red[stride + c] = m2;
        }
    } else {
        auto sum_parts = [&](const float *from) {  // [lanes][cc]
            float v[kMostLanes], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t k = 0; k < kMostLanes; k++) {
                if (k >= lanes) break;
                v[k] = from[k * cc];
            }
#pragma unroll
            for (uint32_t k = 0; k < kMostLanes; k++) {
                if (k >= lanes) break;
                sum[k % 4] += v[k];
            }
            return (sum[0] + sum[1]) + (sum[2] + sum[3]);
        };
        const uint32_t j = threadIdx.x / cc, c = threadIdx.x - j * cc;
        ChannelLanes<SQUARES, HELD> channel(red + c, stride, ty, cc, j, log_lanes, rows);
        float pivot = 0.0f, mean = 0.0f;
        if (j < lanes) {
            pivot = red[c];
            parts[threadIdx.x] = channel.offsets(pivot);
        }
        __syncthreads();
        if (j < lanes) {
            mean = fmaf(sum_parts(parts + c), one_nth, pivot);
            parts[blockDim.x + threadIdx.x] = channel.squares(mean);
        }
        __syncthreads();
        if (j == 0) {
            red[c] = mean;
            red[stride + c] = sum_parts(parts + blockDim.x + c);
        }
    }
    __syncthreads();
}

// Mean and squared deviations of every group's part in a workgroup's channels and rows, from the lanes' (red and parts as for
// join_lanes): done(i, mean, m2, channels) by the first lane of a team, for group i of `groups`.  The channels, of equal size n,
// are joined by M2 = sum M2_c + n sum (mean_c - mean)^2.
template <bool SQUARES, uint32_t HELD, typename F>
__device__ __forceinline__ void group_moments(float *red, float *parts, uint32_t ty, uint32_t cc, uint32_t c0, const LaneRows &rows,
                                              const ClPlan &p, const ClGroups &groups, F done) {
    const uint32_t stride = ty * cc;
    const float n = rows.all;
    join_lanes<SQUARES, HELD>(red, parts, ty, cc, rows);
    const uint32_t team = threadIdx.x / kClTeam, lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const uint32_t lo = max(g * p.per_group.d, c0) - c0, hi = min((g + 1) * p.per_group.d, c0 + cc) - c0;
        constexpr uint32_t kHeld = 5;  // channels a lane keeps in registers between the two sums
        const float pivot = red[lo];
        float sum = 0.0f, m2 = 0.0f, means[kHeld], m2s[kHeld];
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) {
            const uint32_t c = min(lo + lane + k * kClTeam, hi - 1);
            means[k] = red[c];
            m2s[k] = red[stride + c];
        }
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) sum += lo + lane + k * kClTeam < hi ? means[k] - pivot : 0.0f;
        for (uint32_t c = lo + lane + kHeld * kClTeam; c < hi; c += kClTeam) sum += red[c] - pivot;
        const float mean = pivot + team_sum<kClTeam>(sum) / (float)(hi - lo);
#pragma unroll
        for (uint32_t k = 0; k < kHeld; k++) {
            const float d = means[k] - mean;
            m2 += lo + lane + k * kClTeam < hi ? fmaf(n * d, d, m2s[k]) : 0.0f;
        }
        for (uint32_t c = lo + lane + kHeld * kClTeam; c < hi; c += kClTeam) {
            const float d = red[c] - mean;
            m2 += fmaf(n * d, d, red[stride + c]);
        }
        m2 = team_sum<kClTeam>(m2);
        if (lane == 0) done(i, mean, m2, (float)(hi - lo));
    }
}

// Sums over every group's part of two values per channel.
template <typename F>
__device__ __forceinline__ void group_sums(const float *va, const float *vb, uint32_t cc, uint32_t c0, const ClPlan &p,
                                           const ClGroups &groups, F done) {
    const uint32_t team = threadIdx.x / kClTeam, lane = threadIdx.x % kClTeam, teams = blockDim.x / kClTeam;
    for (uint32_t i = team; i < groups.count; i += teams) {
        const uint32_t g = groups.first + i;
        const uint32_t lo = max(g * p.per_group.d, c0) - c0, hi = min((g + 1) * p.per_group.d, c0 + cc) - c0;
        float a = 0.0f, q = 0.0f;
#pragma unroll 4
        for (uint32_t c = lo + lane; c < hi; c += kClTeam) {
            a += va[c];
            q += vb[c];
        }
        a = team_sum<kClTeam>(a);
        q = team_sum<kClTeam>(q);
        if (lane == 0) done(i, a, q);
    }
}

// Sums of a lane's rows, channel by channel: deviations from a pivot and their squares.  The pivot is the first row until it moves
// to the mean of the rows so far.  A lane moves it when it has had 8, 64, 512, ... rows: with n rows in all, of which the pivot is the
// mean of n / 8 or more, the square that `finish` subtracts is at most 8 times what is left, whatever the rows are (with the
// slice's first row as the pivot of all, as many times as the slice has rows: a first row of 0 and 65535 of 100 +- 0.01 in each of
// 16 samples had 1 / sqrt(variance) off by 4.7e-4, now by 6e-7).
template <int VEC>
struct Moments {
    float pivot[VEC], s1[VEC], s2[VEC];
    __device__ __forceinline__ Moments() {
#pragma unroll
        for (int e = 0; e < VEC; e++) pivot[e] = s1[e] = s2[e] = 0.0f;
    }
    __device__ __forceinline__ void add(const float *f) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float d = f[e] - pivot[e];
            s1[e] += d;
            s2[e] = fmaf(d, d, s2[e]);
        }
    }
    __device__ __forceinline__ void move(float n, float one_nth) {  // to the mean of the n rows that were added
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float to = fmaf(s1[e], one_nth, pivot[e]), d = to - pivot[e], rest = fmaf(-n, d, s1[e]);
            s2[e] = fmaf(-d, s1[e] + rest, s2[e]);
            s1[e] = rest;
            pivot[e] = to;
        }
    }
    // s1 and s2 become the mean and the squared deviations from it of n rows (n = 0: nothing)
    __device__ __forceinline__ void finish(float n) {
        const float one_nth = 1.0f / fmaxf(n, 1.0f);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float off = s1[e] * one_nth, m2 = fmaf(-off, s1[e], s2[e]);
            s1[e] = n == 0.0f ? 0.0f : pivot[e] + off;
            s2[e] = m2 < 0.0f ? 0.0f : m2;  // (NaN stays)
        }
    }
};

// ---------------------------------------------------------------------------
// Statistics of a slice of positions: partials [batch][slices][spans][groups], (mean, M2).
// A read of x: 134 MB of float32 (128 channels at 512 x 512) in 23.8 us, 5.6 TB/s, against 6.1 to 7.1 of a plain read; three quarters of
// a wavefront's cycles are waits for it.  The joining at the end counts where there are many channels: 320 at 64 x 64 float16, 16
// samples in 10 us, of which its second sum is 0.4.
// ---------------------------------------------------------------------------
// A lane's walk over its rows first, first + step, ... below `rows`, kClRows at a time and as many on their way.  Requests are made
// without a branch (behind the last row: the last row again, which is in the cache) and stay in order, so that a use waits for
// its own request and not for the ones behind it.
// between(): after every 2 kClRows rows that are not the last.
template <typename Stage, typename Request, typename Use, typename Between>
__device__ __forceinline__ void walk_rows(uint32_t first, uint32_t step, uint32_t rows, Stage (&stage)[2][kClRows], Request request, Use use,
                                          Between between) {
    auto requests = [&](Stage *to, uint32_t row) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++) request(to[i], min(row + i * step, rows - 1));
        __builtin_amdgcn_sched_barrier(0);
    };
    auto uses = [&](Stage *from, uint32_t row) {
#pragma unroll
        for (uint32_t i = 0; i < kClRows; i++)
            if (row + i * step < rows) use(from[i], row + i * step);
    };
    const uint32_t ahead = kClRows * step;
    for (uint32_t row = first; row < rows; row += 2 * ahead) {
        uses(stage[0], row);
        requests(stage[0], row + 2 * ahead);
        uses(stage[1], row + ahead);
        requests(stage[1], row + 3 * ahead);
        if (row + 2 * ahead < rows) between();
    }
}
template <typename Stage, typename Request, typename Use>
__device__ __forceinline__ void walk_rows(uint32_t first, uint32_t step, uint32_t rows, Stage (&stage)[2][kClRows], Request request, Use use) {
    walk_rows(first, step, rows, stage, request, use, [] {});
}
template <typename Stage, typename Request>
__device__ __forceinline__ void first_rows(uint32_t first, uint32_t step, uint32_t rows, Stage (&stage)[2][kClRows], Request request) {
#pragma unroll
    for (uint32_t i = 0; i < 2 * kClRows; i++) request(stage[i / kClRows][i % kClRows], min(first + i * step, rows - 1));
    __builtin_amdgcn_sched_barrier(0);
}

template <typename T, int VEC, bool ADD>
__global__ __launch_bounds__(kClThreads) void cl_stats_kernel(const T *x, const T *chunk, CL_GEOMETRY, float2 *partials, ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t = CL_TILE(VEC, blockIdx.x);
    const uint32_t cc = t.cols * VEC, c0 = t.col0 * VEC;
    Moments<VEC> m;
    if (t.live) {
        const uint32_t c = c0 + t.tx * VEC;
        const T *at = x + (size_t)t.b * positions * channels + c;
        Row<T, VEC> r[2][kClRows], add;
        auto request = [&](Row<T, VEC> &to, uint32_t row) { to.load(at + (size_t)row * channels); };
        if (ADD) add.load(chunk + (size_t)t.b * channels + c);
        first_rows(t.first, t.step, positions, r, request);
        Row<T, VEC> first = r[0][0];
        if (ADD) first.add(add);
        first.floats(m.pivot);
        uint32_t rounds = 0, next = 8 / (2 * kClRows);
        walk_rows(t.first, t.step, positions, r, request, [&](Row<T, VEC> &row, uint32_t) {
            if (ADD) row.add(add);
            float f[VEC];
            row.floats(f);
            m.add(f);
        }, [&] {
            if (++rounds != next) return;
            const float n = (float)(2 * kClRows * rounds);
            m.move(n, 1.0f / n);
            next *= 8;
        });
    }
    const SliceRows of_slices(positions, counts & 0xFFFFu, ty);
    const LaneRows rows(of_slices.each, of_slices.extra(t.slice), ty);
    m.finish(rows.of(t.ty));
    put_channels<VEC>(lds, t, m.s1);
    put_channels<VEC>(lds + ty * cc, t, m.s2);
    const ClGroups groups(p, c0, c0 + cc);
    group_moments<true, VEC == 8 ? 12 : 8>(lds, lds + 2 * ty * cc, ty, cc, c0, rows, p, groups, [&](uint32_t i, float mean, float m2, float) {
        const uint32_t g = groups.first + i, span = p.spans == 1 ? 0 : t.chunk - g * p.per_group.d / VEC / p.tx;
        partials[(((size_t)t.b * p.slices + t.slice) * p.spans + span) * p.groups + g] = make_float2(mean, m2);
    });
}

// ---------------------------------------------------------------------------
// Joining the slices.
// ---------------------------------------------------------------------------
struct ClParts {  // what a launch of sums left
    const float2 *at;
    uint32_t slices, ty;
};

// Mean and squared deviations of `weight` positions of a group of `per` channels.
struct PartMoments {
    float weight = 0.0f, mean = 0.0f, m2 = 0.0f;
    __device__ __forceinline__ void join(const PartMoments &o, float per) {
        const float both = weight + o.weight, share = weight > 0.0f ? o.weight * __builtin_amdgcn_rcpf(both) : 1.0f, d = o.mean - mean;
        m2 += fmaf(per * weight * share * d, d, o.m2);
        mean = fmaf(share, d, mean);
        weight = both;
    }
};

// A lane's part of a group's slices, slices first, first + step, ...: kBatch requests under way at a time.  Statistics: the mean of
// a batch, by the distance from its first, the squared deviations from that mean, and then the batches are joined; no sum has
// another subtracted from it.  Sums (of a gradient): added up.
constexpr uint32_t kBatch = 12;
__device__ __forceinline__ void part_batch(const ClPlan &p, const ClParts &parts, const float2 *at, uint32_t s, uint32_t step, float2 *v) {
#pragma unroll
    for (uint32_t k = 0; k < kBatch; k++) v[k] = at[(size_t)min(s + k * step, parts.slices - 1) * p.groups];
}
__device__ __forceinline__ PartMoments part_moments(const ClPlan &p, const ClParts &parts, const float2 *at, uint32_t first, uint32_t step) {
    const SliceRows rows(p.positions, parts.slices, parts.ty);
    const float per = (float)p.per_group.d;
    PartMoments all;
    for (uint32_t s = first; s < parts.slices; s += kBatch * step) {
        float2 v[kBatch];
        float w[kBatch], off = 0.0f;
        part_batch(p, parts, at, s, step, v);
        PartMoments batch;
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            w[k] = s + k * step < parts.slices ? (float)rows.of(s + k * step) : 0.0f;
            batch.weight += w[k];
            off = fmaf(w[k], v[k].x - v[0].x, off);
        }
        batch.mean = fmaf(off, __builtin_amdgcn_rcpf(batch.weight), v[0].x);  // (every slice has a row)
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            const float d = v[k].x - batch.mean;
            batch.m2 += s + k * step < parts.slices ? fmaf(per * w[k] * d, d, v[k].y) : 0.0f;
        }
        all.join(batch, per);
    }
    return all;
}
__device__ __forceinline__ float2 part_sums(const ClPlan &p, const ClParts &parts, const float2 *at, uint32_t first, uint32_t step) {
    float2 all = make_float2(0.0f, 0.0f);
    for (uint32_t s = first; s < parts.slices; s += kBatch * step) {
        float2 v[kBatch];
        part_batch(p, parts, at, s, step, v);
#pragma unroll
        for (uint32_t k = 0; k < kBatch; k++) {
            all.x += s + k * step < parts.slices ? v[k].x : 0.0f;
            all.y += s + k * step < parts.slices ? v[k].y : 0.0f;
        }
    }
    return all;
}

// By the 32 lanes of every half wavefront, one a group; they share the slices.  red: [kClThreads / 64][3][32].
template <bool STATS>
__device__ __forceinline__ void join_whole_groups(const ClPlan &p, const ClParts &parts, uint32_t b, const ClGroups &groups, float eps,
                                                  float2 *of_group, float (*red)[3][32]) {
    constexpr uint32_t kWaves = kClThreads / kWave;
    const uint32_t lane = threadIdx.x % 32, half = threadIdx.x / 32, halves = blockDim.x / 32, wave = threadIdx.x / kWave;
    const float count = (float)p.positions, per = (float)p.per_group.d;
    for (uint32_t g0 = 0; g0 < groups.count; g0 += 32) {
        const float2 *at = parts.at + (size_t)b * parts.slices * p.groups + groups.first + min(g0 + lane, groups.count - 1);
        if constexpr (STATS) {
            PartMoments mine = part_moments(p, parts, at, half, halves), other;
            other.weight = half_swap(mine.weight);
            other.mean = half_swap(mine.mean);
            other.m2 = half_swap(mine.m2);
            mine.join(other, per);
            if (threadIdx.x % kWave < 32) {
                red[wave][0][lane] = mine.weight;
                red[wave][1][lane] = mine.mean;
                red[wave][2][lane] = mine.m2;
            }
        } else {
            const float2 mine = part_sums(p, parts, at, half, halves);
            const float a = half_pair_sum(mine.x), q = half_pair_sum(mine.y);
            if (threadIdx.x % kWave < 32) {
                red[wave][0][lane] = a;
                red[wave][1][lane] = q;
            }
        }
        __syncthreads();
        if (threadIdx.x < 32 && g0 + lane < groups.count) {
            const uint32_t waves = blockDim.x / kWave;
            if constexpr (STATS) {  // as in part_moments; wavefronts without slices have the weight 0
                float w[kWaves], mean[kWaves], m2[kWaves], off = 0.0f, sum = 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < kWaves; k++) {
                    const uint32_t from = min(k, waves - 1);
                    w[k] = k < waves ? red[from][0][lane] : 0.0f;
                    mean[k] = red[from][1][lane];
                    m2[k] = red[from][2][lane];
                }
#pragma unroll
                for (uint32_t k = 0; k < kWaves; k++) off = fmaf(w[k], mean[k] - mean[0], off);
                const float whole = mean[0] + off / count;
#pragma unroll
                for (uint32_t k = 0; k < kWaves; k++) {
                    const float d = mean[k] - whole;
                    sum += k < waves ? fmaf(per * w[k] * d, d, m2[k]) : 0.0f;
                }
                of_group[g0 + lane] = make_float2(whole, 1.0f / sqrtf(sum / (count * per) + eps));
            } else {
                float a = 0.0f, q = 0.0f;
                for (uint32_t w = 0; w < waves; w++) {
                    a += red[w][0][lane];
                    q += red[w][1][lane];
                }
                of_group[g0 + lane] = make_float2(a / (count * per), q / (count * per));
            }
        }
        __syncthreads();
    }
}

// The same where a group can be spread over several chunks, by a team of TEAM lanes per group.
template <int TEAM>
__device__ __forceinline__ float sum_over(float v) {
    if constexpr (TEAM > 1) v = team_sum<TEAM>(v);
    return v;
}
template <bool STATS, int TEAM>
__device__ __forceinline__ float2 join_spread_group(const ClPlan &p, const ClParts &parts, uint32_t vec, uint32_t b, uint32_t g,
                                                    float eps, uint32_t lane) {
    const uint32_t lo = g * p.per_group.d, hi = lo + p.per_group.d, chunk_channels = p.tx * vec, first = lo / chunk_channels;
    const uint32_t spans = (hi - 1) / chunk_channels - first + 1, count = parts.slices * spans;
    const float2 *at = parts.at + (size_t)b * parts.slices * p.spans * p.groups + g;
    const float total = (float)p.positions * (float)p.per_group.d;
    auto part = [&](uint32_t i) { return at[((size_t)(i / spans) * p.spans + i % spans) * p.groups]; };
    const SliceRows rows(p.positions, parts.slices, parts.ty);
    auto size = [&](uint32_t i) {
        const uint32_t c0 = (first + i % spans) * chunk_channels, s = i / spans;
        return (float)rows.of(s) * (float)(min(hi, c0 + chunk_channels) - max(lo, c0));
    };
    float a = 0.0f, q = 0.0f;
    const float pivot = STATS ? part(0).x : 0.0f;
    for (uint32_t i = lane; i < count; i += TEAM) {
        const float2 v = part(i);
        a = STATS ? fmaf(v.x - pivot, size(i) / total, a) : a + v.x;
        q += v.y;
    }
    a = pivot + sum_over<TEAM>(a);
    if (STATS) {
        q = 0.0f;
        for (uint32_t i = lane; i < count; i += TEAM) {
            const float2 v = part(i);
            const float d = v.x - a;
            q += fmaf(size(i) * d, d, v.y);
        }
    }
    q = sum_over<TEAM>(q);
    return STATS ? make_float2(a, 1.0f / sqrtf(q / total + eps)) : make_float2(a / total, q / total);
}

template <bool STATS>
__device__ __forceinline__ void join_groups(const ClPlan &p, const ClParts &parts, const float2 *joined, uint32_t vec, uint32_t b,
                                            const ClGroups &groups, float eps, float2 *of_group, float (*red)[3][32]) {
    if (joined != nullptr) {
        for (uint32_t i = threadIdx.x; i < groups.count; i += blockDim.x) of_group[i] = joined[(size_t)b * p.groups + groups.first + i];
    } else if (p.spans == 1) {
        join_whole_groups<STATS>(p, parts, b, groups, eps, of_group, red);
    } else {
        for (uint32_t i = threadIdx.x / kClTeam; i < groups.count; i += blockDim.x / kClTeam) {
            const float2 v = join_spread_group<STATS, kClTeam>(p, parts, vec, b, groups.first + i, eps, threadIdx.x % kClTeam);
            if (threadIdx.x % kClTeam == 0) of_group[i] = v;
        }
    }
    __syncthreads();
}

// For groups over more chunks than every workgroup should join by itself: a wavefront per group of a sample.
template <bool STATS>
__global__ __launch_bounds__(kWave) void cl_join_kernel(ClParts parts, float2 *joined, float eps, uint32_t vec, ClPlan p) {
    const uint32_t b = blockIdx.x / p.groups, g = blockIdx.x - b * p.groups;
    const float2 v = join_spread_group<STATS, kWave>(p, parts, vec, b, g, eps, threadIdx.x);
    if (threadIdx.x == 0) joined[blockIdx.x] = v;
}

// ---------------------------------------------------------------------------
// y = act(gamma (h - mean) rstd + beta), and with KEEP the 8-bit codes of h.
// `joined`: the statistics, where cl_join_kernel has been there.  `stats`: receives them, or null.
// The first rows are on their way while a workgroup joins the slices for itself, which saves a launch for that.
// 134 MB of float32 in and out in 42.9 us, 6.3 TB/s; results leave past the caches, where x stays (a pass of 128 channels at
// 512 x 512: 73 us in place of 86, in a state of the kernels before the 67).  With codes the vector instructions bound it, four fifths of the SIMDs' cycles: some 20 an element, of which
// SiLU's exponential and reciprocal count four each; 16 samples of 320 at 64 x 64 float16 in 21.4 us, 4.9 TB/s.
// ---------------------------------------------------------------------------
// A lane's constants, channel by channel: z = (h - mean) mul + off.
template <int VEC>
struct Affine {
    float mean[VEC], mul[VEC], off[VEC];
    __device__ __forceinline__ void request(const float *gamma, const float *beta, uint32_t c) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            mul[e] = gamma[c + e];
            off[e] = beta[c + e];
        }
    }
    __device__ __forceinline__ void take(const ClPlan &p, const float2 *of_group, uint32_t first_group, uint32_t c) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float2 s = of_group[fast_div(c + e, p.per_group) - first_group];
            mean[e] = s.x;
            mul[e] *= s.y;
        }
    }
    template <bool SILU>
    __device__ __forceinline__ void apply(float *f) const {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float z = fmaf(f[e] - mean[e], mul[e], off[e]);
            f[e] = SILU ? silu_f(z) : z;
            // float32 first, then the storage type: some instances would round once, and no two give other bits
            asm volatile("" : "+v"(f[e]));
        }
    }
};

template <typename T, int VEC, bool ADD, bool SILU, bool KEEP>
__global__ __launch_bounds__(kClThreads) void cl_apply_kernel(const T *x, const T *chunk, CL_GEOMETRY, const float *gamma,
                                                              const float *beta, T *y, ClParts parts, const float2 *joined,
                                                              float2 *stats, int8_t *codes, float *scales, float eps, ClPlan p) {
    extern __shared__ float2 of_group[];
    __shared__ float red[kClThreads / kWave][3][32];
    const ClTile t = CL_TILE(VEC, blockIdx.x);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC, c = c0 + t.tx * VEC;
    const size_t first = (size_t)t.b * positions, base = first * channels + c;
    Row<T, VEC> r[2][kClRows], add;
    Affine<VEC> affine;
    auto request = [&](Row<T, VEC> &to, uint32_t row) { to.load(x + base + (size_t)row * channels); };
    if (t.live) {  // on their way while the slices are joined
        if (ADD) add.load(chunk + (size_t)t.b * channels + c);
        first_rows(t.first, t.step, positions, r, request);
        affine.request(gamma, beta, c);
    }
    const ClGroups groups(p, c0, c0 + cc);
    join_groups<true>(p, parts, joined, VEC, t.b, groups, eps, of_group, red);
    if (stats != nullptr && t.slice == 0)  // (the chunks of a spread group have the same values)
        for (uint32_t i = threadIdx.x; i < groups.count; i += blockDim.x) stats[(size_t)t.b * p.groups + groups.first + i] = of_group[i];
    if (!t.live) return;
    affine.take(p, of_group, groups.first, c);
    const uint32_t blocks = (channels + kCodeBlock - 1) / kCodeBlock;
    walk_rows(t.first, t.step, positions, r, request, [&](Row<T, VEC> &row, uint32_t at) {
        if (ADD) row.add(add);
        float f[VEC];
        row.floats(f);
        if constexpr (KEEP)
            keep_codes<VEC>(f, codes + base + (size_t)at * channels, scales + (first + at) * blocks + c / kCodeBlock, t.tx % (kCodeBlock / VEC) == 0);
        affine.template apply<SILU>(f);
        Row<T, VEC>::store(y + base + (size_t)at * channels, f);
    });
}

// LDS of cl_unit_kernel, in floats: the lanes' means and squared deviations [2][ty][cc], what join_lanes needs, and the groups'
// statistics, where a float2 may begin.
struct UnitLds {
    uint32_t parts, of_group;
    __host__ __device__ constexpr UnitLds(uint32_t block, uint32_t ty, uint32_t cc)
        : parts(2 * ty * cc), of_group(parts + 2 * block) {}
    constexpr size_t bytes(size_t groups) const { return of_group * sizeof(float) + groups * sizeof(float2); }
};

// The whole of it where a workgroup has all positions of its chunk (whole groups): K rows a lane.  Latency bounds it: a load, the
// sums through LDS, a store.  Passes in a graph, us, so and in slices: 1280 channels at 8 x 8 float16 5.4 and 10.4, at 16 x 16, 2
// samples (K = 2) 7.8 and 11.1; with the gradient 19.2 and 23.9, of 2560 at 9 x 7 float32 (K = 2) 13.1 and 19.4.
template <typename T, int VEC, int K, bool KEEP>
__global__ __launch_bounds__(kClUnitThreads) void cl_unit_kernel(const T *x, const T *chunk, CL_GEOMETRY, const float *gamma,
                                                                 const float *beta, T *y, float2 *stats, int8_t *codes, float *scales,
                                                                 float eps, int silu, ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t = CL_TILE(VEC, blockIdx.x);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC, c = c0 + t.tx * VEC;
    const size_t base = (size_t)t.b * positions * channels + c;
    Row<T, VEC> r[K];
    Affine<VEC> affine;
    uint32_t each = 0;
#pragma unroll
    for (int i = 1; i <= K; i++) each += i * ty <= positions ? 1 : 0;
    const LaneRows rows(each, positions - each * ty, ty);
    Moments<VEC> m;
    if (t.live) {
#pragma unroll
        for (int i = 0; i < K; i++) r[i].load(x + base + min(t.ty + i * ty, positions - 1) * channels);
        if (chunk != nullptr) {
            Row<T, VEC> add;
            add.load(chunk + (size_t)t.b * channels + c);
            affine.request(gamma, beta, c);
#pragma unroll
            for (int i = 0; i < K; i++) r[i].add(add);
        } else {
            affine.request(gamma, beta, c);
        }
        r[0].floats(m.pivot);  // (every lane has a row)
#pragma unroll
        for (int i = 1; i < K; i++) {
            if (t.ty + i * ty < positions) {
                float f[VEC];
                r[i].floats(f);
                m.add(f);
            }
        }
    }
    m.finish(rows.of(t.ty));
    const UnitLds at_lds(blockDim.x, ty, cc);
    float2 *of_group = reinterpret_cast<float2 *>(lds + at_lds.of_group);
    put_channels<VEC>(lds, t, m.s1);
    if (K > 1) put_channels<VEC>(lds + ty * cc, t, m.s2);
    const ClGroups groups(p, c0, c0 + cc);
    const float n = (float)positions;
    group_moments<(K > 1), 8>(lds, lds + at_lds.parts, ty, cc, c0, rows, p, groups, [&](uint32_t i, float mean, float m2, float members) {
        const float2 v = make_float2(mean, 1.0f / sqrtf(m2 / (n * members) + eps));
        of_group[i] = v;
        if (stats != nullptr) stats[(size_t)t.b * p.groups + groups.first + i] = v;
    });
    __syncthreads();
    if (!t.live) return;
    affine.take(p, of_group, groups.first, c);
#pragma unroll
    for (int i = 0; i < K; i++) {
        const uint32_t at = t.ty + i * ty;
        if (at >= positions) break;
        float f[VEC];
        r[i].floats(f);
        if constexpr (KEEP)
            keep_codes<VEC>(f, codes + base + at * channels, scales + ((size_t)t.b * positions + at) * (channels / kCodeBlock) + c / kCodeBlock,
                            t.tx % (kCodeBlock / VEC) == 0);
        if (silu) affine.template apply<true>(f);
        else affine.template apply<false>(f);
        Row<T, VEC>::store(y + base + at * channels, f);
    }
}

// The 8-bit codes where the lanes of the kernels above are not whole blocks: 32 lanes per block, a read of x of its own.
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
// Gradient.  What its passes read: h from the input, from input and addend, or from the codes.
// ---------------------------------------------------------------------------
enum { kFromX = 0, kFromXAdd = 1, kFromCodes = 2 };

// `h` is x or the codes, `more` the addend or the codes' scales.
template <typename T, int VEC, int FROM>
struct GradRow {
    Row<T, VEC> x, dy;
    __device__ __forceinline__ void load(const T *dyp, const void *h, const void *, size_t at, size_t) {
        x.load(static_cast<const T *>(h) + at);
        dy.load(dyp + at);
    }
    __device__ __forceinline__ void floats(float *f, float *d, const Row<T, VEC> &add) const {
        Row<T, VEC> sum = x;
        if (FROM == kFromXAdd) sum.add(add);
        sum.floats(f);
        dy.floats(d);
    }
};
template <typename T, int VEC>
struct GradRow<T, VEC, kFromCodes> {
    Codes<VEC> q;
    Row<T, VEC> dy;
    __device__ __forceinline__ void load(const T *dyp, const void *h, const void *more, size_t at, size_t scale_at) {
        q.load(static_cast<const int8_t *>(h) + at, static_cast<const float *>(more) + scale_at);
        dy.load(dyp + at);
    }
    __device__ __forceinline__ void floats(float *f, float *d, const Row<T, VEC> &) const {
        q.floats(f);
        dy.floats(d);
    }
};

// d silu(z) / dz = s + z (s - s^2)
__device__ __forceinline__ float silu_slope(float z) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    return fmaf(z, fmaf(-s, s, s), s);
}

// A lane's constants: z = (h - mean) mul + off, mul = rstd gamma.  The sums are of dz, dz (h - mean) and h - mean: rstd
// multiplies the last two when they are whole.
template <int VEC>
struct Normal {
    float mean[VEC], mul[VEC], off[VEC];
    __device__ __forceinline__ void load(const ClPlan &p, const float2 *stats, const float *gammas, const float *betas, uint32_t b, uint32_t c) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float2 s = stats[(size_t)b * p.groups + fast_div(c + e, p.per_group)];
            mean[e] = s.x;
            mul[e] = s.y * gammas[c + e];
            off[e] = betas[c + e];
        }
    }
    template <bool SILU>
    __device__ __forceinline__ void add_sums(const float *h, const float *d, float (*sums)[VEC]) const {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float hc = h[e] - mean[e];
            const float dz = SILU ? d[e] * silu_slope(fmaf(hc, mul[e], off[e])) : d[e];
            sums[0][e] += dz;
            sums[1][e] = fmaf(dz, hc, sums[1][e]);
            sums[2][e] += hc;
        }
    }
};

// A lane's constants for dx = mul dz - low - (h - mean) slope: mul = rstd gamma, low = rstd m1, slope = rstd^2 m2.
template <int VEC>
struct Slope {
    Normal<VEC> normal;
    float low[VEC], slope[VEC];
    __device__ __forceinline__ void set(int e, float rstd, float2 m) {
        low[e] = rstd * m.x;
        slope[e] = rstd * rstd * m.y;
    }
    template <bool SILU>
    __device__ __forceinline__ void apply(float *h, const float *d) const {  // h becomes dx
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float hc = h[e] - normal.mean[e];
            const float dz = SILU ? d[e] * silu_slope(fmaf(hc, normal.mul[e], normal.off[e])) : d[e];
            h[e] = fmaf(normal.mul[e], dz, -low[e]) - hc * slope[e];
        }
    }
};

// dchunk of a channel from its sums: sum_p dx.
__device__ __forceinline__ float chunk_gradient(float2 stat, float gamma, float positions, float2 m, float s1, float su) {
    return stat.y * (gamma * s1 - positions * m.x - m.y * su);
}

// Sums over a slice of positions: per channel S1, S2 and sum_p u (channel_sums [batch][slices][3][channels]), per group
// sum gamma dz and sum gamma dz u (partials, as in cl_stats_kernel).  z is computed again, not kept: it costs instructions, 16 an
// element of which two count four.  16 samples of 320 at 64 x 64, float16 from codes: 63 MB in 20 us, of which the SIMDs issue vector
// instructions three quarters; the rest both wavefronts of a SIMD wait, for memory or a result.
template <typename T, int VEC, int FROM, bool SILU>
__global__ __launch_bounds__(kClThreads) void cl_sums_kernel(const T *dy, const void *h, const void *more, CL_GEOMETRY, const float2 *stats,
                                                             const float *gamma, const float *beta, float2 *partials,
                                                             float *channel_sums, ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t = CL_TILE(VEC, blockIdx.x);
    const uint32_t cc = t.cols * VEC, c0 = t.col0 * VEC;
    float sums[3][VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[0][e] = sums[1][e] = sums[2][e] = 0.0f;
    if (t.live) {
        const uint32_t c = c0 + t.tx * VEC, blocks = (channels + kCodeBlock - 1) / kCodeBlock;
        const size_t first = (size_t)t.b * positions, base = first * channels + c;
        Row<T, VEC> add;
        GradRow<T, VEC, FROM> r[2][kClRows];
        auto request = [&](GradRow<T, VEC, FROM> &to, uint32_t row) {
            to.load(dy, h, more, base + (size_t)row * channels, (first + row) * blocks + c / kCodeBlock);
        };
        if (FROM == kFromXAdd) add.load(static_cast<const T *>(more) + (size_t)t.b * channels + c);
        first_rows(t.first, t.step, positions, r, request);
        Normal<VEC> normal;
        normal.load(p, stats, gamma, beta, t.b, c);
        walk_rows(t.first, t.step, positions, r, request, [&](GradRow<T, VEC, FROM> &row, uint32_t) {
            float f[VEC], d[VEC];
            row.floats(f, d, add);
            normal.template add_sums<SILU>(f, d, sums);
        });
    }
    const uint32_t stride = ty * cc;
#pragma unroll
    for (int q = 0; q < 3; q++) put_channels<VEC>(lds + q * stride, t, sums[q]);
    add_rows<3>(lds, stride, ty, cc);
    float *to = channel_sums + ((size_t)t.b * p.slices + t.slice) * 3 * channels + c0;
    for (uint32_t c = threadIdx.x; c < cc; c += blockDim.x) {
        const float g = gamma[c0 + c], rstd = stats[(size_t)t.b * p.groups + fast_div(c0 + c, p.per_group)].y;
        const float s1 = lds[c], s2 = rstd * lds[stride + c];
        to[c] = s1;
        to[channels + c] = s2;
        to[2 * channels + c] = rstd * lds[2 * stride + c];
        lds[c] = g * s1;
        lds[stride + c] = g * s2;
    }
    __syncthreads();
    const ClGroups groups(p, c0, c0 + cc);
    group_sums(lds, lds + stride, cc, c0, p, groups, [&](uint32_t i, float a, float q) {
        const uint32_t g = groups.first + i, span = p.spans == 1 ? 0 : t.chunk - g * p.per_group.d / VEC / p.tx;
        partials[(((size_t)t.b * p.slices + t.slice) * p.spans + span) * p.groups + g] = make_float2(a, q);
    });
}

// Gradients of gamma and beta (the first `affine_tiles` blocks of `channel_blocks`) and of the addend (the others: a tile of a
// sample each) from the channels' sums: 64 channels a block, its wavefronts share the samples and slices.
struct ClChannelGrads {
    const float *sums;
    float *dgamma, *dbeta;
    void *dchunk;
    uint32_t affine_tiles, batch;
};

template <typename T>
__device__ __forceinline__ void channel_grads(const ClChannelGrads &a, uint32_t block, const float2 *stats, const float *gamma,
                                              const ClParts &parts, const float2 *joined, uint32_t vec, const ClPlan &p,
                                              float (*red)[kClThreads / kWave][kWave]) {
    constexpr uint32_t kAhead = 8;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const uint32_t tiles = (p.channels + kWave - 1) / kWave;
    const bool affine = block < a.affine_tiles;
    const uint32_t job = affine ? block : block - a.affine_tiles;
    const uint32_t b = job / tiles, c = (job - b * tiles) * kWave + lane, at_c = min(c, p.channels - 1);
    const uint32_t count = affine ? a.batch * parts.slices : parts.slices;
    const float *at = a.sums + (size_t)b * parts.slices * 3 * p.channels + at_c;
    float s[3] = {0.0f, 0.0f, 0.0f}, m[2] = {0.0f, 0.0f};
    const uint32_t g = fast_div(at_c, p.per_group);
    const int other = affine ? 1 : 2;  // S2 for the affine gradients, sum_p u for the addend's
    for (uint32_t i0 = wave; i0 < count; i0 += waves * kAhead) {
        float v[2][kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const float *from = at + (size_t)min(i0 + k * waves, count - 1) * 3 * p.channels;
            v[0][k] = from[0];
            v[1][k] = from[other * p.channels];
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            if (i0 + k * waves < count) {
                s[0] += v[0][k];
                s[1] += v[1][k];
            }
        }
    }
    red[0][wave][lane] = s[0];
    red[1][wave][lane] = s[1];
    if (!affine && joined == nullptr && p.spans == 1) {  // the group's means, by the same wavefronts
        const float2 *from = parts.at + (size_t)b * parts.slices * p.groups + g;
#pragma unroll 4
        for (uint32_t i = wave; i < parts.slices; i += waves) {
            const float2 v = from[(size_t)i * p.groups];
            m[0] += v.x;
            m[1] += v.y;
        }
        red[2][wave][lane] = m[0];
        red[3][wave][lane] = m[1];
    }
    __syncthreads();
    if (wave != 0 || c >= p.channels) return;
    float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < 4; q++)
        for (uint32_t w = 0; w < waves; w++) total[q] += red[q][w][lane];
    if (affine) {
        a.dbeta[c] = total[0];
        a.dgamma[c] = total[1];
        return;
    }
    const float n = (float)p.positions * (float)p.per_group.d;
    const float2 means = joined != nullptr ? joined[(size_t)b * p.groups + g]
                         : p.spans == 1    ? make_float2(total[2] / n, total[3] / n)
                                           : join_spread_group<false, 1>(p, parts, vec, b, g, 0.0f, 0);
    Store<T>::store1(static_cast<T *>(a.dchunk) + (size_t)b * p.channels + c,
                     chunk_gradient(stats[(size_t)b * p.groups + g], gamma[c], (float)p.positions, means, total[0], total[1]));
}

// dx of a slice, after the join of the sums as in cl_apply_kernel, and in its first workgroups the channels' gradients (a launch of
// their own took 31 us at 8 samples of 320 channels; here they run beside the rest).  16 samples of 320 at 64 x 64, float16 from codes:
// 105 MB in 21.6 us, for the same instructions (16 an element) and waits.
template <typename T, int VEC, int FROM, bool SILU>
__global__ __launch_bounds__(kClThreads) void cl_dx_kernel(const T *dy, const void *h, const void *more, CL_GEOMETRY, uint32_t channel_blocks,
                                                           const float2 *stats, const float *gamma, const float *beta, T *dx,
                                                           ClParts parts, const float2 *joined, ClChannelGrads grads, ClPlan p) {
    extern __shared__ float2 of_group[];
    __shared__ float red[4][kClThreads / kWave][kWave];
    if (blockIdx.x < channel_blocks) {  // (first, so that they run beside the others)
        channel_grads<T>(grads, blockIdx.x, stats, gamma, parts, joined, VEC, p, red);
        return;
    }
    const ClTile t = CL_TILE(VEC, blockIdx.x - channel_blocks);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC, c = c0 + t.tx * VEC, blocks = (channels + kCodeBlock - 1) / kCodeBlock;
    const size_t first = (size_t)t.b * positions, base = first * channels + c;
    GradRow<T, VEC, FROM> r[2][kClRows];
    Row<T, VEC> add;
    auto request = [&](GradRow<T, VEC, FROM> &to, uint32_t row) {
        to.load(dy, h, more, base + (size_t)row * channels, (first + row) * blocks + c / kCodeBlock);
    };
    Slope<VEC> s;
    if (t.live) {
        if (FROM == kFromXAdd) add.load(static_cast<const T *>(more) + (size_t)t.b * channels + c);
        first_rows(t.first, t.step, positions, r, request);
        s.normal.load(p, stats, gamma, beta, t.b, c);
    }
    const ClGroups groups(p, c0, c0 + cc);
    join_groups<false>(p, parts, joined, VEC, t.b, groups, 0.0f, of_group, reinterpret_cast<float(*)[3][32]>(&red[0][0][0]));
    if (!t.live) return;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const uint32_t g = fast_div(c + e, p.per_group);
        s.set(e, stats[(size_t)t.b * p.groups + g].y, of_group[g - groups.first]);
    }
    walk_rows(t.first, t.step, positions, r, request, [&](GradRow<T, VEC, FROM> &row, uint32_t at) {
        float f[VEC], d[VEC];
        row.floats(f, d, add);
        s.template apply<SILU>(f, d);
        Row<T, VEC>::store(dx + base + (size_t)at * channels, f);
    });
}

// LDS of cl_unit_grads_kernel, in floats: three sums [ty][cc] and gamma S1, gamma S2 [2][cc]; then, where a float2 may begin, the
// groups' means.
struct UnitGradsLds {
    uint32_t sums, weighted, of_group;
    __host__ __device__ constexpr UnitGradsLds(uint32_t ty, uint32_t cc)
        : sums(ty * cc), weighted(3 * sums), of_group((weighted + 2 * cc + 1) / 2 * 2) {}
    constexpr size_t bytes(size_t groups) const { return of_group * sizeof(float) + groups * sizeof(float2); }
};
static_assert(UnitGradsLds(1, 5).of_group == 26 && UnitGradsLds(2, 5).of_group == 40 && UnitGradsLds(3, 7).of_group == 78 &&
              UnitGradsLds(2, 8).of_group == 64, "rounded up to whole float2");

// The whole of it where a workgroup has all positions of its chunk (whole groups): K rows a lane.  channel_sums
// [batch][2][channels]: S1 and S2, for cl_affine_grads_kernel, or, of one sample, dbeta and dgamma themselves (or null).
// 2560 channels at 9 x 7, 2 samples float32: 6.2 us, and 2.1 for dgamma and dbeta.
template <typename T, int VEC, int K, int FROM>
__global__ __launch_bounds__(kClUnitThreads) void cl_unit_grads_kernel(const T *dy, const void *h, const void *more, CL_GEOMETRY,
                                                                       const float2 *stats, const float *gamma, const float *beta,
                                                                       T *dx, float *s1_to, float *s2_to, T *dchunk,
                                                                       uint32_t sample_stride, int silu, ClPlan p) {
    extern __shared__ float lds[];
    const ClTile t = CL_TILE(VEC, blockIdx.x);
    const uint32_t c0 = t.col0 * VEC, cc = t.cols * VEC, c = c0 + t.tx * VEC, blocks = (channels + kCodeBlock - 1) / kCodeBlock;
    const size_t first = (size_t)t.b * positions, base = first * channels + c;
    GradRow<T, VEC, FROM> r[K];
    Row<T, VEC> add;
    Slope<VEC> s;
    float sums[3][VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) sums[0][e] = sums[1][e] = sums[2][e] = 0.0f;
    if (t.live) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            const uint32_t at = min(t.ty + i * ty, positions - 1);
            r[i].load(dy, h, more, base + at * channels, (first + at) * blocks + c / kCodeBlock);
        }
        if (FROM == kFromXAdd) add.load(static_cast<const T *>(more) + (size_t)t.b * channels + c);
        s.normal.load(p, stats, gamma, beta, t.b, c);
#pragma unroll
        for (int i = 0; i < K; i++) {
            if (t.ty + i * ty < positions) {
                float f[VEC], d[VEC];
                r[i].floats(f, d, add);
                if (silu) s.normal.template add_sums<true>(f, d, sums);
                else s.normal.template add_sums<false>(f, d, sums);
            }
        }
    }
    const UnitGradsLds at_lds(ty, cc);
    const uint32_t stride = at_lds.sums;
    float *weighted = lds + at_lds.weighted;
    float2 *of_group = reinterpret_cast<float2 *>(lds + at_lds.of_group);
#pragma unroll
    for (int q = 0; q < 3; q++) put_channels<VEC>(lds + q * stride, t, sums[q]);
    add_rows<3>(lds, stride, ty, cc);
    for (uint32_t k = threadIdx.x; k < cc; k += blockDim.x) {
        const float g = gamma[c0 + k], rstd = stats[(size_t)t.b * p.groups + fast_div(c0 + k, p.per_group)].y;
        const float s1 = lds[k], s2 = rstd * lds[stride + k];
        lds[2 * stride + k] *= rstd;
        weighted[k] = g * s1;
        weighted[cc + k] = g * s2;
        if (s1_to != nullptr) {
            s1_to[(size_t)t.b * sample_stride + c0 + k] = s1;
            s2_to[(size_t)t.b * sample_stride + c0 + k] = s2;
        }
    }
    __syncthreads();
    const ClGroups groups(p, c0, c0 + cc);
    const float n = (float)positions * (float)p.per_group.d;
    group_sums(weighted, weighted + cc, cc, c0, p, groups, [&](uint32_t i, float a, float q) { of_group[i] = make_float2(a / n, q / n); });
    __syncthreads();
    if (dchunk != nullptr) {
        for (uint32_t k = threadIdx.x; k < cc; k += blockDim.x) {
            const uint32_t g = fast_div(c0 + k, p.per_group);
            Store<T>::store1(dchunk + (size_t)t.b * channels + c0 + k,
                             chunk_gradient(stats[(size_t)t.b * p.groups + g], gamma[c0 + k], (float)positions, of_group[g - groups.first],
                                            lds[k], lds[2 * stride + k]));
        }
    }
    if (!t.live) return;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const uint32_t g = fast_div(c + e, p.per_group);
        s.set(e, stats[(size_t)t.b * p.groups + g].y, of_group[g - groups.first]);
    }
#pragma unroll
    for (int i = 0; i < K; i++) {
        const uint32_t at = t.ty + i * ty;
        if (at >= positions) break;
        float f[VEC], d[VEC];
        r[i].floats(f, d, add);
        if (silu) s.template apply<true>(f, d);
        else s.template apply<false>(f, d);
        Row<T, VEC>::store(dx + base + at * channels, f);
    }
}

// dbeta and dgamma: sums over the samples of S1 and S2 ([batch][2][channels]).
__global__ __launch_bounds__(kWave) void cl_affine_grads_kernel(const float *sums, float *dgamma, float *dbeta, uint32_t batch,
                                                                uint32_t channels) {
    const uint32_t c = blockIdx.x * kWave + threadIdx.x;
    if (c >= channels) return;
    float a = 0.0f, q = 0.0f;
#pragma unroll 8
    for (uint32_t b = 0; b < batch; b++) {
        a += sums[(size_t)b * 2 * channels + c];
        q += sums[((size_t)b * 2 + 1) * channels + c];
    }
    dbeta[c] = a;
    dgamma[c] = q;
}

// ---- host ----
// A grid holds less than 2^32 lanes.
bool fits_grid(uint64_t blocks, uint32_t lanes) { return blocks <= 0xFFFFFFFFull / lanes; }
constexpr size_t kClMaxChannels = (size_t)1 << 22;
constexpr uint64_t kClUnitElements = 1u << 28;  // of a sample that workgroups have whole: offsets in it are counted in 32 bits

// The shape's own numbers; false where they are beyond what the kernels count in 32 bits.
bool cl_shape(size_t elt, size_t batch, size_t positions, size_t channels, size_t groups, bool vectors, ClPlan *p, uint32_t *vec) {
    if (positions > 0x7FFFFFFFull || channels > kClMaxChannels || batch > 0x7FFFFFFFull || batch * groups > 0x7FFFFFFFull)
        return false;
    const uint32_t epv = (uint32_t)(16 / elt);
    *vec = vectors && channels % epv == 0 ? epv : 1;
    *p = ClPlan{};
    p->positions = (uint32_t)positions;
    p->channels = (uint32_t)channels;
    p->columns = (uint32_t)(channels / *vec);
    p->groups = (uint32_t)groups;
    p->per_group = make_fast_div((uint32_t)(channels / groups));
    return true;
}

uint32_t cl_lanes(const ClPlan &p) { return (p.tx * p.ty + kWave - 1) / kWave * kWave; }
bool joins(const ClPlan &p) { return p.slices * p.spans > kClMaxParts; }

void finish_plan(ClPlan *p, uint32_t tx, uint32_t ty, uint32_t slices, uint32_t vec) {
    p->tx = tx;
    p->ty = ty;
    p->chunks = (p->columns + tx - 1) / tx;
    p->slices = std::min(slices, (p->positions + ty - 1) / ty);  // (each has a row)
    const uint64_t chunk_channels = (uint64_t)tx * vec;
    p->spans = chunk_channels % p->per_group.d == 0 || p->chunks == 1
                   ? 1 : (uint32_t)std::min<uint64_t>(p->chunks, (p->per_group.d + chunk_channels - 2) / chunk_channels + 1);
    p->by_tx = make_fast_div(tx);
    p->by_slices = make_fast_div(p->slices);
    p->by_chunks = make_fast_div(p->chunks);
}

// Columns of the smallest chunk of whole groups (and, for codes, of whole blocks).
uint64_t whole_columns(const ClPlan &p, uint32_t vec, bool blocks) {
    const uint64_t columns = std::lcm<uint64_t, uint64_t>(p.per_group.d, vec) / vec;
    return blocks ? std::lcm<uint64_t, uint64_t>(columns, std::max<uint32_t>(1, kCodeBlock / vec)) : columns;
}

size_t chunk_channels(const ClPlan &p, uint32_t vec) { return (size_t)std::min(p.tx, p.columns) * vec; }
// What a workgroup of unit_plan asks for of LDS (its chunk is whole groups).
size_t unit_lds(const ClPlan &p, uint32_t vec, bool backward) {
    const uint32_t cc = (uint32_t)chunk_channels(p, vec);
    const size_t groups = cc / p.per_group.d;
    return backward ? UnitGradsLds(p.ty, cc).bytes(groups) : UnitLds(cl_lanes(p), p.ty, cc).bytes(groups);
}

// (a gradient holds two rows for one: of 8 channels each, no more than two fit the registers)
uint32_t unit_max_k(uint32_t vec, bool backward) { return backward && vec == 8 ? 2 : kClUnitMaxK; }

// A workgroup with all positions of some whole groups: K rows a lane; 0 where that is too much for one.
uint32_t unit_plan(ClPlan *p, uint32_t vec, size_t batch, bool backward) {
    const uint32_t max_k = unit_max_k(vec, backward);
    const uint64_t whole = whole_columns(*p, vec, false);
    if (whole > kClUnitThreads || whole * p->positions > kClUnitThreads * max_k) return 0;
    if ((uint64_t)p->positions * p->channels > kClUnitElements) return 0;
    uint64_t tx = whole;  // more of them where they are short
    while (tx * 2 <= p->columns && tx * 2 * p->positions <= 128) tx *= 2;
    const uint64_t chunks = (p->columns + tx - 1) / tx;
    if (chunks > kClMaxCount) return 0;
    uint32_t k = 1;
    while (k * (kClUnitThreads / tx) < p->positions) k *= 2;
    if (k > max_k) return 0;
    finish_plan(p, (uint32_t)tx, (p->positions + k - 1) / k, 1, vec);
    return fits_grid(batch * chunks, cl_lanes(*p)) && unit_lds(*p, vec, backward) <= kClMaxLds ? k : 0;
}

bool slice_plan(ClPlan *p, uint32_t vec, size_t batch) {
    // whole groups and whole code blocks in a chunk where that leaves it short enough, else whole code blocks
    const uint32_t block_columns = kCodeBlock / vec;
    const uint64_t unit = whole_columns(*p, vec, true);
    const uint32_t n = (p->columns + kClMaxTx - 1) / kClMaxTx, even = (p->columns + n - 1) / n;
    const uint64_t whole = (even + unit - 1) / unit * unit;
    const uint32_t tx = n == 1 ? p->columns : whole <= kClThreads ? (uint32_t)whole : (even + block_columns - 1) / block_columns * block_columns;
    const uint32_t ty = std::max<uint32_t>(1, std::min<uint32_t>(kClThreads / tx, p->positions));
    const uint64_t across = (uint64_t)batch * ((p->columns + tx - 1) / tx);
    const uint64_t most = std::max<uint64_t>(1, kClBlocks / across);
    const uint64_t wanted = ((uint64_t)p->positions + (uint64_t)ty * kClRows - 1) / ((uint64_t)ty * kClRows);
    finish_plan(p, tx, ty, (uint32_t)std::min(wanted, most), vec);
    return p->slices <= kClMaxCount && p->chunks <= kClMaxCount && fits_grid(across * p->slices, cl_lanes(*p)) &&
           (!joins(*p) || fits_grid(batch * p->groups, kWave));
}

size_t partial_floats(const ClPlan &p, size_t batch) { return 2 * batch * p.slices * p.spans * p.groups; }
size_t joined_floats(const ClPlan &p, size_t batch) { return 2 * batch * p.groups; }
size_t channel_floats(const ClPlan &p, size_t batch) { return (3 * batch * p.slices * (size_t)p.channels + 1) / 2 * 2; }

// f(std::bool_constant) of a runtime flag, f(std::integral_constant) of a number of rows
template <typename F>
void with_flag(bool flag, F f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}
template <typename F>
void with_rows(uint32_t k, F f) {
    if (k == 1) f(std::integral_constant<int, 1>{});
    else if (k == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
}

template <bool STATS>
float2 *join_launch(const ClPlan &p, const ClParts &parts, float2 *joined, size_t batch, float eps, uint32_t vec, hipStream_t stream) {
    launch(cl_join_kernel<STATS>, dim3((uint32_t)(batch * p.groups)), dim3(kWave), 0, stream, parts, joined, eps, vec, p);
    return joined;
}

template <typename T, int VEC>
int cl_forward(ClPlan p, const ClForward &a, size_t batch, float eps, bool silu, hipStream_t stream) {
    const T *x = static_cast<const T *>(a.x), *chunk = static_cast<const T *>(a.chunk);
    T *y = static_cast<T *>(a.y);
    float2 *stats = reinterpret_cast<float2 *>(a.stats);
    const uint32_t k = unit_plan(&p, VEC, batch, false);
    if (k == 0 && !slice_plan(&p, VEC, batch)) return MSD_ERR_INVALID_VALUE;
    const bool keep_here = a.codes != nullptr && VEC > 1 && p.channels % kCodeBlock == 0 && p.tx * VEC % kCodeBlock == 0;
    if (a.codes != nullptr && !keep_here) {
        const size_t rows = batch * p.positions, blocks = rows * ((p.channels + kCodeBlock - 1) / kCodeBlock);
        launch(cl_codes_kernel<T>, dim3((uint32_t)std::min<size_t>(8192, (blocks + 7) / 8)), dim3(256), 0, stream, x, chunk,
               a.codes, a.scales, rows, p.positions, p.channels);
    }
    if (k != 0) {
        const size_t lds = unit_lds(p, VEC, false);
        with_rows(k, [&](auto rows) {
            with_flag(keep_here, [&](auto keep) {
                if constexpr (VEC > 1 || !keep.value)
                    launch(cl_unit_kernel<T, VEC, rows.value, keep.value>, dim3((uint32_t)(batch * p.chunks)), dim3(cl_lanes(p)), lds, stream,
                           x, chunk, CL_GEOMETRY_OF(p), a.gamma, a.beta, y, stats, a.codes, a.scales, eps, silu, p);
            });
        });
        return launch_status();
    }
    float2 *partials = static_cast<float2 *>(a.workspace), *joined = nullptr;
    const ClParts parts = {partials, p.slices, p.ty};
    const dim3 grid((uint32_t)(batch * p.chunks * p.slices)), block(cl_lanes(p));
    const size_t cc = chunk_channels(p, VEC);
    with_flag(chunk != nullptr, [&](auto add) {
        launch(cl_stats_kernel<T, VEC, add.value>, grid, block, 2 * (p.ty * cc + block.x) * sizeof(float), stream, x, chunk, CL_GEOMETRY_OF(p),
               partials, p);
    });
    if (joins(p)) {
        joined = join_launch<true>(p, parts, stats != nullptr ? stats : partials + partial_floats(p, batch) / 2, batch, eps, VEC, stream);
        stats = nullptr;
    }
    with_flag(chunk != nullptr, [&](auto add) {
        with_flag(silu, [&](auto act) {
            with_flag(keep_here, [&](auto keep) {
                if constexpr (VEC > 1 || !keep.value)
                    launch(cl_apply_kernel<T, VEC, add.value, act.value, keep.value>, grid, block,
                           std::min<size_t>(p.groups, cc) * sizeof(float2), stream, x, chunk, CL_GEOMETRY_OF(p), a.gamma, a.beta, y, parts,
                           joined, stats, a.codes, a.scales, eps, p);
            });
        });
    });
    return launch_status();
}

template <typename T, int VEC, int FROM>
int cl_backward_from(ClPlan p, const ClBackward &a, size_t batch, bool silu, hipStream_t stream) {
    const T *dy = static_cast<const T *>(a.dy);
    const void *h = FROM == kFromCodes ? a.codes : a.x, *more = FROM == kFromCodes ? a.scales : a.chunk;
    T *dx = static_cast<T *>(a.dx), *dchunk = static_cast<T *>(a.dchunk);
    const float2 *stats = reinterpret_cast<const float2 *>(a.stats);
    float *channel_sums = static_cast<float *>(a.workspace);
    const uint32_t tiles = (p.channels + kWave - 1) / kWave;
    if (const uint32_t k = unit_plan(&p, VEC, batch, true)) {
        const size_t lds = unit_lds(p, VEC, true);
        const bool affine = a.dgamma != nullptr, one = batch == 1;
        float *s1 = !affine ? nullptr : one ? a.dbeta : channel_sums, *s2 = !affine ? nullptr : one ? a.dgamma : channel_sums + p.channels;
        with_rows(k, [&](auto rows) {
            if constexpr (VEC < 8 || rows.value <= 2)
                launch(cl_unit_grads_kernel<T, VEC, rows.value, FROM>, dim3((uint32_t)(batch * p.chunks)), dim3(cl_lanes(p)), lds, stream, dy,
                       h, more, CL_GEOMETRY_OF(p), stats, a.gamma, a.beta, dx, s1, s2, dchunk, 2 * p.channels, silu, p);
        });
        if (affine && !one)
            launch(cl_affine_grads_kernel, dim3(tiles), dim3(kWave), 0, stream, channel_sums, a.dgamma, a.dbeta, (uint32_t)batch, p.channels);
        return launch_status();
    }
    if (!slice_plan(&p, VEC, batch)) return MSD_ERR_INVALID_VALUE;
    const size_t affine = a.dgamma != nullptr ? tiles : 0, added = dchunk != nullptr ? batch * tiles : 0;
    if (!fits_grid(affine + added + (uint64_t)batch * p.chunks * p.slices, cl_lanes(p))) return MSD_ERR_INVALID_VALUE;
    float2 *partials = reinterpret_cast<float2 *>(channel_sums + channel_floats(p, batch)), *joined = nullptr;
    const ClParts parts = {partials, p.slices, p.ty};
    const dim3 grid((uint32_t)(batch * p.chunks * p.slices)), block(cl_lanes(p));
    const size_t cc = chunk_channels(p, VEC);
    with_flag(silu, [&](auto act) {
        launch(cl_sums_kernel<T, VEC, FROM, act.value>, grid, block, 3 * p.ty * cc * sizeof(float), stream, dy, h, more,
               CL_GEOMETRY_OF(p), stats, a.gamma, a.beta, partials, channel_sums, p);
    });
    if (joins(p)) joined = join_launch<false>(p, parts, partials + partial_floats(p, batch) / 2, batch, 0.0f, VEC, stream);
    const ClChannelGrads grads = {channel_sums, a.dgamma, a.dbeta, dchunk, (uint32_t)affine, (uint32_t)batch};
    const uint32_t channel_blocks = (uint32_t)(affine + added);
    with_flag(silu, [&](auto act) {
        launch(cl_dx_kernel<T, VEC, FROM, act.value>, dim3(grid.x + channel_blocks), block, std::min<size_t>(p.groups, cc) * sizeof(float2),
               stream, dy, h, more, CL_GEOMETRY_OF(p), channel_blocks, stats, a.gamma, a.beta, dx, parts, joined, grads, p);
    });
    return launch_status();
}

template <typename T, int VEC>
int cl_backward(const ClPlan &p, const ClBackward &a, size_t batch, bool silu, hipStream_t stream) {
    if (a.codes != nullptr) return cl_backward_from<T, VEC, kFromCodes>(p, a, batch, silu, stream);
    if (a.chunk != nullptr) return cl_backward_from<T, VEC, kFromXAdd>(p, a, batch, silu, stream);
    return cl_backward_from<T, VEC, kFromX>(p, a, batch, silu, stream);
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
    size_t most = 16;  // (never nothing)
    for (const bool vectors : {false, true}) {  // (what the operands' alignment allows is not known here)
        ClPlan p;
        uint32_t vec;
        if (!cl_shape(elt, batch, positions, channels, groups, vectors, &p, &vec)) return SIZE_MAX;
        if (unit_plan(&p, vec, batch, backward) != 0) {
            if (backward) most = std::max(most, 2 * batch * channels * sizeof(float));
            continue;
        }
        if (!slice_plan(&p, vec, batch)) return SIZE_MAX;
        most = std::max(most, (partial_floats(p, batch) + (joins(p) ? joined_floats(p, batch) : 0) + (backward ? channel_floats(p, batch) : 0)) * sizeof(float));
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
    if (!cl_shape(sizeof(T), batch, positions, channels, groups, vectors, &p, &vec)) return MSD_ERR_INVALID_VALUE;
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
        if (!fits_grid((most + 255) / 256, 256)) return MSD_ERR_INVALID_VALUE;
        if (most != 0)
            launch(cl_zero_kernel<T>, dim3((uint32_t)((most + 255) / 256)), dim3(256), 0, stream, a.dgamma, a.dbeta,
                   static_cast<T *>(a.dchunk), channels, added);
        return launch_status();
    }
    ClPlan p;
    uint32_t vec;
    const bool vectors = all_aligned16({a.dy, a.x, a.chunk, a.codes, a.dx});
    if (!cl_shape(sizeof(T), batch, positions, channels, groups, vectors, &p, &vec)) return MSD_ERR_INVALID_VALUE;
    return vec == 1 ? cl_backward<T, 1>(p, a, batch, silu, stream) : cl_backward<T, 16 / sizeof(T)>(p, a, batch, silu, stream);
}
template int cl_backward_dispatch<float>(const ClBackward &, size_t, size_t, size_t, size_t, bool, hipStream_t);
template int cl_backward_dispatch<__half>(const ClBackward &, size_t, size_t, size_t, size_t, bool, hipStream_t);

}  // namespace msd
