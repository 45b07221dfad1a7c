// Gradient of LayerNorm for gfx950.  With u = (x - mean) rstd and w = dy gamma, a row gives
//     dx = rstd (w - mean(w) - u mean(w u)) (+ dsum),   dgamma += dy u,   dbeta += dy.
// A row is owned by TL lanes (of one wavefront, or the 256 of a workgroup for long rows), K accesses of N elements each; x and
// dy stay in registers, so each is read once.  mean and rstd come from x again, in two passes over the registers: two
// reductions more per row, where keeping them would change the forward call and add a read.  A lane owns the same columns in
// every row that it handles, so dgamma and dbeta gather in its registers over the rows; a workgroup adds its teams through LDS
// and writes one row of partial sums, and a second launch adds those in order: no atomics, the same bits every time.
//
// Measured: 65536 x 320 float16 with dsum 34 us (168 MB, 4.9 TB/s, the rate of a large copy) and 4.8 for the sums of the partial rows;
// 2049 x 777 float32 with dsum 10.5 us (rows of no whole vectors: single values) and 4.4; 154 x 768 float32 4.3 and 2.3, latency.
#include <algorithm>

#include "msd_device.h"
#include "msd_internal.h"

namespace msd {
namespace {

constexpr uint32_t kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// N elements of T as one access (N = 1: a scalar, for rows of no whole vectors or unaligned tensors).
template <typename T, int N>
struct Piece {
    u32x4 v;
    __device__ __forceinline__ void load(const T *p) { v = load_stream(reinterpret_cast<const u32x4 *>(p)); }
    __device__ __forceinline__ void clear() { v = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void unpack(float *f) const { Store<T>::unpack(v, f); }
    static __device__ __forceinline__ void store(T *p, const float *f) {
        store_stream(reinterpret_cast<u32x4 *>(p), Store<T>::pack(f));
    }
};
template <typename T>
struct Piece<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T *p) { v = *p; }
    __device__ __forceinline__ void clear() { v = T(0.0f); }
    __device__ __forceinline__ void unpack(float *f) const { f[0] = Store<T>::load1(&v); }
    static __device__ __forceinline__ void store(T *p, const float *f) { Store<T>::store1(p, f[0]); }
};

// Sum over a row's team: lanes of a wavefront, or the workgroup (`slots`: kWaves floats of LDS per reduction in flight).
template <int TL>
__device__ __forceinline__ float row_sum(float v, float *slots) {
    if constexpr (TL < (int)kThreads) {
        return team_sum<TL>(v);
    } else {
        return block_sum<kWaves>(v, slots);
    }
}

// Three at once.
template <int TL>
__device__ __forceinline__ void row_sums(float &a, float &b, float &c, float *slots) {
    a = team_sum<TL < (int)kThreads ? TL : kWave>(a);
    b = team_sum<TL < (int)kThreads ? TL : kWave>(b);
    c = team_sum<TL < (int)kThreads ? TL : kWave>(c);
    if constexpr (TL == (int)kThreads) {
        if (threadIdx.x % kWave == 0) {
            slots[threadIdx.x / kWave] = a;
            slots[kWaves + threadIdx.x / kWave] = b;
            slots[2 * kWaves + threadIdx.x / kWave] = c;
        }
        __syncthreads();
        a = b = c = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            a += slots[i];
            b += slots[kWaves + i];
            c += slots[2 * kWaves + i];
        }
    }
}

// The rows of workgroup b: teams of it take rows b * teams + team, and so on by gridDim.x * teams.  Each keeps the next row's
// loads in flight while it works on one.  partial: [gridDim.x][2][dim] or null (dgamma and dbeta not wanted).
template <typename T, int N, int K, int TL>
__global__ __launch_bounds__(kThreads) void ln_grad_kernel(const T *dy, const T *x, const T *dsum, const float *__restrict__ gamma,
                                                           T *dx, float *partial, uint32_t rows, uint32_t dim, float eps,
                                                           float inv_dim) {
    constexpr uint32_t kTeams = kThreads / TL;
    // the columns' sums of the teams, one part of a lane's pieces at a time; before that the slots of the row sums
    __shared__ float lds[2 * kThreads * N];
    const uint32_t team = threadIdx.x / TL, j = threadIdx.x % TL;
    const uint32_t stride = gridDim.x * kTeams;
    float g[K][N], sum_g[K][N], sum_b[K][N];
    bool in[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t col = (k * TL + j) * N;
        in[k] = col < dim;  // (a whole piece: dim is a multiple of N)
#pragma unroll
        for (int e = 0; e < N; e++) {
            g[k][e] = in[k] ? gamma[col + e] : 0.0f;
            sum_g[k][e] = sum_b[k][e] = 0.0f;
        }
    }
    Piece<T, N> px[K], pd[K], ps[K];
    auto fetch = [&](uint32_t row) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t at = (size_t)row * dim + (k * TL + j) * N;
            px[k].clear();
            pd[k].clear();
            ps[k].clear();
            if (in[k]) {
                px[k].load(x + at);
                pd[k].load(dy + at);
                if (dsum != nullptr) ps[k].load(dsum + at);
            }
        }
    };
    uint32_t row = blockIdx.x * kTeams + team;
    // every lane of a workgroup takes the same number of turns (long rows meet at barriers); a team past the last row
    // works on zeros
    const uint32_t first = blockIdx.x * kTeams;
    const uint32_t turns = first < rows ? (rows - first + stride - 1) / stride : 0;
    auto fetch_live = [&](uint32_t r) {
        if (r < rows) {
            fetch(r);
        } else {
#pragma unroll
            for (int k = 0; k < K; k++) {
                px[k].clear();
                pd[k].clear();
                ps[k].clear();
            }
        }
    };
    if (turns != 0) fetch_live(row);
    for (uint32_t turn = 0; turn < turns; turn++, row += stride) {
        float f[K][N], d[K][N], s[K][N];
#pragma unroll
        for (int k = 0; k < K; k++) {
            px[k].unpack(f[k]);
            pd[k].unpack(d[k]);
            ps[k].unpack(s[k]);
        }
        if (turn + 1 < turns) fetch_live(row + stride);
        float *const slots = lds + (turn & 1) * 4 * kWaves;
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < N; e++) t += f[k][e];
        const float mean = row_sum<TL>(t, slots) * inv_dim;
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                f[k][e] = in[k] ? f[k][e] - mean : 0.0f;
                q = fmaf(f[k][e], f[k][e], q);
            }
        float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float w = d[k][e] * g[k][e];
                m1 += w;
                m2 = fmaf(w, f[k][e], m2);
            }
        // (three sums side by side: a row waits for two rounds of reductions in all)
        row_sums<TL>(q, m1, m2, slots + kWaves);
        // (the zeros of a team past the last row: 1 / sqrt(eps) times them is NaN for eps = 0, and the sums over rows take in every team)
        const float rstd = row < rows ? __builtin_amdgcn_rsqf(q * inv_dim + eps) : 0.0f;
        m1 *= inv_dim;
        m2 *= rstd * inv_dim;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                f[k][e] *= rstd;
                sum_g[k][e] = fmaf(d[k][e], f[k][e], sum_g[k][e]);
                sum_b[k][e] += d[k][e];
                d[k][e] *= g[k][e];
            }
        if (row < rows) {
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int e = 0; e < N; e++) s[k][e] = fmaf(rstd, d[k][e] - m1 - f[k][e] * m2, s[k][e]);
                if (in[k]) Piece<T, N>::store(dx + (size_t)row * dim + (k * TL + j) * N, s[k]);
            }
        }
    }
    if (partial == nullptr) return;
    float *const to_g = partial + (size_t)blockIdx.x * 2 * dim, *const to_b = to_g + dim;
#pragma unroll
    for (int k = 0; k < K; k++) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; e++) {
            lds[e * kThreads + threadIdx.x] = sum_g[k][e];
            lds[(N + e) * kThreads + threadIdx.x] = sum_b[k][e];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (uint32_t)TL * N; i += kThreads) {
            const uint32_t e = i % N, lane = i / N, col = (k * TL + lane) * N + e;
            float a = 0.0f, b = 0.0f;
            for (uint32_t t = 0; t < kTeams; t++) {
                a += lds[e * kThreads + t * TL + lane];
                b += lds[(N + e) * kThreads + t * TL + lane];
            }
            if (col < dim) {
                to_g[col] = a;
                to_b[col] = b;
            }
        }
    }
}

// Columns of the partial rows, added in order: 32 columns and 32 runs of rows to a workgroup.
constexpr uint32_t kJoinThreads = 1024, kJoinColumns = 32, kJoinRuns = kJoinThreads / kJoinColumns;
__global__ __launch_bounds__(kJoinThreads) void ln_grad_join_kernel(const float *partial, float *dgamma, float *dbeta, uint32_t parts,
                                                                    uint32_t dim) {
    __shared__ float lds[kJoinRuns][kJoinColumns + 1];
    const uint32_t lane = threadIdx.x % kJoinColumns, run = threadIdx.x / kJoinColumns;
    const uint32_t col = blockIdx.x * kJoinColumns + lane;  // of [dgamma | dbeta]
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < 2 * dim) {
        const uint32_t each = (parts + kJoinRuns - 1) / kJoinRuns, last = min(parts, (run + 1) * each);
        for (uint32_t p = run * each; p < last; p += 8)
#pragma unroll
            for (int i = 0; i < 8; i++) t[i % 4] += p + i < last ? partial[(size_t)(p + i) * 2 * dim + col] : 0.0f;
    }
    lds[run][lane] = (t[0] + t[1]) + (t[2] + t[3]);
    __syncthreads();
    if (run != 0 || col >= 2 * dim) return;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kJoinRuns; i++) sum += lds[i][lane];
    if (col < dim)
        dgamma[col] = sum;
    else
        dbeta[col - dim] = sum;
}

// ---- rows that no team's registers hold: statistics, the columns' sums, dx, each in a pass of its own ----
template <typename T>
__global__ __launch_bounds__(kThreads) void ln_grad_long_stats_kernel(const T *dy, const T *x, const float *__restrict__ gamma,
                                                                      f32x4 *stats, uint32_t rows, uint32_t dim, float eps) {
    __shared__ float lds[4 * kWaves];
    const float inv_dim = 1.0f / (float)dim;
    const T *xr = x + (size_t)blockIdx.x * dim, *dr = dy + (size_t)blockIdx.x * dim;
    float t = 0.0f;
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) t += Store<T>::load1(xr + i);
    const float mean = block_sum<kWaves>(t, lds) * inv_dim;
    float q = 0.0f;
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
        const float d = Store<T>::load1(xr + i) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = __builtin_amdgcn_rsqf(block_sum<kWaves>(q, lds + kWaves) * inv_dim + eps);
    float m1 = 0.0f, m2 = 0.0f;
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
        const float w = Store<T>::load1(dr + i) * gamma[i];
        m1 += w;
        m2 = fmaf(w, (Store<T>::load1(xr + i) - mean) * rstd, m2);
    }
    m1 = block_sum<kWaves>(m1, lds + 2 * kWaves) * inv_dim;
    m2 = block_sum<kWaves>(m2, lds + 3 * kWaves) * inv_dim;
    if (threadIdx.x == 0) stats[blockIdx.x] = f32x4{mean, rstd, m1, m2};
}

// A column per lane; blockIdx.y takes the rows y, y + gridDim.y, ...
template <typename T>
__global__ __launch_bounds__(kThreads) void ln_grad_long_columns_kernel(const T *dy, const T *x, const f32x4 *stats, float *partial,
                                                                        uint32_t rows, uint32_t dim) {
    const uint32_t col = blockIdx.x * kThreads + threadIdx.x;
    if (col >= dim) return;
    float a = 0.0f, b = 0.0f;
    for (uint32_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const f32x4 st = stats[row];
        const float d = Store<T>::load1(dy + (size_t)row * dim + col);
        a = fmaf(d, (Store<T>::load1(x + (size_t)row * dim + col) - st[0]) * st[1], a);
        b += d;
    }
    partial[(size_t)blockIdx.y * 2 * dim + col] = a;
    partial[((size_t)blockIdx.y * 2 + 1) * dim + col] = b;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_grad_long_dx_kernel(const T *dy, const T *x, const T *dsum,
                                                                   const float *__restrict__ gamma, const f32x4 *stats, T *dx,
                                                                   uint32_t dim) {
    const f32x4 st = stats[blockIdx.x];
    const size_t base = (size_t)blockIdx.x * dim;
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
        const float u = (Store<T>::load1(x + base + i) - st[0]) * st[1];
        const float w = Store<T>::load1(dy + base + i) * gamma[i];
        const float s = dsum != nullptr ? Store<T>::load1(dsum + base + i) : 0.0f;
        Store<T>::store1(dx + base + i, fmaf(st[1], w - st[2] - u * st[3], s));
    }
}

// ---- plan ------------------------------------------------------------------
constexpr uint32_t kLongParts = 64;  // runs of rows in the columns' pass over long rows

struct Plan {
    int n, k, tl;     // elements per access, accesses per lane, lanes per row; tl == 0: long rows
    uint32_t blocks;  // workgroups, each with a row of partial sums
};

// Accesses per lane of vectors: four of float16 (32 values in float32, twice, beside the sums over rows) leave a wavefront alone on its
// SIMD.  With three at most, and more lanes to a row, 65536 x 512 and 16384 x 2048 float16 with dsum take 52.5 and 61.0 us, with four
// 68.5 and 68.9.
constexpr int most_accesses(int n, int lanes) { return n == 8 && lanes < 256 ? 3 : 4; }

// The accesses per lane that kernels exist for.
int round_k(int n, uint32_t k, int lanes) {
    if (n > 1) return (int)k <= most_accesses(n, lanes) ? (int)k : 0;
    for (const int have : {1, 2, 4, 8, 16})
        if (k <= (uint32_t)have) return have;
    return 0;
}

Plan make_plan(size_t elt, size_t rows, size_t dim, bool aligned) {
    const int n = aligned && dim * elt % 16 == 0 ? (int)(16 / elt) : 1;
    Plan p{n, 0, 0, kLongParts};
    const size_t pieces = dim / n;
    // the fewest lanes whose registers hold the row, from a quarter of a wavefront on
    for (const int tl : {16, 32, 64, 256}) {
        if (pieces > (size_t)tl * 16 || (n == 1 && tl < 64)) continue;
        p.k = round_k(n, (uint32_t)((pieces + tl - 1) / tl), tl);
        if (p.k == 0) continue;
        p.tl = tl;
        break;
    }
    if (p.tl == 0) return p;
    const size_t teams = kThreads / p.tl, most = (rows + teams - 1) / teams;
    p.blocks = (uint32_t)std::max<size_t>(1, std::min<size_t>(most, 2 * (size_t)chip_info().cus));
    return p;
}

struct Args {
    const void *dy, *x, *dsum;
    const float *gamma;
    void *dx;
    float *partial;
    uint32_t rows, dim;
    float eps;
    hipStream_t stream;
};

template <typename T, int N, int K, int TL>
void launch_rows(const Args &a, uint32_t blocks) {
    launch((ln_grad_kernel<T, N, K, TL>), dim3(blocks), dim3(kThreads), 0, a.stream, static_cast<const T *>(a.dy),
           static_cast<const T *>(a.x), static_cast<const T *>(a.dsum), a.gamma, static_cast<T *>(a.dx), a.partial, a.rows, a.dim,
           a.eps, 1.0f / (float)a.dim);
}

// (the accesses per lane that make_plan gives to a number of lanes)
template <typename T, int TL>
void launch_vectors(const Args &a, const Plan &p) {
    constexpr int N = Store<T>::EPV, kMost = most_accesses(N, TL), kFewer = TL == 256 ? 64 : TL / 2;
    constexpr int kLeast = TL == 16 ? 1 : most_accesses(N, kFewer) * kFewer / TL + 1;
    if constexpr (kLeast <= 1) {
        if (p.k == 1) return launch_rows<T, N, 1, TL>(a, p.blocks);
    }
    if constexpr (kLeast <= 2) {
        if (p.k == 2) return launch_rows<T, N, 2, TL>(a, p.blocks);
    }
    if constexpr (kMost > 3) {
        if (p.k == 4) return launch_rows<T, N, 4, TL>(a, p.blocks);
    }
    launch_rows<T, N, 3, TL>(a, p.blocks);
}

template <typename T, int TL>
void launch_scalars(const Args &a, const Plan &p) {
    if constexpr (TL == 64) {
        switch (p.k) {
            case 1: return launch_rows<T, 1, 1, TL>(a, p.blocks);
            case 2: return launch_rows<T, 1, 2, TL>(a, p.blocks);
            case 4: return launch_rows<T, 1, 4, TL>(a, p.blocks);
            default: break;
        }
    }
    if (p.k == 8) return launch_rows<T, 1, 8, TL>(a, p.blocks);
    launch_rows<T, 1, 16, TL>(a, p.blocks);
}

__global__ __launch_bounds__(kThreads) void ln_grad_zero_kernel(float *dgamma, float *dbeta, uint32_t dim) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i < dim) dgamma[i] = dbeta[i] = 0.0f;
}

}  // namespace

size_t ln_grad_workspace_bytes(size_t elt, size_t rows, size_t dim) {
    if (rows > 0x7FFFFFFFull || dim > 0x3FFFFFFFull) return SIZE_MAX;
    if (rows == 0 || dim == 0) return 0;
    // (room for either alignment: which of the two kernels runs is known only with the pointers)
    size_t need = 0;
    for (const bool aligned : {false, true}) {
        const Plan p = make_plan(elt, rows, dim, aligned);
        need = std::max(need, (size_t)p.blocks * 2 * dim * sizeof(float) + (p.tl == 0 ? rows * sizeof(f32x4) : 0));
    }
    return need;
}

template <typename T>
int ln_grad_dispatch(const LnGrad &g, size_t rows, size_t dim, float eps, hipStream_t stream) {
    if (dim == 0) return MSD_OK;
    if (rows == 0) {
        if (g.dgamma != nullptr)
            launch(ln_grad_zero_kernel, dim3((uint32_t)((dim + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, g.dgamma,
                   g.dbeta, (uint32_t)dim);
        return launch_status();
    }
    const bool aligned = aligned16(g.dy) && aligned16(g.x) && aligned16(g.dx) && aligned16(g.dsum);
    Plan p = make_plan(sizeof(T), rows, dim, aligned);
    const size_t room = (g.workspace_bytes - (p.tl == 0 ? rows * sizeof(f32x4) : 0)) / (2 * dim * sizeof(float));
    p.blocks = (uint32_t)std::min<size_t>(p.blocks, room);
    const bool affine = g.dgamma != nullptr;
    f32x4 *const stats = static_cast<f32x4 *>(g.workspace);
    float *const partial = static_cast<float *>(g.workspace) + (p.tl == 0 ? 4 * rows : 0);
    const Args a{g.dy, g.x, g.dsum, g.gamma, g.dx, affine ? partial : nullptr, (uint32_t)rows, (uint32_t)dim, eps, stream};
    if (p.tl == 0) {
        const T *dy = static_cast<const T *>(g.dy), *x = static_cast<const T *>(g.x);
        launch((ln_grad_long_stats_kernel<T>), dim3(a.rows), dim3(kThreads), 0, stream, dy, x, g.gamma, stats, a.rows, a.dim, eps);
        if (affine)  // (before dx, which may take the place of dy)
            launch((ln_grad_long_columns_kernel<T>), dim3((a.dim + kThreads - 1) / kThreads, p.blocks), dim3(kThreads), 0, stream, dy,
                   x, stats, partial, a.rows, a.dim);
        launch((ln_grad_long_dx_kernel<T>), dim3(a.rows), dim3(kThreads), 0, stream, dy, x, static_cast<const T *>(g.dsum), g.gamma,
               stats, static_cast<T *>(g.dx), a.dim);
    } else if (p.n > 1) {
        switch (p.tl) {
            case 16: launch_vectors<T, 16>(a, p); break;
            case 32: launch_vectors<T, 32>(a, p); break;
            case 64: launch_vectors<T, 64>(a, p); break;
            default: launch_vectors<T, 256>(a, p); break;
        }
    } else if (p.tl == 64) {
        launch_scalars<T, 64>(a, p);
    } else {
        launch_scalars<T, 256>(a, p);
    }
    if (affine)
        launch(ln_grad_join_kernel, dim3((2 * a.dim + kJoinColumns - 1) / kJoinColumns), dim3(kJoinThreads), 0, stream, partial, g.dgamma,
               g.dbeta, p.blocks, a.dim);
    return launch_status();
}

template int ln_grad_dispatch<float>(const LnGrad &, size_t, size_t, float, hipStream_t);
template int ln_grad_dispatch<__half>(const LnGrad &, size_t, size_t, float, hipStream_t);

}  // namespace msd
