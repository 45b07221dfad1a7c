// Gradient of attention for gfx950.  With p as in the forward call (formed again from its log2 sums) and D_i = do_i . out_i,
//     dS_ij = p_ij (do_i . v_j - D_i),   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i p_ij do_i.
// A launch for D (and row norms); dq with a workgroup for rows, over the keys, as the forward call; dk and dv with a workgroup for
// keys, over the rows: one launch or one for each.  Each gradient is owned by one workgroup, so nothing is added by atomics, at the
// price of forming S and dO V^T twice (7 products for 5).  The heads of a key head are rows of the same tiles, so their gradients
// add up in the accumulators.  Where either kind of workgroup is few, its rows or keys are cut into parts, joined by another launch.
//
// Measured (10 d operations for each visible pair):
//   float16, 4 x 4000 causal, 16 heads of 128 on 4: D 41 us (at the rate of a large copy), dk and dv 670 and their join 34, dq 420:
//     595 TFLOP/s.  4 x 4096, 32 heads on 8: 4.08 ms, 674.  dk and dv hold 254 of 256 registers: waits for operands and tiles are
//     36 % of a wavefront's cycles, matrix instructions 42 % of the SIMD's.
//   float16, 8 x 4096, 16 heads of 64: 2.36 ms, 582 TFLOP/s; 2 x 4096 rows over 77 keys, 5 heads of 64: 36 us.
//   float32, 32 sequences of up to 77, 12 heads of 64: 4 and 23 us; a launch's fixed 6, the wavefronts' own first rows, then 5 a tile.
//   float32, 2 x 2048 causal, 8 heads: 67 TFLOP/s with 64 columns, 78 with 128.
//
// float16: dS is rounded to float16 for its product, after a power of two that brings the largest it can be,
// |do_i| max |v_j| + |D_i|, next to 2^14: it keeps 11 bits down to 2^-28 of that, whatever the gradients' size.  Each row of dq
// and each key of dk and dv has a power of its own, from what it sees alone; it follows the largest bound so far, and the sums
// are scaled down where it moves.
#include <algorithm>
#include <type_traits>

#include "attention_tiles.h"

namespace msd {
namespace {

struct Backward {
    AttnShape s;
    AttnView q, k, v, out, dout, dq, dk, dv;
    const float *lse;
    const void *rest;  // [rows][heads][dim] what rounding took from out, or null
    // [rows][heads] what the weights' exponents take (kPShift less the log2 sum), D and |do|, [keys][kv_heads] |v|; the norms null
    // for float32
    float *base, *delta, *norm, *v_norm;
    float *part, *q_part;  // parts > 1: [parts][keys][kv_heads][dk, dv][dim]; q_parts > 1: [q_parts][rows][heads][dim]
    uint32_t total_rows, total_keys, parts, q_parts, kv_blocks;
    bool vec;
};

// kPShift: float16 weights are kept that many powers of two larger where they are an operand themselves (they are at most 1).
template <typename T>
constexpr int kPShift = Frag<T>::kFloat ? 0 : 15;

// 16 lanes to a row of a head.
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attn_grad_rows_kernel(const Backward a) {
    constexpr uint32_t E = 16 / sizeof(T), kTeam = 16;
    const size_t at = (size_t)blockIdx.x * (kAttnThreads / kTeam) + threadIdx.x / kTeam;
    const size_t rows = (size_t)a.total_rows * a.s.heads, keys = a.v_norm != nullptr ? (size_t)a.total_keys * a.s.kv_heads : 0;
    if (at >= rows + keys) return;
    const bool of_keys = at >= rows;
    const size_t item = of_keys ? at - rows : at;
    const uint32_t heads = of_keys ? a.s.kv_heads : a.s.heads;
    const uint32_t row = (uint32_t)(item / heads), head = (uint32_t)(item % heads);
    auto address = [&](const AttnView &v, const int32_t *offsets, uint32_t each) {
        const uint32_t b = offsets != nullptr ? 0 : row / each, i = offsets != nullptr ? row : row % each;
        return static_cast<const T *>(v.at) + b * v.batch + (size_t)i * v.row + head * v.head;
    };
    const T *first, *second;
    if (of_keys) {
        first = second = address(a.v, a.s.k_offsets, a.s.k_rows);
    } else {
        first = address(a.dout, a.s.q_offsets, a.s.q_rows);
        second = address(a.out, a.s.q_offsets, a.s.q_rows);
    }
    const T *const rest = !of_keys && a.rest != nullptr ? static_cast<const T *>(a.rest) + item * a.s.dim : nullptr;
    float dot = 0.0f, square = 0.0f;
    for (uint32_t d = threadIdx.x % kTeam * E; d < a.s.dim; d += kTeam * E) {
        float x[E], y[E];
        Store<T>::unpack(a.vec ? *reinterpret_cast<const u32x4 *>(first + d) : load_chunk<T>(first, d, a.s.dim), x);
        Store<T>::unpack(a.vec ? *reinterpret_cast<const u32x4 *>(second + d) : load_chunk<T>(second, d, a.s.dim), y);
#pragma unroll
        for (uint32_t e = 0; e < E; e++) {
            dot = fmaf(x[e], y[e], dot);
            square = fmaf(x[e], x[e], square);
        }
        if (rest != nullptr) {
            Store<T>::unpack(a.vec ? *reinterpret_cast<const u32x4 *>(rest + d) : load_chunk<T>(rest, d, a.s.dim), y);
#pragma unroll
            for (uint32_t e = 0; e < E; e++) dot = fmaf(x[e], y[e], dot);
        }
    }
    dot = team_sum<16>(dot);
    square = team_sum<16>(square);
    if (threadIdx.x % kTeam != 0) return;
    if (of_keys) {
        a.v_norm[item] = sqrtf(square);
    } else {
        const float lse = a.lse[item];
        a.base[item] = lse == -__builtin_inff() ? lse : (float)kPShift<T> - lse;  // (a row that sees nothing: weights of zero)
        a.delta[item] = dot;
        if (a.norm != nullptr) a.norm[item] = sqrtf(square);
    }
}

// Largest of the (not negative) values of the lanes up to this one.
__device__ __forceinline__ float max_up_to(float v) {
    v = fmaxf(v, dpp_move<0x111>(v));  // from 1, 2, 4 and 8 lanes below, within 16
    v = fmaxf(v, dpp_move<0x112>(v));
    v = fmaxf(v, dpp_move<0x114>(v));
    v = fmaxf(v, dpp_move<0x118>(v));
    // the last lane of the 16 below, for the odd ones of four; the last of the lower 32, for the upper ones
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xA, 0xF, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xC, 0xF, true)));
    return v;
}

// A lane's power of two for dS of up to `bound`; where that lowers any lane's, its sums are to be scaled by `down`.  (A bound of 0, of
// rows that the loss leaves out, says nothing of the size of others.)
struct DsScale {
    int power = 100;
    __device__ __forceinline__ bool lower(float bound, float &down) {
        const int p = bound > 0.0f ? min(power, max(-100, min(100, 14 - __builtin_amdgcn_frexp_expf(bound)))) : power;
        if (__builtin_amdgcn_ballot_w64(p < power) == 0) return false;
        down = ldexpf(1.0f, max(-126, p - power));
        power = p;
        return true;
    }
};

// Whether a sequence's float16 score gradients go into their products in two parts, the rounded value and what it left.  The
// roundings of one part are as large as that of the result itself, 1.41 times it together, where many terms make a sum;
// of few terms, or of few columns (dS sums to zero over the keys, and what is left of such sums is smaller), they come to 1.7 times
// and more.  Longer sequences have the second part in the tiles that the mask cuts alone: 9 products for 7 take 1.2 times as long.
__device__ __forceinline__ bool few_terms(uint32_t lq, uint32_t lk, uint32_t dim) { return min(lq, lk) < 512 || dim <= 48; }

// The part of registers 8 u ... 8 u + 7 that their rounding to `f` left.
__device__ __forceinline__ void left_by(const half8 &f, int u, f32x16 &c) {
#pragma unroll
    for (int j = 0; j < 8; j++) c[8 * u + j] -= (float)f[j];
}
[[maybe_unused]] __device__ __forceinline__ void left_by(const Thirds &, int, f32x16 &) {}

// dq: the forward kernel's tiles of rows over tiles of keys.
template <typename T, int D, int WAVES>
struct ForQ {
    Tile<T, D, WAVES> tiles[2][2];  // [buffer][K, V]
};
template <typename T, int D, int WAVES>
__device__ __forceinline__ void attn_grad_q(const Backward &a, const uint32_t block, ForQ<T, D, WAVES> &lds) {
    typedef typename Frag<T>::type frag;
    typedef typename Frag<T>::operand operand_t;
    typedef Tile<T, D, WAVES> KvTile;
    constexpr uint32_t kOwn = 32 * WAVES;
    constexpr bool kHalf = !Frag<T>::kFloat;
    // Operands from LDS are read a step ahead, in this order: there are registers for that, not for the compiler's choice, which
    // waits for most reads right behind them.
    constexpr bool kAhead = kHalf && D == 128;
    constexpr int R = KvTile::kRows, KD = D / 16, DB = D / 32;
    KvTile(&tiles)[2][2] = lds.tiles;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, h = lane / 32;
    const TileLanes<T, D> lanes;
    const uint32_t rest = fast_div(block, a.s.by_kv_heads), head = block - rest * a.s.kv_heads;
    const uint32_t tiles_at = a.q_parts == 1 ? rest : rest / a.q_parts, part = rest - tiles_at * a.q_parts;
    uint32_t b, tile, q0, lq, k0, lk;
    if (!find_tile(a.s.q_offsets, a.s.batch, a.s.q_rows, a.s.group, kOwn, tiles_at, a.s.q_by_tile, b, tile)) return;
    span(a.s.q_offsets, b, a.s.q_rows, q0, lq);
    span(a.s.k_offsets, b, a.s.k_rows, k0, lk);
    const uint32_t rows = lq * a.s.group;
    if (a.s.causal) tile = (rows + kOwn - 1) / kOwn - 1 - tile;
    const bool packed = a.s.q_offsets != nullptr;
    const uint32_t row = tile * kOwn + wave * 32 + lane % 32;
    const uint32_t i = fast_div(row, a.s.by_group), qh = head * a.s.group + row - i * a.s.group;
    const bool live = row < rows;
    auto seen_by = [&](uint32_t query) -> uint32_t {
        return a.s.causal ? (uint32_t)max((int64_t)0, min((int64_t)lk, (int64_t)query + 1 + lk - lq)) : lk;
    };
    const uint32_t limit = live ? seen_by(i) : 0;
    auto at_row = [&](const AttnView &v) {
        return static_cast<const T *>(v.at) + (packed ? 0 : b * v.batch) + (size_t)(q0 + i) * v.row + qh * v.head;
    };
    const T *kbase = static_cast<const T *>(a.k.at) + (packed ? 0 : b * a.k.batch) + (size_t)k0 * a.k.row + head * a.k.head;
    const T *vbase = static_cast<const T *>(a.v.at) + (packed ? 0 : b * a.v.batch) + (size_t)k0 * a.v.row + head * a.v.head;
    operand_t q[KD], g[KD];
    load_frags<T, D>(live ? at_row(a.q) : nullptr, a.s.dim, a.vec, q);
    load_frags<T, D>(live ? at_row(a.dout) : nullptr, a.s.dim, a.vec, g);
    const size_t place = ((size_t)(packed ? 0 : b) * lq + q0 + i) * a.s.heads + qh;
    const float base = live ? a.base[place] - (float)kPShift<T> : 0.0f, delta = live ? a.delta[place] : 0.0f;
    const float norm = kHalf && live ? a.norm[place] : 0.0f;
    const float *const v_norm = kHalf ? a.v_norm + ((size_t)(packed ? 0 : b) * lk + k0) * a.s.kv_heads + head : nullptr;

    const uint32_t last_row = min(rows, (tile + 1) * kOwn) - 1;
    const uint32_t all = (seen_by(fast_div(last_row, a.s.by_group)) + R - 1) / R, each = (all + a.q_parts - 1) / a.q_parts;
    const uint32_t t0 = min(all, part * each), t1 = min(all, t0 + each);
    const uint32_t wave_row = tile * kOwn + wave * 32;
    const uint32_t wave_limit = wave_row < rows ? seen_by(fast_div(min(rows - 1, wave_row + 31), a.s.by_group)) : 0;
    const uint32_t wave_full = wave_row < rows ? seen_by(fast_div(wave_row, a.s.by_group)) : 0;

    uint32_t k_base[KvTile::kTurn], v_base[KvTile::kTurn];
    const uint32_t k_row = (uint32_t)a.k.row, v_row = (uint32_t)a.v.row;
    KvTile::offsets(k_row, a.s.dim, k_base);
    KvTile::offsets(v_row, a.s.dim, v_base);
    float next_norm = 0.0f;
    auto fetch = [&](uint32_t t, uint32_t buffer) {
        if (kHalf) next_norm = t * R + lane < lk ? v_norm[(size_t)(t * R + lane) * a.s.kv_heads] : 0.0f;
        const T *const kt = kbase + (size_t)t * R * a.k.row, *const vt = vbase + (size_t)t * R * a.v.row;
        const uint32_t n = min(lk - t * R, (uint32_t)R);
        if (a.vec) {
            tiles[buffer][0].request(kt, (uint32_t)(((n - 1) * a.k.row + a.s.dim) * sizeof(T)),
                                     [&](int p) { return KvTile::offset_of(k_base, k_row, p); });
            tiles[buffer][1].request(vt, (uint32_t)(((n - 1) * a.v.row + a.s.dim) * sizeof(T)),
                                     [&](int p) { return KvTile::offset_of(v_base, v_row, p); });
        } else {
            tiles[buffer][0].copy([&](uint32_t r) -> const T * { return r < n ? kt + r * a.k.row : nullptr; }, a.s.dim);
            tiles[buffer][1].copy([&](uint32_t r) -> const T * { return r < n ? vt + r * a.v.row : nullptr; }, a.s.dim);
        }
    };
    const bool few = kHalf && few_terms(lq, lk, a.s.dim);
    f32x16 dq[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) dq[d] = zero16();
    DsScale scale;
    if (t0 < t1) fetch(t0, 0);
    for (uint32_t t = t0; t < t1; t++) {
        const float v_norms = next_norm;  // (of the tile's keys, one to a lane)
        wait_tiles();
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1, (t + 1 - t0) & 1);
        const KvTile &kt = tiles[(t - t0) & 1][0], &vt = tiles[(t - t0) & 1][1];
        const uint32_t first = t * R;
        if (first < wave_limit) {
            auto work = [&](auto with_masked) {  // (apart for tiles with masked pairs, as in the forward call)
                constexpr bool MASKED = decltype(with_masked)::value;
                float by = 1.0f;
                bool odd = false;
                if (kHalf) {
                    float down, v_most;
                    if constexpr (MASKED) {
                        const float upto = __shfl(max_up_to(v_norms), (int)min(limit - first - 1, (uint32_t)R - 1), kWave);
                        v_most = first < limit ? upto : 0.0f;
                    } else {
                        v_most = team_max<64>(v_norms);
                    }
                    if (scale.lower(fmaf(norm, v_most, fabsf(delta)), down)) {
#pragma unroll
                        for (int d = 0; d < DB; d++)
#pragma unroll
                            for (int r = 0; r < 16; r++) dq[d][r] *= down;
                    }
                    by = ldexpf(1.0f, scale.power);
                }
                const float delta_by = delta * by;
#pragma unroll
                for (int n = 0; n < R / 32; n++) {
                    f32x16 s = zero16(), dp = zero16();
                    if constexpr (kAhead) {
                        frag kc = kt.rows(lanes, 32 * n, 0), vc = vt.rows(lanes, 32 * n, 0);
#pragma unroll
                        for (int k = 0; k < KD; k++) {
                            frag kn = kc, vn = vc;
                            if (k + 1 < KD) {
                                kn = kt.rows(lanes, 32 * n, k + 1);
                                vn = vt.rows(lanes, 32 * n, k + 1);
                            }
                            step_end<true>();
                            s = mma(kc, q[k], s);
                            dp = mma(vc, g[k], dp);
                            step_end<true>();
                            kc = kn;
                            vc = vn;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < KD; k++) {
                            s = mma(kt.rows(lanes, 32 * n, k), q[k], s);
                            dp = mma(vt.rows(lanes, 32 * n, k), g[k], dp);
                            step_end<Frag<T>::kFloat>();
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.s.scale2, base)) * fmaf(dp[r], by, -delta_by);
                    if constexpr (MASKED) {
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (first + 32 * n + 8 * (r / 4) + 4 * h + r % 4 >= limit) s[r] = 0.0f;
                    }
                    if constexpr (Frag<T>::kFloat) {
                        operand_t ds[2];
                        to_frag(s, 0, ds[0]);
                        to_frag(s, 1, ds[1]);
                        add_products<MASKED, true, T, D>(kt, lanes, ds, dq, odd);
                        continue;
                    }
                    if constexpr (kAhead && !MASKED) {
                        operand_t ds[2];
                        to_frag(s, 0, ds[0]);
                        to_frag(s, 1, ds[1]);
                        frag c = kt.columns(lanes, 32 * n, 0);
#pragma unroll
                        for (int step = 0; step < 2 * DB; step++) {
                            frag next = c;
                            if (step + 1 < 2 * DB) next = kt.columns(lanes, 32 * n + (step + 1) / DB * 16, (step + 1) % DB);
                            step_end<true>();
                            dq[step % DB] = mma(c, ds[step / DB], dq[step % DB]);
                            step_end<true>();
                            c = next;
                        }
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        operand_t ds[MASKED ? 2 : 1];
                        to_frag(s, u, ds[0]);
                        if constexpr (MASKED) {  // (and what the rounding took away)
                            left_by(ds[0], u, s);
                            to_frag(s, u, ds[1]);
                        }
                        frag k[DB];
#pragma unroll
                        for (int d = 0; d < DB; d++) k[d] = kt.columns(lanes, 32 * n + 16 * u, d);
                        if constexpr (MASKED) leave_out_odd<DB>(k, odd);
#pragma unroll
                        for (const operand_t &w : ds)
#pragma unroll
                            for (int d = 0; d < DB; d++) dq[d] = mma(k[d], w, dq[d]);
                        step_end<D == 128>();
                    }
                }
                if (MASKED && odd) add_odd<T, D, R>(kt, lanes, dq, [&](uint32_t r) { return first + r < limit; });
            };
            if (first + R > wave_full || few)
                work(std::true_type{});
            else
                work(std::false_type{});
        }
    }
    uint32_t thread = threadIdx.x;  // (the row's number is formed again: over the loop there is no register for it)
    asm volatile("" : "+v"(thread));
    const uint32_t own_row = tile * kOwn + thread / kWave * 32 + thread % 32, own_i = fast_div(own_row, a.s.by_group);
    if (own_row >= rows) return;
    T *const to = static_cast<T *>(const_cast<void *>(a.dq.at)) + (packed ? 0 : b * a.dq.batch) + (size_t)(q0 + own_i) * a.dq.row +
                  (head * a.s.group + own_row - own_i * a.s.group) * a.dq.head;
    const float natural = a.s.scale2 * (1.0f / kLog2e), by_q = kHalf ? ldexpf(natural, -scale.power) : natural;
    if (a.q_parts > 1) {
        const size_t own = ((size_t)(packed ? 0 : b) * lq + q0 + own_i) * a.s.heads + head * a.s.group + own_row - own_i * a.s.group;
        store_rows<float, D>(a.q_part + (part * (size_t)a.total_rows * a.s.heads + own) * a.s.dim, dq, by_q, a.s.dim, a.s.dim % 4 == 0);
        return;
    }
    store_rows<T, D>(to, dq, by_q, a.s.dim, a.vec);
}

template <typename T, int D, int WAVES, bool IN_LDS>
struct KeptValues {
    typedef Tile<T, D, WAVES, 32 * WAVES> type;
};
template <typename T, int D, int WAVES>
struct KeptValues<T, D, WAVES, false> {
    struct type {};
};

// dk and dv: a wavefront owns 32 keys as the columns of S = Q K^T; the rows that see them pass by.
template <typename T, int D, int WAVES>
struct ForKv {
    static constexpr bool kVInLds = !Frag<T>::kFloat && D == 128;
    static constexpr int kRows = D == 128 ? 32 : Frag<T>::kTile;  // (64 rows of 128 columns on their way leave too few registers)
    Tile<T, D, WAVES, kRows> tiles[2][2];  // [buffer][Q, dO]
    float stats[2][3][kRows];              // [buffer][base, D, |do|]
    typename KeptValues<T, D, WAVES, kVInLds>::type values;
};
template <typename T, int D, int WAVES>
__device__ __forceinline__ void attn_grad_kv(const Backward &a, const uint32_t block, ForKv<T, D, WAVES> &lds) {
    typedef typename Frag<T>::type frag;
    typedef typename Frag<T>::operand operand_t;
    constexpr uint32_t kOwn = 32 * WAVES;
    typedef Tile<T, D, WAVES, ForKv<T, D, WAVES>::kRows> RowTile;
    constexpr bool kHalf = !Frag<T>::kFloat;
    constexpr int R = RowTile::kRows, KD = D / 16, DB = D / 32;
    constexpr bool kVInLds = ForKv<T, D, WAVES>::kVInLds;
    constexpr int kAtOnce = D == 64 ? DB : 1;  // column blocks whose operands are read, and looked through, at once
    RowTile(&tiles)[2][2] = lds.tiles;
    float(&stats)[2][3][R] = lds.stats;
    auto &values = lds.values;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, h = lane / 32;
    const TileLanes<T, D> lanes;
    const uint32_t rest = fast_div(block, a.s.by_kv_heads), head = block - rest * a.s.kv_heads;
    const uint32_t tiles_at = a.parts == 1 ? rest : rest / a.parts, part = rest - tiles_at * a.parts;
    uint32_t b, tile, q0, lq, k0, lk;
    if (!find_tile(a.s.k_offsets, a.s.batch, a.s.k_rows, 1, kOwn, tiles_at, a.s.k_by_tile, b, tile)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    span_of_all(a.s.q_offsets, b, a.s.q_rows, q0, lq);
    span_of_all(a.s.k_offsets, b, a.s.k_rows, k0, lk);
    const bool packed = a.s.q_offsets != nullptr;
    const uint32_t rows = lq * a.s.group, key = tile * kOwn + wave * 32 + lane % 32;
    const bool live = key < lk;
    // the first row that sees a key
    auto first_row = [&](uint32_t j) -> uint32_t {
        const int64_t query = a.s.causal ? max((int64_t)0, (int64_t)j + lq - lk) : 0;
        return query >= lq ? rows : (uint32_t)query * a.s.group;
    };
    const T *kbase = static_cast<const T *>(a.k.at) + (packed ? 0 : b * a.k.batch) + (size_t)(k0 + key) * a.k.row + head * a.k.head;
    const T *vbase = static_cast<const T *>(a.v.at) + (packed ? 0 : b * a.v.batch) + (size_t)(k0 + key) * a.v.row + head * a.v.head;
    const T *qbase = static_cast<const T *>(a.q.at) + (packed ? 0 : b * a.q.batch) + (size_t)q0 * a.q.row + head * a.s.group * a.q.head;
    const T *gbase = static_cast<const T *>(a.dout.at) + (packed ? 0 : b * a.dout.batch) + (size_t)q0 * a.dout.row + head * a.s.group * a.dout.head;
    const size_t place0 = ((size_t)(packed ? 0 : b) * lq + q0) * a.s.heads + head * a.s.group;
    operand_t k[KD], v[kVInLds ? 1 : KD];
    load_frags<T, D>(live ? kbase : nullptr, a.s.dim, a.vec, k);
    if constexpr (kVInLds) {
        typedef typename KeptValues<T, D, WAVES, true>::type Values;
        const uint32_t key0 = tile * kOwn, n = min(lk - key0, kOwn);
        const T *const from = static_cast<const T *>(a.v.at) + (packed ? 0 : b * a.v.batch) + (size_t)(k0 + key0) * a.v.row + head * a.v.head;
        if (a.vec) {
            uint32_t base[Values::kTurn];
            Values::offsets((uint32_t)a.v.row, a.s.dim, base);
            values.request(from, (uint32_t)(((n - 1) * a.v.row + a.s.dim) * sizeof(T)),
                           [&](int p) { return Values::offset_of(base, (uint32_t)a.v.row, p); });
        } else {
            values.copy([&](uint32_t r) -> const T * { return r < n ? from + r * a.v.row : nullptr; }, a.s.dim);
        }
    } else {
        load_frags<T, D>(live ? vbase : nullptr, a.s.dim, a.vec, v);
    }
    auto value = [&](int c) -> operand_t {
        if constexpr (kVInLds)
            return values.rows(lanes, wave * 32, c);
        else
            return v[c];
    };
    const float v_norm = kHalf && live ? a.v_norm[(((size_t)(packed ? 0 : b) * lk + k0) + key) * a.s.kv_heads + head] : 0.0f;

    const uint32_t wave_key = tile * kOwn + wave * 32;
    const uint32_t own_from = live ? first_row(key) : rows;                              // the lane's rows: [own_from, rows)
    const uint32_t wave_from = wave_key < lk ? first_row(wave_key) : rows;               // the first any key is seen by
    const uint32_t wave_full = wave_key < lk ? first_row(min(lk - 1, wave_key + 31)) : rows; // from here on all are
    // Tiles of rows from the last one back, every parts-th of them: under a mask, too, all workgroups are then at the same rows at a
    // time, and read them from L2 (from the first row on: of the requests of 4 sequences of 4000 26 % were served there, now 69 %).
    const uint32_t from_tile = min(first_row(tile * kOwn), rows) / R, all = (rows + R - 1) / R - from_tile;
    const uint32_t count = all > part ? (all - part + a.parts - 1) / a.parts : 0;
    auto tile_of = [&](uint32_t n) { return from_tile + all - 1 - part - n * a.parts; };

    auto fetch = [&](uint32_t t, uint32_t buffer) {
        const uint32_t i0 = fast_div(t * R, a.s.by_group);  // the query of the tile's first row
        const T *const q = qbase + (size_t)i0 * a.q.row, *const g = gbase + (size_t)i0 * a.dout.row;
        const uint32_t last = min(rows, (t + 1) * R) - 1, n = fast_div(last, a.s.by_group) - i0;
        if (a.vec) {
            uint32_t q_offset[RowTile::kPerThread], g_offset[RowTile::kPerThread];
#pragma unroll
            for (int p = 0; p < RowTile::kPerThread; p++) {
                const uint32_t r = t * R + RowTile::row_of(p), d = RowTile::column_of(p), i = fast_div(r, a.s.by_group), gh = r - i * a.s.group;
                const bool in = r < rows && d < a.s.dim;
                q_offset[p] = in ? (uint32_t)(((i - i0) * a.q.row + gh * a.q.head + d) * sizeof(T)) : kNowhere;
                g_offset[p] = in ? (uint32_t)(((i - i0) * a.dout.row + gh * a.dout.head + d) * sizeof(T)) : kNowhere;
            }
            const uint32_t heads = a.s.group - 1;
            tiles[buffer][0].request(q, (uint32_t)((n * a.q.row + heads * a.q.head + a.s.dim) * sizeof(T)), [&](int p) { return q_offset[p]; });
            tiles[buffer][1].request(g, (uint32_t)((n * a.dout.row + heads * a.dout.head + a.s.dim) * sizeof(T)), [&](int p) { return g_offset[p]; });
        } else {
            auto from = [&](const T *base, const AttnView &v) {
                return [=](uint32_t r) -> const T * {
                    const uint32_t i = fast_div(t * R + r, a.s.by_group), gh = t * R + r - i * a.s.group;
                    return t * R + r < rows ? base + (i - i0) * v.row + gh * v.head : nullptr;
                };
            };
            tiles[buffer][0].copy(from(q, a.q), a.s.dim);
            tiles[buffer][1].copy(from(g, a.dout), a.s.dim);
        }
        if (threadIdx.x < R) {  // (rows behind the last have zeros, as in the tiles: nothing comes of them)
            const uint32_t r = t * R + threadIdx.x, i = fast_div(r, a.s.by_group), at = (i - i0) * a.s.heads + r - i * a.s.group;
            const size_t from = place0 + (size_t)i0 * a.s.heads;
            const uint32_t bytes = (n * a.s.heads + a.s.group) * (uint32_t)sizeof(float), offset = r < rows ? at * (uint32_t)sizeof(float) : kNowhere;
            request_floats(stats[buffer][0], a.base + from, bytes, offset);
            request_floats(stats[buffer][1], a.delta + from, bytes, offset);
            if (kHalf) request_floats(stats[buffer][2], a.norm + from, bytes, offset);
        }
    };
    const bool few = kHalf && few_terms(lq, lk, a.s.dim);
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) dk[d] = dv[d] = zero16();
    DsScale scale;
    if (count != 0)
        fetch(tile_of(0), 0);
    else
        wait_tiles();  // (keys that no row sees: their values are on the way to LDS, which is not given back before they are there)
    for (uint32_t at = 0; at < count; at++) {
        wait_tiles();
        __syncthreads();
        if (at + 1 < count) fetch(tile_of(at + 1), (at + 1) & 1);
        const uint32_t buffer = at & 1, first = tile_of(at) * R;
        const RowTile &qt = tiles[buffer][0], &gt = tiles[buffer][1];
        if (first + R > wave_from && wave_from < rows) {
            auto work = [&](auto with_masked) {
                constexpr bool MASKED = decltype(with_masked)::value;
                float by = 1.0f;
                bool odd = false;
                uint32_t from = own_from;
                if constexpr (MASKED && kVInLds) {  // (formed again: over the loop there is no register for it)
                    uint32_t thread = threadIdx.x;
                    asm volatile("" : "+v"(thread));
                    const uint32_t own = tile * kOwn + thread / kWave * 32 + thread % 32;
                    from = own < lk ? first_row(own) : rows;
                }
                if (kHalf) {
                    // (the tile's rows from the last to the first, one to a lane)
                    float down, norms = stats[buffer][2][R - 1 - lane % R], deltas = fabsf(stats[buffer][1][R - 1 - lane % R]);
                    if constexpr (MASKED) {
                        norms = max_up_to(norms);
                        deltas = max_up_to(deltas);
                        const uint32_t seeing = from > first ? R - min(from - first, (uint32_t)R) : R;  // rows that see the key
                        norms = __shfl(norms, (int)max(seeing, 1u) - 1, kWave);
                        deltas = __shfl(deltas, (int)max(seeing, 1u) - 1, kWave);
                        if (seeing == 0) norms = deltas = 0.0f;
                    } else {
                        norms = team_max<64>(norms);
                        deltas = team_max<64>(deltas);
                    }
                    if (scale.lower(fmaf(norms, v_norm, deltas), down)) {
#pragma unroll
                        for (int d = 0; d < DB; d++)
#pragma unroll
                            for (int r = 0; r < 16; r++) dk[d][r] *= down;
                    }
                    by = ldexpf(1.0f, scale.power - kPShift<T>);
                }
#pragma unroll
                for (int n = 0; n < R / 32; n++) {
                    f32x16 s = zero16(), dp = zero16();
                    if constexpr (kVInLds) {  // (operands are read a step ahead: there are registers for that, not for the compiler's choice)
                        frag qc = qt.rows(lanes, 32 * n, 0), gc = gt.rows(lanes, 32 * n, 0);
                        operand_t vc = value(0);
#pragma unroll
                        for (int c = 0; c < KD; c++) {
                            const int next = c + 1 < KD ? c + 1 : c;
                            frag qn = qc, gn = gc;
                            operand_t vn = vc;
                            if (next != c) {
                                qn = qt.rows(lanes, 32 * n, next);
                                gn = gt.rows(lanes, 32 * n, next);
                                vn = value(next);
                            }
                            step_end<true>();
                            s = mma(qc, k[c], s);
                            dp = mma(gc, vc, dp);
                            step_end<true>();
                            qc = qn;
                            gc = gn;
                            vc = vn;
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < KD; c++) {
                            s = mma(qt.rows(lanes, 32 * n, c), k[c], s);
                            dp = mma(gt.rows(lanes, 32 * n, c), value(c), dp);
                            step_end<Frag<T>::kFloat>();
                        }
                    }
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const f32x4 base = *reinterpret_cast<const f32x4 *>(&stats[buffer][0][32 * n + 8 * g + 4 * h]);
                        const f32x4 delta = *reinterpret_cast<const f32x4 *>(&stats[buffer][1][32 * n + 8 * g + 4 * h]);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int r = 4 * g + j;
                            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.s.scale2, base[j]));
                            dp[r] = s[r] * (kHalf ? fmaf(dp[r], by, -delta[j] * by) : dp[r] - delta[j]);
                        }
                    }
                    if constexpr (MASKED) {
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (first + 32 * n + 8 * (r / 4) + 4 * h + r % 4 < from) s[r] = dp[r] = 0.0f;
                    }
                    if (first + 32 * n + 32 > rows) {  // (zeros behind the last row times an infinite key are NaN)
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (first + 32 * n + 8 * (r / 4) + 4 * h + r % 4 >= rows) s[r] = dp[r] = 0.0f;
                    }
                    if constexpr (Frag<T>::kFloat) {
                        operand_t w[2];
                        to_frag(s, 0, w[0]);
                        to_frag(s, 1, w[1]);
                        add_products<MASKED, D == 64, T, D>(gt, lanes, w, dv, odd);
                        to_frag(dp, 0, w[0]);
                        to_frag(dp, 1, w[1]);
                        add_products<MASKED, D == 64, T, D>(qt, lanes, w, dk, odd);
                        continue;
                    }
                    constexpr int kTimes = MASKED ? 4 : 2;  // (two more are what the rounding took away)
                    operand_t p[kTimes], ds[kTimes];
#pragma unroll
                    for (int u = 0; u < kTimes; u++) {
                        to_frag(s, u % 2, p[u]);
                        to_frag(dp, u % 2, ds[u]);
                        if constexpr (MASKED) {
                            keep_here(p[u]);
                            keep_here(ds[u]);
                            if (u < 2) {
                                left_by(p[u], u, s);
                                left_by(ds[u], u, dp);
                            }
                        }
                    }
                    if constexpr (D == 128 && !MASKED) {
                        // (each operand is read one product ahead: there are registers for that, not for the compiler's choice)
                        auto read = [&](int step) { return (step % 2 == 0 ? gt : qt).columns(lanes, 32 * n + step / (2 * DB) * 16, step / 2 % DB); };
                        frag c = read(0);
#pragma unroll
                        for (int step = 0; step < 4 * DB; step++) {
                            const int u = step / (2 * DB), d = step / 2 % DB;
                            frag next = c;
                            if (step + 1 < 4 * DB) next = read(step + 1);
                            step_end<true>();
                            if (step % 2 == 0)
                                dv[d] = mma(c, p[u], dv[d]);
                            else
                                dk[d] = mma(c, ds[u], dk[d]);
                            c = next;
                            step_end<true>();
                        }
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
#pragma unroll
                        for (int d0 = 0; d0 < DB; d0 += kAtOnce) {
                            frag c[kAtOnce];
#pragma unroll
                            for (int d = 0; d < kAtOnce; d++) c[d] = gt.columns(lanes, 32 * n + 16 * u, d0 + d);
                            if constexpr (MASKED) leave_out_odd<kAtOnce>(c, odd);
#pragma unroll
                            for (int w = u; w < kTimes; w += 2)
#pragma unroll
                                for (int d = 0; d < kAtOnce; d++) dv[d0 + d] = mma(c[d], p[w], dv[d0 + d]);
                            step_end<D == 128>();
#pragma unroll
                            for (int d = 0; d < kAtOnce; d++) c[d] = qt.columns(lanes, 32 * n + 16 * u, d0 + d);
                            if constexpr (MASKED) leave_out_odd<kAtOnce>(c, odd);
#pragma unroll
                            for (int w = u; w < kTimes; w += 2)
#pragma unroll
                                for (int d = 0; d < kAtOnce; d++) dk[d0 + d] = mma(c[d], ds[w], dk[d0 + d]);
                            step_end<D == 128>();
                        }
                    }
                }
                if (MASKED && odd) {
                    auto visible = [&](uint32_t r) { return first + r >= from; };
                    add_odd<T, D, R>(gt, lanes, dv, visible);
                    add_odd<T, D, R>(qt, lanes, dk, visible);
                }
            };
            if (first < wave_full || few)
                work(std::true_type{});
            else
                work(std::false_type{});
        }
    }
    uint32_t thread = threadIdx.x;  // (the key's number is formed again, and the keys' count is a scalar: over the loop there is no
                                    // vector register for them)
    asm volatile("" : "+v"(thread));
    asm volatile("" : "+s"(lk));
    const uint32_t own_key = tile * kOwn + thread / kWave * 32 + thread % 32;
    if (own_key >= lk) return;
    const uint32_t own_b = packed ? 0 : __builtin_amdgcn_readfirstlane(b);
    const uint32_t first_key = __builtin_amdgcn_readfirstlane(k0);
    auto out = [&](const AttnView &to) {
        return static_cast<T *>(const_cast<void *>(to.at)) + own_b * to.batch + (size_t)(first_key + own_key) * to.row + head * to.head;
    };
    const float natural = a.s.scale2 * (1.0f / kLog2e);
    const float by_k = kHalf ? ldexpf(natural, -scale.power) : natural, by_v = ldexpf(1.0f, -kPShift<T>);
    if (a.parts > 1) {
        const size_t place = ((size_t)own_b * lk + first_key + own_key) * a.s.kv_heads + head;
        float *const to = a.part + (part * (size_t)a.total_keys * a.s.kv_heads + place) * 2 * a.s.dim;
        const bool whole = a.s.dim % 4 == 0;
        store_rows<float, D>(to, dk, by_k, a.s.dim, whole);
        store_rows<float, D>(to + a.s.dim, dv, by_v, a.s.dim, whole);
        return;
    }
    store_rows<T, D>(out(a.dk), dk, by_k, a.s.dim, a.vec);
    store_rows<T, D>(out(a.dv), dv, by_v, a.s.dim, a.vec);
}

// The workgroups of dk and dv, then those of dq, which fill up what the former leave; or one kind alone (float16 with 128 columns:
// together they have a few registers too few).
template <typename T, int D, int WAVES, bool KV, bool Q>
__global__ __launch_bounds__(WAVES *kWave, Frag<T>::kFloat || WAVES == 1 ? 1 : 2) void attn_grad_kernel(const Backward a) {
    constexpr size_t kBytes = std::max(KV ? sizeof(ForKv<T, D, WAVES>) : 0, Q ? sizeof(ForQ<T, D, WAVES>) : 0);
    __shared__ __align__(256) char lds[kBytes];
    if constexpr (KV) {
        if (!Q || blockIdx.x < a.kv_blocks) return attn_grad_kv<T, D, WAVES>(a, blockIdx.x, *reinterpret_cast<ForKv<T, D, WAVES> *>(lds));
    }
    if constexpr (Q) attn_grad_q<T, D, WAVES>(a, blockIdx.x - (KV ? a.kv_blocks : 0), *reinterpret_cast<ForQ<T, D, WAVES> *>(lds));
}

// Gradients from their parts, in the parts' order, for a few rows of a head: of dk and dv, or of dq.  V values a lane: 4 where rows
// are whole vectors of the parts and of the gradients, or 1.
constexpr uint32_t kJoinRows = 8;
template <typename T, bool OF_KEYS, int V>
__global__ __launch_bounds__(kAttnThreads) void attn_grad_join_kernel(const Backward a) {
    typedef float floats __attribute__((ext_vector_type(V)));
    const uint32_t heads = OF_KEYS ? a.s.kv_heads : a.s.heads, parts = OF_KEYS ? a.parts : a.q_parts;
    const uint32_t all = blockIdx.x / heads, head = blockIdx.x - all * heads;
    const int32_t *const offsets = OF_KEYS ? a.s.k_offsets : a.s.q_offsets;
    const uint32_t rows = OF_KEYS ? a.s.k_rows : a.s.q_rows;
    uint32_t b, tile, first, count;
    if (!find_tile(offsets, a.s.batch, rows, 1, kJoinRows, all, false, b, tile)) return;
    span(offsets, b, rows, first, count);
    const uint32_t n = min(kJoinRows, count - tile * kJoinRows), row = (OF_KEYS ? 2 : 1) * a.s.dim / V;
    const size_t step = (size_t)(OF_KEYS ? a.total_keys : a.total_rows) * heads * row;
    for (uint32_t at = threadIdx.x; at < n * row; at += kAttnThreads) {
        const uint32_t r = at / row, c = at - r * row;
        const size_t own = first + tile * kJoinRows + r;
        const floats *from = reinterpret_cast<const floats *>(OF_KEYS ? a.part : a.q_part) +
                             (((size_t)(offsets != nullptr ? 0 : b) * count + own) * heads + head) * row + c;
        floats sum = floats(0.0f);
        for (uint32_t p0 = 0; p0 < parts; p0 += 8) {
            floats f[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) f[u] = p0 + u < parts ? from[(p0 + u) * step] : floats(0.0f);
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) sum += f[u];
        }
        const bool first_half = c * V < a.s.dim;
        const AttnView &to = !OF_KEYS ? a.dq : first_half ? a.dk : a.dv;
        T v[V];
#pragma unroll
        for (int e = 0; e < V; e++) Store<T>::store1(v + e, sum[e]);
        T *const out = static_cast<T *>(const_cast<void *>(to.at)) + (offsets != nullptr ? 0 : b * to.batch) + own * to.row + head * to.head +
                       (first_half ? c * V : c * V - a.s.dim);
        __builtin_memcpy(__builtin_assume_aligned(out, sizeof(v)), v, sizeof(v));
    }
}

size_t tiles_of(const int32_t *offsets, size_t batch, size_t rows, size_t times, size_t own) {
    if (offsets == nullptr) return batch * ((rows * times + own - 1) / own);
    return rows * times / own + batch;
}
bool few_rows_and_keys(const AttnProblem &p) { return attn_few(p, p.q_rows, p.heads / p.kv_heads) && attn_few(p, p.k_rows, 1); }
size_t tiles_of_keys(const AttnProblem &p) { return tiles_of(p.k_offsets, p.batch, p.k_rows, 1, attn_rows(few_rows_and_keys(p))); }

// Parts of the rows for dk and dv.  Under a causal mask tiles of keys differ in the rows that see them: cut in two they fill up
// a launch of few rounds.  Few keys and many rows (a prompt's keys, an image's rows) are cut until the chip is full, with
// at least 256 rows in a part on average.
uint32_t row_parts(const AttnProblem &p) {
    const size_t blocks = std::max<size_t>(1, tiles_of_keys(p) * p.kv_heads), once = 2 * (size_t)chip_info().cus;
    const size_t rows = (p.q_offsets != nullptr ? p.q_rows / std::max<size_t>(1, p.batch) : p.q_rows) * (p.heads / p.kv_heads);
    size_t parts = p.causal && blocks <= 4 * once ? 2 : 1;
    parts = std::max(parts, once / blocks);
    return (uint32_t)std::max<size_t>(1, std::min<size_t>(parts, rows / 256));
}

// Parts of the keys for dq, where rows are too few to fill the chip, of at least 256 keys on average.
uint32_t dq_parts(const AttnProblem &p) {
    const size_t own = attn_rows(few_rows_and_keys(p)), cus = chip_info().cus;
    const size_t blocks = std::max<size_t>(1, tiles_of(p.q_offsets, p.batch, p.q_rows, p.heads / p.kv_heads, own) * p.kv_heads);
    const size_t keys = p.k_offsets != nullptr ? p.k_rows / std::max<size_t>(1, p.batch) : p.k_rows;
    if (blocks > cus) return 1;
    return (uint32_t)std::max<size_t>(1, std::min<size_t>((p.k_offsets != nullptr ? 8 : 2) * cus / blocks, keys / 256));
}

// Floats of the workspace: vectors over rows and keys, parts of dk and dv, parts of dq.
struct Room {
    size_t vectors, part, q_part;  // (of one part)
};
Room room_of(const AttnProblem &p) {
    const size_t rows = p.q_offsets == nullptr ? p.batch * p.q_rows : p.q_rows, keys = p.k_offsets == nullptr ? p.batch * p.k_rows : p.k_rows;
    return Room{(3 * rows * p.heads + keys * p.kv_heads + 3) / 4 * 4, (keys * p.kv_heads * 2 * p.dim + 3) / 4 * 4,
                (rows * p.heads * p.dim + 3) / 4 * 4};
}

}  // namespace

size_t attn_grad_workspace_bytes(const AttnProblem &p, bool any_mask) {
    AttnProblem other = p;  // (the bytes go by the sizes, the parts by the mask too)
    other.causal = !p.causal;
    const size_t parts = any_mask ? std::max(row_parts(p), row_parts(other)) : row_parts(p), q_parts = dq_parts(p);
    const Room r = room_of(p);
    return (r.vectors + (parts > 1 ? parts * r.part : 0) + (q_parts > 1 ? q_parts * r.q_part : 0)) * sizeof(float);
}

template <typename T, int D>
static void launch_apart(const Backward &a, uint32_t row_blocks, hipStream_t stream) {
    if (a.kv_blocks != 0) launch((attn_grad_kernel<T, D, kAttnWaves, true, false>), dim3(a.kv_blocks), dim3(kAttnThreads), 0, stream, a);
    if (row_blocks != 0) launch((attn_grad_kernel<T, D, kAttnWaves, false, true>), dim3(row_blocks), dim3(kAttnThreads), 0, stream, a);
}

template <typename T, int V>
static void launch_joins(const AttnProblem &p, const Backward &a, hipStream_t stream) {
    if (a.parts > 1)
        launch((attn_grad_join_kernel<T, true, V>), dim3((uint32_t)(tiles_of(p.k_offsets, p.batch, p.k_rows, 1, kJoinRows) * p.kv_heads)),
               dim3(kAttnThreads), 0, stream, a);
    if (a.q_parts > 1)
        launch((attn_grad_join_kernel<T, false, V>), dim3((uint32_t)(tiles_of(p.q_offsets, p.batch, p.q_rows, 1, kJoinRows) * p.heads)),
               dim3(kAttnThreads), 0, stream, a);
}

template <typename T>
int attn_grad_dispatch(const AttnProblem &p, const AttnGradViews &g, const float *lse, const void *rest, void *workspace, size_t workspace_bytes,
                       hipStream_t stream) {
    const size_t rows = p.q_offsets == nullptr ? p.batch * p.q_rows : p.q_rows, keys = p.k_offsets == nullptr ? p.batch * p.k_rows : p.k_rows;
    float *const base = static_cast<float *>(workspace), *const delta = base + rows * p.heads;
    constexpr bool kHalf = !Frag<T>::kFloat;
    // no more parts than the workspace holds, those of dk and dv first; none of a side without rows, which has no workgroups to join them
    const Room r = room_of(p);
    size_t left = workspace_bytes / sizeof(float) - r.vectors;
    const uint32_t parts = r.part == 0 ? 1 : (uint32_t)std::max<size_t>(1, std::min<size_t>(row_parts(p), left / r.part));
    if (parts > 1) left -= parts * r.part;
    const uint32_t q_parts = r.q_part == 0 ? 1 : (uint32_t)std::max<size_t>(1, std::min<size_t>(dq_parts(p), left / r.q_part));
    float *const part = base + r.vectors, *const q_part = part + (parts > 1 ? parts * r.part : 0);
    const Backward a{attn_shape(p), g.q, g.k, g.v, g.out, g.dout, g.dq, g.dk, g.dv, lse, rest, base, delta,
                     kHalf ? delta + rows * p.heads : nullptr, kHalf ? delta + 2 * rows * p.heads : nullptr, part, q_part, (uint32_t)rows,
                     (uint32_t)keys, parts, q_parts,
                     (uint32_t)(tiles_of_keys(p) * p.kv_heads * parts),
                     attn_vectors(sizeof(T), p, {g.q, g.k, g.v, g.out, g.dout, g.dq, g.dk, g.dv, AttnView{rest, 0, 0, 0}})};
    const size_t items = rows * p.heads + (kHalf ? keys * p.kv_heads : 0);
    if (items != 0)
        launch((attn_grad_rows_kernel<T>), dim3((uint32_t)((items + 15) / 16)), dim3(kAttnThreads), 0, stream, a);
    const bool few = few_rows_and_keys(p);
    const size_t row_blocks = tiles_of(p.q_offsets, p.batch, p.q_rows, p.heads / p.kv_heads, attn_rows(few)) * p.kv_heads * q_parts;
    const dim3 grid((uint32_t)(a.kv_blocks + row_blocks));
    if (grid.x != 0) {
        if (few) {
            launch((attn_grad_kernel<T, 64, 1, true, true>), grid, dim3(kWave), 0, stream, a);
        } else if (p.dim <= 64) {
            // (apart, dq has three wavefronts per SIMD in float16: 5 % faster where there are rounds enough)
            bool apart = false;
            if constexpr (kHalf) {
                apart = grid.x > 8 * chip_info().cus;
                if (apart) launch_apart<T, 64>(a, (uint32_t)row_blocks, stream);
            }
            if (!apart) launch((attn_grad_kernel<T, 64, kAttnWaves, true, true>), grid, dim3(kAttnThreads), 0, stream, a);
        } else if constexpr (!kHalf) {
            launch((attn_grad_kernel<T, 128, kAttnWaves, true, true>), grid, dim3(kAttnThreads), 0, stream, a);
        } else {
            launch_apart<T, 128>(a, (uint32_t)row_blocks, stream);
        }
    }
    if (a.vec)
        launch_joins<T, 4>(p, a, stream);
    else
        launch_joins<T, 1>(p, a, stream);
    return launch_status();
}

template int attn_grad_dispatch<float>(const AttnProblem &, const AttnGradViews &, const float *, const void *, void *, size_t, hipStream_t);
template int attn_grad_dispatch<__half>(const AttnProblem &, const AttnGradViews &, const float *, const void *, void *, size_t, hipStream_t);

}  // namespace msd
