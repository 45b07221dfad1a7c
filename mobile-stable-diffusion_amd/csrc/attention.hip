// Attention for gfx950: out_i = sum_j p_ij v_j, p_ij = softmax over the visible j of scale q_i . k_j, in one pass over the keys with
// a running maximum and sum.  The query heads of a key head are rows of one tile (row = query * group + head in the group), so keys
// and values are read once for all of them, and a single query still has `group` rows.  A wavefront owns 32 rows as the columns of
// S^T = K Q^T: a lane has one row, its maximum and sum need one exchange between the halves, and P^T stays in registers as the
// operand of O^T = V^T P^T.  K and V tiles go through LDS, twice buffered, straight from memory.  Where rows are too few to fill the
// chip, the keys are cut into parts, each with a workgroup of its own, and a second launch joins them.
//
// Measured (4 d operations for each visible pair; a library product of 8192 x 8192 reaches 1100 TFLOP/s in float16, 154 in float32):
//   float16, 4 x 4096, 32 heads of 128 on 8: 1.14 ms, 960 TFLOP/s; 8 x 4096, 16 heads of 64: 0.66 ms, 838.  The two wavefronts of a
//     SIMD wait for each other's matrix and exp2 instructions (38 % of their cycles) and for tiles (22 %).
//   float16, 2 x 4096, 5 heads of 64: 85 us, 500 TFLOP/s: 320 workgroups on 256 CUs (see key_parts).
//   float16, one query of 16 sequences of up to 16385 keys, 32 heads on 8: 104 us and 7 for the join, 4.3 TB/s.
//   float16, 2 x 77, 12 heads of 64: 7.8 us, of which 6.5 are there for one key too: launch, arguments, two reads of memory in a row
//     (queries and the first tile), instructions from no cache; a tile of 64 keys is 0.8.
//   float32, 2 x 2048, 8 heads: 110 TFLOP/s with 64 columns, 106 with 128, causal 77 and 87 (six products for one: 183 at the library's
//     float16 rate; cutting the values of each fragment in three takes more cycles than they do).  One query of 16 sequences of 16384
//     keys, 32 heads of 128 on 8: 1.05 ms, 2.0 TB/s: 32 columns of each product for 4 rows.
#include <algorithm>
#include <type_traits>

#include "attention_tiles.h"

namespace msd {
namespace {

struct Forward {
    AttnShape s;
    AttnView q, k, v, out;
    float *lse;        // [rows of queries][heads] log2 of the weights' sum, or null
    void *rest;        // [rows of queries][heads][dim] what rounding takes from out, or null
    float *part;       // parts > 1: [parts][rows of queries][heads][dim] and behind it their log2 sums [parts][rows][heads]
    float *part_lse;
    uint32_t parts, total_rows;
    bool vec;
};

// A lane's maximum may lag by this much (in powers of two) before the sums are scaled down to it, and float16 weights are
// kept kShift larger, so that they use the type's range: at most 2^(kLag + kShift) = 2^15.
constexpr float kLag = 8.0f;
template <typename T>
constexpr float kShift = Frag<T>::kFloat ? 0.0f : 7.0f;

template <typename T, int D, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, Frag<T>::kFloat || WAVES == 1 ? 1 : 2) void attn_kernel(const Forward a) {
    typedef typename Frag<T>::type frag;
    typedef typename Frag<T>::operand operand_t;
    typedef Tile<T, D, WAVES> KvTile;
    constexpr uint32_t kOwn = 32 * WAVES;
    constexpr int R = KvTile::kRows, KD = D / 16, DB = D / 32;
    __shared__ KvTile tiles[2][2];  // [buffer][K, V]
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, h = lane / 32;
    const TileLanes<T, D> lanes;
    const uint32_t rest = fast_div(blockIdx.x, a.s.by_kv_heads), head = blockIdx.x - rest * a.s.kv_heads;
    const uint32_t tiles_at = a.parts == 1 ? rest : rest / a.parts, part = rest - tiles_at * a.parts;
    uint32_t b, tile, q0, lq, k0, lk;
    if (!find_tile(a.s.q_offsets, a.s.batch, a.s.q_rows, a.s.group, kOwn, tiles_at, a.s.q_by_tile, b, tile)) return;
    span(a.s.q_offsets, b, a.s.q_rows, q0, lq);
    span(a.s.k_offsets, b, a.s.k_rows, k0, lk);
    const uint32_t rows = lq * a.s.group;
    if (a.s.causal) tile = (rows + kOwn - 1) / kOwn - 1 - tile;  // (those that see most keys first)

    const bool packed_q = a.s.q_offsets != nullptr, packed_k = a.s.k_offsets != nullptr;
    // the lane's row: query i of head `qh`; it sees the keys [0, limit)
    const uint32_t row = tile * kOwn + wave * 32 + lane % 32;
    const uint32_t i = fast_div(row, a.s.by_group), qh = head * a.s.group + row - i * a.s.group;
    const bool live = row < rows;
    auto seen_by = [&](uint32_t query) -> uint32_t {
        return a.s.causal ? (uint32_t)max((int64_t)0, min((int64_t)lk, (int64_t)query + 1 + lk - lq)) : lk;
    };
    const uint32_t limit = live ? seen_by(i) : 0;
    const T *qrow = static_cast<const T *>(a.q.at) + (packed_q ? 0 : b * a.q.batch) + (size_t)(q0 + i) * a.q.row + qh * a.q.head;
    const T *kbase = static_cast<const T *>(a.k.at) + (packed_k ? 0 : b * a.k.batch) + (size_t)k0 * a.k.row + head * a.k.head;
    const T *vbase = static_cast<const T *>(a.v.at) + (packed_k ? 0 : b * a.v.batch) + (size_t)k0 * a.v.row + head * a.v.head;
    operand_t q[KD];
    load_frags<T, D>(live ? qrow : nullptr, a.s.dim, a.vec, q);

    // tiles of keys: what the workgroup's last row sees, this part's share of it
    const uint32_t last_row = min(rows, (tile + 1) * kOwn) - 1;
    const uint32_t all = (seen_by(fast_div(last_row, a.s.by_group)) + R - 1) / R, each = (all + a.parts - 1) / a.parts;
    const uint32_t t0 = min(all, part * each), t1 = min(all, t0 + each);
    const uint32_t wave_row = tile * kOwn + wave * 32;
    const uint32_t wave_limit = wave_row < rows ? seen_by(fast_div(min(rows - 1, wave_row + 31), a.s.by_group)) : 0;  // the most any row sees
    const uint32_t wave_full = wave_row < rows ? seen_by(fast_div(wave_row, a.s.by_group)) : 0;                       // what every row sees

    uint32_t k_base[KvTile::kTurn], v_base[KvTile::kTurn];
    const uint32_t k_row = (uint32_t)a.k.row, v_row = (uint32_t)a.v.row;
    KvTile::offsets(k_row, a.s.dim, k_base);
    KvTile::offsets(v_row, a.s.dim, v_base);
    auto fetch = [&](uint32_t t, uint32_t buffer) {
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

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) o[d] = zero16();
    float top = -__builtin_inff(), sum = 0.0f;
    if (t0 < t1) fetch(t0, 0);
    for (uint32_t t = t0; t < t1; t++) {
        wait_tiles();
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1, (t + 1 - t0) & 1);
        const KvTile &kt = tiles[(t - t0) & 1][0], &vt = tiles[(t - t0) & 1][1];
        const uint32_t first = t * R;
        if (first < wave_limit) {
            // (apart for tiles with masked pairs: the tests between their products would keep the others' from overlapping)
            auto work = [&](auto with_masked) {
                constexpr bool MASKED = decltype(with_masked)::value;
                f32x16 s[R / 32];
#pragma unroll
                for (int n = 0; n < R / 32; n++) {
                    s[n] = zero16();
#pragma unroll
                    for (int k = 0; k < KD; k++) s[n] = mma(kt.rows(lanes, 32 * n, k), q[k], s[n]);
                }
                bool odd = false;
                if constexpr (MASKED) {
#pragma unroll
                    for (int n = 0; n < R / 32; n++)
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (first + 32 * n + 8 * (r / 4) + 4 * h + r % 4 >= limit) s[n][r] = -__builtin_inff();
                }
                float most = s[0][0];
#pragma unroll
                for (int n = 0; n < R / 32; n++)
#pragma unroll
                    for (int r = 0; r < 16; r++) most = fmaxf(most, s[n][r]);
                const float now = fmaxf(top, halves_max(most) * a.s.scale2);
                if (__builtin_amdgcn_ballot_w64(now > top + kLag) != 0) {
                    const float down = __builtin_amdgcn_exp2f(top - (now == -__builtin_inff() ? 0.0f : now));
                    sum *= down;
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[d][r] *= down;
                    top = now;
                }
                const float base = kShift<T> - (top == -__builtin_inff() ? 0.0f : top);
#pragma unroll
                for (int n = 0; n < R / 32; n++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], a.s.scale2, base));
                        sum += s[n][r];
                    }
                if constexpr (Frag<T>::kFloat) {
                    operand_t p[2];
                    to_frag(s[0], 0, p[0]);
                    to_frag(s[0], 1, p[1]);
                    add_products<MASKED, true, T, D>(vt, lanes, p, o, odd);
                } else {
#pragma unroll
                    for (int n = 0; n < R / 32; n++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            operand_t p;
                            to_frag(s[n], u, p);
                            frag v[DB];
#pragma unroll
                            for (int d = 0; d < DB; d++) v[d] = vt.columns(lanes, 32 * n + 16 * u, d);
                            if constexpr (MASKED) leave_out_odd<DB>(v, odd);
#pragma unroll
                            for (int d = 0; d < DB; d++) o[d] = mma(v[d], p, o[d]);
                        }
                }
                if (MASKED && odd) add_odd<T, D, R>(vt, lanes, o, [&](uint32_t r) { return first + r < limit; });
            };
            if (first + R > wave_full)
                work(std::true_type{});
            else
                work(std::false_type{});
        }
    }
    sum += half_swap(sum);
    if (!live) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that sees nothing is zero)
    const float lse = sum == 0.0f ? -__builtin_inff() : top - kShift<T> + __builtin_amdgcn_logf(sum);
    const size_t place = ((size_t)(packed_q ? 0 : b) * lq + q0 + i) * a.s.heads + qh;
    if (a.parts > 1) {
        store_rows<float, D>(a.part + (part * (size_t)a.total_rows * a.s.heads + place) * a.s.dim, o, inv, a.s.dim, a.s.dim % 4 == 0);
        if (h == 0) a.part_lse[part * (size_t)a.total_rows * a.s.heads + place] = lse;
        return;
    }
    T *const to = static_cast<T *>(const_cast<void *>(a.out.at)) + (packed_q ? 0 : b * a.out.batch) + (size_t)(q0 + i) * a.out.row + qh * a.out.head;
    T *const rest_to = !Frag<T>::kFloat && a.rest != nullptr ? static_cast<T *>(a.rest) + place * a.s.dim : nullptr;
    store_rows<T, D>(to, o, inv, a.s.dim, a.vec, rest_to);
    if (a.lse != nullptr && h == 0) a.lse[place] = lse;
}

// out = sum of the parts, each weighted by its share of the weights' sum: a wavefront for a row of a head.
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(const Forward a) {
    const size_t at = (size_t)blockIdx.x * kAttnWaves + threadIdx.x / kWave;
    const size_t count = (size_t)a.total_rows * a.s.heads;
    if (at >= count) return;
    const uint32_t row = (uint32_t)(at / a.s.heads), head = (uint32_t)(at % a.s.heads), lane = threadIdx.x % kWave;
    uint32_t b = 0, i = row;
    if (a.s.q_offsets == nullptr) {
        b = row / a.s.q_rows;
        i = row - b * a.s.q_rows;
    } else {  // rows of no sequence stay as they were
        bool inside = false;
        for (uint32_t s = lane; s < a.s.batch; s += kWave) {
            uint32_t first, n;
            span(a.s.q_offsets, s, a.s.q_rows, first, n);
            inside |= row >= first && row - first < n;
        }
        if (__builtin_amdgcn_ballot_w64(inside) == 0) return;
    }
    // a part's share of the weights, one to a lane
    const float l = lane < a.parts ? a.part_lse[lane * count + at] : -__builtin_inff();
    const float most = team_max<64>(l), base = most == -__builtin_inff() ? 0.0f : most;
    const float weight = __builtin_amdgcn_exp2f(l - base), sum = wave_sum(weight);  // (NaN where any is)
    const float share = sum == 0.0f ? 0.0f : weight / sum;
    T *const to = static_cast<T *>(const_cast<void *>(a.out.at)) + b * a.out.batch + (size_t)i * a.out.row + head * a.out.head;
    for (uint32_t d = lane; d < a.s.dim + lane; d += kWave) {  // (all lanes take every turn: each hands out its share)
        float t = 0.0f;
        for (uint32_t p0 = 0; p0 < a.parts; p0 += 8) {
            float f[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; u++)
                f[u] = p0 + u < a.parts && d < a.s.dim ? a.part[((p0 + u) * count + at) * a.s.dim + d] : 0.0f;
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) {
                const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), min(p0 + u, kWave - 1)));
                if (w != 0.0f) t = fmaf(w, f[u], t);
            }
        }
        if (d < a.s.dim) {
            Store<T>::store1(to + d, t);
            if (!Frag<T>::kFloat && a.rest != nullptr) Store<T>::store1(static_cast<T *>(a.rest) + at * a.s.dim + d, t - round_to_storage<T>(t));
        }
    }
    if (a.lse != nullptr && lane == 0) a.lse[at] = sum == 0.0f ? -__builtin_inff() : base + __builtin_amdgcn_logf(sum);
}

}  // namespace

// Whether workgroups of one wavefront do, of up to 64 columns: all of them at once are one to a SIMD, or sequences are so short that
// of four most would have no rows.
bool attn_few(const AttnProblem &p, size_t rows, size_t times) {
    if (p.dim > 64) return false;
    const size_t all = (p.q_offsets == nullptr ? p.batch : 1) * rows * times, tiles = all / 32 + p.batch;
    return tiles * p.kv_heads <= 4 * (size_t)chip_info().cus || all / std::max<size_t>(1, p.batch) <= 48;
}

namespace {

bool attn_few_rows(const AttnProblem &p) { return attn_few(p, p.q_rows, p.heads / p.kv_heads); }

// Tiles of rows: the sequences' own where they are equal, at most this many where only their sum is known here.
size_t row_tiles(const AttnProblem &p) {
    const size_t group = p.heads / p.kv_heads;
    const size_t own = attn_rows(attn_few_rows(p));
    if (p.q_offsets == nullptr) return p.batch * ((p.q_rows * group + own - 1) / own);
    return p.q_rows * group / own + p.batch;
}

// Parts of the keys: workgroups for eight rounds of the chip where the sequences' lengths may differ, for two otherwise, with at
// least 256 keys in a part on average, or 128 as long as all are at work at once; one wavefront joins at most kWave of them.  (Four
// workgroups of one wavefront count as one.)  One query of 32 sequences of 4096 keys, 12 heads of 64, float16: 115 us in one part, 79
// in five; one of 1000 keys, 32 heads of 128 on 8: 15.8 us in parts of 256 keys, 12.1 of 128.  Many rows, float16, heads of 64, calls
// without a profiler (the join, a row to a wavefront, takes 4-byte loads):
//   workgroups                               one part   two parts   three   four
//   320  2 x 4096, 5 heads                      85.2        85.5     91.0   82.0 us  (one is taken)
//   160  1 x 4096, 5 heads                      87.2       106.7     81.8   86.1     (three)
//   160  2 x 1024, 10 heads                     24.3        42.0     37.7   40.7     (three, though the join costs more than they give:
//                                                                                     the rule does not count it)
uint32_t key_parts(const AttnProblem &p) {
    const bool packed = p.k_offsets != nullptr;
    const size_t keys = packed ? p.k_rows / std::max<size_t>(1, p.batch) : p.k_rows;
    const size_t blocks = std::max<size_t>(1, row_tiles(p) * p.kv_heads / (attn_few_rows(p) ? kAttnWaves : 1)), cus = chip_info().cus;
    if (blocks > cus) return 1;
    const size_t parts = std::max(std::min((packed ? 8 : 2) * cus / blocks, keys / 256), std::min(cus / blocks, keys / 128));
    return (uint32_t)std::max<size_t>(1, std::min<size_t>(parts, kWave));
}

size_t total_rows(const AttnProblem &p) { return p.q_offsets == nullptr ? p.batch * p.q_rows : p.q_rows; }

}  // namespace

size_t attn_workspace_bytes(const AttnProblem &p) {
    const uint32_t parts = key_parts(p);
    return parts <= 1 ? 0 : parts * total_rows(p) * p.heads * (p.dim + 1) * sizeof(float);
}

AttnShape attn_shape(const AttnProblem &p) {
    const size_t few = 8 * (size_t)chip_info().cus;
    const size_t own = attn_rows(attn_few(p, p.k_rows, 1)), k_blocks = p.batch * ((p.k_rows + own - 1) / own) * p.kv_heads;
    return AttnShape{p.q_offsets, p.k_offsets, (uint32_t)p.batch, (uint32_t)p.q_rows, (uint32_t)p.k_rows, (uint32_t)p.heads,
                     (uint32_t)p.kv_heads, (uint32_t)(p.heads / p.kv_heads), (uint32_t)p.dim,
                     make_fast_div((uint32_t)(p.heads / p.kv_heads)), make_fast_div((uint32_t)p.kv_heads), p.scale * kLog2e, p.causal,
                     p.causal && row_tiles(p) * p.kv_heads <= few, p.causal && k_blocks <= few};
}

bool attn_vectors(size_t elt, const AttnProblem &p, std::initializer_list<AttnView> views) {
    bool vec = p.dim * elt % 16 == 0;
    for (const AttnView &v : views)
        vec = vec && aligned16(v.at) && v.row * elt % 16 == 0 && v.head * elt % 16 == 0 && v.batch * elt % 16 == 0 &&
              v.row * elt < (size_t(1) << 23) && v.head * elt < (size_t(1) << 29) / p.heads;
    return vec;
}

template <typename T>
int attn_dispatch(const AttnProblem &p, const AttnView &q, const AttnView &k, const AttnView &v, const AttnView &out, float *lse,
                  void *rest, void *workspace, size_t workspace_bytes, hipStream_t stream) {
    const size_t tiles = row_tiles(p);
    if (tiles == 0) return MSD_OK;
    Forward a{attn_shape(p), q, k, v, out, lse, rest, nullptr, nullptr, key_parts(p), (uint32_t)total_rows(p),
              attn_vectors(sizeof(T), p, {q, k, v, out, AttnView{rest, 0, 0, 0}})};
    a.parts = (uint32_t)std::max<size_t>(1, std::min<size_t>(a.parts, workspace_bytes / (total_rows(p) * p.heads * (p.dim + 1) * sizeof(float))));
    if (a.parts > 1) {
        a.part = static_cast<float *>(workspace);
        a.part_lse = a.part + (size_t)a.parts * a.total_rows * p.heads * p.dim;
    }
    const dim3 grid((uint32_t)(tiles * a.parts * p.kv_heads));
    if (attn_few_rows(p))
        launch((attn_kernel<T, 64, 1>), grid, dim3(kWave), 0, stream, a);
    else if (p.dim <= 64)
        launch((attn_kernel<T, 64, kAttnWaves>), grid, dim3(kAttnThreads), 0, stream, a);
    else
        launch((attn_kernel<T, 128, kAttnWaves>), grid, dim3(kAttnThreads), 0, stream, a);
    if (a.parts > 1)
        launch((attn_join_kernel<T>), dim3((uint32_t)((total_rows(p) * p.heads + kAttnWaves - 1) / kAttnWaves)), dim3(kAttnThreads), 0,
               stream, a);
    return launch_status();
}

template int attn_dispatch<float>(const AttnProblem &, const AttnView &, const AttnView &, const AttnView &, const AttnView &, float *,
                                  void *, void *, size_t, hipStream_t);
template int attn_dispatch<__half>(const AttnProblem &, const AttnView &, const AttnView &, const AttnView &, const AttnView &, float *,
                                   void *, void *, size_t, hipStream_t);

}  // namespace msd
