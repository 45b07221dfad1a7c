// Token embedding and its gradient for gfx950.
//     y[i] = scale * table[ids[i]] + positions[i % length]
//     dtable[v] = scale * (sum of dy[i] over the i with ids[i] = v),   dpositions[p] = sum of dy[i] over the i with i % length = p
// Up to 1024 tokens' gradient is one launch (few tokens, below).  More are sorted first (stable, by digits of 9 bits); a wavefront
// then takes kSlab sorted tokens and adds their rows of dy, runs of one token in ascending order in float32.  A run that lies in one
// slab is a row of dtable; a run over several leaves a part in each (padding; a few words are most of a text), and the last
// launch adds those: no atomics, the same bits every time, and no token costs more than its share.  The rows that no token names,
// and the sums over the batch for dpositions, are the work of workgroups beside the sort's, whose few ones mostly wait.
// Tokens outside [0, vocab) have rows of zeros and no gradient.
//
// Measured: 512 x 77 tokens, 50000 rows of 768, float16: rows out 16 us (61 MB written, the rows read again from the caches), the
// gradient's launches 2 x 11 (with the zeros: 77 MB) + 2 x 8, 15 and 11 us, 200 MB at the least.  2 x 77, 1024 columns: 2.9 us, latency.
#include <algorithm>
#include <initializer_list>

#include "msd_device.h"
#include "msd_internal.h"

namespace msd {
namespace {

constexpr uint32_t kThreads = 256;

// ---- forward ---------------------------------------------------------------

// N elements per lane: 16 or 8 bytes, or one element where rows are no whole pieces of those or not aligned to them.
template <typename T, int N>
__device__ __forceinline__ void load_piece(const T *p, float (&f)[N]) {
    T v[N];
    __builtin_memcpy(v, __builtin_assume_aligned(p, sizeof(v)), sizeof(v));
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = Store<T>::load1(v + e);
}
template <typename T, int N>
__device__ __forceinline__ void store_piece(T *p, const float (&f)[N]) {
    T v[N];
#pragma unroll
    for (int e = 0; e < N; e++) Store<T>::store1(v + e, f[e]);
    if constexpr (sizeof(v) == 16) {
        store_stream(reinterpret_cast<u32x4 *>(p), __builtin_bit_cast(u32x4, v));
    } else {
        __builtin_memcpy(__builtin_assume_aligned(p, sizeof(v)), v, sizeof(v));
    }
}

// 1 << shift adjacent lanes to a token.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void embed_kernel(const int64_t *ids, const T *table, const T *positions, T *y, uint32_t tokens,
                                                         uint32_t pieces, uint32_t length, uint32_t vocab, float scale,
                                                         uint32_t shift) {
    const uint32_t token = (blockIdx.x * kThreads + threadIdx.x) >> shift;
    if (token >= tokens) return;
    const int64_t id = ids[token];
    const size_t dim = (size_t)pieces * N;
    const bool known = id >= 0 && id < (int64_t)vocab;
    const T *const row = table + (known ? (size_t)id : 0) * dim;
    const T *const place = positions == nullptr ? nullptr : positions + (size_t)(token % length) * dim;
    for (uint32_t piece = threadIdx.x & ((1u << shift) - 1); piece < pieces; piece += 1u << shift) {
        float f[N], p[N];
        load_piece<T, N>(row + (size_t)piece * N, f);
        if (place != nullptr) {
            load_piece<T, N>(place + (size_t)piece * N, p);
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = known ? fmaf(f[e], scale, p[e]) : p[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = known ? f[e] * scale : 0.0f;
        }
        store_piece<T, N>(y + (size_t)token * dim + (size_t)piece * N, f);
    }
}

// ---- beside the sort ---------------------------------------------------------
constexpr uint32_t kSortThreads = 1024, kSortWaves = kSortThreads / kWave;

// Work of the workgroups behind the sort's own: zeros to dtable, and dpositions' partial sums over runs of the batch.
struct Side {
    char *zeros;             // (null: none in this launch)
    size_t zero_bytes;       // (a share of dtable: whole 16-byte vectors from its beginning on, but for the last)
    uint32_t zero_blocks;
    const void *dy;
    float *position_parts;   // [runs][length][dim], null: none in this launch
    uint32_t batch, length, pieces, run_blocks, runs;
    int piece;               // elements of a piece
};

template <typename T, int N>
__device__ __forceinline__ void positions_parts(const Side &w, uint32_t block) {
    const uint32_t run = block / w.run_blocks;
    const uint64_t count = (uint64_t)w.length * w.pieces, i = (uint64_t)(block - run * w.run_blocks) * kSortThreads + threadIdx.x;
    if (i >= count) return;
    const T *const dy = static_cast<const T *>(w.dy) + i * N;
    const size_t step = (size_t)w.length * w.pieces * N;
    const uint32_t each = (w.batch + w.runs - 1) / w.runs, stop = min(w.batch, (run + 1) * each);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.0f;
    for (uint32_t b = run * each; b < stop; b += 8) {
        float f[8][N];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) load_piece<T, N>(dy + min(b + u, stop - 1) * step, f[u]);
#pragma unroll
        for (uint32_t u = 0; u < 8; u++)
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += b + u < stop ? f[u][e] : 0.0f;
    }
    float *const out = w.position_parts + ((size_t)run * count + i) * N;
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = sum[e];
}

template <typename T>
__device__ __forceinline__ void side_work(const Side &w, uint32_t block) {
    if (block < w.zero_blocks) {
        const size_t at = (size_t)block * kSortThreads + threadIdx.x, step = (size_t)w.zero_blocks * kSortThreads;
        size_t vectors = w.zero_bytes / 16;
        if ((reinterpret_cast<uintptr_t>(w.zeros) & 15u) != 0) vectors = 0;
        for (size_t i = at; i < vectors; i += step) reinterpret_cast<u32x4 *>(w.zeros)[i] = u32x4{0, 0, 0, 0};
        for (size_t i = vectors * (16 / sizeof(T)) + at; i < w.zero_bytes / sizeof(T); i += step)
            Store<T>::store1(reinterpret_cast<T *>(w.zeros) + i, 0.0f);
        return;
    }
    block -= w.zero_blocks;
    constexpr int V = Store<T>::EPV;
    if (w.piece == V)
        positions_parts<T, V>(w, block);
    else if (w.piece == V / 2)
        positions_parts<T, V / 2>(w, block);
    else
        positions_parts<T, 1>(w, block);
}

// ---- sort --------------------------------------------------------------------
constexpr uint32_t kDigitBits = 9, kBins = 1u << kDigitBits;

struct Entry {  // a token and its place
    uint32_t id, at;
};

// Key of token i: its id, or vocab for one outside the table (those come last and are left out).
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, uint32_t i, uint32_t vocab) {
    const int64_t id = ids[i];
    return id >= 0 && id < (int64_t)vocab ? (uint32_t)id : vocab;
}

// How many of a block's tokens have each digit before this one: a wavefront has ROUNDS times 64 neighbouring tokens of the block.
// counts[w][bin] ends as the wavefront's count; rank[r] is the token's place among those of its wavefront
// and digit.  Lanes of a digit find each other by a ballot for each of its bits; the lowest of them moves the counter.
template <uint32_t ROUNDS>
__device__ __forceinline__ void rank_digits(uint16_t (*counts)[kBins], const uint32_t (&digit)[ROUNDS], const bool (&live)[ROUNDS],
                                            uint32_t (&rank)[ROUNDS]) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (uint32_t i = lane; i < kBins; i += kWave) counts[wave][i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        uint64_t same = __builtin_amdgcn_ballot_w64(live[r]);
#pragma unroll
        for (uint32_t bit = 0; bit < kDigitBits; bit++) {
            const bool one = (digit[r] >> bit & 1) != 0;
            const uint64_t ones = __builtin_amdgcn_ballot_w64(one);
            same &= one ? ones : ~ones;
        }
        const uint32_t before = __builtin_popcountll(same & ((1ull << lane) - 1));
        uint32_t base = 0;
        if (live[r]) base = counts[wave][digit[r]];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (live[r] && before == 0) counts[wave][digit[r]] = (uint16_t)(base + __builtin_popcountll(same));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[r] = base + before;
    }
}

// Turns counts[wave][bin] into the count before that wavefront; returns the block's total of bin threadIdx.x (< kBins).
__device__ __forceinline__ uint32_t before_waves(uint16_t (*counts)[kBins]) {
    uint32_t total = 0;
    if (threadIdx.x < kBins)
        for (uint32_t w = 0; w < kSortWaves; w++) {
            const uint32_t c = counts[w][threadIdx.x];
            counts[w][threadIdx.x] = (uint16_t)total;
            total += c;
        }
    return total;
}

// Sum of the values of lower lanes of the first kBins threads; every thread of the workgroup calls it.
__device__ __forceinline__ uint32_t before_bins(uint32_t v, uint32_t *slots) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t up = v;
#pragma unroll
    for (uint32_t d = 1; d < kWave; d *= 2) {
        const uint32_t o = __shfl_up(up, d, kWave);
        if (lane >= d) up += o;
    }
    if (lane == kWave - 1 && wave < kBins / kWave) slots[wave] = up;
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (uint32_t w = 0; w < kBins / kWave; w++)
        if (w < wave) base += slots[w];
    return base + up - v;
}

// Up to ROUNDS * 1024 tokens: one workgroup, all digits, the tokens in LDS between them.
template <typename T, uint32_t ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const int64_t *ids, Entry *sorted, uint32_t tokens, uint32_t vocab,
                                                                  uint32_t digits, const Side side) {
    if (blockIdx.x != 0) return side_work<T>(side, blockIdx.x - 1);
    __shared__ uint16_t counts[kSortWaves][kBins];
    __shared__ uint32_t start[kBins], slots[kBins / kWave];
    __shared__ Entry entries[(kSortThreads * ROUNDS)];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t id[ROUNDS], at[ROUNDS], digit[ROUNDS], rank[ROUNDS];
    bool live[ROUNDS];
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = wave * (kWave * ROUNDS) + r * kWave + lane;
        live[r] = i < tokens;
        at[r] = i;
        id[r] = live[r] ? key_of(ids, i, vocab) : 0;
    }
    for (uint32_t pass = 0; pass < digits; pass++) {
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; r++) digit[r] = id[r] >> (pass * kDigitBits) & (kBins - 1);
        rank_digits<ROUNDS>(counts, digit, live, rank);
        __syncthreads();
        const uint32_t total = before_waves(counts);
        const uint32_t first = before_bins(total, slots);
        if (threadIdx.x < kBins) start[threadIdx.x] = first;
        __syncthreads();
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; r++)
            if (live[r]) entries[start[digit[r]] + counts[wave][digit[r]] + rank[r]] = Entry{id[r], at[r]};
        __syncthreads();
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; r++) {
            const uint32_t i = wave * (kWave * ROUNDS) + r * kWave + lane;
            if (live[r]) {
                const Entry e = entries[i];
                id[r] = e.id;
                at[r] = e.at;
            }
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++)
        if (live[r]) sorted[wave * (kWave * ROUNDS) + r * kWave + lane] = Entry{id[r], at[r]};
}

// A block's tokens in front of a pass: from the ids, or from the pass before.
template <uint32_t ROUNDS>
__device__ __forceinline__ void block_entries(const int64_t *ids, const Entry *from, uint32_t tokens, uint32_t vocab, Entry (&e)[ROUNDS],
                                              bool (&live)[ROUNDS]) {
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = blockIdx.x * (kSortThreads * ROUNDS) + threadIdx.x / kWave * (kWave * ROUNDS) + r * kWave + threadIdx.x % kWave;
        live[r] = i < tokens;
        e[r] = Entry{0, i};
        if (live[r]) e[r] = from != nullptr ? from[i] : Entry{key_of(ids, i, vocab), i};
    }
}

// table[block][bin]: how many of the block's tokens have that digit.
template <typename T, uint32_t ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int64_t *ids, const Entry *from, uint32_t *table, uint32_t tokens,
                                                                  uint32_t vocab, uint32_t shift, uint32_t blocks, const Side side) {
    if (blockIdx.x >= blocks) return side_work<T>(side, blockIdx.x - blocks);
    __shared__ uint32_t bins[kBins];
    if (threadIdx.x < kBins) bins[threadIdx.x] = 0;
    __syncthreads();
    Entry e[ROUNDS];
    bool live[ROUNDS];
    block_entries<ROUNDS>(ids, from, tokens, vocab, e, live);
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++)
        if (live[r]) atomicAdd(&bins[e[r].id >> shift & (kBins - 1)], 1u);  // (whole numbers: any order gives the same)
    __syncthreads();
    if (threadIdx.x < kBins) table[(size_t)blockIdx.x * kBins + threadIdx.x] = bins[threadIdx.x];
}

// Every block adds the table's columns for itself: what lies before it in its bins, and the bins' totals.  That saves a launch, and
// grows with the square of the tokens: a pass over 2^20 takes 21 us, over 2^22 0.16 ms (as long as the sums of 8 columns), over 2^25,
// the most there are, 7.5 ms of a call's 17.6.
template <typename T, uint32_t ROUNDS>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int64_t *ids, const Entry *from, const uint32_t *table, Entry *to,
                                                                  uint32_t tokens, uint32_t vocab, uint32_t shift, uint32_t blocks,
                                                                  const Side side) {
    if (blockIdx.x >= blocks) return side_work<T>(side, blockIdx.x - blocks);
    __shared__ uint16_t counts[kSortWaves][kBins];
    __shared__ uint32_t start[kBins], half[2][kBins], slots[kBins / kWave];
    const uint32_t wave = threadIdx.x / kWave;
    Entry e[ROUNDS];
    bool live[ROUNDS];
    uint32_t digit[ROUNDS], rank[ROUNDS];
    block_entries<ROUNDS>(ids, from, tokens, vocab, e, live);
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) digit[r] = e[r].id >> shift & (kBins - 1);
    rank_digits<ROUNDS>(counts, digit, live, rank);
    // two threads to a bin: the even blocks' counts and the odd ones'
    const uint32_t bin = threadIdx.x % kBins, odd = threadIdx.x / kBins;
    uint32_t all = 0, mine = 0;
#pragma unroll 8
    for (uint32_t b = odd; b < blocks; b += 2) {
        const uint32_t c = table[(size_t)b * kBins + bin];
        all += c;
        mine += b < blockIdx.x ? c : 0;
    }
    if (odd == 1) {
        half[0][bin] = all;
        half[1][bin] = mine;
    }
    __syncthreads();
    if (odd == 0) {
        all += half[0][bin];
        mine += half[1][bin];
    } else {
        all = 0;
    }
    before_waves(counts);
    const uint32_t first = before_bins(all, slots);
    if (odd == 0) start[bin] = first + mine;
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++)
        if (live[r]) to[start[digit[r]] + counts[wave][digit[r]] + rank[r]] = e[r];
}

// ---- sums ----------------------------------------------------------------------
constexpr uint32_t kSlab = 32;  // sorted tokens of a wavefront

// First place in sorted[0, tokens) whose id is at least v; the whole wavefront looks, 64 places at a time.
__device__ __forceinline__ uint32_t first_of(const Entry *sorted, uint32_t tokens, uint32_t v) {
    uint32_t low = 0, high = tokens;  // the answer is in [low, high]
    const uint32_t lane = threadIdx.x % kWave;
    while (high - low > 0) {
        const uint32_t step = (high - low + kWave - 1) / kWave;
        const uint64_t probe = (uint64_t)low + (uint64_t)lane * step;
        const bool below = probe < high && sorted[probe].id < v;
        const uint32_t n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(below));  // (sorted: the first n lanes)
        if (n == 0) return low;
        const uint32_t last = low + (n - 1) * step;  // the last probe below v
        high = (uint32_t)min((uint64_t)high, (uint64_t)last + step);
        low = last + 1;
    }
    return low;
}

// A wavefront's slab and 64 of its pieces (few tokens of long rows are work for many wavefronts): parts[slab][2][dim] receives the
// run that comes in from the slab before, and the one that starts in it and goes on in the next; runs that begin and end here are
// rows of dtable.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void embed_grad_slabs_kernel(const T *dy, const Entry *sorted, T *dtable, float *parts, uint32_t tokens,
                                                                    uint32_t pieces, uint32_t vocab, float scale, uint32_t chunks) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave);
    const uint32_t slab = wave / chunks, p0 = (wave - slab * chunks) * kWave;
    const uint32_t begin = slab * kSlab, lane = threadIdx.x % kWave;
    if (begin >= tokens) return;
    const uint32_t n = min(kSlab, tokens - begin);
    const size_t dim = (size_t)pieces * N;
    const Entry mine = sorted[begin + min(lane, n - 1)];
    const uint32_t before = begin != 0 ? sorted[begin - 1].id : 0xFFFFFFFFu, after = begin + n < tokens ? sorted[begin + n].id : 0xFFFFFFFFu;
    auto id_of = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane(mine.id, i); };
    if (id_of(0) >= vocab) return;  // (those outside the table come last)
    const uint32_t p = min(p0 + lane, pieces - 1);
    const bool in = p0 + lane < pieces;
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.0f;
    auto put = [&](uint32_t id, bool first, bool last) {  // the run of `id` up to here
        if (!in || id >= vocab) return;
        if ((first && before == id) || (last && after == id)) {
            float *const out = parts + ((size_t)slab * 2 + (first && before == id ? 0 : 1)) * dim + (size_t)p * N;
#pragma unroll
            for (int e = 0; e < N; e++) out[e] = sum[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] *= scale;
            store_piece<T, N>(dtable + (size_t)id * dim + (size_t)p * N, sum);
        }
    };
    uint32_t id = id_of(0);
    bool first = true;
    for (uint32_t i0 = 0; i0 < n; i0 += 8) {
        float f[8][N];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
            const uint32_t at = (uint32_t)__builtin_amdgcn_readlane(mine.at, min(i0 + u, n - 1));
            load_piece<T, N>(dy + (size_t)at * dim + (size_t)p * N, f[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
            if (i0 + u >= n) break;
            const uint32_t next = id_of(i0 + u);
            if (next != id) {
                put(id, first, false);
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] = 0.0f;
                id = next;
                first = false;
            }
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += f[u][e];
        }
    }
    put(id, first, true);
}

constexpr uint32_t kJoinLane = 2, kJoinColumns = kJoinLane * kWave;  // columns of a lane, of a workgroup
constexpr uint32_t kJoinAlone = 16;  // slabs behind the first up to which a run is one wavefront's work

// A workgroup for kSortWaves slabs and kJoinColumns columns, a wavefront looking at each slab: it adds the parts of a run that starts
// in its slab and goes on, or, of a long one, all wavefronts a share each.  The workgroups behind `blocks` add dpositions' parts.
template <typename T>
__global__ __launch_bounds__(kSortThreads) void embed_grad_join_kernel(const Entry *sorted, const float *parts, T *dtable, uint32_t tokens,
                                                                       uint32_t dim, uint32_t vocab, float scale, uint32_t columns,
                                                                       uint32_t blocks, const float *position_parts, T *dpositions,
                                                                       uint64_t live, uint64_t count, uint32_t runs) {
    if (blockIdx.x >= blocks) {
        const uint64_t i = (uint64_t)(blockIdx.x - blocks) * kSortThreads + threadIdx.x;
        if (i >= count) return;
        float sum = 0.0f;
        if (i < live) {
#pragma unroll 4
            for (uint32_t r = 0; r < runs; r++) sum += position_parts[(size_t)r * live + i];
        }
        Store<T>::store1(dpositions + i, sum);
        return;
    }
    __shared__ float lds[kSortWaves][kJoinColumns];
    __shared__ uint32_t run_id[kSortWaves], run_slabs[kSortWaves];  // (slabs behind the first that a long run reaches; 0: none)
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t slab0 = blockIdx.x / columns * kSortWaves, col0 = blockIdx.x % columns * kJoinColumns;
    float sum[kJoinLane];
    auto add = [&](size_t part) {
#pragma unroll
        for (uint32_t c = 0; c < kJoinLane; c++) {
            const uint32_t col = col0 + c * kWave + lane;
            sum[c] += col < dim ? parts[part * dim + col] : 0.0f;
        }
    };
    {
        const uint32_t slab = slab0 + wave, begin = slab * kSlab;
        uint32_t id = 0, more = 0;
        if (begin < tokens && begin + kSlab < tokens) {
            id = sorted[begin + kSlab - 1].id;
            const bool here = begin == 0 || sorted[begin - 1].id != id;  // (it starts in this slab)
            if (here && id < vocab && sorted[begin + kSlab].id == id) more = (first_of(sorted, tokens, id + 1) - 1) / kSlab - slab;
        }
        more = __builtin_amdgcn_readfirstlane(more);
        const bool is_long = more > kJoinAlone;
        if (lane == 0) {
            run_id[wave] = id;
            run_slabs[wave] = is_long ? more : 0;
        }
        if (more != 0 && !is_long) {  // most runs: the wavefront's own
#pragma unroll
            for (uint32_t c = 0; c < kJoinLane; c++) sum[c] = 0.0f;
            add((size_t)slab * 2 + 1);
#pragma unroll 4
            for (uint32_t i = 0; i < more; i++) add(((size_t)slab + 1 + i) * 2);
#pragma unroll
            for (uint32_t c = 0; c < kJoinLane; c++) {
                const uint32_t col = col0 + c * kWave + lane;
                if (col < dim) Store<T>::store1(dtable + (size_t)id * dim + col, sum[c] * scale);
            }
        }
    }
    __syncthreads();
    for (uint32_t s = 0; s < kSortWaves; s++) {
        const uint32_t slabs = run_slabs[s], slab = slab0 + s;
        if (slabs == 0) continue;
        const uint32_t each = (slabs + kSortWaves - 1) / kSortWaves, stop = min(slabs, (wave + 1) * each);
#pragma unroll
        for (uint32_t c = 0; c < kJoinLane; c++) sum[c] = 0.0f;
        if (wave == 0) add((size_t)slab * 2 + 1);
        for (uint32_t i = wave * each; i < stop; i += 16) {
            float f[16][kJoinLane];
#pragma unroll
            for (uint32_t u = 0; u < 16; u++)
#pragma unroll
                for (uint32_t c = 0; c < kJoinLane; c++) {
                    const uint32_t col = col0 + c * kWave + lane;
                    f[u][c] = i + u < stop && col < dim ? parts[((size_t)slab + 1 + i + u) * 2 * dim + col] : 0.0f;
                }
#pragma unroll
            for (uint32_t u = 0; u < 16; u++)
#pragma unroll
                for (uint32_t c = 0; c < kJoinLane; c++) sum[c] += f[u][c];
        }
#pragma unroll
        for (uint32_t c = 0; c < kJoinLane; c++) lds[wave][c * kWave + lane] = sum[c];
        __syncthreads();
        if (threadIdx.x < kJoinColumns && col0 + threadIdx.x < dim) {
            float total = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kSortWaves; w++) total += lds[w][threadIdx.x];
            Store<T>::store1(dtable + (size_t)run_id[s] * dim + col0 + threadIdx.x, total * scale);
        }
        __syncthreads();
    }
}

// ---- few tokens ------------------------------------------------------------------
constexpr uint32_t kFewTokens = 1024, kFewBatch = 64, kFewThreads = 512, kFewWaves = kFewThreads / kWave, kFewEach = kFewTokens / kFewWaves;
constexpr uint32_t kZeroRows = 2048, kFewAtOnce = 8;

struct Few {
    uint32_t tokens, length, vocab, positions, pieces;
    uint32_t chunks, sum_blocks, zero_rows, zero_blocks;  // 64 pieces each; chunks for each token; rows of a block of zeros
    FastDiv by_pieces;
    float scale;
};

// Everything in one launch, without a sort: a workgroup for a token and 64 pieces of its row looks at all ids, leaves if the token's
// id occurs before it, and otherwise adds the rows of dy that have the id, a wavefront those of its share of the tokens in ascending
// order.  Other workgroups write the zeros of a range of table rows, but for those that some token names; others again dpositions.
template <typename T, int N>
__global__ __launch_bounds__(kFewThreads) void embed_grad_few_kernel(const int64_t *ids, const T *dy, T *dtable, T *dpositions, const Few f) {
    __shared__ uint32_t keys[kFewTokens];
    __shared__ float sums[kFewWaves][kWave * N];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const size_t dim = (size_t)f.pieces * N;
    uint32_t block = blockIdx.x;
    if (block < f.sum_blocks + f.zero_blocks) {
        for (uint32_t i = threadIdx.x; i < kFewTokens; i += kFewThreads) keys[i] = i < f.tokens ? key_of(ids, i, f.vocab) : f.vocab;
        __syncthreads();
    }
    if (block < f.sum_blocks) {
        const uint32_t token = block / f.chunks, piece = (block - token * f.chunks) * kWave + lane, key = keys[token];
        bool before = false;
        for (uint32_t i = threadIdx.x; i < token; i += kFewThreads) before |= keys[i] == key;
        if (__syncthreads_or(before) != 0 || key == f.vocab) return;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; e++) sum[e] = 0.0f;
        for (uint32_t i0 = wave * kFewEach; i0 < (wave + 1) * kFewEach; i0 += kWave) {
            uint64_t same = __builtin_amdgcn_ballot_w64(keys[i0 + lane] == key);
            while (same != 0) {
                typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) * N < 8 ? 1 : sizeof(T) * N / 4)));
                words v[kFewAtOnce];  // (as they are: a conversion here would wait for each)
#pragma unroll
                for (uint32_t u = 0; u < kFewAtOnce; u++) {
                    v[u] = words(0);
                    if (same == 0) continue;
                    const uint32_t at = i0 + (uint32_t)__builtin_ctzll(same);
                    same &= same - 1;
                    __builtin_memcpy(&v[u], __builtin_assume_aligned(dy + (size_t)at * dim + (size_t)min(piece, f.pieces - 1) * N, sizeof(T) * N),
                                     sizeof(T) * N);
                }
#pragma unroll
                for (uint32_t u = 0; u < kFewAtOnce; u++) {
                    T t[N];
                    __builtin_memcpy(t, &v[u], sizeof(t));
#pragma unroll
                    for (int e = 0; e < N; e++) sum[e] += Store<T>::load1(t + e);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < N; e++) sums[wave][e * kWave + lane] = sum[e];
        __syncthreads();
        if (wave != 0 || piece >= f.pieces) return;
#pragma unroll
        for (int e = 0; e < N; e++) {
            for (uint32_t w = 1; w < kFewWaves; w++) sum[e] += sums[w][e * kWave + lane];
            sum[e] *= f.scale;
        }
        store_piece<T, N>(dtable + (size_t)key * dim + (size_t)piece * N, sum);
        return;
    }
    block -= f.sum_blocks;
    float zero[N];
#pragma unroll
    for (int e = 0; e < N; e++) zero[e] = 0.0f;
    if (block < f.zero_blocks) {
        __shared__ uint32_t named[kZeroRows / 32];
        const uint32_t first = block * f.zero_rows, rows = min(f.zero_rows, f.vocab - first);
        if (threadIdx.x < kZeroRows / 32) named[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < f.tokens; i += kFewThreads) {
            const uint32_t r = keys[i] - first;
            if (keys[i] < f.vocab && r < rows) atomicOr(&named[r / 32], 1u << r % 32);  // (any order gives the same)
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < rows * f.pieces; i += kFewThreads) {
            const uint32_t r = fast_div(i, f.by_pieces);
            if ((named[r / 32] >> r % 32 & 1) == 0) store_piece<T, N>(dtable + (size_t)first * dim + (size_t)i * N, zero);
        }
        return;
    }
    block -= f.zero_blocks;
    const uint32_t i = block * kFewThreads + threadIdx.x;
    if (i >= f.positions * f.pieces) return;
    const uint32_t step = f.length * f.pieces, batch = i < step ? f.tokens / max(1u, f.length) : 0;
    for (uint32_t b = 0; b < batch; b += 8) {
        float v[8][N];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) load_piece<T, N>(dy + ((size_t)min(b + u, batch - 1) * step + i) * N, v[u]);
#pragma unroll
        for (uint32_t u = 0; u < 8; u++)
#pragma unroll
            for (int e = 0; e < N; e++) zero[e] += b + u < batch ? v[u][e] : 0.0f;
    }
    store_piece<T, N>(dpositions + (size_t)i * N, zero);
}

// Whether that launch does.  13 sequences of 77, 1000 rows of 768, float16: 9.0 us, by the sort 18.1; where two thirds of the text are
// one token 12.4 and 19.8; 9 of 61, 8191 rows of 650, float32: 12.2 and 11.4, by the sort 17.7 and 18.9 (with workgroups of 256 threads
// 9.5 and 15.8).  1024 tokens of 4096 columns, 32000 rows: 64 and 50 (each workgroup goes through all ids for 64 pieces of one token).
bool few_tokens(size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim) {
    return tokens <= kFewTokens && tokens * dim <= (size_t(1) << 20) && (positions == 0 || tokens <= kFewBatch * length) &&
           vocab * dim <= (size_t(1) << 35);  // (a launch holds the workgroups of the zeros)
}

uint32_t sort_digits(size_t vocab) {
    uint32_t bits = 1;
    while ((vocab >> bits) != 0) bits++;  // (keys go up to vocab itself)
    return (bits + kDigitBits - 1) / kDigitBits;
}

// Tokens per lane of the sort: four where one would make more workgroups than a chip has CUs by far, whose counts each adds for itself.
uint32_t sort_rounds(size_t tokens) { return tokens <= kSortThreads || (tokens > 4 * kSortThreads && tokens <= 128 * kSortThreads) ? 1 : 4; }

// Workspace: the sorted tokens twice (passes go from one to the other), the digits' table, the parts of runs, those of positions.
struct Layout {
    size_t entries[2], table, parts, position_parts, bytes;
    uint32_t blocks, rounds, digits, runs;
};
Layout layout(size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim) {
    Layout l{};
    auto take = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += (bytes + 255) & ~(size_t)255;
        return at;
    };
    l.rounds = sort_rounds(tokens);
    l.blocks = (uint32_t)((tokens + kSortThreads * l.rounds - 1) / (kSortThreads * l.rounds));
    l.digits = sort_digits(vocab);
    l.entries[0] = take(tokens * sizeof(Entry));
    if (l.blocks > 1) {
        l.entries[1] = take(tokens * sizeof(Entry));
        l.table = take((size_t)l.blocks * kBins * sizeof(uint32_t));
    }
    l.parts = take((tokens + kSlab - 1) / kSlab * 2 * dim * sizeof(float));
    if (positions != 0 && tokens != 0) {
        // runs of the batch: enough lanes for the chip, no fewer than 8 rows each
        const size_t batch = tokens / length, lanes = std::max<size_t>(1, length * dim / 4);
        const size_t want = (512 * (size_t)chip_info().cus + lanes - 1) / lanes;
        l.runs = (uint32_t)std::max<size_t>(1, std::min<size_t>(want, batch / 8));
        l.position_parts = take(l.runs * length * dim * sizeof(float));
    }
    return l;
}

template <typename T, uint32_t ROUNDS>
void sort_tokens(const EmbedGrad &g, const Layout &l, Entry *const (&entries)[2], uint32_t *table, const Entry **sorted, uint32_t tokens,
                 uint32_t vocab, size_t table_bytes, Side side, hipStream_t stream) {
    const uint32_t launches = l.blocks > 1 ? 2 * l.digits : 1;
    // a share of the zeros to every launch, positions' sums to the first
    const size_t share = (table_bytes / 16 + launches - 1) / launches * 16;
    auto next = [&](uint32_t launch) {
        const size_t from = std::min(table_bytes, launch * share);
        side.zeros = static_cast<char *>(g.dtable) + from;
        side.zero_bytes = launch + 1 == launches ? table_bytes - from : std::min(share, table_bytes - from);
        side.zero_blocks = (uint32_t)std::min<size_t>((side.zero_bytes / 16 + 4 * kSortThreads - 1) / (4 * kSortThreads) + 1, 1024);
        if (launch != 0) side.position_parts = nullptr;
        return l.blocks + side.zero_blocks + (side.position_parts != nullptr ? side.run_blocks * side.runs : 0);
    };
    if (l.blocks <= 1) {
        const uint32_t blocks = next(0) + 1 - l.blocks;  // (no tokens: the sort's workgroup finds none)
        launch((sort_small_kernel<T, ROUNDS>), dim3(blocks), dim3(kSortThreads), 0, stream, g.ids, entries[0], tokens, vocab, l.digits, side);
        *sorted = entries[0];
        return;
    }
    const Entry *from = nullptr;
    for (uint32_t pass = 0; pass < l.digits; pass++) {
        Entry *const to = entries[pass % 2];
        const uint32_t counting = next(2 * pass);
        launch((sort_count_kernel<T, ROUNDS>), dim3(counting), dim3(kSortThreads), 0, stream, g.ids, from, table, tokens, vocab,
               pass * kDigitBits, l.blocks, side);
        const uint32_t placing = next(2 * pass + 1);
        launch((sort_place_kernel<T, ROUNDS>), dim3(placing), dim3(kSortThreads), 0, stream, g.ids, from, table, to, tokens, vocab,
               pass * kDigitBits, l.blocks, side);
        from = to;
    }
    *sorted = from;
}

}  // namespace

size_t embed_grad_workspace_bytes(size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim) {
    return layout(tokens, length, vocab, positions, dim).bytes;
}

// Elements per piece: the widest of 16 and 8 bytes that rows are whole ones of, aligned, or 1.
template <typename T>
static int piece_of(size_t dim, std::initializer_list<const void *> at) {
    for (int n = Store<T>::EPV; n >= Store<T>::EPV / 2; n /= 2) {
        bool fits = dim % n == 0;
        for (const void *p : at) fits = fits && reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0;
        if (fits) return n;
    }
    return 1;
}

template <typename T, int N>
static void embed_rows(const int64_t *ids, const void *table, const void *positions, void *y, size_t tokens, size_t length, size_t vocab,
                       size_t dim, float scale, hipStream_t stream) {
    const size_t pieces = dim / N;
    uint32_t shift = 0;
    while (shift < 6 && (size_t(1) << shift) < pieces) shift++;
    launch((embed_kernel<T, N>), dim3((uint32_t)(((tokens << shift) + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, ids,
           static_cast<const T *>(table), static_cast<const T *>(positions), static_cast<T *>(y), (uint32_t)tokens, (uint32_t)pieces,
           (uint32_t)length, (uint32_t)vocab, scale, shift);
}

template <typename T>
int embed_dispatch(const int64_t *ids, const void *table, const void *positions, void *y, size_t tokens, size_t length, size_t vocab,
                   size_t dim, float scale, hipStream_t stream) {
    constexpr int V = Store<T>::EPV;
    switch (piece_of<T>(dim, {table, positions, y})) {
        case V: embed_rows<T, V>(ids, table, positions, y, tokens, length, vocab, dim, scale, stream); break;
        case V / 2: embed_rows<T, V / 2>(ids, table, positions, y, tokens, length, vocab, dim, scale, stream); break;
        default: embed_rows<T, 1>(ids, table, positions, y, tokens, length, vocab, dim, scale, stream); break;
    }
    return launch_status();
}

template <typename T, int N>
static void embed_grad_slabs(const EmbedGrad &g, const Entry *sorted, float *parts, uint32_t tokens, size_t dim, uint32_t vocab, float scale,
                             hipStream_t stream) {
    const uint32_t chunks = (uint32_t)((dim / N + kWave - 1) / kWave), per = kThreads / kWave;
    const size_t waves = (size_t)((tokens + kSlab - 1) / kSlab) * chunks;
    launch((embed_grad_slabs_kernel<T, N>), dim3((uint32_t)((waves + per - 1) / per)), dim3(kThreads), 0, stream, static_cast<const T *>(g.dy), sorted,
           static_cast<T *>(g.dtable), parts, tokens, (uint32_t)(dim / N), vocab, scale, chunks);
}

template <typename T, int N>
static int embed_grad_few(const EmbedGrad &g, size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim, float scale,
                          hipStream_t stream) {
    const size_t pieces = dim / N, row = dim * sizeof(T);
    Few f{};
    f.tokens = (uint32_t)tokens;
    f.length = (uint32_t)length;
    f.vocab = (uint32_t)vocab;
    f.positions = g.dpositions != nullptr ? (uint32_t)positions : 0;
    f.pieces = (uint32_t)pieces;
    f.chunks = (uint32_t)((pieces + kWave - 1) / kWave);
    f.sum_blocks = vocab != 0 ? f.tokens * f.chunks : 0;
    f.zero_rows = (uint32_t)std::max<size_t>(1, std::min<size_t>(kZeroRows, std::clamp<size_t>(vocab * row >> 11, 32 << 10, 256 << 10) / row));
    f.zero_blocks = (uint32_t)((vocab + f.zero_rows - 1) / f.zero_rows);
    f.by_pieces = make_fast_div(f.pieces);
    f.scale = scale;
    const size_t blocks = (size_t)f.sum_blocks + f.zero_blocks + ((size_t)f.positions * pieces + kFewThreads - 1) / kFewThreads;
    launch((embed_grad_few_kernel<T, N>), dim3((uint32_t)blocks), dim3(kFewThreads), 0, stream, g.ids, static_cast<const T *>(g.dy),
           static_cast<T *>(g.dtable), static_cast<T *>(g.dpositions), f);
    return launch_status();
}

template <typename T>
int embed_grad_dispatch(const EmbedGrad &g, size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim, float scale,
                        hipStream_t stream) {
    constexpr int V = Store<T>::EPV;
    if (few_tokens(tokens, length, vocab, positions, dim)) {
        switch (piece_of<T>(dim, {g.dy, g.dtable, g.dpositions})) {
            case V: return embed_grad_few<T, V>(g, tokens, length, vocab, positions, dim, scale, stream);
            case V / 2: return embed_grad_few<T, V / 2>(g, tokens, length, vocab, positions, dim, scale, stream);
            default: return embed_grad_few<T, 1>(g, tokens, length, vocab, positions, dim, scale, stream);
        }
    }
    Layout l = layout(tokens, length, vocab, positions, dim);
    if (l.runs != 0) l.runs = (uint32_t)std::min<size_t>(l.runs, (g.workspace_bytes - l.position_parts) / (length * dim * sizeof(float)));
    char *const base = static_cast<char *>(g.workspace);
    Entry *const entries[2] = {reinterpret_cast<Entry *>(base + l.entries[0]), reinterpret_cast<Entry *>(base + l.entries[1])};
    uint32_t *const table = reinterpret_cast<uint32_t *>(base + l.table);
    float *const parts = reinterpret_cast<float *>(base + l.parts);
    float *const position_parts = reinterpret_cast<float *>(base + l.position_parts);
    const int piece = piece_of<T>(dim, {g.dy, g.dtable});
    Side side{};
    side.dy = g.dy;
    side.piece = piece;
    side.pieces = (uint32_t)(dim / piece);
    if (l.runs != 0) {
        side.position_parts = position_parts;
        side.batch = (uint32_t)(tokens / length);
        side.length = (uint32_t)length;
        side.runs = l.runs;
        side.run_blocks = (uint32_t)((length * side.pieces + kSortThreads - 1) / kSortThreads);
    }
    const Entry *sorted = nullptr;
    const size_t table_bytes = vocab * dim * sizeof(T);
    if (l.rounds == 1)
        sort_tokens<T, 1>(g, l, entries, table, &sorted, (uint32_t)tokens, (uint32_t)vocab, table_bytes, side, stream);
    else
        sort_tokens<T, 4>(g, l, entries, table, &sorted, (uint32_t)tokens, (uint32_t)vocab, table_bytes, side, stream);
    if (tokens != 0 && vocab != 0) {
        if (piece == V)
            embed_grad_slabs<T, V>(g, sorted, parts, (uint32_t)tokens, dim, (uint32_t)vocab, scale, stream);
        else if (piece == V / 2)
            embed_grad_slabs<T, V / 2>(g, sorted, parts, (uint32_t)tokens, dim, (uint32_t)vocab, scale, stream);
        else
            embed_grad_slabs<T, 1>(g, sorted, parts, (uint32_t)tokens, dim, (uint32_t)vocab, scale, stream);
    }
    const uint64_t count = g.dpositions != nullptr ? (uint64_t)positions * dim : 0, live = tokens != 0 ? (uint64_t)length * dim : 0;
    const uint32_t slabs = (uint32_t)((tokens + kSlab - 1) / kSlab), columns = (uint32_t)((dim + kJoinColumns - 1) / kJoinColumns);
    const uint32_t blocks = slabs > 1 && vocab != 0 ? (slabs + kSortWaves - 1) / kSortWaves * columns : 0;  // (one slab has no run that goes on)
    const uint32_t more = (uint32_t)((count + kSortThreads - 1) / kSortThreads);
    if (blocks + more != 0)
        launch((embed_grad_join_kernel<T>), dim3(blocks + more), dim3(kSortThreads), 0, stream, sorted, parts, static_cast<T *>(g.dtable),
               (uint32_t)tokens, (uint32_t)dim, (uint32_t)vocab, scale, columns, blocks, position_parts, static_cast<T *>(g.dpositions), live,
               count, l.runs);
    return launch_status();
}

template int embed_dispatch<float>(const int64_t *, const void *, const void *, void *, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_dispatch<__half>(const int64_t *, const void *, const void *, void *, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_grad_dispatch<float>(const EmbedGrad &, size_t, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_grad_dispatch<__half>(const EmbedGrad &, size_t, size_t, size_t, size_t, size_t, float, hipStream_t);

}  // namespace msd
