// Token embedding and its gradient for gfx950.
//     y[i] = scale * table[ids[i]] + positions[i % length]
//     dtable[v] = scale * (sum of dy[i] over the i with ids[i] = v),   dpositions[p] = sum of dy[i] over the i with i % length = p
// Tokens are few next to what their rows hold, so the gradient first sorts them (stable, by digits of 9 bits) and then every
// row of dtable is written once by one wavefront, which adds its token's rows of dy in ascending order in float32: no atomics,
// the same bits every time.  A token that comes more often than kSlab times (padding; a few words are most of a text) is cut
// into parts, whose sums a second launch adds.  Tokens outside [0, vocab) have rows of zeros and no gradient.
#include <algorithm>

#include "msd_device.h"
#include "msd_internal.h"

namespace msd {
namespace {

constexpr uint32_t kThreads = 256;

// ---- forward ---------------------------------------------------------------

// N elements per lane: a 16-byte vector, or one element where rows are no whole vectors or not aligned to them.
template <typename T, int N>
__device__ __forceinline__ void load_piece(const T *p, float (&f)[N]) {
    if constexpr (N == 1)
        f[0] = Store<T>::load1(p);
    else
        Store<T>::unpack(*reinterpret_cast<const u32x4 *>(p), f);
}
template <typename T, int N>
__device__ __forceinline__ void store_piece(T *p, const float (&f)[N]) {
    if constexpr (N == 1)
        Store<T>::store1(p, f[0]);
    else
        store_stream(reinterpret_cast<u32x4 *>(p), Store<T>::pack(f));
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

// ---- sort --------------------------------------------------------------------
constexpr uint32_t kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr uint32_t kSortRounds = 4;  // tokens per lane
constexpr uint32_t kSortBlock = kSortThreads * kSortRounds;
constexpr uint32_t kDigitBits = 9, kBins = 1u << kDigitBits;

struct Entry {  // a token and its place
    uint32_t id, at;
};

// Key of token i: its id, or vocab for one outside the table (those come last and are left out).
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, uint32_t i, uint32_t vocab) {
    const int64_t id = ids[i];
    return id >= 0 && id < (int64_t)vocab ? (uint32_t)id : vocab;
}

// How many of a block's tokens have each digit before this one: wavefront w has the tokens [w * 256, w * 256 + 256) of the block
// in rounds of 64.  counts[w][bin] ends as the wavefront's count; rank[r] is the token's place among those of its wavefront
// and digit.  Lanes of a digit find each other by a ballot for each of its bits; the lowest of them moves the counter.
__device__ __forceinline__ void rank_digits(uint16_t (*counts)[kBins], const uint32_t (&digit)[kSortRounds],
                                            const bool (&live)[kSortRounds], uint32_t (&rank)[kSortRounds]) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (uint32_t i = lane; i < kBins; i += kWave) counts[wave][i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++) {
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

// Up to kSortBlock tokens: one workgroup, all digits, the tokens in LDS between them.
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const int64_t *ids, Entry *sorted, uint32_t tokens, uint32_t vocab,
                                                                  uint32_t digits) {
    __shared__ uint16_t counts[kSortWaves][kBins];
    __shared__ uint32_t start[kBins], slots[kBins / kWave];
    __shared__ Entry entries[kSortBlock];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t id[kSortRounds], at[kSortRounds], digit[kSortRounds], rank[kSortRounds];
    bool live[kSortRounds];
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++) {
        const uint32_t i = wave * (kWave * kSortRounds) + r * kWave + lane;
        live[r] = i < tokens;
        at[r] = i;
        id[r] = live[r] ? key_of(ids, i, vocab) : 0;
    }
    for (uint32_t pass = 0; pass < digits; pass++) {
#pragma unroll
        for (uint32_t r = 0; r < kSortRounds; r++) digit[r] = id[r] >> (pass * kDigitBits) & (kBins - 1);
        rank_digits(counts, digit, live, rank);
        __syncthreads();
        const uint32_t total = before_waves(counts);
        const uint32_t first = before_bins(total, slots);
        if (threadIdx.x < kBins) start[threadIdx.x] = first;
        __syncthreads();
#pragma unroll
        for (uint32_t r = 0; r < kSortRounds; r++)
            if (live[r]) entries[start[digit[r]] + counts[wave][digit[r]] + rank[r]] = Entry{id[r], at[r]};
        __syncthreads();
#pragma unroll
        for (uint32_t r = 0; r < kSortRounds; r++) {
            const uint32_t i = wave * (kWave * kSortRounds) + r * kWave + lane;
            if (live[r]) {
                const Entry e = entries[i];
                id[r] = e.id;
                at[r] = e.at;
            }
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++)
        if (live[r]) sorted[wave * (kWave * kSortRounds) + r * kWave + lane] = Entry{id[r], at[r]};
}

// A block's tokens in front of a pass: from the ids, or from the pass before.
__device__ __forceinline__ void block_entries(const int64_t *ids, const Entry *from, uint32_t tokens, uint32_t vocab, Entry (&e)[kSortRounds],
                                              bool (&live)[kSortRounds]) {
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++) {
        const uint32_t i = blockIdx.x * kSortBlock + threadIdx.x / kWave * (kWave * kSortRounds) + r * kWave + threadIdx.x % kWave;
        live[r] = i < tokens;
        e[r] = Entry{0, i};
        if (live[r]) e[r] = from != nullptr ? from[i] : Entry{key_of(ids, i, vocab), i};
    }
}

// table[block][bin]: how many of the block's tokens have that digit.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int64_t *ids, const Entry *from, uint32_t *table, uint32_t tokens,
                                                                  uint32_t vocab, uint32_t shift) {
    __shared__ uint32_t bins[kBins];
    if (threadIdx.x < kBins) bins[threadIdx.x] = 0;
    __syncthreads();
    Entry e[kSortRounds];
    bool live[kSortRounds];
    block_entries(ids, from, tokens, vocab, e, live);
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++)
        if (live[r]) atomicAdd(&bins[e[r].id >> shift & (kBins - 1)], 1u);  // (whole numbers: any order gives the same)
    __syncthreads();
    if (threadIdx.x < kBins) table[(size_t)blockIdx.x * kBins + threadIdx.x] = bins[threadIdx.x];
}

// Every block adds the table's columns for itself: what lies before it in its bins, and the bins' totals.
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int64_t *ids, const Entry *from, const uint32_t *table, Entry *to,
                                                                  uint32_t tokens, uint32_t vocab, uint32_t shift) {
    __shared__ uint16_t counts[kSortWaves][kBins];
    __shared__ uint32_t start[kBins], half[2][kBins], slots[kBins / kWave];
    const uint32_t wave = threadIdx.x / kWave;
    Entry e[kSortRounds];
    bool live[kSortRounds];
    uint32_t digit[kSortRounds], rank[kSortRounds];
    block_entries(ids, from, tokens, vocab, e, live);
#pragma unroll
    for (uint32_t r = 0; r < kSortRounds; r++) digit[r] = e[r].id >> shift & (kBins - 1);
    rank_digits(counts, digit, live, rank);
    // two threads to a bin: the even blocks' counts and the odd ones'
    const uint32_t bin = threadIdx.x % kBins, odd = threadIdx.x / kBins;
    uint32_t all = 0, mine = 0;
    for (uint32_t b = odd; b < gridDim.x; b += 2) {
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
    for (uint32_t r = 0; r < kSortRounds; r++)
        if (live[r]) to[start[digit[r]] + counts[wave][digit[r]] + rank[r]] = e[r];
}

// ---- sums ----------------------------------------------------------------------
constexpr uint32_t kSlab = 64;  // sorted tokens of a part; a token that comes more often is long
constexpr uint32_t kRows = 8;   // rows of dtable per wavefront

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

// Adds scale * dy of sorted[from, to) into one row, in order.  A lane has the pieces lane, lane + 64, ...
template <typename T, int N, typename Put>
__device__ __forceinline__ void add_rows(const T *dy, const Entry *sorted, uint32_t from, uint32_t to, uint32_t pieces, Put put) {
    const size_t dim = (size_t)pieces * N;
    for (uint32_t p = threadIdx.x % kWave; p < pieces; p += kWave) {
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; e++) sum[e] = 0.0f;
        uint32_t i = from;
        for (; i + 4 <= to; i += 4) {
            float f[4][N];
#pragma unroll
            for (int u = 0; u < 4; u++) load_piece<T, N>(dy + (size_t)sorted[i + u].at * dim + (size_t)p * N, f[u]);
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] += f[u][e];
        }
        for (; i < to; i++) {
            float f[N];
            load_piece<T, N>(dy + (size_t)sorted[i].at * dim + (size_t)p * N, f);
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += f[e];
        }
        put(p, sum);
    }
}

// Wavefronts [0, ceil(vocab / kRows)): the rows of dtable, long tokens' left out.  The following ceil(tokens / kSlab): the parts
// of long tokens in the sorted tokens' slabs, parts[slab][2][dim]: what comes in from the slab before, and what starts in it.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void embed_grad_rows_kernel(const T *dy, const Entry *sorted, T *dtable, float *parts, uint32_t tokens,
                                                                   uint32_t pieces, uint32_t vocab, float scale) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave);
    const uint32_t owners = (vocab + kRows - 1) / kRows;
    const size_t dim = (size_t)pieces * N;
    if (wave < owners) {
        uint32_t at = __builtin_amdgcn_readfirstlane(first_of(sorted, tokens, wave * kRows));
        for (uint32_t v = wave * kRows; v < min(vocab, (wave + 1) * kRows); v++) {
            // (the row's tokens: at most kSlab of them, or it is left to its parts)
            const uint32_t lane = threadIdx.x % kWave;
            const bool mine = at + lane < tokens && sorted[at + lane].id == v;
            const uint32_t n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine));
            if (n == kSlab && at + kSlab < tokens && sorted[at + kSlab].id == v) {
                at = __builtin_amdgcn_readfirstlane(first_of(sorted, tokens, v + 1));
                continue;
            }
            add_rows<T, N>(dy, sorted, at, at + n, pieces, [&](uint32_t p, const float (&sum)[N]) {
                float f[N];
#pragma unroll
                for (int e = 0; e < N; e++) f[e] = n != 0 ? sum[e] * scale : 0.0f;
                store_piece<T, N>(dtable + (size_t)v * dim + (size_t)p * N, f);
            });
            at += n;
        }
        return;
    }
    const uint32_t slab = wave - owners, begin = slab * kSlab;
    if (begin >= tokens) return;
    const uint32_t end = min(tokens, begin + kSlab);
    auto part = [&](uint32_t from, uint32_t to, uint32_t which) {
        float *const out = parts + ((size_t)slab * 2 + which) * dim;
        add_rows<T, N>(dy, sorted, from, to, pieces, [&](uint32_t p, const float (&sum)[N]) {
#pragma unroll
            for (int e = 0; e < N; e++) out[(size_t)p * N + e] = sum[e];
        });
    };
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t id = begin + lane < end ? sorted[begin + lane].id : 0xFFFFFFFFu;
    const uint32_t first = sorted[begin].id, last = sorted[end - 1].id;
    if (begin != 0 && sorted[begin - 1].id == first && first < vocab) {
        // is it long?  (it starts before this slab)
        const uint32_t from = first_of(sorted, tokens, first);
        if (from + kSlab < tokens && sorted[from + kSlab].id == first)
            part(begin, begin + __builtin_popcountll(__builtin_amdgcn_ballot_w64(id == first)), 0);
        if (first == last) return;
    }
    if (last < vocab) {
        const uint32_t n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(id == last && begin + lane < end));
        const uint32_t from = end - n;
        if (from + kSlab < tokens && sorted[from + kSlab].id == last) part(from, end, 1);
    }
}

// A workgroup for a slab in which a long token starts, and for 64 of its columns: the four wavefronts add a quarter of its parts each.
template <typename T>
__global__ __launch_bounds__(kThreads) void embed_grad_join_kernel(const Entry *sorted, const float *parts, T *dtable, uint32_t tokens,
                                                                   uint32_t dim, uint32_t vocab, float scale) {
    __shared__ float lds[kThreads / kWave][kWave];
    const uint32_t begin = blockIdx.x * kSlab, end = min(tokens, begin + kSlab);
    const uint32_t last = sorted[end - 1].id;
    if (last >= vocab || (begin != 0 && sorted[begin - 1].id == last)) return;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(begin + lane < end && sorted[begin + lane].id == last));
    const uint32_t from = end - n;
    if (from + kSlab >= tokens || sorted[from + kSlab].id != last) return;
    const uint32_t to = first_of(sorted, tokens, last + 1);
    const uint32_t slabs = (to - 1) / kSlab - blockIdx.x;  // after this one
    const uint32_t col = blockIdx.y * kWave + lane;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < dim) {
        if (wave == 0) sum[0] = parts[((size_t)blockIdx.x * 2 + 1) * dim + col];
        const uint32_t each = (slabs + 3) / 4, stop = min(slabs, (wave + 1) * each);
        uint32_t s = wave * each;
        for (; s + 4 <= stop; s += 4)
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) sum[u] += parts[((size_t)blockIdx.x + 1 + s + u) * 2 * dim + col];
        for (; s < stop; s++) sum[0] += parts[((size_t)blockIdx.x + 1 + s) * 2 * dim + col];
    }
    lds[wave][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    __syncthreads();
    if (wave != 0 || col >= dim) return;
    Store<T>::store1(dtable + (size_t)last * dim + col, ((lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane])) * scale);
}

// dpositions: runs of the batch to partial sums [runs][length][dim], one lane a piece of a row; the rows behind `length` are zero.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void positions_parts_kernel(const T *dy, float *parts, uint32_t batch, uint32_t length,
                                                                   uint32_t pieces, uint32_t runs) {
    const uint64_t count = (uint64_t)length * pieces, i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= count) return;
    const size_t dim = (size_t)pieces * N;
    const uint32_t each = (batch + runs - 1) / runs, stop = min(batch, (blockIdx.y + 1) * each);
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.0f;
    uint32_t b = blockIdx.y * each;
    for (; b + 4 <= stop; b += 4) {
        float f[4][N];
#pragma unroll
        for (uint32_t u = 0; u < 4; u++) load_piece<T, N>(dy + ((size_t)(b + u) * length) * dim + (size_t)i * N, f[u]);
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += f[u][e];
    }
    for (; b < stop; b++) {
        float f[N];
        load_piece<T, N>(dy + ((size_t)b * length) * dim + (size_t)i * N, f);
#pragma unroll
        for (int e = 0; e < N; e++) sum[e] += f[e];
    }
    float *const out = parts + ((size_t)blockIdx.y * count + i) * N;
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = sum[e];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void positions_join_kernel(const float *parts, T *dpositions, uint64_t live, uint64_t count,
                                                                  uint32_t runs) {
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= count) return;
    float sum = 0.0f;
    if (i < live)
        for (uint32_t r = 0; r < runs; r++) sum += parts[(size_t)r * live + i];
    Store<T>::store1(dpositions + i, sum);
}

uint32_t sort_digits(size_t vocab) {
    uint32_t bits = 1;
    while ((vocab >> bits) != 0) bits++;  // (keys go up to vocab itself)
    return (bits + kDigitBits - 1) / kDigitBits;
}

// Workspace: the sorted tokens twice (passes go from one to the other), the digits' table, the parts of long tokens, those of positions.
struct Layout {
    size_t entries[2], table, parts, position_parts, bytes;
    uint32_t blocks, digits, runs;
};
Layout layout(size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim) {
    Layout l{};
    auto take = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += (bytes + 255) & ~(size_t)255;
        return at;
    };
    l.blocks = (uint32_t)((tokens + kSortBlock - 1) / kSortBlock);
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

}  // namespace

size_t embed_grad_workspace_bytes(size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim) {
    return layout(tokens, length, vocab, positions, dim).bytes;
}

template <typename T>
int embed_dispatch(const int64_t *ids, const void *table, const void *positions, void *y, size_t tokens, size_t length, size_t vocab,
                   size_t dim, float scale, hipStream_t stream) {
    constexpr int N = Store<T>::EPV;
    const T *t = static_cast<const T *>(table), *p = static_cast<const T *>(positions);
    const bool vectors = dim % N == 0 && aligned16(table) && aligned16(positions) && aligned16(y);
    const size_t pieces = vectors ? dim / N : dim;
    uint32_t shift = 0;
    while (shift < 6 && (size_t(1) << shift) < pieces) shift++;
    const dim3 grid((uint32_t)(((tokens << shift) + kThreads - 1) / kThreads));
    if (vectors)
        launch((embed_kernel<T, N>), grid, dim3(kThreads), 0, stream, ids, t, p, static_cast<T *>(y), (uint32_t)tokens,
               (uint32_t)pieces, (uint32_t)length, (uint32_t)vocab, scale, shift);
    else
        launch((embed_kernel<T, 1>), grid, dim3(kThreads), 0, stream, ids, t, p, static_cast<T *>(y), (uint32_t)tokens,
               (uint32_t)pieces, (uint32_t)length, (uint32_t)vocab, scale, shift);
    return launch_status();
}

template <typename T, int N>
static void embed_grad_rows(const EmbedGrad &g, const Entry *sorted, float *parts, const Layout &l, size_t tokens, size_t length, size_t dim,
                            size_t vocab, float *position_parts, float scale, hipStream_t stream) {
    const T *dy = static_cast<const T *>(g.dy);
    const uint32_t pieces = (uint32_t)(dim / N);
    const size_t waves = (vocab + kRows - 1) / kRows + (tokens + kSlab - 1) / kSlab, per = kThreads / kWave;
    launch((embed_grad_rows_kernel<T, N>), dim3((uint32_t)((waves + per - 1) / per)), dim3(kThreads), 0, stream, dy, sorted,
           static_cast<T *>(g.dtable), parts, (uint32_t)tokens, pieces, (uint32_t)vocab, scale);
    if (g.dpositions != nullptr && tokens != 0)
        launch((positions_parts_kernel<T, N>), dim3((uint32_t)((length * pieces + kThreads - 1) / kThreads), l.runs), dim3(kThreads), 0,
               stream, dy, position_parts, (uint32_t)(tokens / length), (uint32_t)length, pieces, l.runs);
}

template <typename T>
int embed_grad_dispatch(const EmbedGrad &g, size_t tokens, size_t length, size_t vocab, size_t positions, size_t dim, float scale,
                        hipStream_t stream) {
    const Layout l = layout(tokens, length, vocab, positions, dim);
    char *const base = static_cast<char *>(g.workspace);
    Entry *entries[2] = {reinterpret_cast<Entry *>(base + l.entries[0]), reinterpret_cast<Entry *>(base + l.entries[1])};
    uint32_t *const table = reinterpret_cast<uint32_t *>(base + l.table);
    float *const parts = reinterpret_cast<float *>(base + l.parts);
    float *const position_parts = reinterpret_cast<float *>(base + l.position_parts);
    const Entry *sorted = entries[0];
    if (l.blocks == 1) {
        launch(sort_small_kernel, dim3(1), dim3(kSortThreads), 0, stream, g.ids, entries[0], (uint32_t)tokens, (uint32_t)vocab, l.digits);
    } else if (l.blocks > 1) {
        const Entry *from = nullptr;
        for (uint32_t pass = 0; pass < l.digits; pass++) {
            Entry *const to = entries[pass % 2];
            launch(sort_count_kernel, dim3(l.blocks), dim3(kSortThreads), 0, stream, g.ids, from, table, (uint32_t)tokens,
                   (uint32_t)vocab, pass * kDigitBits);
            launch(sort_place_kernel, dim3(l.blocks), dim3(kSortThreads), 0, stream, g.ids, from, table, to, (uint32_t)tokens,
                   (uint32_t)vocab, pass * kDigitBits);
            from = to;
        }
        sorted = from;
    }
    constexpr int N = Store<T>::EPV;
    const bool vectors = dim % N == 0 && aligned16(g.dy) && aligned16(g.dtable);
    if (vectors)
        embed_grad_rows<T, N>(g, sorted, parts, l, tokens, length, dim, vocab, position_parts, scale, stream);
    else
        embed_grad_rows<T, 1>(g, sorted, parts, l, tokens, length, dim, vocab, position_parts, scale, stream);
    if (tokens > kSlab)  // (fewer: no token is long)
        launch((embed_grad_join_kernel<T>), dim3((uint32_t)((tokens + kSlab - 1) / kSlab), (uint32_t)((dim + kWave - 1) / kWave)),
               dim3(kThreads), 0, stream, sorted, parts, static_cast<T *>(g.dtable), (uint32_t)tokens, (uint32_t)dim, (uint32_t)vocab,
               scale);
    if (g.dpositions != nullptr) {
        const uint64_t count = (uint64_t)positions * dim, live = tokens != 0 ? (uint64_t)length * dim : 0;
        launch((positions_join_kernel<T>), dim3((uint32_t)((count + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, position_parts,
               static_cast<T *>(g.dpositions), live, count, l.runs);
    }
    return launch_status();
}

template int embed_dispatch<float>(const int64_t *, const void *, const void *, void *, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_dispatch<__half>(const int64_t *, const void *, const void *, void *, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_grad_dispatch<float>(const EmbedGrad &, size_t, size_t, size_t, size_t, size_t, float, hipStream_t);
template int embed_grad_dispatch<__half>(const EmbedGrad &, size_t, size_t, size_t, size_t, size_t, float, hipStream_t);

}  // namespace msd
