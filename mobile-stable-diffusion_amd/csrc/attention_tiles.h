// What the attention kernels share (attention.hip, attention_grad.hip): fragments of the 32 x 32 x 16 matrix products, tiles of
// rows in LDS that are read by rows and by columns, the way from a workgroup to its sequence.
//
// Products are formed transposed, so that what one leaves in registers is what the next one takes.  With A's rows and B's
// columns both indexed by lane & 31, the accumulator's lane has column lane & 31 and, in register 4 i + j, row 8 i + 4 h + j
// with h = lane / 32.  Registers 8 t ... 8 t + 7 are then, rounded to the storage type, the B operand of the product over
// rows 16 t ... 16 t + 15, if its A operand takes the same rows in the same order.
//
// float32 goes through the same fragments, eight values a lane.  Each value is cut into three bfloat16 (8 bits each, together
// all 24, and the exponents of float32), and six products of those stand for the one of float32: the three left out are below
// 2^-23 of it.  Six products of 32 x 32 x 16 take 192 cycles, the eight of 32 x 32 x 2 in float32 512.
#pragma once

#include <initializer_list>

#include "msd_device.h"
#include "msd_internal.h"

namespace msd {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kAttnThreads = 256, kAttnWaves = kAttnThreads / kWave;
// A workgroup has 1 or 4 wavefronts, each with 32 rows of its own; the tiles that pass by are everyone's.
constexpr uint32_t attn_rows(bool few) { return few ? 32 : 32 * kAttnWaves; }

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Thirds {  // eight float32 as sums of three bfloat16 each
    bf16x8 part[3];
};

// type: a fragment as it is read; operand: as a product's B operand takes it.
template <typename T>
struct Frag;
template <>
struct Frag<__half> {
    typedef half8 type;
    typedef half8 operand;
    static constexpr int kTile = 64;  // rows of a tile in LDS
    static constexpr bool kFloat = false;
};
template <>
struct Frag<float> {
    typedef f32x8 type;
    typedef Thirds operand;
    static constexpr int kTile = 32;
    static constexpr bool kFloat = true;
};

__device__ __forceinline__ f32x16 mma(const half8 &a, const half8 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half8 operand(const half8 &f) { return f; }
template <bool ODD = true>
__device__ __forceinline__ Thirds operand(const f32x8 &f) {
    // ODD: an infinity is the largest finite values and an infinity in the third part, which meets the other operand's first alone:
    // times a zero second or third part of a finite value it would be NaN.  A NaN is in the third part, too.  (Weights and score
    // gradients are not infinite but where the gradient is NaN.)
    constexpr float kMost = 0x1.fffffep127f;
    Thirds t;
    float left[8];
#pragma unroll
    for (int j = 0; j < 8; j++) left[j] = f[j];
#pragma unroll
    for (int n = 0; n < 3; n++) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            w[j] = __float_as_uint(ODD && n < 2 ? __builtin_amdgcn_fmed3f(left[j], -kMost, kMost) : left[j]);
            left[j] -= __uint_as_float(w[j] & 0xFFFF0000u);
        }
        u32x4 packed;
#pragma unroll
        for (int j = 0; j < 4; j++) packed[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);  // (the upper halves)
        t.part[n] = __builtin_bit_cast(bf16x8, packed);
    }
    return t;
}
__device__ __forceinline__ f32x16 mma(const f32x8 &a, const Thirds &b, f32x16 c) {
    const Thirds t = operand(a);
    constexpr int kPairs[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};  // (the small ones first)
#pragma unroll
    for (int n = 0; n < 6; n++)
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(t.part[kPairs[n][0]], b.part[kPairs[n][1]], c, 0, 0, 0);
    return c;
}

// Between steps of products whose operands fill the registers: none is read from LDS ahead of its step (with all of them read
// first there is no room).
template <bool FULL>
__device__ __forceinline__ void step_end() {
    if (FULL) __builtin_amdgcn_sched_barrier(0);
}

// Registers 8 t ... 8 t + 7 of an accumulator as a B operand (float16: rounded to nearest).
__device__ __forceinline__ void to_frag(const f32x16 &c, int t, half8 &b) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __half2 h = __floats2half2_rn(c[8 * t + 2 * j], c[8 * t + 2 * j + 1]);
        typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
        const half2_t v = __builtin_bit_cast(half2_t, h);
        b[2 * j] = v[0];
        b[2 * j + 1] = v[1];
    }
}
__device__ __forceinline__ void to_frag(const f32x16 &c, int t, Thirds &b) {
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = c[8 * t + j];
    b = operand<false>(f);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; i++) z[i] = 0.0f;
    return z;
}

// Keeps the compiler from moving what gives a fragment behind the branches that follow.
__device__ __forceinline__ void keep_here(half8 &f) {
    u32x4 v = __builtin_bit_cast(u32x4, f);
    asm volatile("" : "+v"(v));
    f = __builtin_bit_cast(half8, v);
}

__device__ __forceinline__ void keep_here(Thirds &) {}

// A masked pair's weight is zero, but zero times an infinity or NaN is not.  Where a tile has masked pairs, what its A operands
// hold of those is left out of the product, and `add_odd` puts it back for the pairs that are visible.
template <int N, typename F>
__device__ __forceinline__ bool any_odd(const F (&a)[N]) {
    uint32_t found = 0;
#pragma unroll
    for (int n = 0; n < N; n++) {
        uint32_t w[sizeof(F) / 4];
        __builtin_memcpy(w, &a[n], sizeof(F));
#pragma unroll
        for (uint32_t i = 0; i < sizeof(F) / 4; i++)  // (an exponent of ones, and one more, is the sign's bit)
            found |= sizeof(F) == 16 ? (w[i] & 0x7C007C00u) + 0x04000400u : (w[i] & 0x7F800000u) + 0x00800000u;
    }
    return __builtin_amdgcn_ballot_w64((found & (sizeof(F) == 16 ? 0x80008000u : 0x80000000u)) != 0) != 0;
}
template <int N, typename F>
__device__ __forceinline__ void leave_out_odd(F (&a)[N], bool &odd) {
    if (!any_odd<N>(a)) return;
    odd = true;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (!(__builtin_fabsf((float)a[n][j]) < __builtin_inff())) a[n][j] = 0;
}
template <typename T, int D>
struct TileLanes;

// The infinities and NaN of a tile's columns, one kind at a time as ones against ones at the visible pairs (`visible(row)`: of
// the lane's column and that row of the tile): a positive count puts the value into the sum.
template <typename T, int D, int ROWS, typename Tile, typename Visible>
__device__ __forceinline__ void add_odd(const Tile &tile, const TileLanes<T, D> &lanes, f32x16 (&acc)[D / 32], Visible visible) {
    typedef typename Frag<T>::type frag;
    const uint32_t h = threadIdx.x % kWave / 32;
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS; r0 += 16) {
        frag ones;
#pragma unroll
        for (int j = 0; j < 8; j++) ones[j] = visible(r0 + 8 * (j / 4) + 4 * h + j % 4) ? 1 : 0;
        const typename Frag<T>::operand seen = operand(ones);
#pragma unroll
        for (int d = 0; d < D / 32; d++) {
            const frag one[1] = {tile.columns(lanes, r0, d)}, &a = one[0];
            if (!any_odd<1>(one)) continue;
#pragma unroll 1
            for (int kind = 0; kind < 3; kind++) {
                const float value = kind == 0 ? __builtin_inff() : kind == 1 ? -__builtin_inff() : __builtin_nanf("");
                frag is;
#pragma unroll
                for (int j = 0; j < 8; j++) is[j] = (kind == 2 ? a[j] != a[j] : (float)a[j] == value) ? 1 : 0;
                const f32x16 count = mma(is, seen, zero16());
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (count[i] > 0.0f) acc[d][i] += value;
            }
        }
    }
}

// 16 bytes of a row from column d on, zeros behind its end, for rows that are no whole aligned vectors.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T *row, uint32_t d, uint32_t dim) {
    constexpr int E = 16 / sizeof(T);
    T v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = d + e < dim ? row[d + e] : T(0.0f);
    u32x4 out;
    __builtin_memcpy(&out, v, 16);
    return out;
}

// Operands that a wavefront keeps: 32 rows (its lane's row, or null) as KD fragments.
template <typename T, int D>
__device__ __forceinline__ void load_frags(const T *row, uint32_t dim, bool vec, typename Frag<T>::operand (&f)[D / 16]) {
    const uint32_t h = threadIdx.x % kWave / 32;
    constexpr uint32_t kPer = sizeof(T) / 2, E = 16 / sizeof(T);  // chunks of a fragment, elements of a chunk
    u32x4 v[D / 16 * kPer];
    if (vec) {
#pragma unroll
        for (uint32_t c = 0; c < D / 16 * kPer; c++) {
            const uint32_t d = 16 * (c / kPer) + 8 * h + c % kPer * E;
            v[c] = row != nullptr && d < dim ? *reinterpret_cast<const u32x4 *>(row + d) : u32x4{0, 0, 0, 0};
        }
    } else {
#pragma unroll
        for (uint32_t c = 0; c < D / 16 * kPer; c++)
            v[c] = row != nullptr ? load_chunk<T>(row, 16 * (c / kPer) + 8 * h + c % kPer * E, dim) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
        typename Frag<T>::type one;
        __builtin_memcpy(&one, v + k * kPer, sizeof(one));
        f[k] = operand(one);
    }
}

// float32: acc += a tile's columns times `p`, its 32 rows' weights.  A tile's products are summed by themselves: each product of
// thirds rounds the sum that it goes into, and over 18000 keys twelve of those in the whole sum left 1.9 times the error of
// the plain form in float32, one a tile leaves less than it.
template <bool MASKED, bool APART, typename T, int D, typename Tile>
__device__ __forceinline__ void add_products(const Tile &tile, const TileLanes<T, D> &lanes, const Thirds (&p)[2], f32x16 (&acc)[D / 32], bool &odd) {
    static_assert(Frag<T>::kFloat && Tile::kRows == 32);
#pragma unroll
    for (int d = 0; d < D / 32; d++) {
        f32x16 sum = APART ? zero16() : acc[d];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            typename Frag<T>::type c[1] = {tile.columns(lanes, 16 * u, d)};
            if constexpr (MASKED) leave_out_odd<1>(c, odd);
            sum = mma(c[0], p[u], sum);
        }
        acc[d] = APART ? acc[d] + sum : sum;
        step_end<true>();
    }
}

constexpr uint32_t kNowhere = 0x80000000u;  // an offset behind the end of any rows of a tile (attn_vectors)

// Until what Tile::request asked for is in LDS (this wavefront's part; a barrier makes it everyone's).
__device__ __forceinline__ void wait_tiles() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ u32x4 buffer_resource(const void *from, uint32_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)),
                 (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
// A float of each lane straight from memory, `offset` bytes behind `from`, to one place after the other of LDS; as Tile::request.
__device__ __forceinline__ void request_floats(float *lds, const void *from, uint32_t bytes, uint32_t offset) {
    const u32x4 resource = buffer_resource(from, bytes);
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds));
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(to), "v"(offset), "s"(resource)
                 : "memory");
}

// Rows of 128 float16 are 256 bytes, as many as the banks of LDS are together: see place_of.
template <typename T, int D>
constexpr bool kWideRows = !Frag<T>::kFloat && D == 128;

// What the number of a chunk is crossed with in row r of a tile, so that lanes that read one chunk of neighbouring rows, or
// neighbouring chunks of four rows, meet different banks.  Rows of 256 bytes: four bits, of which four neighbouring rows differ in the
// upper two (reads by columns: four chunks of four rows at a time) and sixteen in all.  With the three bits of the others
// conflicts were two fifths of the time of the kernel for dk and dv.
template <typename T, int D>
__device__ __forceinline__ uint32_t place_of(uint32_t r) {
    return kWideRows<T, D> ? (r & 3) << 2 | (r >> 2 & 3) : r & 7;
}

// Where a lane reads in a tile (below), in bytes from its beginning.  The places differ by more than a constant only in the three
// bits of the chunk's number that the row's number goes into: a few registers, and the rest is in the instructions.  Wide rows: one
// register each, crossed with a constant (a tile begins at a multiple of 256).
template <typename T, int D>
struct TileLanes {
    static constexpr uint32_t kRowBytes = D * sizeof(T);
    uint32_t row[kWideRows<T, D> ? 1 : 4], column[kWideRows<T, D> ? 1 : Frag<T>::kFloat ? 4 : 2];
    __device__ __forceinline__ TileLanes() {
        const uint32_t lane = threadIdx.x % kWave, h = lane / 32, i = lane % 16;
        if constexpr (kWideRows<T, D>) {
            row[0] = lane % 32 * kRowBytes + (h ^ place_of<T, D>(lane)) * 16;
            column[0] = (4 * h + i / 4) * kRowBytes + ((2 * (lane / 16 % 2) + i % 4 / 2) ^ place_of<T, D>(4 * h + i / 4)) * 16 + i % 2 * 8;
            return;
        } else {
            for (uint32_t j = 0; j < 4; j++)
                row[j] = lane % 32 * kRowBytes + (((Frag<T>::kFloat ? 4 * (j / 2) + 2 * h + j % 2 : 2 * j + h) ^ lane % 8) * 16);
        }
        if constexpr (Frag<T>::kFloat) {
            for (uint32_t j = 0; j < 4; j++)
                column[j] = (4 * h + j) * kRowBytes + (lane % 32 / 4 ^ (4 * h + j)) * 16 + lane % 4 * 4;
        } else if constexpr (!kWideRows<T, D>) {
            for (uint32_t j = 0; j < 2; j++)
                column[j] = (4 * h + i / 4) * kRowBytes + ((4 * j + 2 * (lane / 16 % 2) + i % 4 / 2) ^ (4 * h + i / 4)) * 16 + i % 2 * 8;
        }
    }
};

// A tile in LDS: ROWS rows of D values as 16-byte chunks, chunk c of row r at place c ^ place_of(r).
template <typename T, int D, int WAVES, int ROWS = Frag<T>::kTile>
struct Tile {
    static constexpr int kThreads = WAVES * kWave, kRows = ROWS, kChunks = D * (int)sizeof(T) / 16;
    static constexpr int kPerThread = kRows * kChunks / kThreads;
    // places of a thread that lie kTurn apart are kTurn * kStep rows apart, in the same column
    static constexpr int kStep = kThreads / kChunks, kTurn = kStep >= 8 ? 1 : 8 / kStep;
    typedef typename Frag<T>::type frag;
    alignas(kWideRows<T, D> ? 256 : 16) u32x4 data[kRows * kChunks];

    // Row and column of the chunk that belongs at this thread's place number p.
    static __device__ __forceinline__ uint32_t row_of(int p) { return (p * kThreads + threadIdx.x) / kChunks; }
    static __device__ __forceinline__ uint32_t column_of(int p) {
        return ((p * kThreads + threadIdx.x) % kChunks ^ place_of<T, D>(row_of(p))) * (16 / (uint32_t)sizeof(T));
    }
    // Bytes from a tile's first row to this thread's first kTurn chunks, for rows of `row` elements; chunk p is at
    // `offset_of(base, row, p)`.
    static __device__ __forceinline__ void offsets(uint32_t row, uint32_t dim, uint32_t (&base)[kTurn]) {
#pragma unroll
        for (int p = 0; p < kTurn; p++) base[p] = column_of(p) < dim ? (row_of(p) * row + column_of(p)) * (uint32_t)sizeof(T) : kNowhere;
    }
    static __device__ __forceinline__ uint32_t offset_of(const uint32_t (&base)[kTurn], uint32_t row, int p) {
        return base[p % kTurn] + p / kTurn * (kTurn * kStep * (uint32_t)sizeof(T)) * row;
    }
    // Asks for this thread's chunks, `offset(p)` bytes behind `from` (the same in the whole wavefront), straight from memory to
    // LDS; from byte `bytes` on there are zeros.  wait_tiles() and a barrier later they are there.  Written as assembly because
    // the compiler, which knows no more than that these write LDS, would wait for them in front of every read by columns.
    template <typename Offset>
    __device__ __forceinline__ void request(const void *from, uint32_t bytes, Offset offset) {
        const u32x4 resource = buffer_resource(from, bytes);
        const uint32_t first = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * kWave;
        const uint32_t lds = __builtin_amdgcn_readfirstlane(
            (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)data) + first * 16);
#pragma unroll
        for (int p = 0; p < kPerThread; p++) {
            uint32_t m0;  // (the compiler's own; a load takes it when it is issued)
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                         : "=&s"(m0)
                         : "s"(lds + p * kThreads * 16), "v"(offset(p)), "s"(resource)
                         : "memory");
        }
    }
    // The same through registers, for rows that are no whole aligned vectors: `row(r)` is a row's first value, or null for zeros.
    template <typename Row>
    __device__ __forceinline__ void copy(Row row, uint32_t dim) {
#pragma unroll 1
        for (int p = 0; p < kPerThread; p++) {
            const T *const from = row(row_of(p));
            data[p * kThreads + threadIdx.x] = from != nullptr ? load_chunk<T>(from, column_of(p), dim) : u32x4{0, 0, 0, 0};
        }
    }

    typedef __attribute__((address_space(3))) const char *lds_t;
    // (wide rows) A lane's place, crossed with a constant below 256.
    __device__ __forceinline__ lds_t crossed(uint32_t lane, uint32_t with) const {
        return (lds_t)(((uint32_t)(uintptr_t)(lds_t)data + lane) ^ with);
    }
    // A operand by rows: row r0 + (lane & 31), columns 16 k + 8 h ...
    __device__ __forceinline__ frag rows(const TileLanes<T, D> &l, int r0, int k) const {
        const lds_t at = (lds_t)data;
        frag f;
        u32x4 v[sizeof(T) / 2];
        if constexpr (kWideRows<T, D>) {
            v[0] = *(__attribute__((address_space(3))) const u32x4 *)(crossed(l.row[0], 32 * k) + r0 * kChunks * 16);
        } else if constexpr (!Frag<T>::kFloat) {
            v[0] = *(__attribute__((address_space(3))) const u32x4 *)(at + l.row[k % 4] + (r0 * kChunks * 16 + k / 4 * 128));
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++)
                v[i] = *(__attribute__((address_space(3))) const u32x4 *)(at + l.row[k % 2 * 2 + i] + (r0 * kChunks * 16 + k / 2 * 128));
        }
        __builtin_memcpy(&f, v, sizeof(f));
        return f;
    }
    // A operand by columns: column 32 db + (lane & 31), the 16 rows from r0 on in the accumulators' order
    __device__ __forceinline__ frag columns(const TileLanes<T, D> &l, int r0, int db) const {
        const lds_t at = (lds_t)data;
        frag f;
        if constexpr (!Frag<T>::kFloat) {
            // 16 lanes read 4 rows of 16 columns, 8 bytes a lane, and each gets a column of 4
#pragma unroll
            for (int u = 0; u < 2; u++) {
                typedef fp16x4 __attribute__((address_space(3))) *four_t;
                four_t from;
                if constexpr (kWideRows<T, D>)
                    from = (four_t)(crossed(l.column[0], 64 * db ^ 32 * u) + (r0 + 8 * u) * kChunks * 16);
                else
                    from = (four_t)(at + l.column[db % 2] + ((r0 + 8 * u) * kChunks * 16 + db / 2 * 128));
                const fp16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4f16(from);
#pragma unroll
                for (int j = 0; j < 4; j++) f[4 * u + j] = (_Float16)v[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                f[j] = *(__attribute__((address_space(3))) const float *)(at + l.column[j % 4] + ((r0 + j / 4 * 8) * kChunks * 16 + db * 128));
        }
        return f;
    }
};

// a b in float32.  (Left to itself the compiler joins some of these with the rounding to float16 that follows, and other alignments
// have other bits.)
__device__ __forceinline__ float rounded_product(float a, float b) {
    float v = a * b;
    asm volatile("" : "+v"(v));
    return v;
}

// Stores an accumulator's columns: row `to` gets the lane's column times `by`; `left`, if not null, what rounding took from it.
template <typename T, int D>
__device__ __forceinline__ void store_rows(T *to, const f32x16 (&acc)[D / 32], float by, uint32_t dim, bool vec, T *left = nullptr) {
    const uint32_t h = threadIdx.x % kWave / 32;
    if (vec) {
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t col = 32 * d + 8 * g + 4 * h;
                T v[4], l[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float value = rounded_product(acc[d][4 * g + j], by);
                    Store<T>::store1(v + j, value);
                    Store<T>::store1(l + j, value - Store<T>::load1(v + j));
                }
                if (col >= dim) continue;
                __builtin_memcpy(__builtin_assume_aligned(to + col, 4 * sizeof(T)), v, sizeof(v));
                if (left != nullptr) __builtin_memcpy(__builtin_assume_aligned(left + col, 4 * sizeof(T)), l, sizeof(l));
            }
        return;
    }
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const uint32_t col = 32 * d + 8 * (r / 4) + 4 * h + r % 4;
            if (col >= dim) continue;
            const float value = rounded_product(acc[d][r], by);
            Store<T>::store1(to + col, value);
            if (left != nullptr) Store<T>::store1(left + col, value - round_to_storage<T>(value));
        }
}

// Maximum with the lane of the other half.
__device__ __forceinline__ float halves_max(float v) { return fmaxf(v, half_swap(v)); }

struct AttnShape {
    const int32_t *q_offsets, *k_offsets;  // [batch + 1] or null: sequences of equal length
    uint32_t batch, q_rows, k_rows;        // rows of all sequences (of one, without offsets)
    uint32_t heads, kv_heads, group, dim;
    FastDiv by_group, by_kv_heads;
    float scale2;  // scale * log2(e)
    bool causal;
    // Order of equal sequences' tiles.  Tile by tile (of all sequences, the longest first) where the work of tiles differs and a
    // launch is few rounds of the chip's workgroups; otherwise sequence by sequence, which keeps fewer keys in an L2 at a time.
    bool q_by_tile, k_by_tile;
};

AttnShape attn_shape(const AttnProblem &p);
bool attn_few(const AttnProblem &p, size_t rows, size_t times);
// Whether every row of the views is whole aligned 16-byte vectors, and a tile's reach fits 31 bits.
bool attn_vectors(size_t elt, const AttnProblem &p, std::initializer_list<AttnView> views);

// [first, last) of sequence b: within the rows there are, whatever the offsets say.
__device__ __forceinline__ void span(const int32_t *offsets, uint32_t b, uint32_t rows, uint32_t &first, uint32_t &count) {
    if (offsets == nullptr) {
        first = 0;
        count = rows;
        return;
    }
    const int32_t from = max(0, min(offsets[b], (int32_t)rows)), to = max(from, min(offsets[b + 1], (int32_t)rows));
    first = (uint32_t)from;
    count = (uint32_t)(to - from);
}
// The same for a sequence that is the whole wavefront's, in scalar registers.
__device__ __forceinline__ void span_of_all(const int32_t *offsets, uint32_t b, uint32_t rows, uint32_t &first, uint32_t &count) {
    span(offsets, b, rows, first, count);
    first = __builtin_amdgcn_readfirstlane(first);
    count = __builtin_amdgcn_readfirstlane(count);
}

// Tile number `index` of all sequences' tiles, `per` rows each: a sequence has `times` rows for each of its offsets' rows.
// `by_tile`: see AttnShape.  False where there are fewer tiles.  Whole wavefronts look, 64 sequences at a time.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, uint32_t batch, uint32_t rows, uint32_t times, uint32_t per, uint32_t index,
                                          bool by_tile, uint32_t &b, uint32_t &tile) {
    if (offsets == nullptr) {
        const uint32_t tiles = (rows * times + per - 1) / per;
        if (by_tile) {
            tile = index / batch;
            b = index - tile * batch;
            return tile < tiles;
        }
        b = index / tiles;
        tile = index - b * tiles;
        return b < batch;
    }
    const uint32_t lane = threadIdx.x % kWave;
    for (uint32_t b0 = 0; b0 < batch; b0 += kWave) {
        uint32_t first, count = 0;
        if (b0 + lane < batch) span(offsets, b0 + lane, rows, first, count);
        const uint32_t tiles = (count * times + per - 1) / per;
        uint32_t upto = tiles;
#pragma unroll
        for (uint32_t d = 1; d < kWave; d *= 2) {
            const uint32_t o = __shfl_up(upto, d, kWave);
            if (lane >= d) upto += o;
        }
        const uint64_t after = __builtin_amdgcn_ballot_w64(upto > index);
        if (after != 0) {
            const uint32_t at = (uint32_t)__builtin_ctzll(after);
            b = b0 + at;
            tile = index - (uint32_t)__builtin_amdgcn_readlane(upto - tiles, at);
            return true;
        }
        index -= (uint32_t)__builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

}  // namespace msd
