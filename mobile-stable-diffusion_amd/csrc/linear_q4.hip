// Linear layers on a few rows with the weight in 4 bits, for gfx950:
//   w[n, k] = (code[n, k] - 8) scale[n, k / group],  y[m, n] = act_out(act_in(x)[m, k] . w[n, k]^T + bias[n]),  m <= 8
// two codes to a byte (even k in the low half), one scale in the storage type per group of 32, 64 or 128 of them.
#include "msd_device.h"
#include "msd_internal.h"

#include <algorithm>

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
    for (size_t i = 0; i < count && m != 0; i++) {
        if (ns[i] == 0) continue;
        launch(linear_q4_generic_kernel<T>, dim3((uint32_t)((ns[i] + kQ4Threads / kWave - 1) / (kQ4Threads / kWave))),
               dim3(kQ4Threads), 0, stream, static_cast<const T *>(x), packed[i], static_cast<const T *>(scales[i]),
               biases != nullptr ? biases[i] : nullptr, static_cast<T *>(ys[i]), (uint32_t)m, (uint32_t)ns[i], (uint32_t)k,
               (uint32_t)group, act_in, act_out);
    }
    return launch_status();
}
template int linear_q4_dispatch<float>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                       const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);
template int linear_q4_dispatch<__half>(const void *, const uint8_t *const *, const void *const *, const float *const *, void *const *,
                                        const size_t *, size_t, size_t, size_t, size_t, int, int, hipStream_t);

}  // namespace msd
