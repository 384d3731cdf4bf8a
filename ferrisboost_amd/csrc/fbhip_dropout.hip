// Dropout from a counter: out = x / (1 - drop) where element e's bits are at or above
// drop * 2^32, else 0. The bits are a function of (seed, e) alone, so the gradient is
// the same call on the output's gradient and no mask is ever stored.
//
// One pass, each cell read and written once, which bounds it: 100,000 x 1023 cells of
// bfloat16 (409 MB) take 75 us, 5.5 TB/s, where a large copy reaches 4.9; 83 us when the
// output goes through the caches. The hash of a pair of cells is twelve multiplies at a
// quarter of the rate and some twenty other operations, half of that time.
#include "fbhip_heads.h"

namespace fbh {
namespace {

constexpr uint32_t DROP_TPB = 256;
constexpr uint32_t DROP_PIECES = 4;  // 16-byte pieces of a thread, all requested at once

// ODD: the first element's number is odd, so pieces start in the middle of a pair.
template <class T, bool ODD>
__device__ __forceinline__ void drop_piece(Piece<T, 16 / sizeof(T)> &p, uint64_t key,
                                           uint64_t e, uint32_t threshold, float scale) {
    constexpr int N = 16 / sizeof(T);
    uint64_t w = ODD ? drop_word(key, e >> 1) : 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool high = ((i + (ODD ? 1 : 0)) & 1) != 0;
        if (!high) w = drop_word(key, (e + i) >> 1);
        const uint32_t bits = high ? (uint32_t)(w >> 32) : (uint32_t)w;
        p.v[i] = bits >= threshold ? (T)((float)p.v[i] * scale) : (T)0.0f;
    }
}

// PAST: written past the caches.
template <class T, bool ODD, bool PAST>
__global__ __launch_bounds__(DROP_TPB) void dropout_kernel(const T *x, T *out, uint64_t n,
                                                           uint64_t first, uint64_t key,
                                                           uint32_t threshold, float scale) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint64_t base = (uint64_t)blockIdx.x * (DROP_TPB * DROP_PIECES * N) + threadIdx.x * N;
    Piece<T, N> p[DROP_PIECES];
#pragma unroll
    for (uint32_t k = 0; k < DROP_PIECES; k++) {
        const uint64_t i = base + k * (DROP_TPB * N);
        if (i + N <= n) p[k] = load_piece<T, N>(x + i);
    }
#pragma unroll
    for (uint32_t k = 0; k < DROP_PIECES; k++) {
        const uint64_t i = base + k * (DROP_TPB * N);
        if (i + N <= n) {
            drop_piece<T, ODD>(p[k], key, first + i, threshold, scale);
            if constexpr (PAST) stream_piece<T, N>(out + i, p[k]);
            else store_piece<T, N>(out + i, p[k]);
        } else {
            for (uint64_t j = i; j < n; j++)
                out[j] = drop_bits(key, first + j) >= threshold ? (T)((float)x[j] * scale)
                                                                : (T)0.0f;
        }
    }
}

template <class T>
void launch_dropout(const void *x, void *out, uint64_t n, uint64_t first, uint64_t key,
                    uint32_t threshold, float scale, hipStream_t s) {
    const uint64_t cells = DROP_TPB * DROP_PIECES * (16 / sizeof(T));
    const uint64_t blocks = (n + cells - 1) / cells;
    const bool past = n * sizeof(T) >= STREAM_BYTES;
    const auto kernel = (first & 1) ? (past ? dropout_kernel<T, true, true>
                                            : dropout_kernel<T, true, false>)
                                    : (past ? dropout_kernel<T, false, true>
                                            : dropout_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(DROP_TPB), 0, s,
                       static_cast<const T *>(x), static_cast<T *>(out), n, first, key, threshold,
                       scale);
    head_check(hipGetLastError(), "dropout");
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" int fbh_dropout(int device, const void *x, void *out, uint64_t n, uint32_t dtype,
                           double drop, uint64_t seed, uint64_t first, void *stream) {
    return head_guard([&] {
        head_input((x && out) || n == 0, "null argument");
        head_input(n <= 1ull << 35, "more than 2^35 cells");
        head_input(dtype <= FBH_BF16, "unknown cell type");
        const uint32_t threshold = drop_threshold(drop);
        if (n == 0) return;
        const OnDevice on(device);
        const float scale = (float)(1.0 / (1.0 - drop));
        const uint64_t key = drop_key(seed);
        const auto s = static_cast<hipStream_t>(stream);
        if (dtype == FBH_F32) launch_dropout<float>(x, out, n, first, key, threshold, scale, s);
        else if (dtype == FBH_F16)
            launch_dropout<_Float16>(x, out, n, first, key, threshold, scale, s);
        else launch_dropout<__bf16>(x, out, n, first, key, threshold, scale, s);
    });
}
