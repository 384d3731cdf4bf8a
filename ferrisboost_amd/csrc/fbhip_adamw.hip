// AdamW over many parameters at once. For a cell's gradient g, step t:
//   m = b1 m + (1 - b1) g,  s = b2 s + (1 - b2) g^2,
//   w = w (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(s / (1 - b2^t)) + eps).
//
// Moments of 8 bits are small floats under the exponent of the largest of 256 cells, one byte a
// block: m a sign, 4 bits of exponent and 3 of the mantissa, s 5 and 3. They are widened to
// doubles, and m and s of the step, as floats, move the weight before they are rounded again.
// That rounding is a random one, up with the probability of what it cuts off: a step changes s
// by some (1 - b2) s, 0.1 %, where neighbours lie 6 to 12 % apart, so the nearest one would
// hold it where it is, while so its expectation follows. The random bits are those that dropout
// draws for (seed + t, cell).
//
// Shifted so that the block's exponent is 30 (s) or 14 (m) of a float's own, a moment's code
// stands in its upper bits, subnormals included: rounding is one addition and one shift.
#include "fbhip_heads.h"

#include <cmath>

namespace fbh {
namespace {

constexpr uint32_t ADAM_TPB = 256;
constexpr uint32_t ADAM_CHUNK = 256;                // cells of a wave at a time: a block
constexpr uint32_t ADAM_CHUNKS = 4;                 // of a wave in a tile
constexpr uint32_t ADAM_TILE = ADAM_TPB / 64 * ADAM_CHUNKS * ADAM_CHUNK;
constexpr uint32_t ADAM_TENSORS = 64;               // of a launch
constexpr uint64_t ADAM_BLOCKS = 1u << 16;          // of a launch at most
constexpr uint32_t ADAM_TOP_M = 14, ADAM_TOP_S = 30;
constexpr uint32_t ADAM_NAN_M = 0x7F, ADAM_NAN_S = 0xFF;

// What a program keeps on the device: the steps done, and the products of as many betas.
struct Clock {
    int64_t step;
    double decay1, decay2;
};

struct AdamTensor {
    void *param;
    const void *grad;
    float *master;
    uint64_t n, first;
    uint64_t tiles_before;
    float decay;
    uint32_t dtype;
};

struct Adam {
    double beta1, beta2, lr;
    const float *lr_at;
    uint64_t seed;
    void *mean, *square;
    uint8_t *scales;
    Clock *clock;
    uint64_t blocks;  // of scales: [2][blocks]
    uint64_t tiles;
    float eps;
    uint32_t n_tensors;
};

struct AdamLaunch {
    Adam a;
    AdamTensor t[ADAM_TENSORS];
};
static_assert(sizeof(AdamLaunch) <= 4096, "kernel arguments");

// A step's numbers.
struct AdamStep {
    double b1, c1, b2, c2;
    float fb1, fc1, fb2, fc2;
    double lr;
    float size, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    float eps;
    uint64_t key;
};

__device__ __forceinline__ AdamStep adam_step(const Adam &A) {
    AdamStep s;
    s.b1 = A.beta1;
    s.c1 = 1.0 - A.beta1;
    s.b2 = A.beta2;
    s.c2 = 1.0 - A.beta2;
    s.fb1 = (float)s.b1;
    s.fc1 = (float)s.c1;
    s.fb2 = (float)s.b2;
    s.fc2 = (float)s.c2;
    s.lr = A.lr_at ? (double)*A.lr_at : A.lr;
    s.size = (float)(s.lr / (1.0 - A.clock->decay1 * A.beta1));
    s.root = (float)(1.0 / sqrt(1.0 - A.clock->decay2 * A.beta2));
    s.eps = A.eps;
    s.key = drop_mix((A.seed + (uint64_t)A.clock->step + 1) ^ 0x9E3779B97F4A7C15ull);
    return s;
}

__global__ void adam_clock_kernel(Clock *clock, double beta1, double beta2) {
    clock->step++;
    clock->decay1 *= beta1;
    clock->decay2 *= beta2;
}

// ---- The 8-bit floats.
__device__ __forceinline__ double widen_mean(uint32_t code, double scale) {
    const uint32_t mag = code & 0x7F;
    const double v = (double)__uint_as_float(mag << 20) * scale;
    return mag == ADAM_NAN_M ? (double)NAN : (code & 0x80) ? -v : v;
}
__device__ __forceinline__ double widen_square(uint32_t code, double scale) {
    const double v = (double)__uint_as_float(code << 20) * scale;
    return code == ADAM_NAN_S ? (double)NAN : v;
}
// 2^(field - top): what a block's codes are multiplied by.
__device__ __forceinline__ double scale_of(uint32_t field, uint32_t top) {
    const int e = (int)max(field, 1u) - (int)top;
    return __longlong_as_double((long long)(1023 + e) << 52);
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0;
}
// random: 16 bits.
__device__ __forceinline__ uint32_t narrow(float v, uint32_t field, uint32_t top,
                                           uint32_t random) {
    const float y = ldexpf(fabsf(v), (int)top - (int)max(field, 1u));
    return (__float_as_uint(y) + (random << 4)) >> 20;
}
__device__ __forceinline__ uint32_t narrow_mean(float v, uint32_t field, uint32_t random) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t code = narrow(v, field, ADAM_TOP_M, random);
    return ((b & 0x7FFFFFFFu) < 0x7F800000u ? code : ADAM_NAN_M) | (b >> 31 << 7);
}
// (a square above 0 stays above it)
__device__ __forceinline__ uint32_t narrow_square(float v, uint32_t field, uint32_t random) {
    const uint32_t code = narrow(v, field, ADAM_TOP_S, random);
    return !(v < __builtin_huge_valf()) ? ADAM_NAN_S : v > 0.0f ? max(code, 1u) : 0;
}

// The largest of a wave's values, in every lane.
__device__ __forceinline__ uint32_t most_of_lanes(uint32_t v) {
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

// ---- Four cells of a lane.
template <class T>
__device__ __forceinline__ void load_four(const T *p, uint64_t i, uint64_t n, float (&v)[4]) {
    if (i + 4 <= n) {
        const Piece<T, 4> q = load_piece<T, 4>(p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = i + k < n ? (float)p[i + k] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store_four(T *p, uint64_t i, uint64_t n, const float (&v)[4]) {
    if (i + 4 <= n) {
        Piece<T, 4> q;
#pragma unroll
        for (int k = 0; k < 4; k++) q.v[k] = (T)v[k];
        store_piece<T, 4>(p + i, q);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i + k < n) p[i + k] = (T)v[k];
    }
}

template <class T, bool SMALL>
__device__ __forceinline__ void adam_chunk(const Adam &A, const AdamStep &S, const AdamTensor &t,
                                           uint64_t at) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t i = at + lane * 4, flat = t.first + i;
    constexpr bool MASTER = sizeof(T) == 2;
    float *weights = MASTER ? t.master : static_cast<float *>(t.param);
    float g[4], w[4], m[4], s[4];
    load_four(static_cast<const T *>(t.grad), i, t.n, g);
    load_four(weights, i, t.n, w);
    uint32_t *codes_m = nullptr, *codes_s = nullptr;
    if constexpr (SMALL) {
        codes_m = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(A.mean) + flat);
        codes_s = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(A.square) + flat);
        const uint32_t cm = *codes_m, cs = *codes_s;
        const uint64_t block = (t.first + at) / ADAM_CHUNK;
        const double scale_m = scale_of(A.scales[block], ADAM_TOP_M);
        const double scale_s = scale_of(A.scales[A.blocks + block], ADAM_TOP_S);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double gd = (double)g[k];
            m[k] = (float)(widen_mean(cm >> 8 * k & 0xFF, scale_m) * S.b1 + gd * S.c1);
            s[k] = (float)(widen_square(cs >> 8 * k & 0xFF, scale_s) * S.b2 + gd * gd * S.c2);
        }
    } else {
        load_four(static_cast<float *>(A.mean), flat, ~0ull, m);
        load_four(static_cast<float *>(A.square), flat, ~0ull, s);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            m[k] = m[k] * S.fb1 + g[k] * S.fc1;
            s[k] = s[k] * S.fb2 + g[k] * g[k] * S.fc2;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (i + k >= t.n) m[k] = s[k] = 0.0f;
    const float shrink = (float)(1.0 - S.lr * (double)t.decay);
#pragma unroll
    for (int k = 0; k < 4; k++)
        w[k] = w[k] * shrink - S.size * (m[k] / (sqrtf(s[k]) * S.root + S.eps));
    store_four(weights, i, t.n, w);
    if constexpr (MASTER) store_four(static_cast<T *>(t.param), i, t.n, w);
    if constexpr (SMALL) {
        uint32_t most_m = 0, most_s = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            most_m = max(most_m, finite_bits(m[k]));
            most_s = max(most_s, finite_bits(s[k]));
        }
        const uint32_t field_m = most_of_lanes(most_m) >> 23;
        const uint32_t field_s = most_of_lanes(most_s) >> 23;
        uint32_t cm = 0, cs = 0;
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint64_t bits = drop_word(S.key, (flat + k) >> 1);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t r = (uint32_t)(bits >> 32 * j);
                cm |= narrow_mean(m[k + j], field_m, r & 0xFFFF) << 8 * (k + j);
                cs |= narrow_square(s[k + j], field_s, r >> 16) << 8 * (k + j);
            }
        }
        *codes_m = cm;
        *codes_s = cs;
        if (lane == 0) {
            const uint64_t block = (t.first + at) / ADAM_CHUNK;
            A.scales[block] = (uint8_t)field_m;
            A.scales[A.blocks + block] = (uint8_t)field_s;
        }
    } else {
        store_four(static_cast<float *>(A.mean), flat, ~0ull, m);
        store_four(static_cast<float *>(A.square), flat, ~0ull, s);
    }
}

template <bool SMALL>
__global__ __launch_bounds__(ADAM_TPB) void adam_kernel(AdamLaunch L) {
    const Adam &A = L.a;
    const AdamStep S = adam_step(A);
    for (uint64_t tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
        uint32_t lo = 0, hi = A.n_tensors;  // the last one that begins at the tile or before
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (L.t[mid].tiles_before <= tile) lo = mid;
            else hi = mid;
        }
        const AdamTensor &t = L.t[lo];
        const uint64_t begin = (tile - t.tiles_before) * ADAM_TILE +
                               (threadIdx.x / 64) * (ADAM_CHUNKS * ADAM_CHUNK);
        for (uint32_t c = 0; c < ADAM_CHUNKS; c++) {
            const uint64_t at = begin + c * ADAM_CHUNK;
            if (at >= t.n) break;
            if (t.dtype == FBH_F32) adam_chunk<float, SMALL>(A, S, t, at);
            else if (t.dtype == FBH_F16) adam_chunk<_Float16, SMALL>(A, S, t, at);
            else adam_chunk<__bf16, SMALL>(A, S, t, at);
        }
    }
}

// What codes stand for, four cells a thread.
__global__ __launch_bounds__(ADAM_TPB) void adam_moments_kernel(const uint8_t *mean,
                                                                const uint8_t *square,
                                                                const uint8_t *scales, uint64_t n,
                                                                float *out_m, float *out_s) {
    for (uint64_t i = ((uint64_t)blockIdx.x * ADAM_TPB + threadIdx.x) * 4; i < n;
         i += (uint64_t)gridDim.x * ADAM_TPB * 4) {
        const uint64_t block = i / ADAM_CHUNK;
        const double scale_m = scale_of(scales[block], ADAM_TOP_M);
        const double scale_s = scale_of(scales[n / ADAM_CHUNK + block], ADAM_TOP_S);
        const uint32_t cm = *reinterpret_cast<const uint32_t *>(mean + i);
        const uint32_t cs = *reinterpret_cast<const uint32_t *>(square + i);
        Piece<float, 4> m, s;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            m.v[k] = (float)widen_mean(cm >> 8 * k & 0xFF, scale_m);
            s.v[k] = (float)widen_square(cs >> 8 * k & 0xFF, scale_s);
        }
        store_piece<float, 4>(out_m + i, m);
        store_piece<float, 4>(out_s + i, s);
    }
}

bool aligned(const void *p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }

void check_adamw(const fbh_adamw *a) {
    head_input(a, "null argument");
    head_input(a->bits == 8 || a->bits == 32, "bits must be 8 or 32");
    head_input(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0,
               "betas must be in [0, 1)");
    head_input(a->eps >= 1.17549435e-38f && a->eps <= 3.4028235e38f,
               "eps must be a positive normal float");
    head_input(std::isfinite(a->lr) && a->lr >= 0.0, "lr must be finite and not negative");
    head_input(a->n % ADAM_CHUNK == 0 && a->n <= 1ull << 42,
               "n must be a multiple of 256, up to 2^42");
    head_input(a->clock && aligned(a->clock, 8), "the clock must be 8-byte aligned");
    head_input(a->n == 0 || (a->mean && a->square && aligned(a->mean, 16) &&
                             aligned(a->square, 16)),
               "the moments must be 16-byte aligned");
    head_input(a->n == 0 || a->bits == 32 || a->scales, "moments of 8 bits need scales");
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" {

int fbh_adamw_step(int device, const fbh_adamw *a, const fbh_adamw_tensor *tensors,
                   uint64_t n_tensors, void *stream) {
    return head_guard([&] {
        check_adamw(a);
        head_input(tensors || n_tensors == 0, "null argument");
        for (uint64_t i = 0; i < n_tensors; i++) {
            const fbh_adamw_tensor &t = tensors[i];
            if (t.n == 0) continue;
            head_input(t.dtype <= FBH_BF16, "unknown cell type");
            head_input(t.param && t.grad && (t.master || t.dtype == FBH_F32), "null argument");
            head_input(t.first % ADAM_CHUNK == 0 && t.first <= a->n && t.n <= a->n - t.first,
                       "a tensor's moments lie outside the state");
            head_input(std::isfinite(t.weight_decay) && t.weight_decay >= 0.0f,
                       "weight_decay must be finite and not negative");
        }
        const OnDevice on(device);
        const auto s = static_cast<hipStream_t>(stream);
        AdamLaunch L{};
        L.a = Adam{a->beta1, a->beta2, a->lr, a->lr_at, a->seed, a->mean, a->square,
                   static_cast<uint8_t *>(a->scales), static_cast<Clock *>(a->clock),
                   a->n / ADAM_CHUNK, 0, a->eps, 0};
        const auto flush = [&] {
            if (L.a.n_tensors == 0) return;
            const uint64_t blocks = L.a.tiles < ADAM_BLOCKS ? L.a.tiles : ADAM_BLOCKS;
            hipLaunchKernelGGL((a->bits == 8 ? adam_kernel<true> : adam_kernel<false>),
                               dim3((uint32_t)blocks), dim3(ADAM_TPB), 0, s, L);
            head_check(hipGetLastError(), "adamw");
            L.a.n_tensors = 0;
            L.a.tiles = 0;
        };
        for (uint64_t i = 0; i < n_tensors; i++) {
            const fbh_adamw_tensor &t = tensors[i];
            if (t.n == 0) continue;
            L.t[L.a.n_tensors++] = AdamTensor{t.param, t.grad, t.master, t.n, t.first, L.a.tiles,
                                              t.weight_decay, t.dtype};
            L.a.tiles += (t.n + ADAM_TILE - 1) / ADAM_TILE;
            if (L.a.n_tensors == ADAM_TENSORS) flush();
        }
        flush();
        hipLaunchKernelGGL(adam_clock_kernel, dim3(1), dim3(1), 0, s, L.a.clock, a->beta1,
                           a->beta2);
        head_check(hipGetLastError(), "adamw");
    });
}

int fbh_adamw_moments(int device, const fbh_adamw *a, float *mean, float *square, void *stream) {
    return head_guard([&] {
        check_adamw(a);
        head_input(a->bits == 8, "moments of 32 bits are what they are");
        head_input((mean && square) || a->n == 0, "null argument");
        if (a->n == 0) return;
        const OnDevice on(device);
        const uint64_t blocks = (a->n / 4 + ADAM_TPB - 1) / ADAM_TPB;
        hipLaunchKernelGGL(adam_moments_kernel,
                           dim3((uint32_t)(blocks < ADAM_BLOCKS ? blocks : ADAM_BLOCKS)),
                           dim3(ADAM_TPB), 0, static_cast<hipStream_t>(stream),
                           static_cast<const uint8_t *>(a->mean),
                           static_cast<const uint8_t *>(a->square),
                           static_cast<const uint8_t *>(a->scales), a->n, mean, square);
        head_check(hipGetLastError(), "adamw");
    });
}

}  // extern "C"
