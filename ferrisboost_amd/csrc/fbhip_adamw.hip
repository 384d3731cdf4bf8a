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
//
// One pass over parameters, gradients, moments and copies, bound by memory (a large copy: 4.84
// TB/s): 64M cells of float32 with moments in float32 in 339 us (28 bytes a cell, 5.3 TB/s), 120M
// of bfloat16 in 642 (28, 5.2), with moments of 8 bits in 390 (16, 4.9). A launch takes 64
// tensors in its arguments, so nothing is copied to the device before it.
#include "fbhip_heads.h"

#include <algorithm>
#include <cmath>
#include <iterator>
#include <utility>
#include <vector>

namespace fbh {
namespace {

constexpr uint32_t ADAM_TPB = 256;
constexpr uint32_t ADAM_CHUNK = 256;                // cells of a wave at a time: a block
constexpr uint32_t ADAM_CHUNKS = 4;                 // of a wave in a tile
constexpr uint32_t ADAM_TILE = ADAM_TPB / 64 * ADAM_CHUNKS * ADAM_CHUNK;
constexpr uint32_t ADAM_TENSORS = 64, ADAM_FEW = 16;  // of a launch
constexpr uint64_t ADAM_BLOCKS = 1u << 16;          // of a launch at most
// Workgroups up to which they move the clock themselves: 25 of them take 4.6 us so and 5.3 with a
// launch of its own for it, 122 6.2 and 6.1, 244, which queue up at one counter, 8.4 and 7.0.
constexpr uint64_t ADAM_TICKS = 64;
constexpr uint32_t ADAM_TOP_M = 14, ADAM_TOP_S = 30;
constexpr uint32_t ADAM_NAN_M = 0x7F, ADAM_NAN_S = 0xFF;

// What a program keeps on the device: the steps done, the products of as many betas, and how
// many workgroups of a step's last launch are through (0 between steps).
struct Clock {
    int64_t step;
    double decay1, decay2;
    uint64_t done;
};

struct AdamTensor {
    void *param;
    const void *grad;
    float *master;
    uint64_t n, first;
    uint64_t tiles_before;
    float decay;
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
    uint32_t ticks;  // whether this launch moves the clock on
};

// (room for few tensors or many: a call with 16 tensors and 1 KB of arguments takes 3.4 to 4.3 us
// of the host, one with 17 and 3.7 KB 0.1 to 0.4 us more)
template <uint32_t MOST>
struct AdamLaunch {
    Adam a;
    AdamTensor t[MOST];
};
static_assert(sizeof(AdamLaunch<ADAM_TENSORS>) <= 4096, "kernel arguments");
static_assert(ADAM_TENSORS == 64, "a lane each");

// A step's numbers.
struct AdamStep {
    double b1, c1, b2, c2;
    float fb1, fc1, fb2, fc2;
    double lr;
    float size, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    float eps;
    bool tiny_eps;
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
    s.tiny_eps = A.eps < 0x1p-38f;  // (2^25 times the root of the largest subnormal)
    s.key = drop_mix((A.seed + (uint64_t)A.clock->step + 1) ^ 0x9E3779B97F4A7C15ull);
    return s;
}

__device__ __forceinline__ void tick(Clock *clock, double beta1, double beta2) {
    clock->step++;
    clock->decay1 *= beta1;
    clock->decay2 *= beta2;
}
__global__ void adam_clock_kernel(Clock *clock, double beta1, double beta2) {
    tick(clock, beta1, beta2);
}

// ---- The 8-bit floats. A block's exponent field is in a scalar register, so is what its codes
// are multiplied by: 2^(field - top).
__device__ __forceinline__ double scale_of(uint32_t field, uint32_t top) {
    const int e = (int)max(field, 1u) - (int)top;
    return __longlong_as_double((long long)(1023 + e) << 52);
}
// Byte k of a word as a float under the exponents 14 and 30.
__device__ __forceinline__ float mean_float(uint32_t codes, int k) {
    return __uint_as_float((uint32_t)((int32_t)(codes << (24 - 8 * k)) >> 4) & 0x87F00000u);
}
__device__ __forceinline__ float square_float(uint32_t codes, int k) {
    return __uint_as_float((codes >> 8 * k & 0xFF) << 20);
}
// Whether one of four bytes stands for what is not finite.
__device__ __forceinline__ bool has_nan_mean(uint32_t codes) {
    return ((codes & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ bool has_nan_square(uint32_t codes) {
    return (~codes - 0x01010101u) & codes & 0x80808080u;
}
__device__ __forceinline__ bool is_nan_mean(uint32_t codes, int k) {
    return (codes >> 8 * k & 0x7F) == ADAM_NAN_M;
}
__device__ __forceinline__ bool is_nan_square(uint32_t codes, int k) {
    return (codes >> 8 * k & 0xFF) == ADAM_NAN_S;
}

// The largest of a wave's values, in a scalar register.
__device__ __forceinline__ uint32_t most_of_wave(uint32_t v) {
#define FBH_MOST(CTRL, ROWS)                                                                     \
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false))
    FBH_MOST(0x111, 0xF);
    FBH_MOST(0x112, 0xF);
    FBH_MOST(0x114, 0xF);
    FBH_MOST(0x118, 0xF);
    FBH_MOST(0x142, 0xA);
    FBH_MOST(0x143, 0xC);
#undef FBH_MOST
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }
// In branches that hardly ever run: the compiler must not run them for everyone.
__device__ __forceinline__ void seldom() { asm volatile(""); }

// The top bytes of four words.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&t)[4]) {
    const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0703u);
    const uint32_t hi = __builtin_amdgcn_perm(t[3], t[2], 0x07030C0Cu);
    return lo | hi;
}

// ---- Four cells of a lane; WHOLE: all of them are the tensor's.
template <bool WHOLE, class T>
__device__ __forceinline__ void load_four(const T *p, uint32_t left, float (&v)[4]) {
    if (WHOLE || left >= 4) {
        const Piece<T, 4> q = load_piece<T, 4>(p);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (uint32_t)k < left ? (float)p[k] : 0.0f;
    }
}
template <bool WHOLE, class T>
__device__ __forceinline__ void store_four(T *p, uint32_t left, const float (&v)[4]) {
    if (WHOLE || left >= 4) {
        Piece<T, 4> q;
#pragma unroll
        for (int k = 0; k < 4; k++) q.v[k] = (T)v[k];
        store_piece<T, 4>(p, q);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if ((uint32_t)k < left) p[k] = (T)v[k];
    }
}

// m / (sqrt(s) root + eps), by the reciprocal and the square root of the hardware, one unit in
// the last place each: the step is small beside the weight that takes it. The square root may
// lose subnormals, which eps covers unless it is tiny. (Divided and rooted to half a unit the
// 8-bit step was bound by its instructions: 120M cells in 484 us.)
__device__ __forceinline__ void move_by(float (&m)[4], const float (&s)[4], const AdamStep &S) {
    float root[4];
    if (S.tiny_eps) {
        seldom();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool low = s[k] < 0x1p-96f;
            root[k] = __builtin_amdgcn_sqrtf(low ? s[k] * 0x1p64f : s[k]) *
                      (low ? 0x1p-32f : 1.0f);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) root[k] = __builtin_amdgcn_sqrtf(s[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
        m[k] *= __builtin_amdgcn_rcpf(root[k] * S.root + S.eps);
}

// A wave's block of 256 cells, `at` of a tensor's; word: the generator's step times the first
// pair's number of this lane.
template <class T, bool SMALL, bool WHOLE>
__device__ __forceinline__ void adam_chunk(const Adam &A, const AdamStep &S, const AdamTensor &t,
                                           float decay, uint64_t at, uint64_t word) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t flat = t.first + at;
    const uint32_t here = (uint32_t)min(t.n - at, (uint64_t)ADAM_CHUNK);
    const uint32_t left = WHOLE ? 4 : here - min(here, lane * 4);
    constexpr bool MASTER = sizeof(T) == 2;
    float *weights = (MASTER ? t.master : static_cast<float *>(t.param)) + at + lane * 4;
    T *param = static_cast<T *>(t.param) + at + lane * 4;
    float g[4], w[4], m[4], s[4];
    load_four<WHOLE>(static_cast<const T *>(t.grad) + at + lane * 4, left, g);
    load_four<WHOLE>(weights, left, w);
    uint32_t *codes_m = nullptr, *codes_s = nullptr;
    float *mean = nullptr, *square = nullptr;
    const uint64_t block = flat / ADAM_CHUNK;
    if constexpr (SMALL) {
        codes_m = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(A.mean) + flat) + lane;
        codes_s = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(A.square) + flat) + lane;
        const uint32_t cm = *codes_m, cs = *codes_s;
        const double scale_m = scale_of(__builtin_amdgcn_readfirstlane(A.scales[block]),
                                        ADAM_TOP_M) * S.b1;
        const double scale_s = scale_of(__builtin_amdgcn_readfirstlane(A.scales[A.blocks + block]),
                                        ADAM_TOP_S) * S.b2;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // (each product rounded by itself, so that whoever computes them in doubles has
            // the same bytes)
            const double gd = (double)g[k];
            m[k] = (float)((double)mean_float(cm, k) * scale_m + gd * S.c1);
            s[k] = (float)((double)square_float(cs, k) * scale_s + gd * gd * S.c2);
        }
        if (has_nan_mean(cm) || has_nan_square(cs)) {
            seldom();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (is_nan_mean(cm, k)) m[k] = NAN;
                if (is_nan_square(cs, k)) s[k] = NAN;
            }
        }
    } else {
        mean = static_cast<float *>(A.mean) + flat + lane * 4;
        square = static_cast<float *>(A.square) + flat + lane * 4;
        load_four<true>(mean, 4, m);
        load_four<true>(square, 4, s);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            m[k] = m[k] * S.fb1 + g[k] * S.fc1;
            s[k] = s[k] * S.fb2 + g[k] * g[k] * S.fc2;
        }
    }
    if (!WHOLE)
#pragma unroll
        for (int k = 0; k < 4; k++)
            if ((uint32_t)k >= left) m[k] = s[k] = 0.0f;
    float by[4] = {m[0], m[1], m[2], m[3]};
    move_by(by, s, S);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        // (what decays joins the step: 1 - lr decay in float32 would be off by up to 2^-25, a
        // large part of a small decay. An infinite weight stays one: inf - decay * most)
        const float most = __FLT_MAX__, part = __builtin_amdgcn_fmed3f(w[k], -most, most);
        w[k] -= fmaf(decay, part, S.size * by[k]);
        // the 16-bit parameter is this float rounded, not the sum before
        if (MASTER) asm volatile("" : "+v"(w[k]));
    }
    store_four<WHOLE>(weights, left, w);
    if constexpr (MASTER) store_four<WHOLE>(param, left, w);
    if constexpr (SMALL) {
        uint32_t most_m = max(max(size_bits(m[0]), size_bits(m[1])),
                              max(size_bits(m[2]), size_bits(m[3])));
        uint32_t most_s = max(max(size_bits(s[0]), size_bits(s[1])),
                              max(size_bits(s[2]), size_bits(s[3])));
        const bool odd = max(most_m, most_s) >= 0x7F800000u;  // some are not finite
        if (odd) {
            seldom();
            most_m = most_s = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (finite(m[k])) most_m = max(most_m, size_bits(m[k]));
                if (finite(s[k])) most_s = max(most_s, size_bits(s[k]));
            }
        }
        const uint32_t field_m = most_of_wave(most_m) >> 23;
        const uint32_t field_s = most_of_wave(most_s) >> 23;
        const int up_m = (int)ADAM_TOP_M - (int)max(field_m, 1u);
        const int up_s = (int)ADAM_TOP_S - (int)max(field_s, 1u);
        uint32_t tm[4], ts[4];  // codes in the top bytes
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint64_t bits = drop_mix(S.key ^ (word + k / 2 * DROP_STEP));
#pragma unroll
            for (int j = k; j < k + 2; j++) {
                const uint32_t r = (uint32_t)(bits >> 32 * (j - k));
                const uint32_t ym = __float_as_uint(ldexpf(fabsf(m[j]), up_m));
                const uint32_t ys = __float_as_uint(ldexpf(s[j], up_s));
                tm[j] = (ym << 4) + (r << 8 & 0xFFFF00u);
                ts[j] = (ys << 4) + (r >> 8 & 0xFFFF00u);
                // the sign; a square above 0 stays above it
                tm[j] = (tm[j] & 0x7FFFFFFFu) | (__float_as_uint(m[j]) & 0x80000000u);
                ts[j] = max(ts[j], s[j] > 0.0f ? 1u << 24 : 0u);
            }
        }
        if (odd) {
            seldom();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (!finite(m[k])) tm[k] = ADAM_NAN_M << 24;
                if (!finite(s[k])) ts[k] = ADAM_NAN_S << 24;
            }
        }
        *codes_m = top_bytes(tm);
        *codes_s = top_bytes(ts);
        if (lane == 0) {
            A.scales[block] = (uint8_t)field_m;
            A.scales[A.blocks + block] = (uint8_t)field_s;
        }
    } else {
        store_four<true>(mean, 4, m);
        store_four<true>(square, 4, s);
    }
}

template <class T, bool SMALL, uint32_t MOST>
__global__ __launch_bounds__(ADAM_TPB) void adam_kernel(AdamLaunch<MOST> L) {
    const Adam &A = L.a;
    const AdamStep S = adam_step(A);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    for (uint64_t tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
        // the last tensor that begins at the tile or before, by a lane each
        const uint32_t lane = threadIdx.x & 63;
        const uint64_t before = lane < A.n_tensors ? L.t[lane].tiles_before : ~0ull;
        const uint32_t lo = __popcll(__ballot(before <= tile)) - 1;
        const AdamTensor &t = L.t[lo];
        const uint64_t begin = (tile - t.tiles_before) * ADAM_TILE +
                               wave * (ADAM_CHUNKS * ADAM_CHUNK);
        const float decay = (float)(S.lr * (double)t.decay);
        const uint64_t word = ((t.first + begin) / 2 + (threadIdx.x & 63) * 2) * DROP_STEP;
        for (uint32_t c = 0; c < ADAM_CHUNKS; c++) {
            const uint64_t at = begin + c * ADAM_CHUNK, w = word + c * (ADAM_CHUNK / 2) * DROP_STEP;
            if (at + ADAM_CHUNK <= t.n) adam_chunk<T, SMALL, true>(A, S, t, decay, at, w);
            else if (at < t.n) adam_chunk<T, SMALL, false>(A, S, t, decay, at, w);
        }
    }
    if (!A.ticks) return;
    // the last workgroup that is through moves the clock on: all have read it by then (which
    // is all that the count has to order, and no load passes the barrier)
    __syncthreads();
    if (threadIdx.x == 0 &&
        __hip_atomic_fetch_add(&A.clock->done, 1ull, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
        A.clock->done = 0;
        tick(A.clock, A.beta1, A.beta2);
    }
}

// What codes stand for, four cells a thread (120M cells: 10 bytes a cell in 203 us, 5.9 TB/s).
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
            m.v[k] = is_nan_mean(cm, k) ? NAN : (float)((double)mean_float(cm, k) * scale_m);
            s.v[k] = is_nan_square(cs, k) ? NAN
                                          : (float)((double)square_float(cs, k) * scale_s);
        }
        store_piece<float, 4>(out_m + i, m);
        store_piece<float, 4>(out_s + i, s);
    }
}

template <uint32_t MOST>
void launch_most(uint32_t dtype, uint32_t bits, const AdamLaunch<MOST> &L, hipStream_t s) {
    const auto kernel =
        dtype == FBH_F32   ? (bits == 8 ? adam_kernel<float, true, MOST>
                                        : adam_kernel<float, false, MOST>)
        : dtype == FBH_F16 ? (bits == 8 ? adam_kernel<_Float16, true, MOST>
                                        : adam_kernel<_Float16, false, MOST>)
                           : (bits == 8 ? adam_kernel<__bf16, true, MOST>
                                        : adam_kernel<__bf16, false, MOST>);
    const uint64_t blocks = L.a.tiles < ADAM_BLOCKS ? L.a.tiles : ADAM_BLOCKS;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(ADAM_TPB), 0, s, L);
    head_check(hipGetLastError(), "adamw");
}
void launch_adamw(uint32_t dtype, uint32_t bits, const AdamLaunch<ADAM_TENSORS> &L,
                  hipStream_t s) {
    if (L.a.n_tensors > ADAM_FEW) return launch_most(dtype, bits, L, s);
    AdamLaunch<ADAM_FEW> few{};
    few.a = L.a;
    for (uint32_t i = 0; i < L.a.n_tensors; i++) few.t[i] = L.t[i];
    launch_most(dtype, bits, few, s);
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

// That no parameter shares memory with another one, a gradient or the learning rate: what a step
// writes and what it reads would run side by side.
void check_overlaps(const fbh_adamw_tensor *tensors, uint64_t n_tensors, const float *lr_at) {
    using Span = std::pair<uintptr_t, uintptr_t>;
    const auto span = [](const fbh_adamw_tensor &t, const void *p) {
        const auto at = reinterpret_cast<uintptr_t>(p);
        return Span{at, at + t.n * (t.dtype == FBH_F32 ? 4 : 2)};
    };
    std::vector<Span> params;
    params.reserve(n_tensors);
    for (uint64_t i = 0; i < n_tensors; i++)
        if (tensors[i].n) params.push_back(span(tensors[i], tensors[i].param));
    std::sort(params.begin(), params.end());
    for (size_t i = 1; i < params.size(); i++)
        head_input(params[i - 1].second <= params[i].first, "parameters overlap in memory");
    const auto apart = [&](const Span &r) {
        // the first parameter that begins behind what is read; the one before ends last
        const auto behind = std::lower_bound(params.begin(), params.end(), Span{r.second, 0});
        return behind == params.begin() || std::prev(behind)->second <= r.first;
    };
    for (uint64_t i = 0; i < n_tensors; i++)
        head_input(!tensors[i].n || apart(span(tensors[i], tensors[i].grad)),
                   "a gradient overlaps a parameter in memory");
    if (lr_at) {
        const auto at = reinterpret_cast<uintptr_t>(lr_at);
        head_input(apart({at, at + 4}), "the learning rate overlaps a parameter in memory");
    }
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
        check_overlaps(tensors, n_tensors, a->lr_at);
        const OnDevice on(device);
        const auto s = static_cast<hipStream_t>(stream);
        AdamLaunch<ADAM_TENSORS> L{};
        L.a = Adam{a->beta1, a->beta2, a->lr, a->lr_at, a->seed, a->mean, a->square,
                   static_cast<uint8_t *>(a->scales), static_cast<Clock *>(a->clock),
                   a->n / ADAM_CHUNK, 0, a->eps, 0, 0};
        // a launch for every 64 tensors of a type; the clock goes on in the last one, or in a
        // launch of its own
        bool ticked = false;
        uint64_t left = 0;
        for (uint64_t i = 0; i < n_tensors; i++) left += tensors[i].n != 0;
        for (uint32_t dtype = FBH_F32; dtype <= FBH_BF16 && left; dtype++) {
            L.a.n_tensors = 0;
            L.a.tiles = 0;
            const auto launch = [&] {
                if (L.a.n_tensors == 0) return;
                ticked = L.a.ticks = left == 0 && L.a.tiles <= ADAM_TICKS;
                launch_adamw(dtype, a->bits, L, s);
                L.a.n_tensors = 0;
                L.a.tiles = 0;
            };
            for (uint64_t i = 0; i < n_tensors; i++) {
                const fbh_adamw_tensor &t = tensors[i];
                if (t.n == 0 || t.dtype != dtype) continue;
                L.t[L.a.n_tensors++] = AdamTensor{t.param, t.grad, t.master, t.n, t.first,
                                                  L.a.tiles, t.weight_decay};
                L.a.tiles += (t.n + ADAM_TILE - 1) / ADAM_TILE;
                left--;
                if (L.a.n_tensors == ADAM_TENSORS) launch();
            }
            launch();
        }
        if (ticked) return;
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
