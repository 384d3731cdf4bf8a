// Classes drawn from logits and given uniform numbers, with temperature, top-k, top-p and
// min-p.
//
// A class' weight is rint(2^45 exp((l - max) / T)) as a 64-bit integer, at most 2^45, so
// sums of up to 2^18 of them are exact and the same in any order: histograms by LDS
// atomics, partial sums of tiles and prefix sums all agree to the last bit, and which
// class a uniform number falls to does not depend on how a row was cut.
//
// No sort: "ordered by falling logit, equal ones by class, the first k" is a threshold
// key and a number of classes that have it (Cut). It is found from a histogram over
// (max - l) / T, which is monotone in l, then by the digits of the key among the classes
// of the bin that the cut falls into.
#include <algorithm>
#include <cmath>
#include <memory>

#include "fbhip_heads.h"

namespace fbh {
namespace {

constexpr uint32_t SAMPLE_MOST = 262144;  // classes: their weights' sum is below 2^63
constexpr int WEIGHT_BITS = 45;
constexpr uint64_t WEIGHT_ONE = 1ull << WEIGHT_BITS;

struct Draw {
    const float *uniforms;
    fbh_sample_options o;
    int64_t *classes;
    float *log_probs;
    uint64_t n_rows;
    uint32_t n_classes;
};

// A row's options, as whole numbers.
struct RowOptions {
    double inv_t;       // 1 / temperature, 0: the largest logit
    uint32_t k;         // classes that stay by rank
    uint32_t p31;       // top_p * 2^31
    uint64_t least;     // smallest weight that stays by min_p
    uint32_t u31;       // uniform * 2^31
};

__device__ __forceinline__ RowOptions row_options(const Draw &D, uint64_t row) {
    RowOptions r;
    const float t = D.o.temperatures ? D.o.temperatures[row] : D.o.temperature;
    const int32_t k = D.o.top_ks ? D.o.top_ks[row] : D.o.top_k;
    float p = D.o.top_ps ? D.o.top_ps[row] : D.o.top_p;
    float m = D.o.min_ps ? D.o.min_ps[row] : D.o.min_p;
    const float u = D.uniforms[row];
    r.k = t > 0.0f ? (k > 0 ? min((uint32_t)k, D.n_classes) : D.n_classes) : 1;
    r.inv_t = t > 0.0f ? 1.0 / (double)t : 0.0;
    p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;  // (NaN: 1)
    r.p31 = (uint32_t)((double)p * 2147483648.0);
    m = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    r.least = (uint64_t)ceil((double)m * (double)WEIGHT_ONE);
    r.u31 = u > 0.0f ? (uint32_t)fmin((double)u * 2147483648.0, 2147483647.0) : 0;
    return r;
}

// floor((part * total + add) / 2^31)
__device__ __forceinline__ uint64_t share(uint32_t part, uint64_t total, uint32_t add) {
    const uint64_t lo = part * total, sum = lo + add;
    const uint64_t hi = __umul64hi(part, total) + (sum < lo ? 1 : 0);
    return hi << 33 | sum >> 31;
}

// Monotone key of a logit; both zeros have one key.
__device__ __forceinline__ uint32_t logit_key(float f) {
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) == 0) u = 0;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// rint(2^45 e^t) for t <= 0: t = n ln 2 + r, |r| <= ln(2) / 2, the exponential series of
// r up to r^13 (what is left out is below 2^-57), scaled by 2^(n + 45); adding 2^52
// rounds to whole numbers. Below -32 the result is 0.
__device__ __forceinline__ uint64_t weight_of(double t) {
    const double n = rint(t * 0x1.71547652b82fep+0);
    double r = fma(n, -0x1.62e42fefap-1, t);
    r = fma(n, -0x1.cf79abc9e3b3ap-40, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double w = __builtin_amdgcn_ldexp(p, (int)n + WEIGHT_BITS) + 0x1p52;
    return t >= -32.0 ? (uint64_t)__double_as_longlong(w) & 0xFFFFFFFFFFFFFull : 0;
}

struct RowScale {
    float most;
    double top, inv_t;
    __device__ __forceinline__ double z(float l) const {
        return l == most ? 0.0 : ((double)l - top) * inv_t;
    }
    __device__ __forceinline__ uint64_t weight(float l) const { return weight_of(z(l)); }
};

__device__ __forceinline__ float masked_nan(float l) { return l == l ? l : -INFINITY; }

// -------------------------------------------------------------- few classes
constexpr uint32_t GROUP_TPB = 256;
constexpr uint32_t GROUP_MOST = 64;

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int from, int width) {
    const uint32_t lo = __shfl((uint32_t)v, from, width);
    const uint32_t hi = __shfl((uint32_t)(v >> 32), from, width);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64_up(uint64_t v, int by, int width) {
    const uint32_t lo = __shfl_up((uint32_t)v, by, width);
    const uint32_t hi = __shfl_up((uint32_t)(v >> 32), by, width);
    return (uint64_t)hi << 32 | lo;
}

// Up to 64 classes: a lane a class, 64 / G rows a wave. Every lane meets every other
// class of its row once, which gives its rank and the weight before it in the order.
template <class T, int G>
__global__ __launch_bounds__(GROUP_TPB) void sample_group_kernel(const T *logits, Draw D) {
    const uint64_t row = (uint64_t)blockIdx.x * (GROUP_TPB / G) + threadIdx.x / G;
    const int c = threadIdx.x % G;
    const bool in = row < D.n_rows;  // (all lanes stay: they shuffle)
    const uint64_t at = in ? row : 0;
    float l = -INFINITY;
    if (in && c < (int)D.n_classes) l = masked_nan((float)logits[at * D.n_classes + c]);
    const RowOptions O = row_options(D, at);
    float most = l;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, G));
    const RowScale S{most, (double)most, O.inv_t};
    uint64_t w = l == -INFINITY ? 0 : (O.inv_t == 0.0 ? (l == most ? WEIGHT_ONE : 0) : S.weight(l));
    const bool ranks = O.k < D.n_classes || O.p31 < 1u << 31;
    if (__any(ranks)) {
        const uint32_t key = logit_key(l);
        uint32_t rank = 0;
        for (int j = 0; j < (int)D.n_classes; j++) {
            const uint32_t kj = __shfl(key, j, G);
            rank += kj > key || (kj == key && j < c);
        }
        if (rank >= O.k) w = 0;
        uint64_t before = 0, all = 0;
        for (int j = 0; j < (int)D.n_classes; j++) {
            const uint32_t rj = __shfl(rank, j, G);
            const uint64_t wj = shfl64(w, j, G);
            all += wj;
            if (rj < rank) before += wj;
        }
        const uint64_t most_w = share(O.p31, all, 0x7FFFFFFFu);
        if (O.p31 < 1u << 31 && before >= (most_w ? most_w : 1)) w = 0;
    }
    if (w < O.least) w = 0;
    uint64_t cum = w;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        const uint64_t y = shfl64_up(cum, d, G);
        if (c >= d) cum += y;
    }
    const uint64_t total = shfl64(cum, G - 1, G);
    const uint64_t hits = __ballot(cum > share(O.u31, total, 0));
    const int lane0 = (threadIdx.x & 63) - c;
    const uint64_t mine = (hits >> lane0) & (G < 64 ? (1ull << (G & 63)) - 1 : ~0ull);
    if (!in) return;
    if (total == 0) {
        if (c == 0) {
            D.classes[row] = -1;
            if (D.log_probs) D.log_probs[row] = -INFINITY;
        }
    } else if (c == __ffsll((long long)mine) - 1) {
        D.classes[row] = c;
        if (D.log_probs)
            D.log_probs[row] = (float)(S.z(l) - log((double)total / (double)WEIGHT_ONE));
    }
}

// -------------------------------------------------------------- a row a workgroup
constexpr uint32_t NO_BIN = 0xFFFFFFFFu;
constexpr uint32_t MOST_TILES = 64;

template <class T>
struct KeyDigits {  // digits of 8 bits above the ones that all cells of a type share
    static constexpr int last = 0;
};
template <>
struct KeyDigits<_Float16> {
    static constexpr int last = 8;
};
template <>
struct KeyDigits<__bf16> {
    static constexpr int last = 16;
};

template <int TPB>
struct RowShared {
    static constexpr uint32_t BINS = TPB == 64 ? 256 : 1024;
    static constexpr uint32_t LIST = TPB == 64 ? 256 : 2048;
    uint64_t wt[BINS];
    uint32_t ct[BINS];
    uint32_t list[LIST];
    uint64_t tile_w[MOST_TILES];
    uint32_t tile_ties[MOST_TILES];
    float wave_most[TPB / 64];
    uint32_t wave_at[TPB / 64];
    uint64_t wave_w[TPB / 64];
    uint32_t wave_ties[TPB / 64];
    uint32_t bin, n_list;
    uint32_t before_ct;
    uint64_t before_wt;
    uint64_t target;
    uint64_t total;
    uint32_t tile, ties;
};

// What stays: classes of larger keys, and the first `ties` classes of this one.
struct Cut {
    uint32_t key, ties;
};

// One row. All threads of the workgroup call every function; a barrier stands between
// a write and its readers.
template <class T, int TPB>
struct SampleRow {
    static constexpr int N = 16 / sizeof(T);
    using Shared = RowShared<TPB>;
    Shared &sh;
    const T *row;
    uint32_t n;
    RowScale S;
    float per_nat;

    template <class F>
    __device__ __forceinline__ void each(F &&f) const {
        for (uint32_t i = threadIdx.x * N; i < n; i += TPB * N) {
            if (i + N <= n) {
                const Piece<T, N> p = load_piece<T, N>(row + i);
#pragma unroll
                for (int j = 0; j < N; j++) f(i + j, masked_nan((float)p.v[j]));
            } else {
                for (uint32_t j = i; j < n; j++) f(j, masked_nan((float)row[j]));
            }
        }
    }

    // The largest logit and its first class.
    __device__ __forceinline__ void largest(float &most, uint32_t &at) const {
        most = -INFINITY;
        at = NO_BIN;
        each([&](uint32_t i, float l) {
            if (l > most) {
                most = l;
                at = i;
            }
        });
        for (int d = 1; d < 64; d <<= 1) {
            const float m = __shfl_xor(most, d);
            const uint32_t a = __shfl_xor(at, d);
            if (m > most || (m == most && a < at)) {
                most = m;
                at = a;
            }
        }
        if constexpr (TPB > 64) {
            if ((threadIdx.x & 63) == 0) {
                sh.wave_most[threadIdx.x / 64] = most;
                sh.wave_at[threadIdx.x / 64] = at;
            }
            __syncthreads();
            for (int w = 0; w < TPB / 64; w++) {
                const float m = sh.wave_most[w];
                const uint32_t a = sh.wave_at[w];
                if (m > most || (m == most && a < at)) {
                    most = m;
                    at = a;
                }
            }
        }
    }

    // Bins of (max - l) / T, 32 over all of them: monotone, as each step of it is.
    __device__ __forceinline__ uint32_t bin_of(float l) const {
        const float d = l == S.most ? 0.0f : (S.most - l) * per_nat;
        return (uint32_t)fminf(d, (float)(Shared::BINS - 1));
    }

    __device__ __forceinline__ void clear(uint32_t bins) {
        __syncthreads();
        for (uint32_t b = threadIdx.x; b < bins; b += TPB) {
            sh.ct[b] = 0;
            sh.wt[b] = 0;
        }
        __syncthreads();
    }
    __device__ __forceinline__ void count(uint32_t bin, uint64_t w) {
        atomicAdd(&sh.ct[bin], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wt[bin]), (unsigned long long)w);
    }

    // The first bin at which the counts reach k (or the weights reach `weight`), and
    // what stands before it, on top of sh.before_*. NO_BIN: they never do.
    __device__ __forceinline__ void find(uint32_t bins, bool by_count, uint32_t k,
                                         uint64_t weight) {
        __syncthreads();
        if (threadIdx.x < 64) {
            const uint32_t each = bins / 64, b0 = threadIdx.x * each;
            uint32_t c = 0;
            uint64_t w = 0;
            for (uint32_t b = 0; b < each; b++) {
                c += sh.ct[b0 + b];
                w += sh.wt[b0 + b];
            }
            uint32_t cc = c;
            uint64_t ww = w;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = __shfl_up(cc, d);
                const uint64_t z = shfl64_up(ww, d, 64);
                if ((int)threadIdx.x >= d) {
                    cc += y;
                    ww += z;
                }
            }
            uint32_t bc = sh.before_ct;
            uint64_t bw = sh.before_wt;
            const bool reach = by_count ? bc + cc >= k : bw + ww >= weight;
            const uint64_t hits = __ballot(reach);
            if (threadIdx.x == 0) sh.bin = NO_BIN;
            if (hits && (int)threadIdx.x == __ffsll((long long)hits) - 1) {
                bc += cc - c;
                bw += ww - w;
                uint32_t b = b0;
                for (; b < b0 + each - 1; b++) {
                    if (by_count ? bc + sh.ct[b] >= k : bw + sh.wt[b] >= weight) break;
                    bc += sh.ct[b];
                    bw += sh.wt[b];
                }
                sh.bin = b;
                sh.before_ct = bc;
                sh.before_wt = bw;
            }
        }
        __syncthreads();
    }

    // The cut inside bin `bin` of `inside` classes, with sh.before_* standing before it.
    __device__ __forceinline__ Cut refine(uint32_t bin, uint32_t inside, bool by_count,
                                          uint32_t k, uint64_t weight) {
        const bool listed = inside <= Shared::LIST;
        if (listed) {
            if (threadIdx.x == 0) sh.n_list = 0;
            __syncthreads();
            each([&](uint32_t, float l) {
                if (l != -INFINITY && bin_of(l) == bin)
                    sh.list[atomicAdd(&sh.n_list, 1u)] = logit_key(l);
            });
        }
        uint32_t prefix = 0;
        for (int shift = 24; shift >= KeyDigits<T>::last; shift -= 8) {
            clear(256);
            const auto take = [&](uint32_t key) {
                if (shift == 24 || key >> (shift + 8) == prefix)
                    count(255 - ((key >> shift) & 255), S.weight(key_logit(key)));
            };
            if (listed)
                for (uint32_t i = threadIdx.x; i < inside; i += TPB) take(sh.list[i]);
            else
                each([&](uint32_t, float l) {
                    if (l != -INFINITY && bin_of(l) == bin) take(logit_key(l));
                });
            find(256, by_count, k, weight);
            prefix = prefix << 8 | (255 - sh.bin);
        }
        if constexpr (KeyDigits<T>::last > 0) {
            constexpr int L = KeyDigits<T>::last;
            const bool positive = prefix >> (31 - L);
            prefix = prefix << L | (positive ? 0u : (1u << L) - 1);
        }
        Cut cut{prefix, 0};
        if (by_count) cut.ties = k - sh.before_ct;
        else {
            const uint64_t w = S.weight(key_logit(prefix)), left = weight - sh.before_wt;
            cut.ties = (uint32_t)((left + w - 1) / w);
        }
        return cut;
    }
};

template <class T, int TPB>
__global__ __launch_bounds__(TPB) void sample_row_kernel(const T *logits, Draw D) {
    __shared__ RowShared<TPB> sh;
    constexpr int N = 16 / sizeof(T);
    const uint64_t r = blockIdx.x;
    const uint32_t n = D.n_classes;
    const RowOptions O = row_options(D, r);
    SampleRow<T, TPB> R{sh, logits + r * n, n, {}, 0.0f};
    float most;
    uint32_t most_at;
    R.largest(most, most_at);
    if (most == -INFINITY || O.inv_t == 0.0 || O.k == 1) {
        if (threadIdx.x == 0) {
            const bool none = most == -INFINITY;
            D.classes[r] = none ? -1 : (int64_t)most_at;
            if (D.log_probs) D.log_probs[r] = none ? -INFINITY : 0.0f;
        }
        return;
    }
    R.S = RowScale{most, (double)most, O.inv_t};
    R.per_nat = (float)(O.inv_t * (RowShared<TPB>::BINS / 32));

    Cut cut{0, 0};
    uint64_t tie_w = 0;
    if (O.k < n || O.p31 < 1u << 31) {
        R.clear(RowShared<TPB>::BINS);
        R.each([&](uint32_t, float l) {
            if (l != -INFINITY) R.count(R.bin_of(l), R.S.weight(l));
        });
        if (threadIdx.x == 0) {
            sh.before_ct = 0;
            sh.before_wt = 0;
        }
        // (refine() reuses the bins, so top-p looks for its bin first, among all
        // classes and, once their weight is known, among the first k.)
        __syncthreads();
        uint64_t all = 0;
        for (uint32_t b = threadIdx.x & 63; b < RowShared<TPB>::BINS; b += 64) all += sh.wt[b];
        for (int d = 1; d < 64; d <<= 1)
            all += (uint64_t)__shfl_xor((uint32_t)(all >> 32), d) * 0x100000000ull +
                   __shfl_xor((uint32_t)all, d);
        uint32_t k_bin = NO_BIN, k_inside = 0, k_before = 0;
        uint64_t k_weight = 0;
        if (O.k < n) {
            R.find(RowShared<TPB>::BINS, true, O.k, 0);
            k_bin = sh.bin;
            if (k_bin != NO_BIN) {
                k_inside = sh.ct[k_bin];
                k_before = sh.before_ct;
                k_weight = sh.before_wt;
            }
        }
        if (k_bin != NO_BIN) {
            cut = R.refine(k_bin, k_inside, true, O.k, 0);
            tie_w = R.S.weight(key_logit(cut.key));
            all = sh.before_wt + cut.ties * tie_w;
        }
        if (O.p31 < 1u << 31) {
            uint64_t weight = share(O.p31, all, 0x7FFFFFFFu);
            if (weight == 0) weight = 1;
            // The bins again, unless they still stand.
            if (k_bin != NO_BIN) {
                if (weight > k_weight) {  // in the bin of the k-th class
                    __syncthreads();
                    if (threadIdx.x == 0) {
                        sh.before_ct = k_before;
                        sh.before_wt = k_weight;
                    }
                    cut = R.refine(k_bin, k_inside, false, 0, weight);
                } else {
                    R.clear(RowShared<TPB>::BINS);
                    R.each([&](uint32_t, float l) {
                        if (l != -INFINITY) R.count(R.bin_of(l), R.S.weight(l));
                    });
                    if (threadIdx.x == 0) {
                        sh.before_ct = 0;
                        sh.before_wt = 0;
                    }
                    R.find(RowShared<TPB>::BINS, false, 0, weight);
                    const uint32_t bin = sh.bin, inside = sh.ct[bin];
                    cut = R.refine(bin, inside, false, 0, weight);
                }
            } else {
                __syncthreads();
                if (threadIdx.x == 0) {
                    sh.before_ct = 0;
                    sh.before_wt = 0;
                }
                R.find(RowShared<TPB>::BINS, false, 0, weight);
                const uint32_t bin = sh.bin, inside = sh.ct[bin];
                cut = R.refine(bin, inside, false, 0, weight);
            }
            tie_w = R.S.weight(key_logit(cut.key));
        }
        if (tie_w < O.least) cut.ties = 0;
    }

    // The staying weight, tile by tile of TPB pieces (in class order).
    const auto piece_sums = [&](uint32_t i, uint64_t &w, uint32_t &ties) {
        w = 0;
        ties = 0;
        const auto one = [&](float l) {
            const uint32_t key = logit_key(l);
            if (l == -INFINITY || key < cut.key) return;
            if (key == cut.key) {
                ties++;
                return;
            }
            const uint64_t v = R.S.weight(l);
            if (v >= O.least) w += v;
        };
        if (i + N <= n) {
            const Piece<T, N> p = load_piece<T, N>(R.row + i);
#pragma unroll
            for (int j = 0; j < N; j++) one(masked_nan((float)p.v[j]));
        } else {
            for (uint32_t j = i; j < n; j++) one(masked_nan((float)R.row[j]));
        }
    };
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < MOST_TILES; t += TPB) {
        sh.tile_w[t] = 0;
        sh.tile_ties[t] = 0;
    }
    __syncthreads();
    const uint32_t tiles = (n + TPB * N - 1) / (TPB * N);
    for (uint32_t t = 0; t < tiles; t++) {
        uint64_t w;
        uint32_t ties;
        piece_sums((t * TPB + threadIdx.x) * N, w, ties);
        for (int d = 32; d; d >>= 1) {
            w += (uint64_t)__shfl_xor((uint32_t)(w >> 32), d) * 0x100000000ull +
                 __shfl_xor((uint32_t)w, d);
            ties += __shfl_xor(ties, d);
        }
        if ((threadIdx.x & 63) == 0) {
            if (w)
                atomicAdd(reinterpret_cast<unsigned long long *>(&sh.tile_w[t]),
                          (unsigned long long)w);
            if (ties) atomicAdd(&sh.tile_ties[t], ties);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint64_t total = 0;
        uint32_t left = cut.ties;
        for (uint32_t t = 0; t < tiles; t++) {
            const uint32_t k = min(left, sh.tile_ties[t]);
            left -= k;
            total += sh.tile_w[t] + k * tie_w;
        }
        const uint64_t target = share(O.u31, total, 0);
        uint64_t before = 0;
        left = cut.ties;
        uint32_t t = 0;
        for (; t < tiles; t++) {
            const uint32_t k = min(left, sh.tile_ties[t]);
            const uint64_t w = sh.tile_w[t] + k * tie_w;
            if (before + w > target) break;
            before += w;
            left -= k;
        }
        sh.tile = t;
        sh.ties = left;
        sh.target = target - before;
        sh.total = total;
    }
    __syncthreads();
    // The tile that holds the target: its pieces' sums in order, then the piece.
    const uint32_t i0 = (sh.tile * TPB + threadIdx.x) * N;
    uint64_t w;
    uint32_t ties;
    piece_sums(i0, w, ties);
    uint64_t cw = w;
    uint32_t ct = ties;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = shfl64_up(cw, d, 64);
        const uint32_t z = __shfl_up(ct, d);
        if ((threadIdx.x & 63) >= (uint32_t)d) {
            cw += y;
            ct += z;
        }
    }
    if ((threadIdx.x & 63) == 63) {
        sh.wave_w[threadIdx.x / 64] = cw;
        sh.wave_ties[threadIdx.x / 64] = ct;
    }
    __syncthreads();
    for (uint32_t v = 0; v < threadIdx.x / 64; v++) {
        cw += sh.wave_w[v];
        ct += sh.wave_ties[v];
    }
    const uint64_t behind = cw + min(ct, sh.ties) * tie_w;
    uint64_t before = cw - w + min(ct - ties, sh.ties) * tie_w;
    if (before <= sh.target && sh.target < behind) {
        uint32_t seen = ct - ties;
        for (uint32_t j = i0; j < min(i0 + N, n); j++) {
            const float l = masked_nan((float)R.row[j]);
            const uint32_t key = logit_key(l);
            if (l == -INFINITY || key < cut.key) continue;
            uint64_t v;
            if (key == cut.key) v = seen++ < sh.ties ? tie_w : 0;
            else {
                v = R.S.weight(l);
                if (v < O.least) v = 0;
            }
            before += v;
            if (before > sh.target) {
                D.classes[r] = j;
                if (D.log_probs)
                    D.log_probs[r] =
                        (float)(R.S.z(l) - log((double)sh.total / (double)WEIGHT_ONE));
                break;
            }
        }
    }
}

template <class T>
void launch_sample(const void *logits, const Draw &D, hipStream_t s) {
    const auto *l = static_cast<const T *>(logits);
    if (D.n_classes <= GROUP_MOST) {
        uint32_t g = 2;
        while (g < D.n_classes) g *= 2;
        const uint64_t blocks = (D.n_rows + GROUP_TPB / g - 1) / (GROUP_TPB / g);
        head_input(blocks < 1u << 24, "too many rows");
        const dim3 grid((uint32_t)blocks), tpb(GROUP_TPB);
        if (g == 2) hipLaunchKernelGGL((sample_group_kernel<T, 2>), grid, tpb, 0, s, l, D);
        else if (g == 4) hipLaunchKernelGGL((sample_group_kernel<T, 4>), grid, tpb, 0, s, l, D);
        else if (g == 8) hipLaunchKernelGGL((sample_group_kernel<T, 8>), grid, tpb, 0, s, l, D);
        else if (g == 16) hipLaunchKernelGGL((sample_group_kernel<T, 16>), grid, tpb, 0, s, l, D);
        else if (g == 32) hipLaunchKernelGGL((sample_group_kernel<T, 32>), grid, tpb, 0, s, l, D);
        else hipLaunchKernelGGL((sample_group_kernel<T, 64>), grid, tpb, 0, s, l, D);
    } else {
        head_input(D.n_rows < 1u << 22, "too many rows");
        const dim3 grid((uint32_t)D.n_rows);
        if (D.n_classes <= 2048)
            hipLaunchKernelGGL((sample_row_kernel<T, 64>), grid, dim3(64), 0, s, l, D);
        else if (D.n_classes <= 16384)
            hipLaunchKernelGGL((sample_row_kernel<T, 256>), grid, dim3(256), 0, s, l, D);
        else hipLaunchKernelGGL((sample_row_kernel<T, 1024>), grid, dim3(1024), 0, s, l, D);
    }
    head_check(hipGetLastError(), "sampling");
}

void sample(const void *logits, uint32_t dtype, const Draw &D, hipStream_t s) {
    if (dtype == FBH_F32) launch_sample<float>(logits, D, s);
    else if (dtype == FBH_F16) launch_sample<_Float16>(logits, D, s);
    else launch_sample<__bf16>(logits, D, s);
}

void check_sample(const void *logits, uint64_t n_rows, uint32_t n_classes, const float *uniforms,
                  const fbh_sample_options *options, const int64_t *classes) {
    head_input(options && ((logits && uniforms && classes) || n_rows == 0), "null argument");
    head_input(n_classes >= 1 && n_classes <= SAMPLE_MOST, "n_classes must be in 1..=262144");
    head_input(n_rows <= 1ull << 40, "too many rows");
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" {

int fbh_sample_classes(int device, const void *logits, uint64_t n_rows, uint32_t n_classes,
                       uint32_t dtype, const float *uniforms, const fbh_sample_options *options,
                       int64_t *classes, float *log_probs, void *stream) {
    return head_guard([&] {
        check_sample(logits, n_rows, n_classes, uniforms, options, classes);
        head_input(dtype <= FBH_BF16, "unknown cell type");
        if (n_rows == 0) return;
        const OnDevice on(device);
        sample(logits, dtype, Draw{uniforms, *options, classes, log_probs, n_rows, n_classes},
               static_cast<hipStream_t>(stream));
    });
}

int fbh_sample_classes_host(int device, const float *logits, uint64_t n_rows, uint32_t n_classes,
                            const float *uniforms, const fbh_sample_options *options,
                            int64_t *classes, float *log_probs) {
    return head_guard([&] {
        check_sample(logits, n_rows, n_classes, uniforms, options, classes);
        head_input(!options->temperatures && !options->top_ks && !options->top_ps &&
                       !options->min_ps,
                   "options of each row's own are taken from device memory alone");
        if (n_rows == 0) return;
        const OnDevice on(device);
        hipStream_t s = nullptr;
        head_check(keep_stream(&s), "stream");
        uint8_t *block = nullptr;
        const auto end = [&](void *) {
            (void)hipStreamSynchronize(s);
            keep_free(KeepKind::device, block);
            (void)keep_stream_back(device, s);
        };
        const std::unique_ptr<void, decltype(end)> own(s, end);
        const uint64_t l_bytes = (4 * n_rows * n_classes + 255) & ~255ull;
        const uint64_t u_bytes = (4 * n_rows + 255) & ~255ull;
        head_check(keep_alloc(KeepKind::device, reinterpret_cast<void **>(&block),
                              l_bytes + 2 * u_bytes + 8 * n_rows),
                   "device allocation");
        auto *d_u = reinterpret_cast<float *>(block + l_bytes);
        auto *d_p = reinterpret_cast<float *>(block + l_bytes + u_bytes);
        auto *d_c = reinterpret_cast<int64_t *>(block + l_bytes + 2 * u_bytes);
        head_check(hipMemcpyAsync(block, logits, 4 * n_rows * n_classes, hipMemcpyHostToDevice, s),
                   "logit upload");
        head_check(hipMemcpyAsync(d_u, uniforms, 4 * n_rows, hipMemcpyHostToDevice, s),
                   "uniform upload");
        sample(block, FBH_F32, Draw{d_u, *options, d_c, d_p, n_rows, n_classes}, s);
        head_check(hipMemcpyAsync(classes, d_c, 8 * n_rows, hipMemcpyDeviceToHost, s),
                   "class download");
        if (log_probs)
            head_check(hipMemcpyAsync(log_probs, d_p, 4 * n_rows, hipMemcpyDeviceToHost, s),
                       "probability download");
        head_check(hipStreamSynchronize(s), "sampling");
    });
}

}  // extern "C"
