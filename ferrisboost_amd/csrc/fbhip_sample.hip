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
#include <type_traits>

#include "fbhip_heads.h"

namespace fbh {
namespace {

template <int N>
using Int = std::integral_constant<int, N>;

constexpr uint32_t SAMPLE_MOST = 262144;  // classes: their weights' sum is below 2^63
constexpr uint32_t NO_BIN = 0xFFFFFFFFu;
constexpr int WEIGHT_BITS = 45;
constexpr uint64_t WEIGHT_ONE = 1ull << WEIGHT_BITS;

// A row's options, as whole numbers.
struct RowOptions {
    double inv_t;       // 1 / temperature; 0 where that is infinite, and where k is 1 for the
                        // largest logit's sake
    uint32_t k;         // classes that stay by rank (1 for the largest logit)
    uint32_t p31;       // top_p * 2^31
    uint64_t least;     // smallest weight that stays by min_p
    __host__ __device__ bool cuts(uint32_t n) const { return k < n || p31 < 1u << 31; }
};

__host__ __device__ inline RowOptions whole_options(float t, int32_t k, float p, float m,
                                                    uint32_t n) {
    RowOptions r;
    r.k = t > 0.0f ? (k > 0 && (uint32_t)k < n ? (uint32_t)k : n) : 1;
    r.inv_t = t > 0.0f ? 1.0 / (double)t : 0.0;
    r.p31 = p < 1.0f ? (p > 0.0f ? (uint32_t)((double)p * 2147483648.0) : 0) : 1u << 31;
    r.least = m > 0.0f ? (m < 1.0f ? (uint64_t)ceil((double)m * (double)WEIGHT_ONE) : WEIGHT_ONE)
                       : 0;
    return r;
}

struct Draw {
    const float *uniforms;
    fbh_sample_options o;
    RowOptions all;     // of every row, where none has options of its own
    bool own;           // some have
    int64_t *classes;
    float *log_probs;
    uint64_t n_rows;
    uint32_t n_classes;
};

__device__ __forceinline__ RowOptions row_options(const Draw &D, uint64_t row) {
    if (!D.own) return D.all;
    return whole_options(D.o.temperatures ? D.o.temperatures[row] : D.o.temperature,
                         D.o.top_ks ? D.o.top_ks[row] : D.o.top_k,
                         D.o.top_ps ? D.o.top_ps[row] : D.o.top_p,
                         D.o.min_ps ? D.o.min_ps[row] : D.o.min_p, D.n_classes);
}

// uniform * 2^31
__device__ __forceinline__ uint32_t uniform31(float u) {
    return u > 0.0f ? (uint32_t)fmin((double)u * 2147483648.0, 2147483647.0) : 0;
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

__device__ __forceinline__ void put_class(const Draw &D, uint64_t row, int64_t c, double z,
                                          uint64_t total) {
    D.classes[row] = c;
    if (D.log_probs)
        D.log_probs[row] =
            c < 0 ? -INFINITY : (float)(z - log((double)total / (double)WEIGHT_ONE));
}

// What stays: classes of larger keys, and the first `ties` classes of this one.
struct Cut {
    uint32_t key, ties;
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int from, int width = 64) {
    const uint32_t lo = __shfl((uint32_t)v, from, width);
    const uint32_t hi = __shfl((uint32_t)(v >> 32), from, width);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64_up(uint64_t v, int by, int width = 64) {
    const uint32_t lo = __shfl_up((uint32_t)v, by, width);
    const uint32_t hi = __shfl_up((uint32_t)(v >> 32), by, width);
    return (uint64_t)hi << 32 | lo;
}
// Sums over a wave's lanes up to each, by moves between lanes that take no LDS: within rows
// of 16, then the last lane of a row to the next one, then of a half to the other.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
    return (uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 |
           moved<CTRL, ROWS>((uint32_t)v);
}
template <class U>
__device__ __forceinline__ U scan_wave(U v) {
    v += moved<0x111, 0xF>(v);
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);
    v += moved<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t at_lane(uint32_t v, uint32_t lane) {
    return __builtin_amdgcn_readlane(v, lane);
}
__device__ __forceinline__ uint64_t at_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)at_lane((uint32_t)(v >> 32), lane) << 32 | at_lane((uint32_t)v, lane);
}
// The largest of a wave's values.
__device__ __forceinline__ float most_of_wave(float v) {
    const auto step = [&](auto ctrl, auto rows) {
        v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(
                         __float_as_int(v), __float_as_int(v), decltype(ctrl)::value,
                         decltype(rows)::value, 0xF, false)));
    };
    step(Int<0x111>{}, Int<0xF>{});
    step(Int<0x112>{}, Int<0xF>{});
    step(Int<0x114>{}, Int<0xF>{});
    step(Int<0x118>{}, Int<0xF>{});
    step(Int<0x142>{}, Int<0xA>{});
    step(Int<0x143>{}, Int<0xC>{});
    return __int_as_float((int)at_lane((uint32_t)__float_as_int(v), 63));
}

// -------------------------------------------------------------- a row a thread
constexpr uint32_t THREAD_MOST = 8;

// Up to 8 classes: a thread a row, whose logits it holds; ranks and the weights before a
// class from every pair of them. Bound by arithmetic: V exponentials and a logarithm of
// doubles a row: 500k rows of 4 take 9 us, and 17 with a lane a class, where each row's
// options and logarithm take a whole wave's instructions.
template <class T, int V>
__global__ __launch_bounds__(256) void sample_thread_kernel(const T *logits, Draw D) {
    const uint64_t row = blockIdx.x * 256ull + threadIdx.x;
    if (row >= D.n_rows) return;
    const Piece<T, V> p = load_piece<T, V>(logits + row * V);
    const RowOptions O = row_options(D, row);
    float l[V];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        l[i] = masked_nan((float)p.v[i]);
        most = fmaxf(most, l[i]);
    }
    const RowScale S{most, (double)most, O.inv_t};
    uint64_t w[V];
#pragma unroll
    for (int i = 0; i < V; i++)
        w[i] = l[i] == -INFINITY ? 0 : S.weight(l[i]);
    if (O.cuts(V)) {
        uint32_t rank[V];
        uint64_t all = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            rank[i] = 0;
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j != i) rank[i] += l[j] > l[i] || (l[j] == l[i] && j < i);
            if (rank[i] >= O.k) w[i] = 0;
            all += w[i];
        }
        if (O.p31 < 1u << 31) {
            uint64_t most_w = share(O.p31, all, 0x7FFFFFFFu);
            if (most_w == 0) most_w = 1;
            uint64_t stay[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                uint64_t before = 0;
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (j != i && rank[j] < rank[i]) before += w[j];
                stay[i] = before < most_w ? w[i] : 0;
            }
#pragma unroll
            for (int i = 0; i < V; i++) w[i] = stay[i];
        }
    }
    uint64_t total = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (w[i] < O.least) w[i] = 0;
        total += w[i];
    }
    const uint64_t target = share(uniform31(D.uniforms[row]), total, 0);
    int c = -1;
    float at = most;
    uint64_t cum = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        cum += w[i];
        if (c < 0 && cum > target) {
            c = i;
            at = l[i];
        }
    }
    put_class(D, row, c, S.z(at), total);
}

// -------------------------------------------------------------- a lane a class
constexpr uint32_t GROUP_TPB = 256;
constexpr uint32_t GROUP_MOST = 64;

// Up to 64 classes: a lane a class, 64 / G rows a wave. Where a row cuts, its classes are
// sorted over its lanes by compare and exchange (10 to 21 steps), which gives their ranks and,
// in that order, the weights before them. Bound by instructions: 500k rows of 40 classes, a
// wave each, take 226 us uncut and 405 with top-p (904 with every lane meeting every class
// of its row in turn).
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
    const int lane0 = (threadIdx.x & 63) - c;  // the row's lanes
    const uint64_t lanes = G < 64 ? (1ull << (G & 63)) - 1 : ~0ull;
    const auto of_row = [&](bool b) { return (__ballot(b) >> lane0) & lanes; };
    // one class by rank: the first of the largest logit
    const int first = __ffsll((long long)of_row(l == most)) - 1;
    uint64_t w = 0;
    if (l != -INFINITY) w = O.k == 1 ? (c == first ? WEIGHT_ONE : 0) : S.weight(l);
    if (__any(O.k != 1 && O.cuts(D.n_classes))) {
        // falling logits, equal ones by class
        uint64_t e = (uint64_t)logit_key(l) << 32 | (uint32_t)~c;
#pragma unroll
        for (int size = 2; size <= G; size <<= 1)
#pragma unroll
            for (int by = size / 2; by; by >>= 1) {
                const uint32_t lo = __shfl_xor((uint32_t)e, by, G);
                const uint32_t hi = __shfl_xor((uint32_t)(e >> 32), by, G);
                const uint64_t other = (uint64_t)hi << 32 | lo;
                const bool larger = ((c & by) == 0) == ((c & size) == 0);
                if ((e > other) != larger) e = other;
            }
        const int who = (int)~(uint32_t)e;  // the class of rank c
        const uint32_t rank =
            (uint32_t)__builtin_amdgcn_ds_permute((lane0 + who) << 2, c);
        if (rank >= O.k) w = 0;
        const uint64_t ws = shfl64(w, who, G);
        uint64_t upto = ws;
#pragma unroll
        for (int d = 1; d < G; d <<= 1) {
            const uint64_t y = shfl64_up(upto, d, G);
            if (c >= d) upto += y;
        }
        const uint64_t most_w = share(O.p31, shfl64(upto, G - 1, G), 0x7FFFFFFFu);
        const uint32_t stay = __popcll(of_row(upto - ws < (most_w ? most_w : 1)));
        if (O.k != 1 && O.p31 < 1u << 31 && rank >= stay) w = 0;
    }
    if (w < O.least) w = 0;
    uint64_t cum = w;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        const uint64_t y = shfl64_up(cum, d, G);
        if (c >= d) cum += y;
    }
    const uint64_t total = shfl64(cum, G - 1, G);
    const uint64_t mine = of_row(cum > share(uniform31(D.uniforms[at]), total, 0));
    if (!in) return;
    if (total == 0) {
        if (c == 0) put_class(D, row, -1, 0.0, 0);
    } else if (c == __ffsll((long long)mine) - 1) {
        put_class(D, row, c, S.z(l), total);
    }
}

// -------------------------------------------------------------- a row a wave
constexpr uint32_t WAVE_BINS = 256;
constexpr uint32_t WAVE_MOST = 1024;

// Up to 64 R classes: a wave a row, which lies in registers, R classes side by side a
// lane. The cut's bin is found from a histogram in LDS; the bin's classes (with top-k of at
// most 64, all up to the cut) then take a lane each. Four waves a workgroup, with nothing
// in common: LDS operations of one wave complete in order. Bound by instructions, about a
// thousand a row: 20k rows of 500, top 50, take 35 us (158 with bins and digits in LDS and a
// row read four times).
struct WaveShared {
    uint64_t wt[WAVE_BINS];
    uint32_t ct[WAVE_BINS];
    uint32_t keys[64];
    uint32_t classes[64];
};

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <class T, int R>
__global__ __launch_bounds__(256) void sample_wave_kernel(const T *logits, Draw D) {
    __shared__ WaveShared shared[4];
    WaveShared &sh = shared[threadIdx.x / 64];
    const uint64_t row = blockIdx.x * 4ull + threadIdx.x / 64;
    if (row >= D.n_rows) return;
    const uint32_t lane = threadIdx.x & 63, n = D.n_classes, c0 = lane * R;
    const T *from = logits + row * n;
    const RowOptions O = row_options(D, row);

    float l[R];
    if (c0 + R <= n) {
        constexpr int N = R * sizeof(T) > 16 ? 16 / sizeof(T) : R;
#pragma unroll
        for (int i = 0; i < R; i += N) {
            const Piece<T, N> p = load_piece<T, N>(from + c0 + i);
#pragma unroll
            for (int j = 0; j < N; j++) l[i + j] = masked_nan((float)p.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++)
            l[i] = c0 + i < n ? masked_nan((float)from[c0 + i]) : -INFINITY;
    }
    float mine = l[0];
#pragma unroll
    for (int i = 1; i < R; i++) mine = fmaxf(mine, l[i]);
    const float most = most_of_wave(mine);
    if (most == -INFINITY || O.k == 1) {
        const uint64_t has = __ballot(mine == most);
        if (lane == (uint32_t)__ffsll((long long)has) - 1) {
            int at = 0;
#pragma unroll
            for (int i = R - 1; i >= 0; i--)
                if (l[i] == most) at = i;
            put_class(D, row, most == -INFINITY ? -1 : (int64_t)(c0 + at), 0.0, WEIGHT_ONE);
        }
        return;
    }
    const RowScale S{most, (double)most, O.inv_t};
    const float per_nat = (float)(O.inv_t * (WAVE_BINS / 32));
    uint32_t bins[R];  // of (max - l) / T, 32 over all of them; masked classes behind them
    const auto set_bins = [&] {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const float d = l[i] == most ? 0.0f : (most - l[i]) * per_nat;
            bins[i] = l[i] == -INFINITY ? WAVE_BINS
                                        : (uint32_t)fminf(d, (float)(WAVE_BINS - 1));
        }
    };
    const uint32_t target31 = uniform31(D.uniforms[row]);

    uint64_t w[R];
    bool weighed = false;
    const auto weigh = [&] {
#pragma unroll
        for (int i = 0; i < R; i++) w[i] = l[i] == -INFINITY ? 0 : S.weight(l[i]);
        weighed = true;
    };
    // The first bin at which the counts (the weights) reach k (weight); what stands before.
    const auto find = [&](bool by_count, uint32_t k, uint64_t weight, uint32_t &before_c,
                          uint64_t &before_w, uint32_t &inside) {
        uint32_t c[WAVE_BINS / 64];
        uint64_t v[WAVE_BINS / 64];
        uint32_t cs = 0;
        uint64_t vs = 0;
#pragma unroll
        for (int b = 0; b < (int)WAVE_BINS / 64; b++) {
            c[b] = sh.ct[lane * (WAVE_BINS / 64) + b];
            v[b] = by_count ? 0 : sh.wt[lane * (WAVE_BINS / 64) + b];
            cs += c[b];
            vs += v[b];
        }
        const uint32_t cc = scan_wave(cs);
        const uint64_t vv = by_count ? 0 : scan_wave(vs);
        const uint64_t hits = __ballot(by_count ? cc >= k : vv >= weight);
        if (!hits) return NO_BIN;
        const int who = __ffsll((long long)hits) - 1;
        uint32_t bc = cc - cs, bin = 0;
        uint64_t bv = vv - vs;
        bool found = false;
#pragma unroll
        for (int b = 0; b < (int)WAVE_BINS / 64; b++)
            if (!found) {
                inside = c[b];
                bin = lane * (WAVE_BINS / 64) + b;
                if (by_count ? bc + c[b] >= k : bv + v[b] >= weight) found = true;
                else {
                    bc += c[b];
                    bv += v[b];
                }
            }
        before_c = at_lane(bc, who);
        before_w = at_lane(bv, who);
        inside = at_lane(inside, who);
        return at_lane(bin, who);
    };
    // Classes with take(i) to lanes, in class order; at most 64 of them.
    const auto gather = [&](auto &&take) {
        uint32_t some = 0;
#pragma unroll
        for (int i = 0; i < R; i++) some += take(i);
        uint32_t at = scan_wave(some) - some;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (take(i)) {
                sh.keys[at] = logit_key(l[i]);
                sh.classes[at] = c0 + i;
                at++;
            }
        wave_fence();
    };
    // This lane's place among `members` lanes by falling key, equal ones by lane.
    const auto rank_of = [&](uint32_t key, uint32_t members) {
        uint32_t rank = 0;
        // (lanes behind the last member hold key 0, below any class')
        for (uint32_t j0 = 0; j0 < members; j0 += 8)
#pragma unroll
            for (uint32_t j = j0; j < j0 + 8; j++) {
                const uint32_t kj = at_lane(key, j);
                rank += kj > key || (kj == key && j < lane);
            }
        return rank;
    };
    // The cut among classes of one bin by bisection of their keys, where they are too many
    // for a lane each.
    const auto bisect = [&](uint32_t bin, bool by_count, uint32_t k, uint64_t weight,
                            uint32_t before_c, uint64_t before_w) {
        uint32_t lo = 0, hi = 0xFFFFFFFFu;  // the cut's key: the largest with enough at or above
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            uint32_t c = 0;
            uint64_t v = 0;
#pragma unroll
            for (int i = 0; i < R; i++)
                if (bins[i] == bin && logit_key(l[i]) >= mid) {
                    c++;
                    if (!by_count) v += w[i];
                }
            const bool enough =
                by_count ? before_c + at_lane(scan_wave(c), 63) >= k
                         : before_w + at_lane(scan_wave(v), 63) >= weight;
            if (enough) lo = mid;
            else hi = mid - 1;
        }
        uint32_t c = 0;
        uint64_t v = 0;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (bins[i] == bin && logit_key(l[i]) > lo) {
                c++;
                if (!by_count) v += w[i];
            }
        Cut cut{lo, 0};
        if (by_count) cut.ties = k - before_c - at_lane(scan_wave(c), 63);
        else {
            const uint64_t one = S.weight(key_logit(lo));
            const uint64_t left = weight - before_w - at_lane(scan_wave(v), 63);
            cut.ties = (uint32_t)((left + one - 1) / one);
        }
        return cut;
    };
    const auto cut_in = [&](uint32_t bin, uint32_t inside, bool by_count, uint32_t k,
                            uint64_t weight, uint32_t before_c, uint64_t before_w) {
        if (inside > 64) return bisect(bin, by_count, k, weight, before_c, before_w);
        gather([&](int i) { return bins[i] == bin; });
        const uint32_t key = lane < inside ? sh.keys[lane] : 0;
        const uint32_t rank = rank_of(key, inside);
        wave_fence();
        // by rank: the keys, and what they add up to
        if (lane < inside) sh.keys[rank] = key;
        wave_fence();
        const uint32_t sorted = lane < inside ? sh.keys[lane] : 0;
        const uint64_t v =
            lane < inside && !by_count ? S.weight(key_logit(sorted)) : 0;
        const uint64_t upto = by_count ? 0 : before_w + scan_wave(v);
        const uint64_t hits = __ballot(
            lane < inside && (by_count ? before_c + lane + 1 >= k : upto >= weight));
        const uint32_t who = (uint32_t)__ffsll((long long)hits) - 1;
        const uint32_t at = at_lane(sorted, who);
        const uint64_t same = __ballot(lane < inside && sorted == at);
        wave_fence();
        return Cut{at, who - ((uint32_t)__ffsll((long long)same) - 1) + 1};
    };
    const auto histogram = [&](bool weights) {
        wave_fence();
#pragma unroll
        for (int b = 0; b < (int)WAVE_BINS / 64; b++) {
            sh.ct[lane + 64 * b] = 0;
            if (weights) sh.wt[lane + 64 * b] = 0;
        }
        wave_fence();
#pragma unroll
        for (int i = 0; i < R; i++)
            if (bins[i] < WAVE_BINS) {
                atomicAdd(&sh.ct[bins[i]], 1u);
                if (weights)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wt[bins[i]]),
                              (unsigned long long)w[i]);
            }
        wave_fence();
    };

    Cut cut{0, 0};
    uint64_t tie_w = 0;
    if (O.cuts(n)) {
        uint32_t before_c = 0, inside = 0;
        uint64_t before_w = 0;
        set_bins();
        if (O.k <= 64 && O.k < n) {
            histogram(false);
            const uint32_t bin = find(true, O.k, 0, before_c, before_w, inside);
            const uint32_t members = before_c + inside;
            if (bin != NO_BIN && members <= 64) {
                // All that can stay has a lane each, in class order.
                gather([&](int i) { return bins[i] <= bin; });
                const uint32_t key = lane < members ? sh.keys[lane] : 0;
                const uint32_t rank = rank_of(key, members);
                const float v = key_logit(key);
                uint64_t kept = lane < members && rank < O.k ? S.weight(v) : 0;
                if (O.p31 < 1u << 31) {
                    if (lane < members) sh.wt[rank] = kept;
                    wave_fence();
                    const uint64_t s = lane < members ? sh.wt[lane] : 0;
                    const uint64_t upto = scan_wave(s);
                    uint64_t weight = share(O.p31, at_lane(upto, 63), 0x7FFFFFFFu);
                    if (weight == 0) weight = 1;
                    const uint32_t stay = __popcll(__ballot(lane < members && upto - s < weight));
                    if (rank >= stay) kept = 0;
                }
                if (kept < O.least) kept = 0;
                const uint64_t cum = scan_wave(kept);
                const uint64_t total = at_lane(cum, 63);
                const uint64_t hits = __ballot(cum > share(target31, total, 0));
                if (lane == (uint32_t)__ffsll((long long)hits) - 1)
                    put_class(D, row, sh.classes[lane], S.z(v), total);
                return;
            }
        }
        weigh();
        histogram(true);
        uint32_t k_bin = NO_BIN, k_inside = 0, k_c = 0;
        uint64_t k_w = 0;
        if (O.k < n) {
            k_bin = find(true, O.k, 0, k_c, k_w, k_inside);
            if (k_bin != NO_BIN) {
                cut = cut_in(k_bin, k_inside, true, O.k, 0, k_c, 0);
                tie_w = S.weight(key_logit(cut.key));
            }
        }
        if (O.p31 < 1u << 31) {
            uint64_t mine_w = 0;
#pragma unroll
            for (int i = 0; i < R; i++)
                if (logit_key(l[i]) > cut.key) mine_w += w[i];
            const uint64_t all = at_lane(scan_wave(mine_w), 63) + cut.ties * tie_w;
            uint64_t weight = share(O.p31, all, 0x7FFFFFFFu);
            if (weight == 0) weight = 1;
            const uint32_t bin = find(false, 0, weight, before_c, before_w, inside);
            cut = cut_in(bin, inside, false, 0, weight, 0, before_w);
            tie_w = S.weight(key_logit(cut.key));
        }
        if (tie_w < O.least) cut.ties = 0;
    }
    if (!weighed) weigh();

    // The staying weights in class order.
    uint32_t ties = 0;
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const uint32_t key = logit_key(l[i]);
        if (key < cut.key || w[i] < O.least) w[i] = 0;
        if (key == cut.key) {
            ties++;
            w[i] = 0;
        }
        sum += w[i];
    }
    const uint32_t ties0 = scan_wave(ties) - ties;  // before this lane
    const uint32_t kept = ties0 < cut.ties ? min(cut.ties - ties0, ties) : 0;
    sum += kept * tie_w;
    const uint64_t cum = scan_wave(sum);
    const uint64_t total = at_lane(cum, 63);
    const uint64_t target = share(target31, total, 0);
    const uint64_t hits = __ballot(cum > target);
    if (lane == (uint32_t)__ffsll((long long)hits) - 1) {
        uint64_t at = cum - sum;
        uint32_t seen = 0;
        int c = -1;
        float v = most;
#pragma unroll
        for (int i = 0; i < R; i++) {
            at += logit_key(l[i]) == cut.key ? (seen++ < kept ? tie_w : 0) : w[i];
            if (c < 0 && at > target) {
                c = (int)c0 + i;
                v = l[i];
            }
        }
        put_class(D, row, c, S.z(v), total);
    }
}

// -------------------------------------------------------------- a row a workgroup
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

// Classes in a list: falling logits first, equal ones by class, as one number falls.
__device__ __forceinline__ uint64_t entry_of(float l, uint32_t c) {
    return (uint64_t)logit_key(l) << 32 | (uint32_t)~c;
}
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ uint32_t entry_class(uint64_t e) { return ~(uint32_t)e; }

constexpr uint32_t ROW_BINS = 1024;
// Bins of max - l: monotone, as each step of it is.
__device__ __forceinline__ uint32_t weight_bin(float l, float most, float per) {
    const float d = l == most ? 0.0f : (most - l) * per;
    return (uint32_t)fminf(d, (float)(ROW_BINS - 1));
}

struct TileWork;

template <int TPB>
struct RowShared {
    static constexpr uint32_t BINS = ROW_BINS;
    static constexpr uint32_t LIST = 2048;
    static constexpr uint32_t MOST_K = TPB / 2;  // of the classes found by the threads' largest
    uint64_t wt[BINS];
    uint32_t ct[BINS];
    uint64_t list[LIST];
    uint64_t tile_w[MOST_TILES];
    uint32_t tile_ties[MOST_TILES];
    float wave_most[TPB / 64];
    uint64_t wave_w[TPB / 64];
    uint32_t wave_ties[TPB / 64];
    uint32_t bin, n_list;
    uint32_t before_ct;
    uint64_t before_wt;
    uint64_t target;
    uint64_t total;
    uint32_t tile, ties;
};

// The thread's piece of a tile, masked classes (and ones behind the last) as -inf.
template <class T>
__device__ __forceinline__ void tile_piece(const T *row, uint32_t n, uint32_t i,
                                           float (&l)[16 / sizeof(T)]) {
    constexpr int N = 16 / sizeof(T);
    if (i + N <= n) {
        const Piece<T, N> p = load_piece<T, N>(row + i);
#pragma unroll
        for (int j = 0; j < N; j++) l[j] = masked_nan((float)p.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) l[j] = i + j < n ? masked_nan((float)row[i + j]) : -INFINITY;
    }
}

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
    float per;  // bins of a unit of logits

    // f(class of the first, logits) for the thread's pieces; ones behind the last class, and
    // NaN, as -inf.
    template <class F>
    __device__ __forceinline__ void pieces(F &&f) const {
        const uint32_t step = TPB * N, whole = n / step * step;  // (all threads have a piece)
        uint32_t i = threadIdx.x * N;
        const auto batch = [&](auto pieces) {
            constexpr int B = decltype(pieces)::value;
            Piece<T, N> p[B];
#pragma unroll
            for (int b = 0; b < B; b++) p[b] = load_piece<T, N>(row + i + b * step);
#pragma unroll
            for (int b = 0; b < B; b++) {
                float l[N];
#pragma unroll
                for (int j = 0; j < N; j++) l[j] = masked_nan((float)p[b].v[j]);
                f(i + b * step, l);
            }
            i += B * step;
        };
        while (i + 4 * step <= whole + threadIdx.x * N) batch(Int<4>{});
        while (i < whole) batch(Int<1>{});
        if (i < n) {
            float l[N];
            tile_piece<T>(row, n, i, l);
            f(i, l);
        }
    }
    // f(class, logit) for the thread's classes.
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

    // The least of all threads' values.
    __device__ __forceinline__ float least(float v) {
        const float m = -most_of_wave(-v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.wave_most[threadIdx.x / 64] = m;
        __syncthreads();
        float all = sh.wave_most[0];
        for (int w = 1; w < TPB / 64; w++) all = fminf(all, sh.wave_most[w]);
        return all;
    }

    // The largest logit, and the thread's own largest.
    __device__ __forceinline__ float largest(float &own) {
        own = -INFINITY;
        pieces([&](uint32_t, const float *l) {
#pragma unroll
            for (int j = 0; j < N; j++) own = fmaxf(own, l[j]);
        });
        return -least(-own);
    }
    // The first class of this logit.
    __device__ __forceinline__ uint32_t first_of(float most) {
        if (threadIdx.x == 0) sh.n_list = NO_BIN;
        __syncthreads();
        pieces([&](uint32_t i, const float *l) {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (l[j] == most) atomicMin(&sh.n_list, i + j);
        });
        __syncthreads();
        return sh.n_list;
    }

    __device__ __forceinline__ uint32_t bin_of(float l) const {
        return weight_bin(l, S.most, per);
    }

    __device__ __forceinline__ void clear(uint32_t bins) {
        __syncthreads();
        for (uint32_t b = threadIdx.x; b < bins; b += TPB) {
            sh.ct[b] = 0;
            sh.wt[b] = 0;
        }
        __syncthreads();
    }
    __device__ __forceinline__ void add_weight(uint32_t bin, uint64_t w) {
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wt[bin]), (unsigned long long)w);
    }
    __device__ __forceinline__ void before(uint32_t ct, uint64_t wt) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.before_ct = ct;
            sh.before_wt = wt;
        }
    }

    // The sum of all threads' values, and with `upto` that of the threads up to this one.
    __device__ __forceinline__ uint64_t sum(uint64_t v, uint64_t *upto = nullptr) {
        const uint64_t x = scan_wave(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) sh.wave_w[threadIdx.x / 64] = x;
        __syncthreads();
        uint64_t all = 0, mine = x;
        for (uint32_t w = 0; w < TPB / 64; w++) {
            const uint64_t y = sh.wave_w[w];
            all += y;
            if (w < threadIdx.x / 64) mine += y;
        }
        if (upto) *upto = mine;
        return all;
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
            const uint32_t cc = scan_wave(c);
            const uint64_t ww = scan_wave(w);
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

    // The cut inside bin `bin`, whose classes are in the list (n_list of them, or, with
    // n_list NO_BIN, are to be read again), with sh.before_* standing before it.
    __device__ __forceinline__ Cut refine(uint32_t bin, uint32_t n_list, bool by_count, uint32_t k,
                                          uint64_t weight) {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= KeyDigits<T>::last; shift -= 8) {
            clear(256);
            const auto take = [&](uint32_t key) {
                if (shift == 24 || key >> (shift + 8) == prefix) {
                    const uint32_t b = 255 - ((key >> shift) & 255);
                    atomicAdd(&sh.ct[b], 1u);
                    add_weight(b, S.weight(key_logit(key)));
                }
            };
            if (n_list != NO_BIN)
                for (uint32_t i = threadIdx.x; i < n_list; i += TPB) take(entry_key(sh.list[i]));
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

    // From a row's bins of weights: the bin that top-p cuts, with sh.before_* before it, and
    // the weight that it asks for.
    template <class W>
    __device__ __forceinline__ uint32_t weight_cut(const W &work, const RowOptions &O,
                                                   uint64_t *asked) {
        clear(Shared::BINS);
        for (uint32_t b = threadIdx.x; b < Shared::BINS; b += TPB) sh.wt[b] = work.wt[b];
        return weight_cut(O, asked);
    }
    __device__ __forceinline__ uint32_t weight_cut(const RowOptions &O, uint64_t *asked) {
        before(0, 0);
        __syncthreads();
        uint64_t all = 0;
        for (uint32_t b = threadIdx.x; b < Shared::BINS; b += TPB) all += sh.wt[b];
        uint64_t weight = share(O.p31, sum(all), 0x7FFFFFFFu);
        if (weight == 0) weight = 1;
        find(Shared::BINS, false, 0, weight);
        if (asked) *asked = weight;
        return sh.bin;
    }

    // The classes of logits at or above `from`, in the list; how many, NO_BIN if too many.
    __device__ __forceinline__ uint32_t gather_from(float from) {
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        pieces([&](uint32_t i, const float *l) {
            float m = l[0];
#pragma unroll
            for (int j = 1; j < N; j++) m = fmaxf(m, l[j]);
            if (m < from) return;
#pragma unroll
            for (int j = 0; j < N; j++)
                if (l[j] >= from) {
                    const uint32_t at = atomicAdd(&sh.n_list, 1u);
                    if (at < Shared::LIST) sh.list[at] = entry_of(l[j], i + j);
                }
        });
        __syncthreads();
        return sh.n_list <= Shared::LIST ? sh.n_list : NO_BIN;
    }

    // The classes that `take`, in the list; how many they are, NO_BIN if too many.
    template <class F>
    __device__ __forceinline__ uint32_t gather(F &&take) {
        __syncthreads();
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        each([&](uint32_t c, float l) {
            if (l != -INFINITY && take(c, l)) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < Shared::LIST) sh.list[at] = entry_of(l, c);
            }
        });
        __syncthreads();
        return sh.n_list <= Shared::LIST ? sh.n_list : NO_BIN;
    }
};

// The draw among the first k classes, which are all in the list of m. Their order is every
// entry's rank among the list; sums in it and by class then need only k numbers.
template <class T, int TPB>
__device__ __forceinline__ void draw_listed(SampleRow<T, TPB> &R, const Draw &D, uint64_t row,
                                            const RowOptions &O, uint32_t m) {
    auto &sh = R.sh;
    uint64_t *weights = sh.wt;   // by rank
    uint32_t *classes = sh.ct;
    for (uint32_t i = threadIdx.x; i < m; i += TPB) {
        const uint64_t e = sh.list[i];
        uint32_t rank = 0;
#pragma unroll 16
        for (uint32_t j = 0; j < m; j++) rank += sh.list[j] > e;
        if (rank < O.k) {
            weights[rank] = R.S.weight(key_logit(entry_key(e)));
            classes[rank] = entry_class(e);
        }
    }
    __syncthreads();
    const uint32_t i = threadIdx.x, k = min(O.k, m);
    uint64_t w = i < k ? weights[i] : 0;
    const uint32_t c = i < k ? classes[i] : 0;
    if (O.p31 < 1u << 31) {
        uint64_t upto;
        const uint64_t all = R.sum(w, &upto);
        uint64_t weight = share(O.p31, all, 0x7FFFFFFFu);
        if (weight == 0) weight = 1;
        if (upto - w >= weight) w = 0;
    }
    if (w < O.least) w = 0;
    const uint64_t total = R.sum(w);  // (its barriers stand before the writes)
    if (i < k) weights[i] = w;
    __syncthreads();
    const uint64_t target = share(uniform31(D.uniforms[row]), total, 0);
    uint64_t before = 0;
    if (w)
#pragma unroll 16
        for (uint32_t j = 0; j < k; j++) before += classes[j] < c ? weights[j] : 0;
    if (w && before <= target && target < before + w) {
        const float l = (float)R.row[c];
        put_class(D, row, c, R.S.z(l), total);
    }
}

// ---- Few rows of many classes: a row's tiles (of 1024 pieces) go to a workgroup each. Three
// launches find what the row's own workgroup finds pass by pass, the largest logit, the
// histogram of weights, and the tiles' sums with a list of the cut's bin; the row kernel
// then begins at its last steps. (1 x 50000 bfloat16, top-p: 46 us in one workgroup, whose
// one CU is bound by the exponentials of doubles; 28 in four launches.) Rows whose options do not take a
// histogram of weights (few classes by rank, or more than the row kernel lists) are left to
// the row kernel altogether.
constexpr uint32_t TILE_TPB = 1024;
constexpr uint32_t TILE_BINS = 1024;
constexpr uint32_t TILE_LIST = 2048;

struct TileWork {  // of one row
    uint64_t wt[TILE_BINS];
    uint64_t list[TILE_LIST];
    uint64_t tile_w[MOST_TILES];
    float most[MOST_TILES];
    uint32_t n_list, reserved;
};

// Whether the tiles' launches do a row's passes.
__device__ __forceinline__ bool tiled(const RowOptions &O, uint32_t n) { return O.k >= n; }

__device__ __forceinline__ float row_most(const TileWork &W, uint32_t tiles) {
    float m = (threadIdx.x & 63) < tiles ? W.most[threadIdx.x & 63] : -INFINITY;
    return most_of_wave(m);
}

// grid (tiles, rows)
template <class T>
__global__ __launch_bounds__(TILE_TPB) void tile_most_kernel(const T *logits, Draw D,
                                                             TileWork *work) {
    __shared__ float waves[TILE_TPB / 64];
    constexpr int N = 16 / sizeof(T);
    const uint64_t r = blockIdx.y;
    const RowOptions O = row_options(D, r);
    if (!tiled(O, D.n_classes)) return;
    TileWork &W = work[r];
    if (blockIdx.x == 0) {
        W.wt[threadIdx.x] = 0;
        if (threadIdx.x == 0) W.n_list = 0;
    }
    float l[N];
    tile_piece<T>(logits + r * D.n_classes, D.n_classes, (blockIdx.x * TILE_TPB + threadIdx.x) * N, l);
    float m = l[0];
#pragma unroll
    for (int j = 1; j < N; j++) m = fmaxf(m, l[j]);
    m = most_of_wave(m);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x / 64] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < TILE_TPB / 64; w++) m = fmaxf(m, waves[w]);
        W.most[blockIdx.x] = m;
    }
}

template <class T>
__global__ __launch_bounds__(TILE_TPB) void tile_weights_kernel(const T *logits, Draw D,
                                                                TileWork *work) {
    __shared__ uint64_t wt[TILE_BINS];
    constexpr int N = 16 / sizeof(T);
    const uint64_t r = blockIdx.y;
    const RowOptions O = row_options(D, r);
    if (!tiled(O, D.n_classes) || O.p31 == 1u << 31) return;
    TileWork &W = work[r];
    wt[threadIdx.x] = 0;
    const float most = row_most(W, gridDim.x);
    const RowScale S{most, (double)most, O.inv_t};
    const float per = (float)(O.inv_t * (TILE_BINS / 32));
    __syncthreads();
    float l[N];
    tile_piece<T>(logits + r * D.n_classes, D.n_classes, (blockIdx.x * TILE_TPB + threadIdx.x) * N, l);
#pragma unroll
    for (int j = 0; j < N; j++)
        if (l[j] != -INFINITY) {
            const uint64_t w = S.weight(l[j]);
            if (w)
                atomicAdd(reinterpret_cast<unsigned long long *>(&wt[weight_bin(l[j], most, per)]),
                          (unsigned long long)w);
        }
    __syncthreads();
    if (wt[threadIdx.x])
        atomicAdd(reinterpret_cast<unsigned long long *>(&W.wt[threadIdx.x]),
                  (unsigned long long)wt[threadIdx.x]);
}

template <class T>
__global__ __launch_bounds__(TILE_TPB) void tile_sums_kernel(const T *logits, Draw D,
                                                             TileWork *work) {
    __shared__ RowShared<TILE_TPB> sh;
    constexpr int N = 16 / sizeof(T);
    const uint64_t r = blockIdx.y;
    const RowOptions O = row_options(D, r);
    if (!tiled(O, D.n_classes)) return;
    TileWork &W = work[r];
    const uint32_t i = (blockIdx.x * TILE_TPB + threadIdx.x) * N;
    float l[N];
    tile_piece<T>(logits + r * D.n_classes, D.n_classes, i, l);
    const float most = row_most(W, gridDim.x);
    SampleRow<T, TILE_TPB> R{sh, logits + r * D.n_classes, D.n_classes,
                             RowScale{most, (double)most, O.inv_t},
                             (float)(O.inv_t * (TILE_BINS / 32))};
    uint32_t bin = NO_BIN;
    if (O.p31 < 1u << 31) bin = R.weight_cut(W, O, nullptr);
    uint64_t w = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (l[j] == -INFINITY) continue;
        const uint32_t b = R.bin_of(l[j]);
        if (b < bin) {
            const uint64_t v = R.S.weight(l[j]);
            if (v >= O.least) w += v;
        } else if (b == bin) {
            const uint32_t at = atomicAdd(&W.n_list, 1u);
            if (at < TILE_LIST) W.list[at] = entry_of(l[j], i + j);
        }
    }
    w = R.sum(w);
    if (threadIdx.x == 0) W.tile_w[blockIdx.x] = w;
}

// More classes: a row a workgroup. 256 x 131071 bfloat16, top 200, take 44 us: two passes
// over 67 MB (12 us each, one row a CU) and the list's ranks and sums; by weight alone 148,
// bound by two exponentials of doubles a class.
//
// TILED: rows whose passes the tiles' launches have done take their results.
template <class T, int TPB, bool TILED>
__global__ __launch_bounds__(TPB) void sample_row_kernel(const T *logits, Draw D,
                                                         const TileWork *work) {
    __shared__ RowShared<TPB> sh;
    constexpr int N = 16 / sizeof(T);
    constexpr uint32_t BINS = RowShared<TPB>::BINS;
    const uint64_t r = blockIdx.x;
    const uint32_t n = D.n_classes;
    const RowOptions O = row_options(D, r);
    SampleRow<T, TPB> R{sh, logits + r * n, n, {}, 0.0f};
    const uint32_t tiles = (n + TPB * N - 1) / (TPB * N);
    const bool done = TILED && tiled(O, n);
    float own = -INFINITY;
    const float most = done ? row_most(work[r], tiles) : R.largest(own);
    if (most == -INFINITY || O.k == 1) {
        const int64_t c = most == -INFINITY ? -1 : (int64_t)R.first_of(most);
        if (threadIdx.x == 0) put_class(D, r, c, 0.0, WEIGHT_ONE);
        return;
    }
    R.S = RowScale{most, (double)most, O.inv_t};

    // Few classes by rank: k of the threads' own largest logits are at or above the k-th of
    // them, so the first k classes of the row are too. One more pass lists those.
    if (O.k < n && O.k <= RowShared<TPB>::MOST_K) {
        const float least = R.least(own == -INFINITY ? INFINITY : own);
        R.per = most > least ? (float)BINS / (most - least) : 0.0f;
        R.clear(BINS);
        if (own != -INFINITY) atomicAdd(&sh.ct[R.bin_of(own)], 1u);
        R.before(0, 0);
        R.find(BINS, true, O.k, 0);
        const uint32_t bin = sh.bin;
        if (bin != NO_BIN) {
            // the least of the largest ones in the bins up to the k-th's
            const float from = R.least(own != -INFINITY && R.bin_of(own) <= bin ? own : INFINITY);
            const uint32_t m = R.gather_from(from);
            if (m != NO_BIN) {
                draw_listed(R, D, r, O, m);
                return;
            }
        }
    }
    R.per = (float)(O.inv_t * (BINS / 32));  // 32 (max - l) / T over all bins

    // tile sums: TPB pieces of N classes a tile, in class order
    for (uint32_t t = threadIdx.x; t < MOST_TILES; t += TPB) {
        sh.tile_w[t] = done && t < tiles ? work[r].tile_w[t] : 0;
        sh.tile_ties[t] = 0;
    }
    // Adds up, tile by tile, what f(class, logit, weight, ties) finds in a piece.
    const auto sum_tiles = [&](auto &&f) {
        __syncthreads();
        for (uint32_t t = 0; t < tiles; t++) {
            uint64_t w = 0;
            uint32_t ties = 0;
            const uint32_t i = (t * TPB + threadIdx.x) * N;
            if (i + N <= n) {
                const Piece<T, N> p = load_piece<T, N>(R.row + i);
#pragma unroll
                for (int j = 0; j < N; j++) f(i + j, masked_nan((float)p.v[j]), w, ties);
            } else {
                for (uint32_t j = i; j < n; j++) f(j, masked_nan((float)R.row[j]), w, ties);
            }
            w = scan_wave(w);
            ties = scan_wave(ties);
            if ((threadIdx.x & 63) == 63) {
                if (w)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sh.tile_w[t]),
                              (unsigned long long)w);
                if (ties) atomicAdd(&sh.tile_ties[t], ties);
            }
        }
        __syncthreads();
    };
    // A class' part in a sum once the cut is known.
    Cut cut{0, 0};
    uint64_t tie_w = 0;
    const auto staying = [&](float l, uint64_t &w, uint32_t &ties) {
        const uint32_t key = logit_key(l);
        if (l == -INFINITY || key < cut.key) return;
        if (key == cut.key) {
            ties++;
            return;
        }
        const uint64_t v = R.S.weight(l);
        if (v >= O.least) w += v;
    };

    if (O.k < n) {
        // Many classes by rank: both cuts from one histogram, then digits of the key.
        const auto histogram = [&] {
            R.clear(BINS);
            R.each([&](uint32_t, float l) {
                if (l != -INFINITY) {
                    const uint32_t b = R.bin_of(l);
                    atomicAdd(&sh.ct[b], 1u);
                    R.add_weight(b, R.S.weight(l));
                }
            });
            R.before(0, 0);
        };
        histogram();
        __syncthreads();
        uint64_t all = 0;
        for (uint32_t b = threadIdx.x; b < BINS; b += TPB) all += sh.wt[b];
        all = R.sum(all);
        R.find(BINS, true, O.k, 0);
        const uint32_t k_bin = sh.bin;
        if (k_bin != NO_BIN) {
            const uint32_t inside = sh.ct[k_bin];
            const uint32_t m =
                inside <= RowShared<TPB>::LIST
                    ? R.gather([&](uint32_t, float l) { return R.bin_of(l) == k_bin; })
                    : NO_BIN;
            cut = R.refine(k_bin, m, true, O.k, 0);
            tie_w = R.S.weight(key_logit(cut.key));
            all = sh.before_wt + cut.ties * tie_w;
        }
        if (O.p31 < 1u << 31) {
            uint64_t weight = share(O.p31, all, 0x7FFFFFFFu);
            if (weight == 0) weight = 1;
            if (k_bin != NO_BIN) histogram();  // (refine() has used the bins)
            else R.before(0, 0);
            R.find(BINS, false, 0, weight);
            const uint32_t bin = sh.bin, inside = sh.ct[bin];
            const uint32_t m =
                inside <= RowShared<TPB>::LIST
                    ? R.gather([&](uint32_t, float l) { return R.bin_of(l) == bin; })
                    : NO_BIN;
            cut = R.refine(bin, m, false, 0, weight);
            tie_w = R.S.weight(key_logit(cut.key));
        }
        if (tie_w < O.least) cut.ties = 0;
        sum_tiles([&](uint32_t, float l, uint64_t &w, uint32_t &t) { staying(l, w, t); });
    } else if (O.p31 < 1u << 31) {
        // By weight alone: a histogram finds the cut's bin; one pass then sums the bins
        // before it and lists its own classes, whose digits find the cut.
        uint64_t weight;
        uint32_t bin, m;
        if (done) {
            bin = R.weight_cut(work[r], O, &weight);
            m = work[r].n_list <= RowShared<TPB>::LIST ? work[r].n_list : NO_BIN;
            if (m != NO_BIN)
                for (uint32_t i = threadIdx.x; i < m; i += TPB) sh.list[i] = work[r].list[i];
        } else {
            R.clear(BINS);
            R.each([&](uint32_t, float l) {
                if (l != -INFINITY) R.add_weight(R.bin_of(l), R.S.weight(l));
            });
            bin = R.weight_cut(O, &weight);
            if (threadIdx.x == 0) sh.n_list = 0;
            sum_tiles([&](uint32_t c, float l, uint64_t &w, uint32_t &) {
                if (l == -INFINITY) return;
                const uint32_t b = R.bin_of(l);
                if (b < bin) {
                    const uint64_t v = R.S.weight(l);
                    if (v >= O.least) w += v;
                } else if (b == bin) {
                    const uint32_t at = atomicAdd(&sh.n_list, 1u);
                    if (at < RowShared<TPB>::LIST) sh.list[at] = entry_of(l, c);
                }
            });
            m = sh.n_list <= RowShared<TPB>::LIST ? sh.n_list : NO_BIN;
        }
        cut = R.refine(bin, m, false, 0, weight);
        tie_w = R.S.weight(key_logit(cut.key));
        if (tie_w < O.least) cut.ties = 0;
        const auto one = [&](uint32_t c, float l) {
            uint64_t w = 0;
            uint32_t ties = 0;
            staying(l, w, ties);
            const uint32_t t = c / (TPB * N);
            if (w)
                atomicAdd(reinterpret_cast<unsigned long long *>(&sh.tile_w[t]),
                          (unsigned long long)w);
            if (ties) atomicAdd(&sh.tile_ties[t], ties);
        };
        if (m != NO_BIN) {
            for (uint32_t i = threadIdx.x; i < m; i += TPB)
                one(entry_class(sh.list[i]), key_logit(entry_key(sh.list[i])));
        } else {
            R.each([&](uint32_t c, float l) {
                if (l != -INFINITY && R.bin_of(l) == bin) one(c, l);
            });
        }
        __syncthreads();
    } else if (done) {
        __syncthreads();
    } else {
        sum_tiles([&](uint32_t, float l, uint64_t &w, uint32_t &t) { staying(l, w, t); });
    }

    if (threadIdx.x == 0) {
        uint64_t total = 0;
        uint32_t left = cut.ties;
        for (uint32_t t = 0; t < tiles; t++) {
            const uint32_t k = min(left, sh.tile_ties[t]);
            left -= k;
            total += sh.tile_w[t] + k * tie_w;
        }
        const uint64_t target = share(uniform31(D.uniforms[r]), total, 0);
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
    const uint32_t i0 = (sh.tile * TPB + threadIdx.x) * N, i1 = min(i0 + N, n);
    uint64_t w = 0;
    uint32_t ties = 0;
    for (uint32_t j = i0; j < i1; j++) staying(masked_nan((float)R.row[j]), w, ties);
    uint64_t cw = scan_wave(w);
    uint32_t ct = scan_wave(ties);
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
        for (uint32_t j = i0; j < i1; j++) {
            const float l = masked_nan((float)R.row[j]);
            uint64_t v = 0;
            uint32_t tie = 0;
            staying(l, v, tie);
            if (tie) v = seen++ < sh.ties ? tie_w : 0;
            before += v;
            if (before > sh.target) {
                put_class(D, r, j, R.S.z(l), sh.total);
                break;
            }
        }
    }
}

uint64_t sample_bytes(uint64_t n_rows, uint32_t n_classes) {
    return sample_tiled_rows(n_rows, n_classes) * sizeof(TileWork);
}

// One launch's rows; work is NULL where the call has no workspace.
template <class T>
void launch_sample(const void *logits, const Draw &D, TileWork *work, hipStream_t s) {
    const uint32_t v = D.n_classes;
    const auto *l = static_cast<const T *>(logits);
    const uint64_t n = D.n_rows;
    if (v <= THREAD_MOST) {
        const dim3 grid((uint32_t)((n + 255) / 256)), tpb(256);
        if (v == 1) hipLaunchKernelGGL((sample_thread_kernel<T, 1>), grid, tpb, 0, s, l, D);
        else if (v == 2) hipLaunchKernelGGL((sample_thread_kernel<T, 2>), grid, tpb, 0, s, l, D);
        else if (v == 3) hipLaunchKernelGGL((sample_thread_kernel<T, 3>), grid, tpb, 0, s, l, D);
        else if (v == 4) hipLaunchKernelGGL((sample_thread_kernel<T, 4>), grid, tpb, 0, s, l, D);
        else if (v == 5) hipLaunchKernelGGL((sample_thread_kernel<T, 5>), grid, tpb, 0, s, l, D);
        else if (v == 6) hipLaunchKernelGGL((sample_thread_kernel<T, 6>), grid, tpb, 0, s, l, D);
        else if (v == 7) hipLaunchKernelGGL((sample_thread_kernel<T, 7>), grid, tpb, 0, s, l, D);
        else hipLaunchKernelGGL((sample_thread_kernel<T, 8>), grid, tpb, 0, s, l, D);
    } else if (v <= GROUP_MOST) {
        const uint32_t g = v <= 16 ? 16 : v <= 32 ? 32 : 64;
        const uint64_t blocks = (n + GROUP_TPB / g - 1) / (GROUP_TPB / g);
        const dim3 grid((uint32_t)blocks), tpb(GROUP_TPB);
        if (g == 16) hipLaunchKernelGGL((sample_group_kernel<T, 16>), grid, tpb, 0, s, l, D);
        else if (g == 32) hipLaunchKernelGGL((sample_group_kernel<T, 32>), grid, tpb, 0, s, l, D);
        else hipLaunchKernelGGL((sample_group_kernel<T, 64>), grid, tpb, 0, s, l, D);
    } else if (v <= WAVE_MOST) {
        const dim3 grid((uint32_t)((n + 3) / 4)), tpb(256);
        if (v <= 128) hipLaunchKernelGGL((sample_wave_kernel<T, 2>), grid, tpb, 0, s, l, D);
        else if (v <= 256) hipLaunchKernelGGL((sample_wave_kernel<T, 4>), grid, tpb, 0, s, l, D);
        else if (v <= 512) hipLaunchKernelGGL((sample_wave_kernel<T, 8>), grid, tpb, 0, s, l, D);
        else hipLaunchKernelGGL((sample_wave_kernel<T, 16>), grid, tpb, 0, s, l, D);
    } else {
        const dim3 grid((uint32_t)n);
        if (v <= SAMPLE_TILE_CLASSES)
            hipLaunchKernelGGL((sample_row_kernel<T, 256, false>), grid, dim3(256), 0, s, l, D,
                               nullptr);
        else if (!work || (!D.own && D.all.k < v))
            hipLaunchKernelGGL((sample_row_kernel<T, 1024, false>), grid, dim3(1024), 0, s, l, D,
                               nullptr);
        else {
            constexpr uint32_t cells = TILE_TPB * 16 / sizeof(T);
            const dim3 tiles((v + cells - 1) / cells, (uint32_t)n);
            hipLaunchKernelGGL((tile_most_kernel<T>), tiles, dim3(TILE_TPB), 0, s, l, D, work);
            if (D.own || D.all.p31 < 1u << 31)
                hipLaunchKernelGGL((tile_weights_kernel<T>), tiles, dim3(TILE_TPB), 0, s, l, D,
                                   work);
            hipLaunchKernelGGL((tile_sums_kernel<T>), tiles, dim3(TILE_TPB), 0, s, l, D, work);
            hipLaunchKernelGGL((sample_row_kernel<T, 1024, true>), grid, dim3(1024), 0, s, l, D,
                               work);
        }
    }
    head_check(hipGetLastError(), "sampling");
}

void sample(const void *logits, uint32_t dtype, const Draw &D, void *work, hipStream_t s) {
    const uint64_t row_bytes = (uint64_t)D.n_classes * (dtype == FBH_F32 ? 4 : 2);
    sample_launches(D.n_rows, D.n_classes, [&](uint64_t r, uint64_t rows, bool tiled) {
        Draw d = D;
        d.n_rows = rows;
        d.uniforms += r;
        d.classes += r;
        if (d.log_probs) d.log_probs += r;
        if (d.o.temperatures) d.o.temperatures += r;
        if (d.o.top_ks) d.o.top_ks += r;
        if (d.o.top_ps) d.o.top_ps += r;
        if (d.o.min_ps) d.o.min_ps += r;
        const auto *from = static_cast<const uint8_t *>(logits) + r * row_bytes;
        auto *w = tiled ? static_cast<TileWork *>(work) : nullptr;
        if (dtype == FBH_F32) launch_sample<float>(from, d, w, s);
        else if (dtype == FBH_F16) launch_sample<_Float16>(from, d, w, s);
        else launch_sample<__bf16>(from, d, w, s);
    });
}

Draw draw_of(const float *uniforms, const fbh_sample_options *o, int64_t *classes,
             float *log_probs, uint64_t n_rows, uint32_t n_classes) {
    return {uniforms, *o, whole_options(o->temperature, o->top_k, o->top_p, o->min_p, n_classes),
            o->temperatures || o->top_ks || o->top_ps || o->min_ps, classes, log_probs, n_rows,
            n_classes};
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

uint64_t fbh_sample_bytes(uint64_t n_rows, uint32_t n_classes) {
    return sample_bytes(n_rows, n_classes);
}

int fbh_sample_classes(int device, const void *logits, uint64_t n_rows, uint32_t n_classes,
                       uint32_t dtype, const float *uniforms, const fbh_sample_options *options,
                       int64_t *classes, float *log_probs, void *work, uint64_t work_bytes,
                       void *stream) {
    return head_guard([&] {
        check_sample(logits, n_rows, n_classes, uniforms, options, classes);
        head_input(dtype <= FBH_BF16, "unknown cell type");
        if (n_rows == 0) return;
        const uint64_t need = sample_bytes(n_rows, n_classes);
        head_input(work_bytes >= need && (work || need == 0), "the workspace is too small");
        head_input(need == 0 || reinterpret_cast<uintptr_t>(work) % 8 == 0,
                   "the workspace is not aligned to 8 bytes");
        const OnDevice on(device);
        sample(logits, dtype,
               draw_of(uniforms, options, classes, log_probs, n_rows, n_classes), work,
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
        const uint64_t c_bytes = (8 * n_rows + 255) & ~255ull;
        head_check(keep_alloc(KeepKind::device, reinterpret_cast<void **>(&block),
                              l_bytes + 2 * u_bytes + c_bytes +
                                  sample_bytes(n_rows, n_classes)),
                   "device allocation");
        auto *d_u = reinterpret_cast<float *>(block + l_bytes);
        auto *d_p = reinterpret_cast<float *>(block + l_bytes + u_bytes);
        auto *d_c = reinterpret_cast<int64_t *>(block + l_bytes + 2 * u_bytes);
        head_check(hipMemcpyAsync(block, logits, 4 * n_rows * n_classes, hipMemcpyHostToDevice, s),
                   "logit upload");
        head_check(hipMemcpyAsync(d_u, uniforms, 4 * n_rows, hipMemcpyHostToDevice, s),
                   "uniform upload");
        sample(block, FBH_F32, draw_of(d_u, options, d_c, d_p, n_rows, n_classes),
               block + l_bytes + 2 * u_bytes + c_bytes, s);
        head_check(hipMemcpyAsync(classes, d_c, 8 * n_rows, hipMemcpyDeviceToHost, s),
                   "class download");
        if (log_probs)
            head_check(hipMemcpyAsync(log_probs, d_p, 4 * n_rows, hipMemcpyDeviceToHost, s),
                       "probability download");
        head_check(hipStreamSynchronize(s), "sampling");
    });
}

}  // extern "C"
