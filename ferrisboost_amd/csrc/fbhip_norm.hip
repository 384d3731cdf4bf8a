// Layer norm: y = (x - mean) * r * w + b over the cells of a row, r = 1 / sqrt(variance + eps),
// and its gradients. With h = (x - mean) * r and d = g * w for the output's gradient g:
//   dx = r * (d - mean(d) - h * mean(d * h)),  dw = sum over rows of g * h,  db = sum of g.
//
// A row is held in registers by G lanes of C cells each, so that every cell is read once, and
// the next one is on its way meanwhile: bound by memory (bfloat16, against 4.84 TB/s of a large
// copy: forward 32768 x 4096 in 102 us, 5.3 TB/s, 1M x 60 in 47, 4096 x 30000 in 109; gradients
// of 32768 x 4096 in 154 us and 5 for the parts of the weights' sums, 5.2 TB/s, 100k x 64 in 11
// and 4). Loads that were widened as they came, and cells read one by one at a row's end, had
// the gradient of 32768 x 4096 wait for each row: 258 us.
//
// A row's sums are taken in f32 in a tree whose shape depends on the width alone; the variance
// is the mean square of differences from the mean, and what the mean's rounding leaves in them
// (their own sum) is taken out: rows far from 0 keep their cells' accuracy.
#include "fbhip_heads.h"

#include <algorithm>

namespace fbh {
namespace {

constexpr uint32_t NORM_MAX_DIM = 32768;

struct Norm {
    const void *weight, *bias;
    uint64_t n_rows;
    uint32_t dim, weight_type;
    float eps;
};

// Sums of K values over G lanes that follow one another (a power of two), in every one of
// them. More than a wave: through LDS, where `buffer` alternates so that no wave writes what
// another still reads.
template <uint32_t G, uint32_t K>
struct GroupSum {
    static constexpr uint32_t WAVES = G > 64 ? G / 64 : 1;
    float part[2][WAVES][K];
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}

template <int V>
struct Int {
    static constexpr int value = V;
};

// The sum over groups of G <= 64 lanes, in every lane: neighbours, pairs, then mirrored quads
// and eights (their lanes all hold the same by then), rows of 16 and halves exchanged.
template <uint32_t G>
__device__ __forceinline__ float sum_of_lanes(float v) {
    if (G >= 2) v = dpp_add<0xB1>(v);
    if (G >= 4) v = dpp_add<0x4E>(v);
    if (G >= 8) v = dpp_add<0x141>(v);
    if (G >= 16) v = dpp_add<0x140>(v);
    if (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                        false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                        false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

template <uint32_t G, uint32_t K>
__device__ __forceinline__ void sum_of_group(float (&v)[K], GroupSum<G, K> &lds, uint32_t buffer) {
#pragma unroll
    for (uint32_t k = 0; k < K; k++) v[k] = sum_of_lanes<(G < 64 ? G : 64)>(v[k]);
    if constexpr (G > 64) {
        constexpr uint32_t W = G / 64;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (uint32_t k = 0; k < K; k++) lds.part[buffer][threadIdx.x / 64][k] = v[k];
        __syncthreads();
        // each lane takes one wave's sum, and the lanes of a group of W add them
#pragma unroll
        for (uint32_t k = 0; k < K; k++)
            v[k] = sum_of_lanes<W>(lds.part[buffer][threadIdx.x % W][k]);
    }
}

// A lane's cells: pieces of N that lie G * N cells apart. A row's last piece starts at dim - N
// wherever its lane's place is, so that every piece is whole: the `twice` first cells of it
// are the lane's before it too, take no part in sums, and are stored by both with the same
// value. Pieces behind the row are empty. (Rows of fewer cells than a piece have N = 1.)
template <uint32_t N_, uint32_t G, uint32_t C>
struct Place {
    static constexpr uint32_t N = N_, P = C / N_;
    uint32_t dim;
    __device__ __forceinline__ uint32_t begin(uint32_t p) const {
        return (p * G + threadIdx.x % G) * N;
    }
    __device__ __forceinline__ bool empty(uint32_t p) const { return begin(p) >= dim; }
    __device__ __forceinline__ uint32_t column(uint32_t p) const {
        return min(begin(p), dim - N);
    }
    __device__ __forceinline__ uint32_t twice(uint32_t p) const { return begin(p) - column(p); }
    // Whether the lane has cells that take no part.
    __device__ __forceinline__ bool ragged() const {
        bool r = false;
#pragma unroll
        for (uint32_t p = 0; p < P; p++) r |= begin(p) + N > dim;
        return r;
    }
    // (of lanes with such cells)
    __device__ __forceinline__ bool counts(uint32_t i) const {
        return !empty(i / N) && i % N >= twice(i / N);
    }
};

// Cells as they lie in memory, in words, so that a load is waited for where they are taken.
template <class T, class L>
struct Raw {
    static constexpr uint32_t BYTES = L::N * sizeof(T), WORDS = (BYTES + 3) / 4;
    uint32_t w[L::P][WORDS];

    __device__ __forceinline__ void load(const T *row, L at) {
#pragma unroll
        for (uint32_t p = 0; p < L::P; p++)
            if (!at.empty(p)) __builtin_memcpy(w[p], row + at.column(p), BYTES);
    }
    __device__ __forceinline__ float cell(uint32_t i) const {
        T t;
        __builtin_memcpy(&t, reinterpret_cast<const char *>(w[i / L::N]) + i % L::N * sizeof(T),
                         sizeof(T));
        return (float)t;
    }
};

template <class L, uint32_t C>
struct Cells {
    float v[C];

    template <class T>
    __device__ __forceinline__ void take(const Raw<T, L> &r) {
#pragma unroll
        for (uint32_t i = 0; i < C; i++) v[i] = r.cell(i);
    }
    __device__ __forceinline__ void load_typed(const void *p, uint32_t type, L at) {
        const auto load = [&](auto t) {
            Raw<decltype(t), L> r = {};
            r.load(static_cast<const decltype(t) *>(p), at);
            take(r);
        };
        if (type == FBH_F32) load(float{});
        else if (type == FBH_F16) load(_Float16{});
        else load(__bf16{});
    }
    __device__ __forceinline__ void fill(float f) {
#pragma unroll
        for (uint32_t i = 0; i < C; i++) v[i] = f;
    }
};

// f(cell) of the lane's cells to a row.
template <class T, class L, class F>
__device__ __forceinline__ void store_cells(T *row, L at, F &&f) {
#pragma unroll
    for (uint32_t p = 0; p < L::P; p++)
        if (!at.empty(p)) {
            Piece<T, L::N> q;
#pragma unroll
            for (uint32_t i = 0; i < L::N; i++) q.v[i] = (T)f(p * L::N + i);
            store_piece<T, L::N>(row + at.column(p), q);
        }
}

// Sums of f(cell) over the lane's cells that take part; with care in those few lanes that have
// others.
template <uint32_t K, uint32_t C, class L, class F>
__device__ __forceinline__ void sum_cells(float (&s)[K], L at, bool ragged, F &&f) {
#pragma unroll
    for (uint32_t k = 0; k < K; k++) s[k] = 0.0f;
    if (!ragged) {
#pragma unroll
        for (uint32_t i = 0; i < C; i++) f(i, s);
    } else {
        asm volatile("" : "+s"(at.dim));  // (what is asked of it here is not kept in registers)
#pragma unroll
        for (uint32_t i = 0; i < C; i++)
            if (at.counts(i)) f(i, s);
    }
}

template <uint32_t G>
constexpr uint32_t norm_threads() {
    return G > 256 ? G : 256;
}

template <class T, uint32_t N, uint32_t G, uint32_t C>
__global__ __launch_bounds__(norm_threads<G>()) void norm_kernel(Norm A, const T *x, T *out,
                                                                 float *stats) {
    using L = Place<N, G, C>;
    constexpr uint32_t ROWS = norm_threads<G>() / G;
    __shared__ GroupSum<G, 1> first;
    __shared__ GroupSum<G, 2> second;
    const L at{A.dim};
    const bool ragged = at.ragged();
    const float inv_n = 1.0f / (float)A.dim;
    const uint64_t step = (uint64_t)gridDim.x * ROWS;
    uint64_t r = (uint64_t)blockIdx.x * ROWS, row = r + threadIdx.x / G;
    // the next row's cells are on their way while this one's are worked on, where there are
    // registers for both
    constexpr bool AHEAD = C * (2 * sizeof(T) + 8) / 4 <= 208;
    Raw<T, L> next = {};
    if (AHEAD && row < A.n_rows) next.load(x + row * A.dim, at);
    Cells<L, C> w, b;
    w.fill(1.0f);
    b.fill(0.0f);
    if (A.weight) w.load_typed(A.weight, A.weight_type, at);
    if (A.bias) b.load_typed(A.bias, A.weight_type, at);
    for (uint32_t turn = 0; r < A.n_rows; r += step, row += step, turn ^= 1) {
        Raw<T, L> c = {};  // (widened where it is used: half the registers)
        if constexpr (AHEAD) {
            c = next;
            if (row + step < A.n_rows) next.load(x + (row + step) * A.dim, at);
        } else {
            if (row < A.n_rows) c.load(x + row * A.dim, at);
        }
        float s1[1], s2[2];
        sum_cells<1, C>(s1, at, ragged, [&](uint32_t i, float (&s)[1]) { s[0] += c.cell(i); });
        sum_of_group<G, 1>(s1, first, turn);
        const float mean = s1[0] * inv_n;
        sum_cells<2, C>(s2, at, ragged, [&](uint32_t i, float (&s)[2]) {
            const float d = c.cell(i) - mean;
            s[0] += d;
            s[1] = fmaf(d, d, s[1]);
        });
        sum_of_group<G, 2>(s2, second, turn);
        const float rest = s2[0] * inv_n;
        // (of equal cells, by rounding, the variance may be below 0; NaN stays)
        const float var = s2[1] * inv_n - rest * rest;
        const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + A.eps);
        if (row >= A.n_rows) continue;  // (all of a group's lanes, and with G > 64 never)
        store_cells(out + row * A.dim, at, [&](uint32_t i) {
            return fmaf((c.cell(i) - mean - rest) * rstd, w.v[i], b.v[i]);
        });
        if (stats && threadIdx.x % G == 0) {
            stats[2 * row] = mean + rest;
            stats[2 * row + 1] = rstd;
        }
    }
}

// f(cells of a piece, lanes of a row, cells of a lane) by the row's cells: few lanes, so that all
// of them have cells (1M rows of 60 bfloat16 in 16 lanes 68 us, in 8 41 to 47), but no more than
// 16 cells of a lane while rows still fit the device's workgroups, as sums over more cells cost
// their registers: waves or, from 512 lanes on, the next row on its way (gradients of 8192 x
// 16384 bfloat16: 512 lanes of 32 cells 170 us, 1024 of 16, with half the registers each, 208).
template <class T, class F>
void with_shape(uint32_t dim, F &&f) {
    constexpr uint32_t N = 16 / sizeof(T);
    if (dim < N) return f(Int<1>{}, Int<4>{}, Int<2>{});
    const Int<N> n;
    if (dim <= 4 * 8) f(n, Int<4>{}, Int<8>{});
    else if (dim <= 8 * 8) f(n, Int<8>{}, Int<8>{});
    else if (dim <= 16 * 8) f(n, Int<16>{}, Int<8>{});
    else if (dim <= 16 * 16) f(n, Int<16>{}, Int<16>{});
    else if (dim <= 64 * 8) f(n, Int<64>{}, Int<8>{});
    else if (dim <= 64 * 16) f(n, Int<64>{}, Int<16>{});
    else if (dim <= 256 * 8) f(n, Int<256>{}, Int<8>{});
    else if (dim <= 256 * 16) f(n, Int<256>{}, Int<16>{});
    else if (dim <= 512 * 16) f(n, Int<512>{}, Int<16>{});
    else if (dim <= 512 * 32) f(n, Int<512>{}, Int<32>{});
    else f(n, Int<512>{}, Int<64>{});
}
template <class F>
void with_type(uint32_t dtype, F &&f) {
    if (dtype == FBH_F32) f(float{});
    else if (dtype == FBH_F16) f(_Float16{});
    else f(__bf16{});
}

// ------------------------------------------------------------------- gradient
// Workgroups go through rows in turn and hold their sums of dw and db in registers; each
// writes its part, and the parts are added in order.
constexpr uint32_t SPLIT_DIM = 16384;  // wider rows' sums have no room in registers
// Rows that are added up in f32, one after the other: of more the parts' sums are taken in
// several batches of rows (65024 of 32768 cells, say), so that what rounding leaves has a bound.
// (With 256 a launch's end comes often enough to be seen: 20,000 x 20,000 in 780 us, in one batch
// 761; 2^25 x 8 in 676 and 650.)
constexpr uint64_t CHAIN = 1024;

struct NormGrad {
    uint64_t n_rows;
    uint32_t dim, weight_type, groups;
    const void *weight;
    const float *stats;
    float *parts;  // [groups][2][dim], or for wide rows [n_rows]: what the mean leaves out
    void *dweight, *dbias;  // of the only workgroup, which needs no parts
};

// Cell `at` of a weight's or bias' gradient, where one is wanted.
__device__ __forceinline__ void store_weight(void *out, uint32_t type, uint32_t at, float v) {
    if (!out) return;
    if (type == FBH_F32) static_cast<float *>(out)[at] = v;
    else if (type == FBH_F16) static_cast<_Float16 *>(out)[at] = (_Float16)v;
    else static_cast<__bf16 *>(out)[at] = (__bf16)v;
}

template <class T, uint32_t N, uint32_t G, uint32_t C, bool SUMS>
__global__ __launch_bounds__(norm_threads<G>()) void norm_grad_kernel(NormGrad A, const T *g,
                                                                      const T *x, T *dx) {
    using L = Place<N, G, C>;
    constexpr uint32_t ROWS = norm_threads<G>() / G;
    constexpr bool AHEAD = C * (4 * sizeof(T) + (SUMS ? 12 : 4)) / 4 <= 208;
    __shared__ GroupSum<G, 3> lds;
    const L at{A.dim};
    const bool ragged = at.ragged();
    const float inv_n = 1.0f / (float)A.dim;
    const uint64_t step = (uint64_t)gridDim.x * ROWS;
    uint64_t r = (uint64_t)blockIdx.x * ROWS, row = r + threadIdx.x / G;
    Raw<T, L> next_x = {}, next_g = {};
    float next_mean = 0.0f, next_rstd = 0.0f;
    const auto load = [&](uint64_t row, Raw<T, L> &c, Raw<T, L> &d, float &mean, float &rstd) {
        if (row < A.n_rows) {
            c.load(x + row * A.dim, at);
            d.load(g + row * A.dim, at);
            mean = A.stats[2 * row];
            rstd = A.stats[2 * row + 1];
        }
    };
    if (AHEAD) load(row, next_x, next_g, next_mean, next_rstd);
    Cells<L, C> w, dw, db;
    w.fill(1.0f);
    if (A.weight) w.load_typed(A.weight, A.weight_type, at);
    if (SUMS) {
        dw.fill(0.0f);
        db.fill(0.0f);
    }
    for (uint32_t turn = 0; r < A.n_rows; r += step, row += step, turn ^= 1) {
        Raw<T, L> c = {}, d = {};  // (widened where they are used)
        float mean = 0.0f, rstd = 0.0f;
        if constexpr (AHEAD) {
            c = next_x;
            d = next_g;
            mean = next_mean;
            rstd = next_rstd;
            load(row + step, next_x, next_g, next_mean, next_rstd);
        } else {
            load(row, c, d, mean, rstd);
        }
        float s[3];
        sum_cells<3, C>(s, at, ragged, [&](uint32_t i, float (&s)[3]) {
            const float e = d.cell(i) * w.v[i], f = c.cell(i) - mean;
            s[0] += f;
            s[1] += e;
            s[2] = fmaf(e, f, s[2]);
        });
        sum_of_group<G, 3>(s, lds, turn);
        if (row >= A.n_rows) continue;  // (all of a group's lanes, and with G > 64 never)
        const float rest = s[0] * inv_n, a = s[1] * inv_n;
        const float b = (s[2] * inv_n - a * rest) * rstd;  // mean(d * h)
        if (!SUMS && A.parts && threadIdx.x % G == 0) A.parts[row] = rest;
        if (SUMS)
#pragma unroll
            for (uint32_t i = 0; i < C; i++) {
                const float h = (c.cell(i) - mean - rest) * rstd;
                dw.v[i] = fmaf(d.cell(i), h, dw.v[i]);
                db.v[i] += d.cell(i);
            }
        if (dx)
            store_cells(dx + row * A.dim, at, [&](uint32_t i) {
                const float h = (c.cell(i) - mean - rest) * rstd;
                return fmaf(-h, b, d.cell(i) * w.v[i] - a) * rstd;
            });
    }
    if constexpr (SUMS) {
        if (!A.parts && !A.dweight && !A.dbias) return;
        const auto put = [&](uint32_t which, uint32_t col, float v) {
            if (A.parts) A.parts[((uint64_t)blockIdx.x * 2 + which) * A.dim + col] = v;
            else store_weight(which ? A.dbias : A.dweight, A.weight_type, col, v);
        };
        if constexpr (ROWS == 1) {
#pragma unroll
            for (uint32_t i = 0; i < C; i++)
                if (!at.empty(i / N)) {
                    put(0, at.column(i / N) + i % N, dw.v[i]);
                    put(1, at.column(i / N) + i % N, db.v[i]);
                }
        } else {
            // the workgroup's rows, added in their order, a quarter of the cells at a time
            constexpr uint32_t Q = C > 4 ? C / 4 : 1;
            __shared__ float sums[2][ROWS][G * Q];
#pragma unroll
            for (uint32_t q = 0; q < C / Q; q++) {
                __syncthreads();
#pragma unroll
                for (uint32_t k = 0; k < Q; k++) {
                    sums[0][threadIdx.x / G][k * G + threadIdx.x % G] = dw.v[q * Q + k];
                    sums[1][threadIdx.x / G][k * G + threadIdx.x % G] = db.v[q * Q + k];
                }
                __syncthreads();
                for (uint32_t j = threadIdx.x; j < 2 * G * Q; j += norm_threads<G>()) {
                    const uint32_t slot = j % (G * Q), which = j / (G * Q);
                    float p[4] = {};  // (in doubles: 100k x 64 in 12.3 us, so in 11.6)
#pragma unroll
                    for (uint32_t k = 0; k < ROWS; k++) p[k % 4] += sums[which][k][slot];
                    const float t = (p[0] + p[1]) + (p[2] + p[3]);
                    const uint32_t i = q * Q + slot / G;
                    const uint32_t begin = ((i / N) * G + slot % G) * N;
                    if (begin < A.dim) put(which, min(begin, A.dim - N) + i % N, t);
                }
            }
        }
    }
}

// dw and db of rows of more than 16384 cells, from the rows once more: four columns a thread,
// four rows at a time, the rows cut into `groups` equal parts. A thread's columns start at
// dim - 4 at the latest.
template <class T>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormGrad A, const T *g, const T *x,
                                                           const float *rests, float *parts) {
    const uint32_t begin = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (begin >= A.dim) return;
    const uint32_t col = min(begin, A.dim - 4);
    const uint64_t each = (A.n_rows + A.groups - 1) / A.groups;
    const uint64_t first = blockIdx.y * each, end = min(first + each, A.n_rows);
    float dw[4] = {}, db[4] = {};
    const auto add = [&](const Piece<T, 4> &gp, const Piece<T, 4> &xp, uint64_t r) {
        const float mean = A.stats[2 * r], rstd = A.stats[2 * r + 1], rest = rests[r];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float d = (float)gp.v[i];
            dw[i] = fmaf(d, ((float)xp.v[i] - mean - rest) * rstd, dw[i]);
            db[i] += d;
        }
    };
    uint64_t r = first;
    for (; r + 4 <= end; r += 4) {
        Piece<T, 4> gp[4], xp[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            gp[k] = load_piece<T, 4>(g + (r + k) * A.dim + col);
            xp[k] = load_piece<T, 4>(x + (r + k) * A.dim + col);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) add(gp[k], xp[k], r + k);
    }
    for (; r < end; r++)
        add(load_piece<T, 4>(g + r * A.dim + col), load_piece<T, 4>(x + r * A.dim + col), r);
    float *out = parts + (uint64_t)blockIdx.y * 2 * A.dim;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        out[col + i] = dw[i];
        out[A.dim + col + i] = db[i];
    }
}

// The parts' sums, in doubles, and those of the batches before (`batches`, where there are
// several): COLUMNS columns a workgroup, 256 / COLUMNS threads a column, each
// of which takes a part in as many; their sums are then added in order. Few columns need many
// threads each (64 cells and 1024 parts: 4.0 us, 8 columns a workgroup), many whole cache lines
// (16384 cells and 512 parts, 67 MB: 41.7 us with 8 columns).
template <uint32_t COLUMNS>
__global__ __launch_bounds__(256) void norm_join_kernel(const float *parts, uint32_t dim,
                                                        uint32_t groups, uint32_t weight_type,
                                                        void *dweight, void *dbias,
                                                        double *batches, bool first, bool last) {
    constexpr uint32_t THREADS = 256 / COLUMNS;
    __shared__ double sums[THREADS][COLUMNS + 1];
    const uint32_t lane = threadIdx.x % COLUMNS, k = threadIdx.x / COLUMNS;
    const uint32_t j = blockIdx.x * COLUMNS + lane;  // of 2 * dim
    double t = 0.0;
    if (j < 2 * dim) {
        uint32_t p = k;
        for (; p + 7 * THREADS < groups; p += 8 * THREADS) {
            float v[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)
                v[i] = parts[(uint64_t)(p + i * THREADS) * 2 * dim + j];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) t += (double)v[i];
        }
        for (; p < groups; p += THREADS) t += (double)parts[(uint64_t)p * 2 * dim + j];
    }
    sums[k][lane] = t;
    __syncthreads();
    if (k != 0 || j >= 2 * dim) return;
    for (uint32_t i = 1; i < THREADS; i++) t += sums[i][lane];
    if (!first) t += batches[j];
    if (!last) batches[j] = t;
    else if (j < dim) store_weight(dweight, weight_type, j, (float)t);
    else store_weight(dbias, weight_type, j - dim, (float)t);
}

// ------------------------------------------------------------------- host side
uint32_t rows_of_group(uint32_t dim) {
    uint32_t rows = 1;
    with_shape<float>(dim, [&](auto, auto g, auto) {
        constexpr uint32_t G = decltype(g)::value;
        rows = norm_threads<G>() / G;
    });
    return rows;
}

// Whether one workgroup takes all rows, twice as many as it holds at once, and writes the
// weights' gradients itself, without a second launch (in us on the device, and with: 64 x 60
// 5.0 and 5.9, 128 x 60 6.5 and 5.8; 8 x 1000 6.8 and 6.7, 16 x 1000 9.6 and 6.7; 2 x 4000 7.9
// and 8.6, 4 x 4000 10.8 and 8.5; a launch less is 5 us less of the host's).
bool grad_alone(uint64_t n_rows, uint32_t dim) {
    return dim <= 4096 && n_rows <= 2 * rows_of_group(dim);
}

// Parts of the weights' sums, a workgroup's each: as many workgroups as the device holds at a
// time, fewer where their parts would be large beside the rows (in us, bfloat16 gradients of
// 4096 cells: 512 rows with 512 parts 24.2, with 128 14.4; 2048 rows with 512 parts 25.9, with
// 256 21.8), and 128 while there are rows for them (128 rows: 10.2, with 32 parts 12.7).
uint32_t grad_groups(uint64_t n_rows, uint32_t dim) {
    if (grad_alone(n_rows, dim)) return 1;
    const uint64_t most = dim <= 256 ? 1024 : dim <= 4096 ? 512 : dim <= SPLIT_DIM ? 256 : 64;
    const uint32_t rows = rows_of_group(dim);
    const uint64_t n = std::max<uint64_t>((n_rows + rows - 1) / rows, 1);
    return (uint32_t)std::min({n, most, std::max<uint64_t>(n / (rows == 1 ? 8 : 4), 128)});
}

// How the rows are cut for the weights' sums: one batch, or several, whose sums in doubles take
// the place of two parts.
struct Batches {
    uint32_t groups;
    uint64_t rows;  // of a batch

    Batches(uint64_t n_rows, uint32_t dim) : groups(grad_groups(n_rows, dim)), rows(n_rows) {
        const uint64_t turn = rows_of_group(dim) * CHAIN;
        if (n_rows <= groups * turn) return;
        groups -= 2;  // (of 64 and more)
        const uint64_t n = (n_rows + groups * turn - 1) / (groups * turn);
        rows = (n_rows + n - 1) / n;
    }
};

uint64_t padded_rows(uint64_t n) { return (n + 3) / 4 * 4; }

uint64_t grad_bytes(const fbh_norm *a) {
    if (grad_alone(a->n_rows, a->dim)) return 0;
    uint64_t b = (uint64_t)grad_groups(a->n_rows, a->dim) * 2 * a->dim * 4;
    if (a->dim > SPLIT_DIM) b += padded_rows(a->n_rows) * 4;
    return b;
}

// Workgroups of a launch at most: they go through the rows in turn, and the more of them there
// are the more often the weights are read (4096 x 30000 bfloat16: 109 us with 256, 155 with
// 4096), but small rows' latencies overlap better (1M x 60: 114 and 47).
uint64_t norm_blocks(uint32_t dim) { return dim <= 8192 ? 4096 : dim <= SPLIT_DIM ? 1024 : 256; }

void check_norm(const fbh_norm *a) {
    head_input(a, "null argument");
    head_input(a->dtype <= FBH_BF16, "unknown cell type");
    head_input(a->weight_type <= FBH_BF16, "unknown weight type");
    head_input(a->dim >= 1 && a->dim <= NORM_MAX_DIM, "dim must be in 1..=32768");
    head_input(a->n_rows <= (1ull << 40) / a->dim, "more than 2^40 cells");
    head_input(a->eps >= 1.17549435e-38f && a->eps <= 3.4028235e38f,
               "eps must be a positive normal float");
}

// Bytes of the rows, of their statistics and of a weight.
uint64_t cell_bytes(uint32_t type) { return type == FBH_F32 ? 4 : 2; }
uint64_t row_bytes(const fbh_norm *a) { return a->n_rows * a->dim * cell_bytes(a->dtype); }
uint64_t stats_bytes(const fbh_norm *a) { return a->n_rows * 8; }
uint64_t weight_bytes(const fbh_norm *a) { return a->dim * cell_bytes(a->weight_type); }

template <class K, class... A>
void launch(K kernel, uint64_t blocks, uint32_t threads, hipStream_t s, A... args) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(threads), 0, s, args...);
    head_check(hipGetLastError(), "layer norm");
}

template <class T>
void launch_norm(const fbh_norm *a, const void *x, const void *weight, const void *bias, void *out,
                 float *stats, hipStream_t s) {
    const Norm A{weight, bias, a->n_rows, a->dim, a->weight_type, a->eps};
    with_shape<T>(a->dim, [&](auto n, auto g, auto c) {
        constexpr uint32_t N = decltype(n)::value, G = decltype(g)::value, C = decltype(c)::value;
        constexpr uint32_t ROWS = norm_threads<G>() / G;
        const uint64_t blocks = (a->n_rows + ROWS - 1) / ROWS;
        launch(norm_kernel<T, N, G, C>, std::min(blocks, norm_blocks(a->dim)), norm_threads<G>(),
               s, A, static_cast<const T *>(x), static_cast<T *>(out), stats);
    });
}

template <class T>
void launch_norm_grad(const fbh_norm *a, const T *g, const T *x, const float *stats,
                      const void *weight, T *dx, void *dweight, void *dbias, float *work,
                      hipStream_t s) {
    const bool sums = dweight || dbias, split = a->dim > SPLIT_DIM;
    const bool alone = grad_alone(a->n_rows, a->dim);
    const Batches cut(a->n_rows, a->dim);
    const bool several = sums && cut.rows < a->n_rows;
    double *batches = nullptr;
    float *parts = work;
    if (split && sums) parts += padded_rows(a->n_rows);
    if (several) {
        batches = reinterpret_cast<double *>(parts);
        parts += 4 * a->dim;
    }
    NormGrad A{a->n_rows, a->dim, a->weight_type, cut.groups, weight, stats, nullptr,
               alone ? dweight : nullptr, alone ? dbias : nullptr};
    const auto rows = [&](uint64_t first) {
        with_shape<T>(a->dim, [&](auto nn, auto gg, auto cc) {
            constexpr uint32_t N = decltype(nn)::value, G = decltype(gg)::value;
            constexpr uint32_t C = decltype(cc)::value;
            constexpr bool SUMS = G * C <= SPLIT_DIM;
            const uint64_t most = norm_blocks(a->dim);
            const uint64_t blocks = SUMS ? cut.groups : std::clamp<uint64_t>(A.n_rows, 1, most);
            launch(norm_grad_kernel<T, N, G, C, SUMS>, blocks, norm_threads<G>(), s, A,
                   g + first * a->dim, x + first * a->dim, dx ? dx + first * a->dim : dx);
        });
    };
    if (split || !sums) {
        A.parts = split && sums ? work : nullptr;
        rows(0);
    }
    if (!sums) return;
    uint64_t first = 0;
    do {
        A.n_rows = std::min(cut.rows, a->n_rows - first);
        A.stats = stats + 2 * first;
        if (split) {
            hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((a->dim + 1023) / 1024, cut.groups),
                               dim3(256), 0, s, A, g + first * a->dim, x + first * a->dim,
                               work + first, parts);
            head_check(hipGetLastError(), "layer norm");
        } else {
            A.parts = alone ? nullptr : parts;
            rows(first);
            if (alone) return;
        }
        const uint64_t end = first + A.n_rows;
        const uint32_t columns = a->dim <= 512 ? 8 : 32;
        launch(columns == 8 ? norm_join_kernel<8> : norm_join_kernel<32>,
               (2 * a->dim + columns - 1) / columns, 256, s, parts, a->dim, cut.groups,
               a->weight_type, dweight, dbias, batches, first == 0, end == a->n_rows);
        first = end;
    } while (first < a->n_rows);
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" {

int fbh_layer_norm(int device, const fbh_norm *a, const void *x, const void *weight,
                   const void *bias, void *out, float *stats, void *stream) {
    return head_guard([&] {
        check_norm(a);
        head_input((x && out) || a->n_rows == 0, "null argument");
        if (a->n_rows == 0) return;
        const uint64_t rows = row_bytes(a), each = stats_bytes(a), cells = weight_bytes(a);
        head_input(out == x || !overlap(out, rows, x, rows), "out must be x or apart from it");
        head_input(!overlap(out, rows, weight, cells) && !overlap(out, rows, bias, cells),
                   "out must not overlap a weight");
        head_input(!overlap(stats, each, x, rows) && !overlap(stats, each, out, rows) &&
                       !overlap(stats, each, weight, cells) && !overlap(stats, each, bias, cells),
                   "stats must not overlap another tensor");
        const OnDevice on(device);
        const auto s = static_cast<hipStream_t>(stream);
        with_type(a->dtype, [&](auto t) {
            launch_norm<decltype(t)>(a, x, weight, bias, out, stats, s);
        });
    });
}

uint64_t fbh_layer_norm_grad_bytes(const fbh_norm *a) {
    uint64_t bytes = 0;
    (void)head_guard([&] {
        check_norm(a);
        bytes = grad_bytes(a);
    });
    return bytes;
}

int fbh_layer_norm_grad(int device, const fbh_norm *a, const void *grad, const void *x,
                        const float *stats, const void *weight, void *dx, void *dweight,
                        void *dbias, void *work, uint64_t work_bytes, void *stream) {
    return head_guard([&] {
        check_norm(a);
        head_input((grad && x && stats) || a->n_rows == 0, "null argument");
        if (dweight || dbias) {
            const uint64_t need = grad_bytes(a);
            head_input(need == 0 || (work && work_bytes >= need), "the workspace is too small");
            head_input(need == 0 || reinterpret_cast<uintptr_t>(work) % 16 == 0,
                       "the workspace must be 16-byte aligned");
        }
        const uint64_t rows = row_bytes(a);
        head_input(!overlap(dx, rows, grad, rows) && !overlap(dx, rows, x, rows),
                   "dx must not be grad or x, nor overlap them");
        head_input(!overlap(dx, rows, stats, stats_bytes(a)) &&
                       !overlap(dx, rows, weight, weight_bytes(a)),
                   "dx must not overlap stats or weight");
        if (!dx && !dweight && !dbias) return;
        const OnDevice on(device);
        const auto s = static_cast<hipStream_t>(stream);
        with_type(a->dtype, [&](auto t) {
            using T = decltype(t);
            launch_norm_grad<T>(a, static_cast<const T *>(grad), static_cast<const T *>(x), stats,
                                weight, static_cast<T *>(dx), dweight, dbias,
                                static_cast<float *>(work), s);
        });
    });
}

}  // extern "C"
