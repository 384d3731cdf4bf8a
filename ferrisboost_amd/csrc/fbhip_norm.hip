// Layer norm: y = (x - mean) * r * w + b over the cells of a row, r = 1 / sqrt(variance + eps),
// and its gradients. With h = (x - mean) * r and d = g * w for the output's gradient g:
//   dx = r * (d - mean(d) - h * mean(d * h)),  dw = sum over rows of g * h,  db = sum of g.
//
// A row is held in registers by G lanes of C cells each, so that every cell is read once. Its
// sums are taken in f32 in a tree whose shape depends on the width alone; the variance is the
// mean square of differences from the mean, and what the mean's rounding leaves in them (their
// own sum) is taken out: rows far from 0 keep their cells' accuracy.
#include "fbhip_heads.h"

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

// A lane's cells: pieces of N that lie G * N cells apart. What is behind the row's end reads
// as 0.
template <class T, uint32_t G, uint32_t C>
struct Cells {
    static constexpr uint32_t N = 16 / sizeof(T);
    static constexpr uint32_t P = C / N;
    float v[C];

    static __device__ __forceinline__ uint32_t column(uint32_t p) {
        return (p * G + threadIdx.x % G) * N;
    }
    template <class U>
    __device__ __forceinline__ void load(const U *row, uint32_t dim) {
#pragma unroll
        for (uint32_t p = 0; p < P; p++) {
            const uint32_t c = column(p);
            if (c + N <= dim) {
                const Piece<U, N> q = load_piece<U, N>(row + c);
#pragma unroll
                for (uint32_t i = 0; i < N; i++) v[p * N + i] = (float)q.v[i];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    v[p * N + i] = c + i < dim ? (float)row[c + i] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void load_typed(const void *p, uint32_t type, uint32_t dim) {
        if (type == FBH_F32) load(static_cast<const float *>(p), dim);
        else if (type == FBH_F16) load(static_cast<const _Float16 *>(p), dim);
        else load(static_cast<const __bf16 *>(p), dim);
    }
    __device__ __forceinline__ void fill(float f) {
#pragma unroll
        for (uint32_t i = 0; i < C; i++) v[i] = f;
    }
    // What lies behind the row's end.
    __device__ __forceinline__ void fill_behind(float f, uint32_t dim) {
#pragma unroll
        for (uint32_t p = 0; p < P; p++) {
            const uint32_t c = column(p);
            if (c + N > dim)
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    if (c + i >= dim) v[p * N + i] = f;
        }
    }
    __device__ __forceinline__ void store(T *row, uint32_t dim) const {
#pragma unroll
        for (uint32_t p = 0; p < P; p++) {
            const uint32_t c = column(p);
            if (c + N <= dim) {
                Piece<T, N> q;
#pragma unroll
                for (uint32_t i = 0; i < N; i++) q.v[i] = (T)v[p * N + i];
                store_piece<T, N>(row + c, q);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    if (c + i < dim) row[c + i] = (T)v[p * N + i];
            }
        }
    }
};

template <uint32_t G>
constexpr uint32_t norm_threads() {
    return G > 256 ? G : 256;
}

template <class T, uint32_t G, uint32_t C>
__global__ __launch_bounds__(norm_threads<G>()) void norm_kernel(Norm A, const T *x, T *out,
                                                                 float *stats) {
    constexpr uint32_t ROWS = norm_threads<G>() / G;
    __shared__ GroupSum<G, 1> first;
    __shared__ GroupSum<G, 2> second;
    Cells<T, G, C> w, b;
    if (A.weight) w.load_typed(A.weight, A.weight_type, A.dim);
    else w.fill(1.0f);
    if (A.bias) b.load_typed(A.bias, A.weight_type, A.dim);
    else b.fill(0.0f);
    const float n = (float)A.dim;
    uint32_t turn = 0;
    for (uint64_t r = (uint64_t)blockIdx.x * ROWS; r < A.n_rows;
         r += (uint64_t)gridDim.x * ROWS, turn ^= 1) {
        const uint64_t row = r + threadIdx.x / G;
        const bool in = row < A.n_rows;  // (all of a group's lanes, and with G > 64 always)
        Cells<T, G, C> c;
        if (in) c.load(x + row * A.dim, A.dim);
        else c.fill(0.0f);
        float s1[1] = {0.0f};
#pragma unroll
        for (uint32_t i = 0; i < C; i++) s1[0] += c.v[i];
        sum_of_group<G, 1>(s1, first, turn);
        const float mean = s1[0] / n;
        c.fill_behind(mean, A.dim);
        float s2[2] = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            c.v[i] -= mean;
            s2[0] += c.v[i];
            s2[1] += c.v[i] * c.v[i];
        }
        sum_of_group<G, 2>(s2, second, turn);
        const float rest = s2[0] / n;
        const float rstd = 1.0f / sqrtf((s2[1] / n - rest * rest) + A.eps);
#pragma unroll
        for (uint32_t i = 0; i < C; i++) c.v[i] = (c.v[i] - rest) * rstd * w.v[i] + b.v[i];
        if (in) {
            c.store(out + row * A.dim, A.dim);
            if (stats && threadIdx.x % G == 0) {
                stats[2 * row] = mean + rest;
                stats[2 * row + 1] = rstd;
            }
        }
    }
}

// Lanes and cells a lane of a row, by its cells.
template <class T, class F>
void with_shape(uint32_t dim, F &&f) {
    if (dim <= 4 * 8) f(Int<4>{}, Int<8>{});
    else if (dim <= 16 * 8) f(Int<16>{}, Int<8>{});
    else if (dim <= 16 * 16) f(Int<16>{}, Int<16>{});
    else if (dim <= 64 * 8) f(Int<64>{}, Int<8>{});
    else if (dim <= 64 * 16) f(Int<64>{}, Int<16>{});
    else if (dim <= 256 * 8) f(Int<256>{}, Int<8>{});
    else if (dim <= 256 * 16) f(Int<256>{}, Int<16>{});
    else if (dim <= 1024 * 8) f(Int<1024>{}, Int<8>{});
    else if (dim <= 1024 * 16) f(Int<1024>{}, Int<16>{});
    else f(Int<1024>{}, Int<32>{});
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
constexpr uint32_t GRAD_GROUPS = 512;
constexpr uint32_t SPLIT_DIM = 16384;  // wider rows' sums have no room in registers

struct NormGrad {
    uint64_t n_rows;
    uint32_t dim, weight_type, groups;
    const void *weight;
    const float *stats;
    float *parts;  // [groups][2][dim], or for wide rows [n_rows]: what the mean leaves out
};

template <class T, uint32_t G, uint32_t C, bool SUMS>
__global__ __launch_bounds__(norm_threads<G>()) void norm_grad_kernel(NormGrad A, const T *g,
                                                                      const T *x, T *dx) {
    constexpr uint32_t ROWS = norm_threads<G>() / G;
    __shared__ GroupSum<G, 3> lds;
    Cells<T, G, C> w, dw, db;
    if (A.weight) w.load_typed(A.weight, A.weight_type, A.dim);
    else w.fill(1.0f);
    if (SUMS) {
        dw.fill(0.0f);
        db.fill(0.0f);
    }
    const float n = (float)A.dim;
    uint32_t turn = 0;
    for (uint64_t r = (uint64_t)blockIdx.x * ROWS; r < A.n_rows;
         r += (uint64_t)gridDim.x * ROWS, turn ^= 1) {
        const uint64_t row = r + threadIdx.x / G;
        const bool in = row < A.n_rows;
        Cells<T, G, C> c, d;
        float mean = 0.0f, rstd = 0.0f;
        if (in) {
            c.load(x + row * A.dim, A.dim);
            d.load(g + row * A.dim, A.dim);
            mean = A.stats[2 * row];
            rstd = A.stats[2 * row + 1];
        } else {
            c.fill(0.0f);
            d.fill(0.0f);
        }
        c.fill_behind(mean, A.dim);
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            c.v[i] -= mean;
            const float e = d.v[i] * w.v[i];
            s[0] += c.v[i];
            s[1] += e;
            s[2] += e * c.v[i];
        }
        sum_of_group<G, 3>(s, lds, turn);
        const float rest = s[0] / n, a = s[1] / n;
        const float b = (s[2] / n - a * rest) * rstd;  // mean(d * h)
        if (!SUMS && A.parts && in && threadIdx.x % G == 0) A.parts[row] = rest;
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            const float h = (c.v[i] - rest) * rstd;
            if (SUMS) {
                dw.v[i] += d.v[i] * h;
                db.v[i] += d.v[i];
            }
            c.v[i] = (d.v[i] * w.v[i] - a - h * b) * rstd;
        }
        if (in && dx) c.store(dx + row * A.dim, A.dim);
    }
    if constexpr (SUMS) {
        if (!A.parts) return;
        constexpr uint32_t N = Cells<T, G, C>::N;
        float *out = A.parts + (uint64_t)blockIdx.x * 2 * A.dim;
        if constexpr (ROWS == 1) {
#pragma unroll
            for (uint32_t i = 0; i < C; i++) {
                const uint32_t col = Cells<T, G, C>::column(i / N) + i % N;
                if (col < A.dim) {
                    out[col] = dw.v[i];
                    out[A.dim + col] = db.v[i];
                }
            }
        } else {
            // the workgroup's rows, added in their order
            __shared__ float sums[2][ROWS][G * C / 4];
#pragma unroll
            for (uint32_t q = 0; q < 4; q++) {  // a quarter of the cells at a time
                __syncthreads();
#pragma unroll
                for (uint32_t k = 0; k < C / 4; k++) {
                    const uint32_t at = k * G + threadIdx.x % G;
                    sums[0][threadIdx.x / G][at] = dw.v[q * (C / 4) + k];
                    sums[1][threadIdx.x / G][at] = db.v[q * (C / 4) + k];
                }
                __syncthreads();
                for (uint32_t j = threadIdx.x; j < 2 * G * C / 4; j += norm_threads<G>()) {
                    const uint32_t at = j % (G * C / 4), which = j / (G * C / 4);
                    float t = 0.0f;
                    for (uint32_t k = 0; k < ROWS; k++) t += sums[which][k][at];
                    const uint32_t i = q * (C / 4) + at / G;
                    const uint32_t col = ((i / N) * G + at % G) * N + i % N;
                    if (col < A.dim) out[which * A.dim + col] = t;
                }
            }
        }
    }
}

// dw and db of wide rows: a thread a column, the rows cut into `groups` equal parts.
template <class T>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormGrad A, const T *g, const T *x,
                                                           const float *rests, float *parts) {
    const uint32_t col = blockIdx.x * 256 + threadIdx.x;
    if (col >= A.dim) return;
    const uint64_t each = (A.n_rows + A.groups - 1) / A.groups;
    const uint64_t begin = blockIdx.y * each, end = min(begin + each, A.n_rows);
    float dw = 0.0f, db = 0.0f;
    for (uint64_t r = begin; r < end; r++) {
        const float d = (float)g[r * A.dim + col];
        const float h = ((float)x[r * A.dim + col] - A.stats[2 * r] - rests[r]) *
                        A.stats[2 * r + 1];
        dw += d * h;
        db += d;
    }
    float *out = parts + (uint64_t)blockIdx.y * 2 * A.dim;
    out[col] = dw;
    out[A.dim + col] = db;
}

// The parts' sums, in doubles: 16 columns a workgroup, each part's cells to one of 16 threads.
__global__ __launch_bounds__(256) void norm_join_kernel(const float *parts, uint32_t dim,
                                                        uint32_t groups, uint32_t weight_type,
                                                        void *dweight, void *dbias) {
    __shared__ double sums[16][17];
    const uint32_t lane = threadIdx.x % 16, k = threadIdx.x / 16;
    const uint32_t j = blockIdx.x * 16 + lane;  // of 2 * dim
    double t = 0.0;
    if (j < 2 * dim)
        for (uint32_t p = k; p < groups; p += 16) t += (double)parts[(uint64_t)p * 2 * dim + j];
    sums[k][lane] = t;
    __syncthreads();
    if (k != 0 || j >= 2 * dim) return;
    for (uint32_t i = 1; i < 16; i++) t += sums[i][lane];
    void *out = j < dim ? dweight : dbias;
    const uint32_t at = j < dim ? j : j - dim;
    if (!out) return;
    if (weight_type == FBH_F32) static_cast<float *>(out)[at] = (float)t;
    else if (weight_type == FBH_F16) static_cast<_Float16 *>(out)[at] = (_Float16)(float)t;
    else static_cast<__bf16 *>(out)[at] = (__bf16)(float)t;
}

// ------------------------------------------------------------------- host side
uint32_t rows_of_group(uint32_t dim) {
    uint32_t rows = 1;
    with_shape<float>(dim, [&](auto g, auto) {
        constexpr uint32_t G = decltype(g)::value;
        rows = norm_threads<G>() / G;
    });
    return rows;
}

uint32_t grad_groups(uint64_t n_rows, uint32_t dim) {
    const uint64_t most = (n_rows + rows_of_group(dim) - 1) / rows_of_group(dim);
    return (uint32_t)(most < GRAD_GROUPS ? (most ? most : 1) : GRAD_GROUPS);
}

uint64_t padded_rows(uint64_t n) { return (n + 3) / 4 * 4; }

uint64_t grad_bytes(const fbh_norm *a) {
    uint64_t b = (uint64_t)grad_groups(a->n_rows, a->dim) * 2 * a->dim * 4;
    if (a->dim > SPLIT_DIM) b += padded_rows(a->n_rows) * 4;
    return b;
}

void check_norm(const fbh_norm *a) {
    head_input(a, "null argument");
    head_input(a->dtype <= FBH_BF16, "unknown cell type");
    head_input(a->weight_type <= FBH_BF16, "unknown weight type");
    head_input(a->dim >= 1 && a->dim <= NORM_MAX_DIM, "dim must be in 1..=32768");
    head_input(a->n_rows <= (1ull << 40) / a->dim, "more than 2^40 cells");
    head_input(a->eps >= 1.17549435e-38f && a->eps <= 3.4028235e38f,
               "eps must be a positive normal float");
}

template <class K, class... A>
void launch(K kernel, uint64_t blocks, uint32_t threads, hipStream_t s, A... args) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(threads), 0, s, args...);
    head_check(hipGetLastError(), "layer norm");
}

template <class T>
void launch_norm(const fbh_norm *a, const void *x, const void *weight, const void *bias, void *out,
                 float *stats, hipStream_t s) {
    const Norm A{weight, bias, a->n_rows, a->dim, a->weight_type, a->eps};
    with_shape<T>(a->dim, [&](auto g, auto c) {
        constexpr uint32_t G = decltype(g)::value, C = decltype(c)::value;
        constexpr uint32_t ROWS = norm_threads<G>() / G;
        const uint64_t blocks = (a->n_rows + ROWS - 1) / ROWS;
        launch(norm_kernel<T, G, C>, blocks < 2048 ? blocks : 2048, norm_threads<G>(), s, A,
               static_cast<const T *>(x), static_cast<T *>(out), stats);
    });
}

template <class T>
void launch_norm_grad(const fbh_norm *a, const T *g, const T *x, const float *stats,
                      const void *weight, T *dx, void *dweight, void *dbias, float *work,
                      hipStream_t s) {
    const bool sums = dweight || dbias, split = a->dim > SPLIT_DIM;
    const uint32_t groups = grad_groups(a->n_rows, a->dim);
    NormGrad A{a->n_rows, a->dim, a->weight_type, groups, weight, stats, sums ? work : nullptr};
    with_shape<T>(a->dim, [&](auto gg, auto cc) {
        constexpr uint32_t G = decltype(gg)::value, C = decltype(cc)::value;
        constexpr bool SUMS = G * C <= SPLIT_DIM;
        launch(norm_grad_kernel<T, G, C, SUMS>, groups, norm_threads<G>(), s, A, g, x, dx);
    });
    if (!sums) return;
    float *parts = work;
    if (split) {
        parts = work + padded_rows(a->n_rows);
        hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((a->dim + 255) / 256, groups), dim3(256),
                           0, s, A, g, x, work, parts);
        head_check(hipGetLastError(), "layer norm");
    }
    launch(norm_join_kernel, (2 * a->dim + 15) / 16, 256, s, parts, a->dim, groups,
           a->weight_type, dweight, dbias);
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
            head_input(work && work_bytes >= grad_bytes(a), "the workspace is too small");
            head_input(reinterpret_cast<uintptr_t>(work) % 16 == 0,
                       "the workspace must be 16-byte aligned");
        }
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
