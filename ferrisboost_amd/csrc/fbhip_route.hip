// Rows handed to experts by their ids and brought back. A position is a row and a column of an
// id matrix; positions are sorted by id, stably, those without an expert behind all others:
//   order   the positions in that order
//   place   the row of a position in it, or -1 - row for one without an expert
//   starts  the first row of every expert, and the end of the last one's
//
// The sort is one counting pass, as there are at most 1024 ids: counts of the ids in chunks of
// positions, their sums over the chunks before, and places from both. All orders are fixed.
#include "fbhip_heads.h"

namespace fbh {
namespace {

constexpr uint32_t ROUTE_MAX_EXPERTS = 1024;
constexpr uint32_t ROUTE_TPB = 512;
constexpr uint32_t ROUTE_WAVES = ROUTE_TPB / 64;
constexpr uint32_t ROUTE_CHUNK = 4096;   // positions of a chunk at least
constexpr uint32_t ROUTE_CHUNKS = 1024;  // chunks at most
constexpr uint32_t ROUTE_MAX_DIM = 32768;
constexpr uint64_t ROUTE_BLOCKS = 1u << 20;  // of a launch at most

struct Route {
    const void *ids;
    uint32_t n, n_experts, bits;
    uint32_t chunks, each;  // chunks, and positions of a wave of one
    int32_t *order, *place, *starts;
    uint32_t *counts;  // [n_experts + 1][chunks]
    uint32_t *totals;  // [n_experts + 1]
};

template <int ID>
__device__ __forceinline__ uint32_t expert_at(const Route &R, uint32_t pos) {
    return min(load_id<ID>(R.ids, pos), R.n_experts);
}

template <int ID>
__global__ __launch_bounds__(ROUTE_TPB) void route_count_kernel(Route R) {
    __shared__ uint32_t c[ROUTE_MAX_EXPERTS + 1];
    for (uint32_t e = threadIdx.x; e <= R.n_experts; e += ROUTE_TPB) c[e] = 0;
    __syncthreads();
    const uint64_t begin = (uint64_t)blockIdx.x * ROUTE_WAVES * R.each;
    const uint32_t end = (uint32_t)min(begin + ROUTE_WAVES * R.each, (uint64_t)R.n);
    for (uint64_t i = begin + threadIdx.x; i < end; i += ROUTE_TPB)
        atomicAdd(&c[expert_at<ID>(R, (uint32_t)i)], 1u);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= R.n_experts; e += ROUTE_TPB)
        R.counts[(uint64_t)e * R.chunks + blockIdx.x] = c[e];
}

// The sum of the values of lower lanes.
__device__ __forceinline__ uint32_t before_in_wave(uint32_t v, uint32_t *all) {
    uint32_t x = v;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if ((threadIdx.x & 63) >= (uint32_t)d) x += y;
    }
    *all = __shfl(x, 63);
    return x - v;
}

// An expert's counts to the positions before them among its own; its total.
__global__ __launch_bounds__(64) void route_scan_kernel(Route R) {
    uint32_t *c = R.counts + (uint64_t)blockIdx.x * R.chunks;
    uint32_t sum = 0;
    for (uint32_t b = 0; b < R.chunks; b += 64) {
        const uint32_t i = b + threadIdx.x;
        uint32_t all;
        const uint32_t at = before_in_wave(i < R.chunks ? c[i] : 0, &all);
        if (i < R.chunks) c[i] = sum + at;
        sum += all;
    }
    if (threadIdx.x == 0) R.totals[blockIdx.x] = sum;
}

template <int ID>
__global__ __launch_bounds__(ROUTE_TPB) void route_place_kernel(Route R) {
    __shared__ uint32_t base[ROUTE_MAX_EXPERTS + 1];
    __shared__ uint32_t seen[ROUTE_WAVES][ROUTE_MAX_EXPERTS + 1];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    for (uint32_t e = threadIdx.x; e <= R.n_experts; e += ROUTE_TPB)
        for (uint32_t k = 0; k < ROUTE_WAVES; k++) seen[k][e] = 0;
    if (w == 0) {  // where each expert's positions begin
        uint32_t sum = 0;
        for (uint32_t b = 0; b <= R.n_experts; b += 64) {
            const uint32_t e = b + lane;
            uint32_t all;
            const uint32_t at = before_in_wave(e <= R.n_experts ? R.totals[e] : 0, &all);
            if (e <= R.n_experts) {
                base[e] = sum + at;
                if (blockIdx.x == 0) R.starts[e] = (int32_t)(sum + at);
            }
            sum += all;
        }
    }
    __syncthreads();
    const uint64_t begin = ((uint64_t)blockIdx.x * ROUTE_WAVES + w) * R.each;
    const uint64_t end = min(begin + R.each, (uint64_t)R.n);
    for (uint64_t i = begin + lane; i < end; i += 64)
        atomicAdd(&seen[w][expert_at<ID>(R, (uint32_t)i)], 1u);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e <= R.n_experts; e += ROUTE_TPB) {
        uint32_t at = base[e] + R.counts[(uint64_t)e * R.chunks + blockIdx.x];
        for (uint32_t k = 0; k < ROUTE_WAVES; k++) {
            const uint32_t c = seen[k][e];
            seen[k][e] = at;
            at += c;
        }
    }
    __syncthreads();
    // a wave's rounds are one after the other, a lane's place in its round is the number of
    // lower lanes with its expert
    for (uint64_t i0 = begin; i0 < end; i0 += 64) {
        const uint64_t i = i0 + lane;
        const bool in = i < end;
        const uint32_t e = in ? expert_at<ID>(R, (uint32_t)i) : 0;
        const uint32_t at = take_places(&seen[w][e], in, same_digit(in, e, R.bits));
        if (in) {
            R.order[at] = (int32_t)i;
            R.place[i] = e < R.n_experts ? (int32_t)at : -1 - (int32_t)at;
        }
    }
}

// ------------------------------------------------------------------- rows
// A row's pieces go to G = 2^lg_g lanes; the last one starts at dim - VEC, so that no piece is
// partial: the cells it shares with the one before are written twice, with the same value.
struct Rows {
    const int32_t *place;
    const float *weights;
    uint64_t n_rows;
    uint32_t n_columns, dim, pieces, lg_g;
    uint32_t n_places;  // n_rows * n_columns, which every place is below
};

__device__ __forceinline__ uint32_t place_row(const Rows &R, int32_t place) {
    return min((uint32_t)(place < 0 ? -1 - place : place), R.n_places - 1);
}

// f(row, lane of the row) for every row: a launch has fewer than 2^32 threads.
template <class F>
__device__ __forceinline__ void for_rows(const Rows &R, F &&f) {
    const uint32_t rows = 256 >> R.lg_g;
    for (uint64_t row = (uint64_t)blockIdx.x * rows + (threadIdx.x >> R.lg_g); row < R.n_rows;
         row += (uint64_t)gridDim.x * rows)
        f(row, threadIdx.x & ((1u << R.lg_g) - 1));
}

template <class T, int VEC>
__device__ __forceinline__ void to_experts_row(Rows R, const T *x, T *out, uint64_t row, uint32_t lane) {
    const int32_t *place = R.place + row * R.n_columns;
    for (uint32_t p = lane; p < R.pieces; p += 1u << R.lg_g) {
        const uint32_t c = min(p * VEC, R.dim - VEC);
        const Piece<T, VEC> v = load_piece<T, VEC>(x + row * R.dim + c);
        for (uint32_t j = 0; j < R.n_columns; j++) {
            const int32_t a = place[j];
            Piece<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = a < 0 ? (T)0.0f : v.v[i];
            store_piece<T, VEC>(out + (uint64_t)place_row(R, a) * R.dim + c, o);
        }
    }
}
template <class T, int VEC>
__global__ __launch_bounds__(256) void to_experts_kernel(Rows R, const T *x, T *out) {
    for_rows(R, [&](uint64_t row, uint32_t lane) {
        to_experts_row<T, VEC>(R, x, out, row, lane);
    });
}

template <class T, int VEC>
__device__ __forceinline__ void from_experts_row(Rows R, const T *y, T *out, uint64_t row, uint32_t lane) {
    const int32_t *place = R.place + row * R.n_columns;
    const float *weights = R.weights + row * R.n_columns;
    for (uint32_t p = lane; p < R.pieces; p += 1u << R.lg_g) {
        const uint32_t c = min(p * VEC, R.dim - VEC);
        float s[VEC] = {};
        for (uint32_t j = 0; j < R.n_columns; j++) {
            const int32_t a = place[j];
            if (a < 0) continue;
            const Piece<T, VEC> v = load_piece<T, VEC>(y + (uint64_t)place_row(R, a) * R.dim + c);
            const float f = R.weights ? weights[j] : 1.0f;
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] += f * (float)v.v[i];
        }
        Piece<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; i++) o.v[i] = (T)s[i];
        store_piece<T, VEC>(out + row * R.dim + c, o);
    }
}
template <class T, int VEC>
__global__ __launch_bounds__(256) void from_experts_kernel(Rows R, const T *y, T *out) {
    for_rows(R, [&](uint64_t row, uint32_t lane) {
        from_experts_row<T, VEC>(R, y, out, row, lane);
    });
}

// The gradients of from_experts: dy = weight * g to the place, dweight = <g, y> there.
template <class T, int VEC>
__device__ __forceinline__ void from_experts_grad_row(Rows R, const T *g, const T *y, T *dy, float *dweights, uint64_t row, uint32_t lane) {
    for (uint32_t j = 0; j < R.n_columns; j++) {
        const int32_t a = R.place[row * R.n_columns + j];
        const float w = R.weights ? R.weights[row * R.n_columns + j] : 1.0f;
        const uint64_t at = (uint64_t)place_row(R, a) * R.dim;
        float dot = 0.0f;
        for (uint32_t p = lane; p < R.pieces; p += 1u << R.lg_g) {
            const uint32_t c = min(p * VEC, R.dim - VEC);
            const Piece<T, VEC> v = load_piece<T, VEC>(g + row * R.dim + c);
            Piece<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = a < 0 ? (T)0.0f : (T)(w * (float)v.v[i]);
            if (dy) store_piece<T, VEC>(dy + at + c, o);
            if (!dweights || a < 0) continue;
            const Piece<T, VEC> u = load_piece<T, VEC>(y + at + c);
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (c + i >= p * VEC) dot += (float)v.v[i] * (float)u.v[i];
        }
        if (!dweights) continue;
        for (uint32_t d = 1u << R.lg_g; d >>= 1;) dot += __shfl_xor(dot, d);
        if (lane == 0) dweights[row * R.n_columns + j] = dot;
    }
}
template <class T, int VEC>
__global__ __launch_bounds__(256) void from_experts_grad_kernel(Rows R, const T *g, const T *y, T *dy, float *dweights) {
    for_rows(R, [&](uint64_t row, uint32_t lane) {
        from_experts_grad_row<T, VEC>(R, g, y, dy, dweights, row, lane);
    });
}

// ------------------------------------------------------------------- host side
template <class K, class... A>
void launch(K kernel, uint64_t blocks, uint32_t threads, hipStream_t s, A... args) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(threads), 0, s, args...);
    head_check(hipGetLastError(), "experts");
}

void check_route(uint64_t n, uint32_t n_experts) {
    head_input(n <= 0x7FFFFFFFull, "more than 2147483647 positions");
    head_input(n_experts >= 1 && n_experts <= ROUTE_MAX_EXPERTS, "n_experts must be in 1..=1024");
}

uint64_t route_chunks(uint64_t n) {
    const uint64_t c = (n + ROUTE_CHUNK - 1) / ROUTE_CHUNK;
    return c < 1 ? 1 : c > ROUTE_CHUNKS ? ROUTE_CHUNKS : c;
}

uint64_t route_bytes(uint64_t n, uint32_t n_experts) {
    return (n_experts + 1) * (route_chunks(n) + 1) * 4;
}

template <int ID>
void launch_route(const Route &R, hipStream_t s) {
    launch(route_count_kernel<ID>, R.chunks, ROUTE_TPB, s, R);
    launch(route_scan_kernel, R.n_experts + 1, 64, s, R);
    launch(route_place_kernel<ID>, R.chunks, ROUTE_TPB, s, R);
}

Rows rows_of(const int32_t *place, const float *weights, uint64_t n_rows, uint32_t n_columns,
             uint32_t dim, uint32_t dtype) {
    head_input(dtype <= FBH_BF16, "unknown cell type");
    head_input(dim >= 1 && dim <= ROUTE_MAX_DIM, "dim must be in 1..=32768");
    head_input(n_columns >= 1, "no columns");
    head_input(n_rows <= 0x7FFFFFFFull / n_columns, "more than 2147483647 positions");
    head_input(place || n_rows == 0, "null argument");
    Rows R{place, weights, n_rows, n_columns, dim, 0, 0, (uint32_t)(n_rows * n_columns)};
    const uint32_t v = piece_cells(dim, dtype);
    R.pieces = (dim + v - 1) / v;
    while (R.lg_g < 6 && (1u << R.lg_g) < R.pieces) R.lg_g++;
    return R;
}

// f(a cell, cells of a piece)
template <class F>
void with_pieces(uint32_t dim, uint32_t dtype, F &&f) {
    const auto vec = [&](auto t) {
        const uint32_t v = piece_cells(dim, dtype);
        if constexpr (sizeof(t) == 2)
            if (v == 8) return f(t, std::integral_constant<int, 8>{});
        if (v == 4) return f(t, std::integral_constant<int, 4>{});
        if (v == 2) return f(t, std::integral_constant<int, 2>{});
        f(t, std::integral_constant<int, 1>{});
    };
    if (dtype == FBH_F32) vec(float{});
    else if (dtype == FBH_F16) vec(_Float16{});
    else vec(__bf16{});
}

uint64_t row_blocks(const Rows &R) {
    const uint32_t rows = 256 >> R.lg_g;
    const uint64_t blocks = (R.n_rows + rows - 1) / rows;
    return blocks < ROUTE_BLOCKS ? blocks : ROUTE_BLOCKS;
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" {

uint64_t fbh_route_bytes(uint64_t n_positions, uint32_t n_experts) {
    uint64_t bytes = 0;
    (void)head_guard([&] {
        check_route(n_positions, n_experts);
        bytes = route_bytes(n_positions, n_experts);
    });
    return bytes;
}

int fbh_route(int device, const void *ids, uint32_t id_type, uint64_t n_positions,
              uint32_t n_experts, int32_t *order, int32_t *place, int32_t *starts, void *work,
              uint64_t work_bytes, void *stream) {
    return head_guard([&] {
        check_route(n_positions, n_experts);
        head_input(id_type <= FBH_ID_F32, "unknown id type");
        head_input((ids && order && place) || n_positions == 0, "null argument");
        head_input(starts, "null argument");
        head_input(work && work_bytes >= route_bytes(n_positions, n_experts),
                   "the workspace is too small");
        head_input(reinterpret_cast<uintptr_t>(work) % 4 == 0,
                   "the workspace must be 4-byte aligned");
        const OnDevice on(device);
        Route R{ids, (uint32_t)n_positions, n_experts, 0, 0, 0, order, place, starts, nullptr,
                nullptr};
        while ((1u << R.bits) <= n_experts) R.bits++;
        R.chunks = (uint32_t)route_chunks(n_positions);
        const uint64_t waves = (uint64_t)R.chunks * ROUTE_WAVES;
        R.each = (uint32_t)(((n_positions + waves - 1) / waves + 63) / 64 * 64);
        R.counts = static_cast<uint32_t *>(work);
        R.totals = R.counts + (uint64_t)(n_experts + 1) * R.chunks;
        const auto s = static_cast<hipStream_t>(stream);
        if (id_type == FBH_ID_I32) launch_route<FBH_ID_I32>(R, s);
        else if (id_type == FBH_ID_I64) launch_route<FBH_ID_I64>(R, s);
        else launch_route<FBH_ID_F32>(R, s);
    });
}

int fbh_to_experts(int device, const void *x, const int32_t *place, uint64_t n_rows,
                   uint32_t n_columns, uint32_t dim, uint32_t dtype, void *out, void *stream) {
    return head_guard([&] {
        const Rows R = rows_of(place, nullptr, n_rows, n_columns, dim, dtype);
        head_input((x && out) || n_rows == 0, "null argument");
        if (n_rows == 0) return;
        const OnDevice on(device);
        with_pieces(dim, dtype, [&](auto t, auto v) {
            using T = decltype(t);
            launch(to_experts_kernel<T, decltype(v)::value>, row_blocks(R), 256,
                   static_cast<hipStream_t>(stream), R, static_cast<const T *>(x),
                   static_cast<T *>(out));
        });
    });
}

int fbh_from_experts(int device, const void *y, const int32_t *place, const float *weights,
                     uint64_t n_rows, uint32_t n_columns, uint32_t dim, uint32_t dtype, void *out,
                     void *stream) {
    return head_guard([&] {
        const Rows R = rows_of(place, weights, n_rows, n_columns, dim, dtype);
        head_input((y && out) || n_rows == 0, "null argument");
        if (n_rows == 0) return;
        const OnDevice on(device);
        with_pieces(dim, dtype, [&](auto t, auto v) {
            using T = decltype(t);
            launch(from_experts_kernel<T, decltype(v)::value>, row_blocks(R), 256,
                   static_cast<hipStream_t>(stream), R, static_cast<const T *>(y),
                   static_cast<T *>(out));
        });
    });
}

int fbh_from_experts_grad(int device, const void *grad, const void *y, const int32_t *place,
                          const float *weights, uint64_t n_rows, uint32_t n_columns, uint32_t dim,
                          uint32_t dtype, void *dy, float *dweights, void *stream) {
    return head_guard([&] {
        const Rows R = rows_of(place, weights, n_rows, n_columns, dim, dtype);
        head_input((grad && (y || !dweights)) || n_rows == 0, "null argument");
        if (n_rows == 0 || (!dy && !dweights)) return;
        const OnDevice on(device);
        with_pieces(dim, dtype, [&](auto t, auto v) {
            using T = decltype(t);
            launch(from_experts_grad_kernel<T, decltype(v)::value>, row_blocks(R), 256,
                   static_cast<hipStream_t>(stream), R, static_cast<const T *>(grad),
                   static_cast<const T *>(y), static_cast<T *>(dy), dweights);
        });
    });
}

}  // extern "C"
