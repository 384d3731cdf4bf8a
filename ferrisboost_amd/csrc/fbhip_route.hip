// Rows handed to experts by their ids and brought back. A position is a row and a column of an
// id matrix; positions are sorted by id, stably, those without an expert behind all others:
//   order   the positions in that order
//   place   the row of a position in it, or -1 - row for one without an expert
//   starts  the first row of every expert, and the end of the last one's
//
// The sort is one counting pass, as there are at most 1024 ids: counts of the ids in chunks of
// positions, their sums over the chunks before, and places from both; up to 4096 positions take
// one workgroup and launch. All orders are fixed. 2M positions of 511 ids take 20.8 us (5.6 +
// 3.7 + 13.4 by themselves) where memory would take 5: each launch's workgroups are all on the
// device at once, and its time is what one of them takes from its loads to its stores. Of the last
// launch waves wait 64 % (LDS counters, round after round, and barriers), and vector instructions,
// most of them the search for equal ids, take 40 %; `order` in runs of 8 positions costs 22.4 MB of
// writes for 16.
#include "fbhip_heads.h"

#include <algorithm>
#include <type_traits>

namespace fbh {
namespace {

constexpr uint32_t ROUTE_MAX_EXPERTS = 1024;
constexpr uint32_t ROUTE_TPB = 512;
constexpr uint32_t ROUTE_WAVES = ROUTE_TPB / 64;
// Positions that one workgroup sorts by itself, in one launch (in us, 511 experts: 4000 positions
// 6.9, in three launches 8.0; 1000 positions 3.7 and 7.5).
constexpr uint32_t ROUTE_ONE = 4096;
constexpr uint32_t ROUTE_MAX_DIM = 32768;
constexpr uint64_t ROUTE_BLOCKS = 1u << 20;  // of a launch at most

struct Route {
    const void *ids;
    uint32_t id_type, n, n_experts, chunks;
    int32_t *order, *place, *starts;
    uint32_t *counts;  // [chunks][n_experts + 1]
    uint32_t *totals;  // [n_experts + 1]
};

// The experts of ROUNDS positions from `first` on, `apart` from one another (behind the last
// one: `none`).
template <uint32_t ROUNDS>
__device__ __forceinline__ void load_experts(const Route &R, uint64_t first, uint32_t apart,
                                             uint32_t none, uint32_t (&e)[ROUNDS]) {
    const auto load = [&](auto id) {
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; r++) {
            const uint64_t i = first + r * apart;
            e[r] = i < R.n ? min(load_id<decltype(id)::value>(R.ids, i), R.n_experts) : none;
        }
    };
    if (R.id_type == FBH_ID_I32) load(std::integral_constant<int, FBH_ID_I32>{});
    else if (R.id_type == FBH_ID_I64) load(std::integral_constant<int, FBH_ID_I64>{});
    else load(std::integral_constant<int, FBH_ID_F32>{});
}

// A workgroup's chunk has ROUNDS positions a thread; a wave's follow one another, 64 a round.
template <uint32_t ROUNDS>
__global__ __launch_bounds__(ROUTE_TPB) void route_count_kernel(Route R) {
    __shared__ uint32_t c[ROUTE_MAX_EXPERTS + 1];
    uint32_t e[ROUNDS];
    load_experts<ROUNDS>(R, (uint64_t)blockIdx.x * (ROUTE_TPB * ROUNDS) + threadIdx.x, ROUTE_TPB,
                         ~0u, e);
    for (uint32_t x = threadIdx.x; x <= R.n_experts; x += ROUTE_TPB) c[x] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++)
        if (e[r] != ~0u) atomicAdd(&c[e[r]], 1u);
    __syncthreads();
    for (uint32_t x = threadIdx.x; x <= R.n_experts; x += ROUTE_TPB)
        R.counts[(uint64_t)blockIdx.x * (R.n_experts + 1) + x] = c[x];
}

// The experts' counts to the positions before them among their own, and their totals: 16 experts
// a workgroup, its threads a 64th of the chunks of one each.
constexpr uint32_t SCAN_EXPERTS = 16, SCAN_PARTS = 64;
__global__ __launch_bounds__(SCAN_EXPERTS *SCAN_PARTS) void route_scan_kernel(Route R) {
    __shared__ uint32_t sums[SCAN_PARTS][SCAN_EXPERTS + 1];
    const uint32_t part = threadIdx.x / SCAN_EXPERTS, mine = threadIdx.x % SCAN_EXPERTS;
    const uint32_t x = blockIdx.x * SCAN_EXPERTS + mine, row = R.n_experts + 1;
    const uint32_t each = (R.chunks + SCAN_PARTS - 1) / SCAN_PARTS;
    const uint32_t begin = min(part * each, R.chunks), end = min(begin + each, R.chunks);
    uint32_t sum = 0, first[8];
    if (x < row) {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
            first[k] = begin + k < end ? R.counts[(uint64_t)(begin + k) * row + x] : 0;
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) sum += first[k];
#pragma unroll 8
        for (uint32_t c = begin + 8; c < end; c++) sum += R.counts[(uint64_t)c * row + x];
    }
    sums[part][mine] = sum;
    __syncthreads();
    {  // a wave an expert, a lane a part
        const uint32_t lane = threadIdx.x % SCAN_PARTS, e = threadIdx.x / SCAN_PARTS;
        const uint32_t v = sums[lane][e], upto = scan_wave(v);
        sums[lane][e] = upto - v;
        const uint32_t y = blockIdx.x * SCAN_EXPERTS + e;
        if (lane == SCAN_PARTS - 1 && y < row) R.totals[y] = upto;
    }
    __syncthreads();
    if (x >= row) return;
    uint32_t at = sums[part][mine];
#pragma unroll
    for (uint32_t k = 0; k < 8; k++) {
        if (begin + k < end) R.counts[(uint64_t)(begin + k) * row + x] = at;
        at += first[k];
    }
    for (uint32_t c = begin + 8; c < end; c++) {
        const uint32_t v = R.counts[(uint64_t)c * row + x];
        R.counts[(uint64_t)c * row + x] = at;
        at += v;
    }
}

// The sums of lower threads' values, of two at a time.
__device__ __forceinline__ void before_in_group(uint32_t (&v)[2], uint32_t (*sums)[2]) {
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    uint32_t upto[2];
#pragma unroll
    for (int k = 0; k < 2; k++) upto[k] = scan_wave(v[k]);
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < 2; k++) sums[w][k] = upto[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
        v[k] = upto[k] - v[k];
        for (uint32_t u = 0; u < w; u++) v[k] += sums[u][k];
    }
}

// A chunk is sorted in LDS first: what a wave then writes of `order` are a few runs and not 64
// cells apart (16M positions of 64 experts: 70 us straight from the ranks). ONE: the only
// workgroup, which needs no counts. BITS: of the experts' numbers, known so that the search for
// equal ones in a wave has no loop, a thread has one of up to 512 experts (2M positions of 511
// with room for 1024: 14.7 us), and workgroups of few take little LDS.
template <uint32_t ROUNDS, uint32_t BITS, bool ONE>
__global__ __launch_bounds__(ROUTE_TPB) void route_place_kernel(Route R) {
    constexpr uint32_t ROOM = BITS > 10 ? ROUTE_MAX_EXPERTS + 1 : 1u << BITS;
    constexpr uint32_t EACH = (ROOM + ROUTE_TPB - 1) / ROUTE_TPB;  // experts a thread
    constexpr uint32_t CHUNK = ROUTE_TPB * ROUNDS;
    __shared__ uint32_t seen[ROUTE_WAVES][ROOM];
    __shared__ uint32_t shift[ROOM];  // from places in the chunk to those in all
    __shared__ uint32_t sorted[CHUNK];  // a position's number in the chunk, and its expert
    __shared__ uint32_t sums[ROUTE_WAVES][2];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    const uint64_t begin = (uint64_t)blockIdx.x * CHUNK;
    const uint32_t here = (uint32_t)min((uint64_t)CHUNK, R.n - min(begin, (uint64_t)R.n));
    const uint32_t first = w * (64 * ROUNDS) + lane;
    uint32_t e[ROUNDS], rank[ROUNDS], total[EACH], before[EACH], own[EACH];
    load_experts<ROUNDS>(R, begin + first, 64, 0, e);
    if (!ONE)
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) {
            const uint32_t x = threadIdx.x * EACH + k;
            total[k] = x <= R.n_experts ? R.totals[x] : 0;
            before[k] = x <= R.n_experts
                            ? R.counts[(uint64_t)blockIdx.x * (R.n_experts + 1) + x] : 0;
        }
    for (uint32_t x = lane; x <= R.n_experts; x += 64) seen[w][x] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // (a wave's LDS operations complete in order, and only it touches its counters)
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const bool in = first + r * 64 < here;
        rank[r] = take_places(&seen[w][e[r]], in, same_digit(in, e[r], BITS));
    }
    __syncthreads();
    // where the experts begin, in the chunk and in all, and each wave's positions of them
    uint32_t at[2] = {0, 0};
#pragma unroll
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t x = threadIdx.x * EACH + k;
        own[k] = 0;
        if (x <= R.n_experts)
#pragma unroll
            for (uint32_t v = 0; v < ROUTE_WAVES; v++) own[k] += seen[v][x];
        if (ONE) {
            total[k] = own[k];
            before[k] = 0;
        }
        at[0] += own[k];
        at[1] += total[k];
    }
    before_in_group(at, sums);
#pragma unroll
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t x = threadIdx.x * EACH + k;
        if (x <= R.n_experts) {
            if (blockIdx.x == 0) R.starts[x] = (int32_t)at[1];
            shift[x] = at[1] + before[k] - at[0];
            uint32_t to = at[0], c[ROUTE_WAVES];
#pragma unroll
            for (uint32_t v = 0; v < ROUTE_WAVES; v++) c[v] = seen[v][x];
#pragma unroll
            for (uint32_t v = 0; v < ROUTE_WAVES; v++) {
                seen[v][x] = to;
                to += c[v];
            }
        }
        at[0] += own[k];
        at[1] += total[k];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = first + r * 64;
        if (i >= here) continue;
        const uint32_t to = seen[w][e[r]] + rank[r], row = to + shift[e[r]];
        sorted[to] = i | e[r] << 16;
        R.place[begin + i] = e[r] < R.n_experts ? (int32_t)row : -1 - (int32_t)row;
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < here; j += ROUTE_TPB) {
        const uint32_t v = sorted[j];
        R.order[j + shift[v >> 16]] = (int32_t)(begin + (v & 0xFFFF));
    }
}

// ------------------------------------------------------------------- rows
// Bound by memory (65,536 rows of 1024 bfloat16 cells with 2 columns: to the experts 63 us, 402
// MB, 6.4 TB/s, most of them writes that the last-level cache takes; back 94 us, 4.3 TB/s, rows
// read from everywhere; a copy reaches 4.84). A row's pieces go to G = 2^lg_g lanes; the last one
// starts at dim - VEC, so that no piece is partial: the cells it shares with the one before are
// written twice, with the same value.
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
__device__ __forceinline__ void to_experts_row(const Rows &R, const T *x, T *out, uint64_t row,
                                               uint32_t lane) {
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

// K columns of a row side by side, so that their pieces are on their way together.
template <int K>
struct Columns {
    uint64_t at[K];   // the first cells of the places
    float weight[K];  // 0 without a place
    bool is[K];

    __device__ __forceinline__ Columns(const Rows &R, uint64_t row, uint32_t first) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint64_t i = row * R.n_columns + first + k;
            const bool in = first + k < R.n_columns;
            const int32_t a = in ? R.place[i] : -1;
            is[k] = a >= 0;
            at[k] = (uint64_t)place_row(R, a) * R.dim;
            weight[k] = !is[k] ? 0.0f : R.weights ? R.weights[i] : 1.0f;
        }
    }
};

template <class T, int VEC, int K>
__device__ __forceinline__ void from_experts_row(const Rows &R, const T *__restrict__ y,
                                                 T *__restrict__ out, uint64_t row,
                                                 uint32_t lane) {
    // (one batch of columns: their places are read once)
    const Columns<K> only(R, row, 0);
#pragma unroll 2
    for (uint32_t p = lane; p < R.pieces; p += 1u << R.lg_g) {
        const uint32_t c = min(p * VEC, R.dim - VEC);
        float s[VEC] = {};
        const auto add = [&](const Columns<K> &C) {
            Piece<T, VEC> v[K] = {};
#pragma unroll
            for (int k = 0; k < K; k++)
                if (C.is[k]) v[k] = load_piece<T, VEC>(y + C.at[k] + c);
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < VEC; i++) s[i] += C.weight[k] * (float)v[k].v[i];
        };
        add(only);
        for (uint32_t j = K; j < R.n_columns; j += K) add(Columns<K>(R, row, j));
        Piece<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; i++) o.v[i] = (T)s[i];
        store_piece<T, VEC>(out + row * R.dim + c, o);
    }
}
template <class T, int VEC, int K>
__global__ __launch_bounds__(256) void from_experts_kernel(Rows R, const T *__restrict__ y,
                                                           T *__restrict__ out) {
    for_rows(R, [&](uint64_t row, uint32_t lane) {
        from_experts_row<T, VEC, K>(R, y, out, row, lane);
    });
}

// The gradients of from_experts: dy = weight * g to the place, dweight = <g, y> there; a row of
// g is read once for K columns, and not once for each, and two pieces of a lane are on their
// way (30,001 rows of 515 float32 cells with 4 columns: 141 -> 124 -> 119 us, 4.7 TB/s).
template <class T, int VEC, int K>
__device__ __forceinline__ void from_experts_grad_row(const Rows &R, const T *__restrict__ g,
                                                      const T *__restrict__ y,
                                                      T *__restrict__ dy,
                                                      float *__restrict__ dweights, uint64_t row,
                                                      uint32_t lane) {
    for (uint32_t j = 0; j < R.n_columns; j += K) {
        const Columns<K> C(R, row, j);
        float dot[K] = {};
#pragma unroll 2
        for (uint32_t p = lane; p < R.pieces; p += 1u << R.lg_g) {
            const uint32_t c = min(p * VEC, R.dim - VEC), twice = p * VEC - c;
            const Piece<T, VEC> v = load_piece<T, VEC>(g + row * R.dim + c);
            Piece<T, VEC> u[K] = {};
            if (dweights)
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (C.is[k]) u[k] = load_piece<T, VEC>(y + C.at[k] + c);
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (j + k >= R.n_columns) continue;
                if (dy) {
                    Piece<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        o.v[i] = C.is[k] ? (T)(C.weight[k] * (float)v.v[i]) : (T)0.0f;
                    store_piece<T, VEC>(dy + C.at[k] + c, o);
                }
                // (cells that the piece before has too count once)
                if (C.is[k])
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        if ((uint32_t)i >= twice) dot[k] += (float)v.v[i] * (float)u[k].v[i];
            }
        }
        if (!dweights) continue;
#pragma unroll
        for (int k = 0; k < K; k++) {
            for (uint32_t d = 1u << R.lg_g; d >>= 1;) dot[k] += __shfl_xor(dot[k], d);
            if (lane == 0 && j + k < R.n_columns) dweights[row * R.n_columns + j + k] = dot[k];
        }
    }
}
template <class T, int VEC, int K>
__global__ __launch_bounds__(256) void from_experts_grad_kernel(Rows R, const T *__restrict__ g,
                                                                const T *__restrict__ y,
                                                                T *__restrict__ dy,
                                                                float *__restrict__ dweights) {
    for_rows(R, [&](uint64_t row, uint32_t lane) {
        from_experts_grad_row<T, VEC, K>(R, g, y, dy, dweights, row, lane);
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

// Positions a thread: more of them where the device is full without, as a chunk's counts are
// written and read besides (in us, 2 and 8 a thread: 65k positions of 511 experts 8.9 and 12.7,
// 524k 13.8 and 14.1, 1M 19.2 and 16.5; of 64 experts 524k 10.8 and 12.7, 1M 15.2 and 13.7).
uint32_t route_rounds(uint64_t n) {
    if (n <= ROUTE_ONE) return n <= ROUTE_TPB ? 1 : n <= 2 * ROUTE_TPB ? 2 : 8;
    return n <= 512 * 2 * ROUTE_TPB ? 2 : 8;
}
uint64_t route_chunks(uint64_t n) {
    const uint64_t chunk = (uint64_t)ROUTE_TPB * route_rounds(n);
    return (n + chunk - 1) / chunk;
}
uint64_t route_bytes(uint64_t n, uint32_t n_experts) {
    return n <= ROUTE_ONE ? 0 : (n_experts + 1) * (route_chunks(n) + 1) * 4;
}

void launch_route(const Route &R, hipStream_t s) {
    const uint32_t rounds = route_rounds(R.n);
    if (R.n > ROUTE_ONE) {
        launch(rounds == 2 ? route_count_kernel<2> : route_count_kernel<8>, R.chunks, ROUTE_TPB,
               s, R);
        launch(route_scan_kernel, R.n_experts / SCAN_EXPERTS + 1, SCAN_EXPERTS * SCAN_PARTS, s, R);
    }
    const auto place = [&](auto b) {
        constexpr uint32_t B = decltype(b)::value;
        launch(R.n > ROUTE_ONE ? (rounds == 2 ? route_place_kernel<2, B, false>
                                              : route_place_kernel<8, B, false>)
               : rounds == 1   ? route_place_kernel<1, B, true>
               : rounds == 2   ? route_place_kernel<2, B, true>
                               : route_place_kernel<8, B, true>,
               R.chunks, ROUTE_TPB, s, R);
    };
    // (numbers up to n_experts, which stands for none)
    if (R.n_experts < 16) place(std::integral_constant<uint32_t, 4>{});
    else if (R.n_experts < 128) place(std::integral_constant<uint32_t, 7>{});
    else if (R.n_experts < 512) place(std::integral_constant<uint32_t, 9>{});
    else place(std::integral_constant<uint32_t, 11>{});
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

// f(columns side by side)
template <class F>
void with_columns(uint32_t n_columns, F &&f) {
    if (n_columns == 1) f(std::integral_constant<int, 1>{});
    else if (n_columns == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
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
        const uint64_t need = route_bytes(n_positions, n_experts);
        head_input(need == 0 || (work && work_bytes >= need), "the workspace is too small");
        head_input(need == 0 || reinterpret_cast<uintptr_t>(work) % 4 == 0,
                   "the workspace must be 4-byte aligned");
        const OnDevice on(device);
        Route R{ids, id_type, (uint32_t)n_positions, n_experts,
                (uint32_t)std::max<uint64_t>(route_chunks(n_positions), 1), order, place, starts,
                static_cast<uint32_t *>(work), nullptr};
        if (need) R.totals = R.counts + (uint64_t)(n_experts + 1) * R.chunks;
        launch_route(R, static_cast<hipStream_t>(stream));
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
            with_columns(n_columns, [&](auto k) {
                launch(from_experts_kernel<T, decltype(v)::value, decltype(k)::value>,
                       row_blocks(R), 256, static_cast<hipStream_t>(stream), R,
                       static_cast<const T *>(y), static_cast<T *>(out));
            });
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
            with_columns(n_columns, [&](auto k) {
                launch(from_experts_grad_kernel<T, decltype(v)::value, decltype(k)::value>,
                       row_blocks(R), 256, static_cast<hipStream_t>(stream), R,
                       static_cast<const T *>(grad), static_cast<const T *>(y),
                       static_cast<T *>(dy), dweights);
            });
        });
    });
}

}  // extern "C"
