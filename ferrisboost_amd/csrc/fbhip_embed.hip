// Embeddings of ids: rows of a table looked up, as they are or summed over a row's
// columns, and the table's gradient by sorted tokens.
//
// Every column's ids have their own part of the table (first[t] .. first[t + 1]), as a
// model's trees have their own leaves and its categorical columns their own codes. A
// position (row, column) whose id is outside its column, or that the counter-based
// generator drops, takes and gives nothing.
#include <algorithm>
#include <type_traits>

#include "fbhip_heads.h"

namespace fbh {
namespace {

constexpr uint32_t NO_TOKEN = 0xFFFFFFFFu;
constexpr uint32_t EMB_TPB = 256;
constexpr uint32_t EMB_MAX_DIM = 32768;
constexpr uint32_t EMB_MAX_COLUMNS = 32768;

// The positions of a call: ids, columns and what is dropped.
struct Positions {
    const void *ids;
    const uint32_t *first;
    uint64_t n_rows;
    uint32_t n_columns, n_tokens;
    uint64_t key;
    uint32_t threshold;
};

template <int ID>
__device__ __forceinline__ uint32_t load_id(const void *ids, uint64_t at) {
    if (ID == FBH_ID_I32) {
        const int32_t v = static_cast<const int32_t *>(ids)[at];
        return (uint32_t)v;  // (negative: above any column)
    } else if (ID == FBH_ID_I64) {
        const int64_t v = static_cast<const int64_t *>(ids)[at];
        return (uint64_t)v < NO_TOKEN ? (uint32_t)v : NO_TOKEN;
    } else {
        const float v = static_cast<const float *>(ids)[at];
        const uint32_t u = v >= 0.0f && v < 4294967040.0f ? (uint32_t)v : NO_TOKEN;
        return (float)u == v ? u : NO_TOKEN;
    }
}

// The table row of a position, or NO_TOKEN.
template <int ID, bool DROP>
__device__ __forceinline__ uint32_t token_at(const Positions &P, uint64_t pos, uint32_t column) {
    const uint32_t id = load_id<ID>(P.ids, pos);
    uint32_t base = 0, size = P.n_tokens;
    if (P.first) {
        base = P.first[column];
        size = P.first[column + 1] - base;
    }
    bool ok = id < size && id < P.n_tokens && base < P.n_tokens - id;
    if (DROP) ok = ok && drop_bits(P.key, pos) >= P.threshold;
    return ok ? base + id : NO_TOKEN;
}

// l / d for l + d below 2^31 and l * d below 2^32 (d > 1: m = ceil(2^32 / d)).
struct Divisor {
    uint32_t d, m;
};
Divisor divisor(uint32_t d) {
    return {d, d > 1 ? (uint32_t)((0x100000000ull + d - 1) / d) : 0u};
}
__device__ __forceinline__ uint32_t divide(uint32_t l, Divisor v) {
    return v.d > 1 ? __umulhi(l, v.m) : l;
}

// ------------------------------------------------------------------- looked up
constexpr uint32_t ROW_PIECES = 4;  // pieces of a thread, all requested at once

// out[pos] = s * table[token(pos)]: the output in pieces of VEC cells, flat over the
// workgroups. A vector's last piece starts at dim - VEC, so that no piece is partial;
// the cells it shares with the piece before are written twice, with the same value.
template <class T, int VEC, int ID, bool DROP>
__global__ __launch_bounds__(EMB_TPB) void embed_rows_kernel(Positions P, const T *table, T *out,
                                                             uint32_t dim, Divisor pieces,
                                                             Divisor columns, float s) {
    const uint64_t block = blockIdx.x + (uint64_t)blockIdx.y * gridDim.x;
    const uint64_t base = block * (EMB_TPB * ROW_PIECES);
    const uint64_t n_pos = P.n_rows * P.n_columns;
    const uint64_t pos0 = base / pieces.d;
    const uint32_t rem0 = (uint32_t)(base - pos0 * pieces.d);
    const uint32_t col0 = (uint32_t)(pos0 % columns.d);
    uint64_t at[ROW_PIECES];
    uint32_t tok[ROW_PIECES], cell[ROW_PIECES];
#pragma unroll
    for (uint32_t k = 0; k < ROW_PIECES; k++) {
        const uint32_t l = rem0 + k * EMB_TPB + threadIdx.x;
        const uint32_t q = divide(l, pieces);
        at[k] = pos0 + q;
        cell[k] = min((l - q * pieces.d) * VEC, dim - VEC);
        const uint32_t c = col0 + q;
        tok[k] = at[k] < n_pos
                     ? token_at<ID, DROP>(P, at[k], c - divide(c, columns) * columns.d)
                     : NO_TOKEN;
    }
    Piece<T, VEC> p[ROW_PIECES];
#pragma unroll
    for (uint32_t k = 0; k < ROW_PIECES; k++)
        p[k] = load_piece<T, VEC>(table + (uint64_t)(tok[k] == NO_TOKEN ? 0 : tok[k]) * dim +
                                  cell[k]);
#pragma unroll
    for (uint32_t k = 0; k < ROW_PIECES; k++) {
        if (at[k] >= n_pos) continue;
#pragma unroll
        for (int i = 0; i < VEC; i++)
            p[k].v[i] = tok[k] == NO_TOKEN ? (T)0.0f : (T)((float)p[k].v[i] * s);
        store_piece<T, VEC>(out + at[k] * dim + cell[k], p[k]);
    }
}

// ------------------------------------------------------------------- summed
// out[row] = s * (sum over columns of table[token]). Column t goes to sum t % 8 and the
// eight sums are added in a tree, in both kernels, so a row's result does not depend on
// the rows beside it.
__device__ __forceinline__ float tree8(const float *a) {
    return ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
}

// A workgroup takes 256 / G rows, G = 2^lg_g lanes a row; the tokens of 2^lg_c columns at
// a time are found by all threads in turn and kept in LDS, so that an id is decoded (and
// its bits drawn) once and not by every lane of its row.
template <class T, int VEC, int ID, bool DROP>
__global__ __launch_bounds__(EMB_TPB) void embed_sum_kernel(Positions P, const T *table, T *out,
                                                            uint32_t dim, uint32_t n_pieces,
                                                            uint32_t lg_g, uint32_t lg_c,
                                                            float s) {
    extern __shared__ uint32_t toks[];
    const uint32_t rows = EMB_TPB >> lg_g, cols = 1u << lg_c, pitch = cols + 4;
    const uint64_t row0 = (uint64_t)blockIdx.x * rows;
    const uint32_t r = threadIdx.x >> lg_g;
    const uint32_t piece = blockIdx.y * (1u << lg_g) + (threadIdx.x & ((1u << lg_g) - 1));
    const bool live = row0 + r < P.n_rows && piece < n_pieces;
    const uint32_t cell = min(piece * VEC, dim - VEC);
    const T *from = table + (live ? cell : 0);
    float a[VEC][8];
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) a[i][j] = 0.0f;
    for (uint32_t t0 = 0; t0 < P.n_columns; t0 += cols) {
        for (uint32_t i = threadIdx.x; i < rows << lg_c; i += EMB_TPB) {
            const uint32_t rr = i >> lg_c, t = t0 + (i & (cols - 1));
            toks[rr * pitch + (i & (cols - 1))] =
                row0 + rr < P.n_rows && t < P.n_columns
                    ? token_at<ID, DROP>(P, (row0 + rr) * P.n_columns + t, t)
                    : NO_TOKEN;
        }
        __syncthreads();
        const uint32_t most = min(cols, P.n_columns - t0);
        if (live)
            for (uint32_t c = 0; c < most; c += 8) {
                uint32_t tok[8];
                Piece<T, VEC> p[8];
                *reinterpret_cast<uint4 *>(tok) =
                    *reinterpret_cast<const uint4 *>(&toks[r * pitch + c]);
                *reinterpret_cast<uint4 *>(tok + 4) =
                    *reinterpret_cast<const uint4 *>(&toks[r * pitch + c + 4]);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    p[j] = load_piece<T, VEC>(from +
                                              (uint64_t)(tok[j] == NO_TOKEN ? 0 : tok[j]) * dim);
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        a[i][j] += tok[j] == NO_TOKEN ? 0.0f : (float)p[j].v[i];
            }
        __syncthreads();
    }
    if (!live) return;
    Piece<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; i++) o.v[i] = (T)(tree8(a[i]) * s);
    store_piece<T, VEC>(out + (row0 + r) * dim + cell, o);
}

// Few rows: the eight sums of a row side by side, a workgroup a row and 2^lg_g pieces.
template <class T, int VEC, int ID, bool DROP>
__global__ void embed_sum_few_kernel(Positions P, const T *table, T *out, uint32_t dim,
                                     uint32_t n_pieces, uint32_t lg_g, float s) {
    extern __shared__ float sums[];
    const uint64_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x & ((1u << lg_g) - 1), j = threadIdx.x >> lg_g;
    const uint32_t piece = (blockIdx.y << lg_g) + lane;
    const bool live = piece < n_pieces;
    const uint32_t cell = live ? min(piece * VEC, dim - VEC) : 0;
    float a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) a[i] = 0.0f;
    for (uint32_t t0 = j; t0 < P.n_columns; t0 += 64) {
        uint32_t tok[8];
        Piece<T, VEC> p[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            const uint32_t t = t0 + 8 * k;
            tok[k] = t < P.n_columns ? token_at<ID, DROP>(P, row * P.n_columns + t, t) : NO_TOKEN;
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
            p[k] = load_piece<T, VEC>(table + (uint64_t)(tok[k] == NO_TOKEN ? 0 : tok[k]) * dim +
                                      cell);
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
#pragma unroll
            for (int i = 0; i < VEC; i++) a[i] += tok[k] == NO_TOKEN ? 0.0f : (float)p[k].v[i];
    }
    float *mine = sums + ((j << lg_g) + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; i++) mine[i] = a[i];
    __syncthreads();
    if (j || !live) return;
    Piece<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        float b[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) b[k] = sums[((k << lg_g) + lane) * VEC + i];
        o.v[i] = (T)(tree8(b) * s);
    }
    store_piece<T, VEC>(out + row * dim + cell, o);
}

// ------------------------------------------------------------------- gradient
// Positions are sorted by token, stably (radix passes of at most 8 bits), so each
// token's positions stand together in their own order; then runs of equal tokens are
// summed in f32. The sorted positions are cut into chunks of equal length: a run inside
// one chunk goes to the table, the parts of longer runs are joined in chunk order. All
// orders are fixed, so the gradient is the same in every call.
constexpr uint32_t SORT_TPB = 256;
constexpr uint32_t SORT_ROUNDS = 16;
constexpr uint32_t SORT_ITEMS = SORT_TPB * SORT_ROUNDS;
constexpr uint32_t SORT_WAVES = SORT_TPB / 64;

// What a pass sorts: positions decoded from the ids (pass 0), or the pass before's output.
struct SortFrom {
    const uint32_t *keys, *vals;
    uint32_t n;       // positions
    uint32_t shift, bits;
    uint32_t per_row; // pooled: the columns of a row, whose positions share its gradient
};

template <int ID, bool DROP, bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const Positions &P, const SortFrom &S, uint32_t i) {
    if (!FIRST) return S.keys[i];
    const uint32_t tok = token_at<ID, DROP>(P, i, P.n_columns > 1 ? i % P.n_columns : 0);
    return tok == NO_TOKEN ? P.n_tokens : tok;  // the last key of all
}

// counts[digit * blocks + block]
template <int ID, bool DROP, bool FIRST>
__global__ __launch_bounds__(SORT_TPB) void sort_count_kernel(Positions P, SortFrom S,
                                                              uint32_t *counts) {
    __shared__ uint32_t c[256];
    c[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * SORT_ITEMS, mask = (1u << S.bits) - 1;
#pragma unroll 4
    for (uint32_t r = 0; r < SORT_ROUNDS; r++) {
        const uint32_t i = base + r * SORT_TPB + threadIdx.x;
        if (i < S.n)
            atomicAdd(&c[(sort_key<ID, DROP, FIRST>(P, S, i) >> S.shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x <= mask) counts[(uint64_t)threadIdx.x * gridDim.x + blockIdx.x] = c[threadIdx.x];
}

// A digit's counts to the positions before them in its own part; its total.
__global__ __launch_bounds__(SORT_TPB) void sort_scan_kernel(uint32_t *counts, uint32_t blocks,
                                                             uint32_t *totals) {
    __shared__ uint32_t wave[SORT_WAVES];
    uint32_t *mine = counts + (uint64_t)blockIdx.x * blocks;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < blocks; b0 += SORT_TPB) {
        const uint32_t b = b0 + threadIdx.x;
        const uint32_t v = b < blocks ? mine[b] : 0;
        uint32_t x = v;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(x, d);
            if ((threadIdx.x & 63) >= (uint32_t)d) x += y;
        }
        if ((threadIdx.x & 63) == 63) wave[threadIdx.x / 64] = x;
        __syncthreads();
        uint32_t add = before;
        for (uint32_t w = 0; w < SORT_WAVES; w++) {
            if (w < threadIdx.x / 64) add += wave[w];
            before += wave[w];
        }
        if (b < blocks) mine[b] = add + x - v;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Items of equal digits keep their order: a wave's 16 rounds are one after the other, a
// lane's place in its round is the number of lower lanes with its digit, and the waves'
// counts are summed up in wave order.
template <int ID, bool DROP, bool FIRST>
__global__ __launch_bounds__(SORT_TPB) void sort_scatter_kernel(Positions P, SortFrom S,
                                                                const uint32_t *counts,
                                                                const uint32_t *totals,
                                                                uint32_t *keys, uint32_t *vals) {
    __shared__ uint32_t base[256];
    __shared__ uint32_t seen[SORT_WAVES][256];
    __shared__ uint32_t wave_sum[SORT_WAVES];
    const uint32_t mask = (1u << S.bits) - 1, lane = threadIdx.x & 63, w = threadIdx.x / 64;
    {
        const uint32_t v = threadIdx.x <= mask ? totals[threadIdx.x] : 0;
        uint32_t x = v;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(x, d);
            if (lane >= (uint32_t)d) x += y;
        }
        if (lane == 63) wave_sum[w] = x;
        for (uint32_t k = 0; k < SORT_WAVES; k++) seen[k][threadIdx.x] = 0;
        __syncthreads();
        uint32_t add = 0;
        for (uint32_t k = 0; k < w; k++) add += wave_sum[k];
        if (threadIdx.x <= mask)
            base[threadIdx.x] =
                add + x - v + counts[(uint64_t)threadIdx.x * gridDim.x + blockIdx.x];
    }
    const uint32_t first = blockIdx.x * SORT_ITEMS + w * (SORT_ROUNDS * 64) + lane;
    uint32_t key[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
    for (uint32_t r = 0; r < SORT_ROUNDS; r++) {
        const uint32_t i = first + r * 64;
        key[r] = i < S.n ? sort_key<ID, DROP, FIRST>(P, S, i) : 0;
    }
    // (a wave's LDS operations complete in order, and only it touches its counters)
#pragma unroll
    for (uint32_t r = 0; r < SORT_ROUNDS; r++) {
        const bool in = first + r * 64 < S.n;
        const uint32_t digit = (key[r] >> S.shift) & mask;
        uint64_t same = __ballot(in);
        for (uint32_t b = 0; b < S.bits; b++) {
            const bool one = (digit >> b) & 1;
            const uint64_t ones = __ballot(one);
            same &= one ? ones : ~ones;
        }
        const uint32_t below = __popcll(same & ((1ull << lane) - 1));
        volatile uint32_t *count = &seen[w][digit];
        uint32_t before = 0;
        if (in) before = *count;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) *count = before + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[r] = before + below;
    }
    __syncthreads();
    if (threadIdx.x <= mask) {
        uint32_t at = base[threadIdx.x];
        for (uint32_t k = 0; k < SORT_WAVES; k++) {
            const uint32_t c = seen[k][threadIdx.x];
            seen[k][threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < SORT_ROUNDS; r++) {
        const uint32_t i = first + r * 64;
        if (i >= S.n) continue;
        const uint32_t at = seen[w][(key[r] >> S.shift) & mask] + rank[r];
        keys[at] = key[r];
        vals[at] = FIRST ? (S.per_row > 1 ? i / S.per_row : i) : S.vals[i];
    }
}

// 16-byte pieces of zeros, and the rest in bytes.
__global__ __launch_bounds__(256) void zero_kernel(uint8_t *p, uint64_t bytes) {
    const uint64_t head = min(bytes, (uint64_t)(-(intptr_t)p & 15));
    const uint64_t pieces = (bytes - head) / 16;
    const uint64_t at = blockIdx.x * 256ull + threadIdx.x, step = gridDim.x * 256ull;
    for (uint64_t i = at; i < pieces; i += step)
        *reinterpret_cast<uint4 *>(p + head + 16 * i) = make_uint4(0, 0, 0, 0);
    if (at < head) p[at] = 0;
    if (at < bytes - head - 16 * pieces) p[head + 16 * pieces + at] = 0;
}

struct Runs {
    const uint32_t *keys, *vals;
    uint32_t n, chunk;  // sorted positions, and a chunk's (a multiple of 8)
    uint32_t n_tokens, dim, n_pieces, lg_g;
    float s;
    float *parts;       // [2 * chunks][dim]
};

// A chunk's sums, 2^lg_g lanes a chunk. Part 2c holds the run that chunk c continues,
// part 2c + 1 the one that starts in it and goes on behind it.
template <class T, int VEC>
__global__ __launch_bounds__(EMB_TPB) void grad_runs_kernel(Runs R, const T *grad, T *table) {
    const uint32_t c = (blockIdx.x * EMB_TPB + threadIdx.x) >> R.lg_g;
    const uint32_t piece =
        (blockIdx.y << R.lg_g) + (threadIdx.x & ((1u << R.lg_g) - 1));
    const uint64_t c0 = (uint64_t)c * R.chunk;
    if (c0 >= R.n || piece >= R.n_pieces) return;
    const uint32_t c1 = (uint32_t)min((uint64_t)R.n, c0 + R.chunk);
    const uint32_t cell = min(piece * VEC, R.dim - VEC);
    const T *from = grad + cell;
    uint32_t key = R.keys[c0];
    bool starts = c0 == 0 || R.keys[c0 - 1] != key;
    float a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) a[i] = 0.0f;
    const auto flush = [&](bool ends) {
        if (key >= R.n_tokens) return;
        if (starts && ends) {
            Piece<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = (T)(a[i] * R.s);
            store_piece<T, VEC>(table + (uint64_t)key * R.dim + cell, o);
        } else {
            Piece<float, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = a[i];
            store_piece<float, VEC>(R.parts + (2ull * c + (starts ? 1 : 0)) * R.dim + cell, o);
        }
    };
    for (uint32_t i0 = (uint32_t)c0; i0 < c1; i0 += 8) {
        uint32_t k[8];
        Piece<T, VEC> p[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            const uint32_t i = min(i0 + j, c1 - 1);
            k[j] = R.keys[i];
            // (positions that give nothing are read from the first row, and not used)
            const uint32_t v = k[j] < R.n_tokens ? R.vals[i] : 0;
            p[j] = load_piece<T, VEC>(from + (uint64_t)v * R.dim);
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            if (i0 + j >= c1) break;
            if (k[j] != key) {
                flush(true);
                key = k[j];
                starts = true;
#pragma unroll
                for (int i = 0; i < VEC; i++) a[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) a[i] += (float)p[j].v[i];
        }
    }
    flush(c1 == R.n || R.keys[c1] != key);
}

constexpr uint32_t JOIN_SHORT = 16;  // parts that one chunk's lanes join by themselves

// Joins the parts of the runs that start in a chunk and go on behind it.
template <class T, int VEC>
__global__ __launch_bounds__(EMB_TPB) void grad_join_kernel(Runs R, T *table) {
    __shared__ uint32_t longs[EMB_TPB], n_longs;
    __shared__ float sums[EMB_TPB * VEC];
    const uint32_t lanes = 1u << R.lg_g, groups = EMB_TPB >> R.lg_g;
    const uint32_t g = threadIdx.x >> R.lg_g, lane = threadIdx.x & (lanes - 1);
    const uint32_t piece = (blockIdx.y << R.lg_g) + lane;
    const bool live = piece < R.n_pieces;
    const uint32_t cell = live ? min(piece * VEC, R.dim - VEC) : 0;
    const uint32_t chunks = (uint32_t)(((uint64_t)R.n + R.chunk - 1) / R.chunk);
    if (threadIdx.x == 0) n_longs = 0;
    __syncthreads();

    // the number of chunks behind c whose first position still has this key
    const auto behind = [&](uint32_t c, uint32_t key, uint32_t most) {
        uint32_t n = 0;
        while (n < most && c + 1 + n < chunks && R.keys[(uint64_t)(c + 1 + n) * R.chunk] == key)
            n++;
        return n;
    };
    const auto write = [&](uint32_t key, const float *a) {
        Piece<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; i++) o.v[i] = (T)(a[i] * R.s);
        store_piece<T, VEC>(table + (uint64_t)key * R.dim + cell, o);
    };

    const uint32_t c = blockIdx.x * groups + g;
    const uint64_t c0 = (uint64_t)c * R.chunk, c1 = c0 + R.chunk;
    if (c1 < R.n) {
        const uint32_t key = R.keys[c1 - 1];
        const bool starts = R.keys[c0] != key || c0 == 0 || R.keys[c0 - 1] != key;
        if (key < R.n_tokens && starts && R.keys[c1] == key) {
            const uint32_t n = behind(c, key, JOIN_SHORT);
            if (n == JOIN_SHORT) {
                if (lane == 0) longs[atomicAdd(&n_longs, 1u)] = c;
            } else if (live) {
                float a[VEC];
                Piece<float, VEC> p = load_piece<float, VEC>(R.parts + (2ull * c + 1) * R.dim + cell);
#pragma unroll
                for (int i = 0; i < VEC; i++) a[i] = p.v[i];
                for (uint32_t k = 1; k <= n; k++) {
                    p = load_piece<float, VEC>(R.parts + 2ull * (c + k) * R.dim + cell);
#pragma unroll
                    for (int i = 0; i < VEC; i++) a[i] += p.v[i];
                }
                write(key, a);
            }
        }
    }
    __syncthreads();
    // Long runs, by all of the workgroup: part k to group k % groups, then the groups'
    // sums in order. (Which run comes first changes nothing.)
    const uint32_t n_runs = n_longs;
    for (uint32_t r = 0; r < n_runs; r++) {
        const uint32_t lc = longs[r];
        const uint32_t key = R.keys[(uint64_t)(lc + 1) * R.chunk - 1];
        // the run's last chunk: doubling steps, then halves
        uint32_t lo = lc + JOIN_SHORT, hi = lo + 1, step = 1;
        while (hi < chunks && R.keys[(uint64_t)hi * R.chunk] == key) {
            lo = hi;
            step *= 2;
            hi = min(lo + step, chunks);
        }
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (R.keys[(uint64_t)mid * R.chunk] == key) lo = mid;
            else hi = mid;
        }
        const uint32_t n = lo - lc + 1;
        float a[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) a[i] = 0.0f;
        if (live)
            for (uint32_t k0 = g; k0 < n; k0 += 4 * groups) {
                Piece<float, VEC> p[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t k = min(k0 + j * groups, n - 1);
                    p[j] = load_piece<float, VEC>(
                        R.parts + (2ull * (lc + k) + (k ? 0 : 1)) * R.dim + cell);
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; j++)
                    if (k0 + j * groups < n)
#pragma unroll
                        for (int i = 0; i < VEC; i++) a[i] += p[j].v[i];
            }
#pragma unroll
        for (int i = 0; i < VEC; i++) sums[threadIdx.x * VEC + i] = a[i];
        __syncthreads();
        if (g == 0 && live) {
            for (uint32_t k = 1; k < groups; k++)
#pragma unroll
                for (int i = 0; i < VEC; i++) a[i] += sums[((k << R.lg_g) + lane) * VEC + i];
            write(key, a);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------- host side
uint32_t lg_at_least(uint64_t n) {
    uint32_t l = 0;
    while ((1ull << l) < n) l++;
    return l;
}

void check_embed(const fbh_embed *e) {
    head_input(e, "null argument");
    head_input(e->dtype <= FBH_BF16, "unknown cell type");
    head_input(e->id_type <= FBH_ID_F32, "unknown id type");
    head_input(e->dim >= 1 && e->dim <= EMB_MAX_DIM, "dim must be in 1..=32768");
    head_input(e->n_columns >= 1, "no columns");
    head_input(!e->first || e->n_columns <= EMB_MAX_COLUMNS,
               "at most 32768 columns with parts of their own");
    head_input(e->n_tokens >= 1 && e->n_tokens <= 0x7FFFFFFFu,
               "n_tokens must be in 1..=2147483647");
    head_input(e->ids || e->n_rows == 0, "null argument");
    head_input(e->n_rows <= (1ull << 40) / e->n_columns, "more than 2^40 positions");
    (void)drop_threshold(e->drop);
}

Positions positions_of(const fbh_embed *e) {
    Positions P{e->ids, e->first, e->n_rows, e->n_columns, e->n_tokens, drop_key(e->seed),
                drop_threshold(e->drop)};
    if (!e->pooled && !e->first) {  // a flat list
        P.n_rows *= P.n_columns;
        P.n_columns = 1;
    }
    return P;
}

float scale_of(const fbh_embed *e) { return (float)((double)e->scale / (1.0 - e->drop)); }

// Cells of a piece: the largest power of two up to 16 bytes and the vector's width.
uint32_t piece_cells(uint32_t dim, uint32_t dtype) {
    uint32_t v = dtype == FBH_F32 ? 4 : 8;
    while (v > dim) v /= 2;
    return v;
}

template <class T, int VEC, int ID, bool DROP>
void launch_embed(const fbh_embed *e, const void *table, void *out, hipStream_t s) {
    const Positions P = positions_of(e);
    const uint32_t pieces = (e->dim + VEC - 1) / VEC;
    const auto *tab = static_cast<const T *>(table);
    auto *to = static_cast<T *>(out);
    const float sc = scale_of(e);
    if (!e->pooled) {
        const uint64_t blocks =
            (P.n_rows * P.n_columns * pieces + EMB_TPB * ROW_PIECES - 1) / (EMB_TPB * ROW_PIECES);
        const uint32_t bx = (uint32_t)std::min<uint64_t>(blocks, 1u << 22);
        const uint64_t by = (blocks + bx - 1) / bx;
        head_input(by <= 65535, "too many cells");
        hipLaunchKernelGGL((embed_rows_kernel<T, VEC, ID, DROP>), dim3(bx, (uint32_t)by),
                           dim3(EMB_TPB), 0, s, P, tab, to, e->dim, divisor(pieces),
                           divisor(P.n_columns), sc);
    } else if (P.n_rows * pieces < 64 * EMB_TPB) {
        const uint32_t lg_g = std::min(lg_at_least(pieces), 5u);
        hipLaunchKernelGGL((embed_sum_few_kernel<T, VEC, ID, DROP>),
                           dim3((uint32_t)P.n_rows, (pieces + (1u << lg_g) - 1) >> lg_g),
                           dim3(8u << lg_g), (size_t)(8u << lg_g) * VEC * sizeof(float), s, P, tab,
                           to, e->dim, pieces, lg_g, sc);
    } else {
        const uint32_t lg_g = std::min(lg_at_least(pieces), 6u), rows = EMB_TPB >> lg_g;
        const uint32_t lg_c =
            std::min(std::max(lg_at_least(P.n_columns), 3u), lg_at_least(4096 / rows));
        const uint64_t blocks = (P.n_rows + rows - 1) / rows;
        head_input(blocks < 1u << 24, "too many rows");
        hipLaunchKernelGGL((embed_sum_kernel<T, VEC, ID, DROP>),
                           dim3((uint32_t)blocks, (pieces + (1u << lg_g) - 1) >> lg_g),
                           dim3(EMB_TPB), (size_t)rows * ((1u << lg_c) + 4) * 4, s, P, tab, to,
                           e->dim, pieces, lg_g, lg_c, sc);
    }
    head_check(hipGetLastError(), "embedding");
}

template <int N>
using Int = std::integral_constant<int, N>;

// Calls f(a cell, Int<VEC>) for the cells and pieces of a call.
template <class F>
void with_cells(uint32_t dtype, uint32_t vec, F &&f) {
    const auto pieces = [&](auto cell) {
        if constexpr (sizeof(cell) == 2)
            if (vec == 8) return f(cell, Int<8>{});
        if (vec == 4) return f(cell, Int<4>{});
        if (vec == 2) return f(cell, Int<2>{});
        return f(cell, Int<1>{});
    };
    if (dtype == FBH_F32) pieces(float{});
    else if (dtype == FBH_F16) pieces(_Float16{});
    else pieces(__bf16{});
}

// Calls f(Int<id type>, whether positions are dropped).
template <class F>
void with_ids(uint32_t id_type, bool drop, F &&f) {
    const auto go = [&](auto dropped) {
        if (id_type == FBH_ID_I32) f(Int<FBH_ID_I32>{}, dropped);
        else if (id_type == FBH_ID_I64) f(Int<FBH_ID_I64>{}, dropped);
        else f(Int<FBH_ID_F32>{}, dropped);
    };
    if (drop) go(std::true_type{});
    else go(std::false_type{});
}

// The gradient's workspace: two lists of sorted positions, a pass' counts, runs' parts.
struct GradPlan {
    uint32_t n = 0, passes = 0, bits = 0, blocks = 0, vec = 0, pieces = 0, lg_g = 0, chunk = 0,
             chunks = 0;
    uint64_t keys[2], vals[2], counts = 0, totals = 0, parts = 0, bytes = 0;
};

GradPlan grad_plan(const fbh_embed *e) {
    GradPlan G;
    const uint64_t n = e->n_rows * e->n_columns;
    head_input(n <= 0x7FFFFFFFull, "a gradient takes at most 2^31 - 1 positions");
    G.n = (uint32_t)n;
    const uint32_t key_bits = lg_at_least((uint64_t)e->n_tokens + 1);  // n_tokens: nothing
    G.passes = (key_bits + 7) / 8;
    G.bits = (key_bits + G.passes - 1) / G.passes;
    G.blocks = (uint32_t)((n + SORT_ITEMS - 1) / SORT_ITEMS);
    G.vec = piece_cells(e->dim, e->dtype);
    G.pieces = (e->dim + G.vec - 1) / G.vec;
    G.lg_g = std::min(lg_at_least(G.pieces), 6u);
    // Chunks for every thread that the device runs at once (256 CUs of 2048), of 16 to
    // 256 positions.
    const uint64_t lanes = (uint64_t)((G.pieces + (1u << G.lg_g) - 1) >> G.lg_g) << G.lg_g;
    const uint64_t c = (n * lanes + (256 * 2048 - 1)) / (256 * 2048);
    G.chunk = (uint32_t)((std::min<uint64_t>(std::max<uint64_t>(c, 16), 256) + 7) & ~7ull);
    G.chunks = (uint32_t)((n + G.chunk - 1) / G.chunk);
    const auto take = [&](uint64_t bytes) {
        const uint64_t at = G.bytes;
        G.bytes = (at + bytes + 255) & ~255ull;
        return at;
    };
    for (int i = 0; i < 2; i++) {
        G.keys[i] = take(4 * n);
        G.vals[i] = take(4 * n);
    }
    G.counts = take(4ull * (1u << G.bits) * G.blocks);
    G.totals = take(4 * 256);
    G.parts = take(8ull * G.chunks * e->dim);
    return G;
}

void embed_grad(const fbh_embed *e, const void *grad, void *table, void *work, hipStream_t s) {
    Positions P{e->ids, e->first, e->n_rows, e->n_columns, e->n_tokens, drop_key(e->seed),
                drop_threshold(e->drop)};
    if (!e->first) {
        P.n_rows *= P.n_columns;
        P.n_columns = 1;
    }
    const uint64_t bytes =
        (uint64_t)e->n_tokens * e->dim * (e->dtype == FBH_F32 ? 4 : 2);
    hipLaunchKernelGGL(zero_kernel, dim3((uint32_t)std::min<uint64_t>((bytes + 4095) / 4096, 4096)),
                       dim3(256), 0, s, static_cast<uint8_t *>(table), bytes);
    head_check(hipGetLastError(), "table gradient");
    const GradPlan G = grad_plan(e);
    if (G.n == 0) return;
    auto *w = static_cast<uint8_t *>(work);
    const auto list = [&](uint64_t at) { return reinterpret_cast<uint32_t *>(w + at); };
    uint32_t *counts = list(G.counts), *totals = list(G.totals);
    for (uint32_t pass = 0; pass < G.passes; pass++) {
        const uint32_t to = pass & 1;
        const SortFrom S{list(G.keys[1 - to]), list(G.vals[1 - to]), G.n, pass * G.bits, G.bits,
                         e->pooled ? e->n_columns : 1};
        uint32_t *keys = list(G.keys[to]), *vals = list(G.vals[to]);
        const auto go = [&](auto id, auto drop, auto first) {
            constexpr int ID = decltype(id)::value;
            constexpr bool DROP = decltype(drop)::value, FIRST = decltype(first)::value;
            hipLaunchKernelGGL((sort_count_kernel<ID, DROP, FIRST>), dim3(G.blocks), dim3(SORT_TPB),
                               0, s, P, S, counts);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(1u << G.bits), dim3(SORT_TPB), 0, s, counts,
                               G.blocks, totals);
            hipLaunchKernelGGL((sort_scatter_kernel<ID, DROP, FIRST>), dim3(G.blocks),
                               dim3(SORT_TPB), 0, s, P, S, counts, totals, keys, vals);
        };
        if (pass == 0)
            with_ids(e->id_type, e->drop > 0.0,
                     [&](auto id, auto drop) { go(id, drop, std::true_type{}); });
        else go(Int<FBH_ID_I32>{}, std::false_type{}, std::false_type{});
        head_check(hipGetLastError(), "token sort");
    }
    const uint32_t at = (G.passes - 1) & 1;
    const Runs R{list(G.keys[at]), list(G.vals[at]), G.n, G.chunk, e->n_tokens, e->dim, G.pieces,
                 G.lg_g, scale_of(e), reinterpret_cast<float *>(w + G.parts)};
    with_cells(e->dtype, G.vec, [&](auto one, auto vec) {
        using T = decltype(one);
        constexpr int VEC = decltype(vec)::value;
        const uint32_t groups = EMB_TPB >> G.lg_g;
        const dim3 grid((G.chunks + groups - 1) / groups,
                        (G.pieces + (1u << G.lg_g) - 1) >> G.lg_g);
        hipLaunchKernelGGL((grad_runs_kernel<T, VEC>), grid, dim3(EMB_TPB), 0, s, R,
                           static_cast<const T *>(grad), static_cast<T *>(table));
        hipLaunchKernelGGL((grad_join_kernel<T, VEC>), grid, dim3(EMB_TPB), 0, s, R,
                           static_cast<T *>(table));
    });
    head_check(hipGetLastError(), "table gradient");
}

}  // namespace
}  // namespace fbh

using namespace fbh;

extern "C" {

int fbh_embed_rows(int device, const fbh_embed *e, const void *table, void *out, void *stream) {
    return head_guard([&] {
        check_embed(e);
        if (e->n_rows == 0) return;
        head_input(table && out, "null argument");
        const OnDevice on(device);
        const auto s = static_cast<hipStream_t>(stream);
        with_cells(e->dtype, piece_cells(e->dim, e->dtype), [&](auto cell, auto vec) {
            with_ids(e->id_type, e->drop > 0.0, [&](auto id, auto drop) {
                launch_embed<decltype(cell), decltype(vec)::value, decltype(id)::value,
                             decltype(drop)::value>(e, table, out, s);
            });
        });
    });
}

uint64_t fbh_embed_grad_bytes(const fbh_embed *e) {
    uint64_t bytes = 0;
    (void)head_guard([&] {
        check_embed(e);
        bytes = grad_plan(e).bytes;
    });
    return bytes;
}

int fbh_embed_grad(int device, const fbh_embed *e, const void *grad, void *table, void *work,
                   uint64_t work_bytes, void *stream) {
    return head_guard([&] {
        check_embed(e);
        head_input(table && (grad || e->n_rows == 0), "null argument");
        const uint64_t need = grad_plan(e).bytes;
        head_input(work_bytes >= need && (work || need == 0), "the workspace is too small");
        const OnDevice on(device);
        embed_grad(e, grad, table, work, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
