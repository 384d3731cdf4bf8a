// Embeddings of ids: rows of a table looked up, as they are or summed over a row's
// columns, and the table's gradient by sorted tokens.
//
// Every column's ids have their own part of the table (first[t] .. first[t + 1]), as a
// model's trees have their own leaves and its categorical columns their own codes. A
// position (row, column) whose id is outside its column, or that the counter-based
// generator drops, takes and gives nothing.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fbhip_heads.h"

namespace fbh {
namespace {

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

// A column's part of the table, inside it whatever `first` says.
struct Part {
    uint32_t base, size;
};
__device__ __forceinline__ Part part_of(const Positions &P, uint32_t column) {
    if (!P.first) return {0, P.n_tokens};
    const uint32_t base = min(P.first[column], P.n_tokens);
    return {base, min(P.first[column + 1] - base, P.n_tokens - base)};
}

// The table row of a position, or NO_TOKEN.
template <bool DROP>
__device__ __forceinline__ uint32_t token_of(const Positions &P, Part part, uint32_t id,
                                             uint32_t bits) {
    return id < part.size && (!DROP || bits >= P.threshold) ? part.base + id : NO_TOKEN;
}
template <int ID, bool DROP>
__device__ __forceinline__ uint32_t token_at(const Positions &P, uint64_t pos, uint32_t column) {
    return token_of<DROP>(P, part_of(P, column), load_id<ID>(P.ids, pos),
                          DROP ? drop_bits(P.key, pos) : 0);
}
// The bits of two positions of a thread whose neighbours in the wave hold the next columns,
// from an even one on; rows of an even number of columns start with an even position.
template <bool DROP>
__device__ __forceinline__ void bits_of_two(const Positions &P, const uint64_t (&pos)[2],
                                            uint32_t (&bits)[2]) {
    if (!DROP) return;
    if (P.n_columns % 2 == 0) drop_bits_of_neighbours(P.key, pos, bits);
    else
        for (int k = 0; k < 2; k++) bits[k] = drop_bits(P.key, pos[k]);
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
constexpr uint32_t ROW_BLOCK = EMB_TPB * ROW_PIECES;

// out[pos] = s * table[token(pos)]: the output in pieces of VEC cells, flat over the
// workgroups, whose positions' tokens are found once and kept in LDS. Bound by the output:
// 2M x 20 ids and vectors of 32 bytes take 201 us (1.44 GB, 7.2 TB/s; a fill reaches 6.9)
// after 26 us of reading the ids where a pass before has left these in the last-level cache,
// and 320 to 335 in all where they come from memory. A vector's last piece starts at
// dim - VEC, so that no piece is partial; the cells it shares with the piece before are
// written twice, with the same value.
// PAST: written past the caches (a parameter, as the compiler would join the two stores of a
// branch into an ordinary one).
template <class T, int VEC, int ID, bool DROP, bool PAST>
__global__ __launch_bounds__(EMB_TPB) void embed_rows_kernel(Positions P, const T *table, T *out,
                                                             uint32_t dim, Divisor pieces,
                                                             Divisor columns, float s,
                                                             uint64_t block0) {
    __shared__ uint32_t toks[ROW_BLOCK + 1];
    const uint64_t base = (block0 + blockIdx.x) * ROW_BLOCK;
    const uint64_t n_pos = P.n_rows * P.n_columns;
    const uint64_t pos0 = base / pieces.d;
    const uint32_t rem0 = (uint32_t)(base - pos0 * pieces.d);
    const uint32_t col0 = (uint32_t)(pos0 % columns.d);
    const uint32_t n = divide(rem0 + ROW_BLOCK - 1, pieces) + 1;  // positions of the block
    for (uint32_t q = threadIdx.x; q < n; q += EMB_TPB) {
        const uint32_t c = col0 + q;
        toks[q] = pos0 + q < n_pos ? token_at<ID, DROP>(P, pos0 + q,
                                                        c - divide(c, columns) * columns.d)
                                   : NO_TOKEN;
    }
    __syncthreads();
    uint32_t q[ROW_PIECES], tok[ROW_PIECES], cell[ROW_PIECES];
    Piece<T, VEC> p[ROW_PIECES];
#pragma unroll
    for (uint32_t k = 0; k < ROW_PIECES; k++) {
        const uint32_t l = rem0 + k * EMB_TPB + threadIdx.x;
        q[k] = divide(l, pieces);
        cell[k] = min((l - q[k] * pieces.d) * VEC, dim - VEC);
        tok[k] = toks[q[k]];
        p[k] = load_piece<T, VEC>(table + (uint64_t)(tok[k] == NO_TOKEN ? 0 : tok[k]) * dim +
                                  cell[k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < ROW_PIECES; k++) {
        if (pos0 + q[k] >= n_pos) continue;
        if (tok[k] == NO_TOKEN) p[k] = Piece<T, VEC>{};
        if (s != 1.0f)  // (the same for all: unscaled vectors are moved as they are)
#pragma unroll
            for (int i = 0; i < VEC; i++) p[k].v[i] = (T)((float)p[k].v[i] * s);
        T *to = out + (pos0 + q[k]) * dim + cell[k];
        if constexpr (PAST) stream_piece<T, VEC>(to, p[k]);
        else store_piece<T, VEC>(to, p[k]);
    }
}

// Ids that come from memory while their vectors are written past the caches wait behind
// those writes, and what is written waits for them. So they are read into the last-level
// cache first, a part of the rows at a time that it holds (TOUCH_BYTES of ids): 1.28 GB out
// take 405 -> 320 to 335 us as vectors of 32 bytes. Where the ids are few beside the vectors it
// costs a little: 221 -> 228 us for vectors of 128 bytes, 220 -> 225 for 256.
constexpr uint64_t TOUCH_BYTES = 160ull << 20;

__global__ __launch_bounds__(256) void touch_kernel(const uint8_t *p, uint64_t pieces) {
    uint32_t x = 0;
    const uint64_t step = gridDim.x * 256ull;
    uint64_t i = blockIdx.x * 256ull + threadIdx.x;
    for (; i + 3 * step < pieces; i += 4 * step) {
        Piece<uint32_t, 4> q[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            q[k] = load_piece<uint32_t, 4>(reinterpret_cast<const uint32_t *>(p + 16 * (i + k * step)));
#pragma unroll
        for (int k = 0; k < 4; k++) x ^= q[k].v[0] ^ q[k].v[1] ^ q[k].v[2] ^ q[k].v[3];
    }
    for (; i < pieces; i += step) x ^= *reinterpret_cast<const uint32_t *>(p + 16 * i);
    asm volatile("" ::"v"(x));  // (the loads' only use)
}

// ------------------------------------------------------------------- summed
// out[row] = s * (sum over columns of table[token]). Column t goes to sum t % 4 and the
// four sums are added in pairs, in both kernels, so a row's result does not depend on the
// rows beside it. (Eight sums take 32 registers more: 100k rows of 100 trees, 64 cells of
// bfloat16, 74 us against 66.)
constexpr uint32_t SUMS = 4;
__device__ __forceinline__ float join_sums(const float *a) {
    return (a[0] + a[1]) + (a[2] + a[3]);
}

// Bound by the gathered bytes and the instructions that unpack and add them, about 35 us each
// of the 66 that 100k rows of 100 trees, 64 cells of bfloat16, take (1.15 GB from the L2s,
// where one column's part of the table stays while all rows go through it).
//
// A workgroup takes 256 / G rows, G = 2^lg_g lanes a row; the tokens of 2^lg_c columns at
// a time are found by all threads in turn and kept in LDS, so that an id is decoded (and
// its bits drawn) once and not by every lane of its row. BUFFER: what is kept are their
// rows' byte offsets, and the table is read by buffer loads.
template <class T, int VEC, int ID, bool DROP, bool BUFFER>
__global__ __launch_bounds__(EMB_TPB) void embed_sum_kernel(Positions P, const T *table, T *out,
                                                            uint32_t dim, uint32_t n_pieces,
                                                            uint32_t lg_g, uint32_t lg_c,
                                                            float s) {
    extern __shared__ uint32_t toks[];
    const uint32_t rows = EMB_TPB >> lg_g, cols = 1u << lg_c, pitch = cols + 4;
    const uint64_t row0 = (blockIdx.x + (uint64_t)blockIdx.z * gridDim.x) * rows;
    const uint32_t r = threadIdx.x >> lg_g;
    const uint32_t piece = blockIdx.y * (1u << lg_g) + (threadIdx.x & ((1u << lg_g) - 1));
    const bool live = row0 + r < P.n_rows && piece < n_pieces;
    const uint32_t cell = live ? min(piece * VEC, dim - VEC) : 0;
    const uint32_t row_bytes = dim * (uint32_t)sizeof(T), cell_bytes = cell * (uint32_t)sizeof(T);
    const auto rsrc = buffer_of(table, BUFFER ? P.n_tokens * row_bytes : 0);
    const T *from = table + cell;
    float a[VEC][SUMS];
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (uint32_t j = 0; j < SUMS; j++) a[i][j] = 0.0f;
    for (uint32_t t0 = 0; t0 < P.n_columns; t0 += cols) {
        for (uint32_t i0 = threadIdx.x; i0 < rows << lg_c; i0 += 4 * EMB_TPB) {
            uint32_t id[4];
            Part part[4];
            // (always a load, as in column_ids_kernel. A workgroup of few rows and columns has
            // fewer positions than a step takes, 32 at least: the break below keeps to them)
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint32_t i = i0 + k * EMB_TPB, t = min(t0 + (i & (cols - 1)), P.n_columns - 1);
                id[k] = load_id<ID>(P.ids, min(row0 + (i >> lg_c), P.n_rows - 1) * P.n_columns + t);
                part[k] = part_of(P, t);
            }
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const uint32_t i = i0 + k * EMB_TPB, rr = i >> lg_c, t = t0 + (i & (cols - 1));
                if (rr >= rows) break;
                const uint32_t bits =
                    DROP ? drop_bits(P.key, (row0 + rr) * P.n_columns + t) : 0;
                uint32_t tok = token_of<DROP>(P, part[k], id[k], bits);
                if (row0 + rr >= P.n_rows || t >= P.n_columns) tok = NO_TOKEN;
                if (BUFFER) tok = tok == NO_TOKEN ? NO_OFFSET : tok * row_bytes;
                toks[rr * pitch + (i & (cols - 1))] = tok;
            }
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
                if constexpr (BUFFER) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        p[j] = load_offset<T, VEC>(rsrc, tok[j] + cell_bytes);
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int i = 0; i < VEC; i++) a[i][j % SUMS] += (float)p[j].v[i];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        p[j] = load_piece<T, VEC>(
                            from + (uint64_t)(tok[j] == NO_TOKEN ? 0 : tok[j]) * dim);
#pragma unroll
                    for (int j = 0; j < 8; j++)
#pragma unroll
                        for (int i = 0; i < VEC; i++)
                            a[i][j % SUMS] += tok[j] == NO_TOKEN ? 0.0f : (float)p[j].v[i];
                }
            }
        __syncthreads();
    }
    if (!live) return;
    Piece<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; i++) o.v[i] = (T)(join_sums(a[i]) * s);
    store_piece<T, VEC>(out + (row0 + r) * dim + cell, o);
}

// Few rows: the sums of a row side by side, a workgroup a row and 2^lg_g pieces.
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
    constexpr uint32_t AHEAD = 16;  // columns requested at once
    for (uint32_t t0 = j; t0 < P.n_columns; t0 += AHEAD * SUMS) {
        uint32_t tok[AHEAD];
        Piece<T, VEC> p[AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; k++) {
            const uint32_t t = min(t0 + SUMS * k, P.n_columns - 1);
            tok[k] = token_at<ID, DROP>(P, row * P.n_columns + t, t);
            if (t0 + SUMS * k >= P.n_columns) tok[k] = NO_TOKEN;
        }
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; k++)
            p[k] = load_piece<T, VEC>(table + (uint64_t)(tok[k] == NO_TOKEN ? 0 : tok[k]) * dim +
                                      cell);
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; k++)
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
        float b[SUMS];
#pragma unroll
        for (uint32_t k = 0; k < SUMS; k++) b[k] = sums[((k << lg_g) + lane) * VEC + i];
        o.v[i] = (T)(join_sums(b) * s);
    }
    store_piece<T, VEC>(out + row * dim + cell, o);
}

// ------------------------------------------------------------------- gradient
// Positions are sorted by token, stably (radix passes of at most 8 bits), so each
// token's positions stand together in their own order; then runs of equal tokens are
// summed in f32. The sorted positions are cut into chunks of equal length: a run inside
// one chunk goes to the table, the parts of longer runs are joined in chunk order. All
// orders are fixed, so the gradient is the same in every call. A part of a sum is held in
// f32 (up to 256 positions here, up to 384 blocks of 8 where columns are summed); what joins
// parts, whose number grows with the positions of a token, is held in f64.
constexpr uint32_t SORT_TPB = 256;
constexpr uint32_t SORT_ROUNDS = 16;  // of a thread's positions; 1 where they are few
constexpr uint32_t SORT_WAVES = SORT_TPB / 64;

// What a pass sorts: positions decoded from the ids (pass 0), or the pass before's output.
struct SortFrom {
    const uint32_t *keys, *vals;
    uint32_t n;       // positions
    uint32_t shift, bits;
    uint32_t per_row; // pooled: the columns of a row, whose positions share its gradient
    uint32_t blocks;
    // The table's zeros, for the tokens without a position: a third beside each launch of
    // the first pass (the blocks behind its own), which leave most of the device idle.
    // (32768 positions, a table of 102 MB: 17 us by themselves.)
    uint8_t *zeros;
    uint64_t zero_bytes;
};

constexpr uint32_t ZERO_BLOCKS = 1024;

// Part `part` of three of the zeros, by ZERO_BLOCKS workgroups: 16-byte pieces, and what is
// left before and behind them in bytes.
__device__ __forceinline__ void zero_part(const SortFrom &S, uint32_t part, uint32_t block) {
    const uint64_t each = (S.zero_bytes / 3 + 15) & ~15ull, from = min(part * each, S.zero_bytes);
    uint8_t *p = S.zeros + from;
    const uint64_t bytes = part == 2 ? S.zero_bytes - from : min(each, S.zero_bytes - from);
    const uint64_t head = min(bytes, (uint64_t)(-(intptr_t)p & 15));
    const uint64_t pieces = (bytes - head) / 16;
    const uint64_t at = block * (uint64_t)SORT_TPB + threadIdx.x,
                   step = ZERO_BLOCKS * (uint64_t)SORT_TPB;
    for (uint64_t i = at; i < pieces; i += step)
        *reinterpret_cast<uint4 *>(p + head + 16 * i) = make_uint4(0, 0, 0, 0);
    if (at < head) p[at] = 0;
    if (at < bytes - head - 16 * pieces) p[head + 16 * pieces + at] = 0;
}

template <int ID, bool DROP, bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const Positions &P, const SortFrom &S, uint32_t i) {
    if (!FIRST) return S.keys[i];
    const uint32_t tok = token_at<ID, DROP>(P, i, P.n_columns > 1 ? i % P.n_columns : 0);
    return tok == NO_TOKEN ? P.n_tokens : tok;  // the last key of all
}

// counts[digit * blocks + block]
template <int ID, bool DROP, bool FIRST, uint32_t ROUNDS>
__global__ __launch_bounds__(SORT_TPB) void sort_count_kernel(Positions P, SortFrom S,
                                                              uint32_t *counts) {
    if (blockIdx.x >= S.blocks) return zero_part(S, 0, blockIdx.x - S.blocks);
    __shared__ uint32_t c[256];
    c[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (SORT_TPB * ROUNDS), mask = (1u << S.bits) - 1;
#pragma unroll 4
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = base + r * SORT_TPB + threadIdx.x;
        if (i < S.n)
            atomicAdd(&c[(sort_key<ID, DROP, FIRST>(P, S, i) >> S.shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x <= mask) counts[(uint64_t)threadIdx.x * S.blocks + blockIdx.x] = c[threadIdx.x];
}

// A digit's counts to the positions before them in its own part; its total.
__global__ __launch_bounds__(SORT_TPB) void sort_scan_kernel(SortFrom S, uint32_t *counts,
                                                             uint32_t *totals) {
    if (blockIdx.x >> S.bits) return zero_part(S, 1, blockIdx.x - (1u << S.bits));
    const uint32_t blocks = S.blocks;
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
template <int ID, bool DROP, bool FIRST, uint32_t ROUNDS>
__global__ __launch_bounds__(SORT_TPB) void sort_scatter_kernel(Positions P, SortFrom S,
                                                                const uint32_t *counts,
                                                                const uint32_t *totals,
                                                                uint32_t *keys, uint32_t *vals) {
    if (blockIdx.x >= S.blocks) return zero_part(S, 2, blockIdx.x - S.blocks);
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
                add + x - v + counts[(uint64_t)threadIdx.x * S.blocks + blockIdx.x];
    }
    const uint32_t first = (blockIdx.x * SORT_WAVES + w) * (ROUNDS * 64) + lane;
    uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = first + r * 64;
        key[r] = i < S.n ? sort_key<ID, DROP, FIRST>(P, S, i) : 0;
    }
    // (a wave's LDS operations complete in order, and only it touches its counters)
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const bool in = first + r * 64 < S.n;
        const uint32_t digit = (key[r] >> S.shift) & mask;
        rank[r] = take_places(&seen[w][digit], in, same_digit(in, digit, S.bits));
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
    for (uint32_t r = 0; r < ROUNDS; r++) {
        const uint32_t i = first + r * 64;
        if (i >= S.n) continue;
        const uint32_t at = seen[w][(key[r] >> S.shift) & mask] + rank[r];
        keys[at] = key[r];
        vals[at] = FIRST ? (S.per_row > 1 ? i / S.per_row : i) : S.vals[i];
    }
}

// ---- Up to 64k positions: one radix pass, of the tokens' high bits and with one position a
// thread so that its launches are short, parts them into buckets; then each bucket is
// sorted in a workgroup. (32768 positions, 50000 tokens of 2 KB: two passes of 16 positions
// a thread and a pass of zeros took 75 us; workgroups that each
// look for their own tokens among all positions 39; workgroups that count all positions
// and place 1024 of them, instead of the pass' three launches, 39 alone.)
constexpr uint32_t FEW_MOST = 65536;     // positions
constexpr uint32_t FEW_TPB = 512;
constexpr uint32_t FEW_WAVES = FEW_TPB / 64;
constexpr uint32_t FEW_RANGE_BITS = 10;  // tokens of a bucket: at most two a thread
constexpr uint32_t FEW_BUCKET_BITS = 8;

struct Few {
    uint32_t n_tokens, shift;    // 2^shift tokens a bucket
    const uint32_t *totals;      // of the buckets
    const uint32_t *part_keys, *part_vals;
    uint32_t *keys, *vals;
};

// The sum of the values of lower threads; *all gets the sum of all.
__device__ __forceinline__ uint32_t sum_below(uint32_t v, uint32_t *wave_sum, uint32_t *all) {
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    uint32_t x = v;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= (uint32_t)d) x += y;
    }
    if (lane == 63) wave_sum[w] = x;
    __syncthreads();
    uint32_t sum = x - v;
    *all = 0;
    for (uint32_t k = 0; k < FEW_WAVES; k++) {
        if (k < w) sum += wave_sum[k];
        *all += wave_sum[k];
    }
    return sum;
}

__global__ __launch_bounds__(FEW_TPB) void few_sort_kernel(Few F) {
    extern __shared__ uint32_t seen[];  // [wave][token]: counts, then places
    __shared__ uint32_t wave_sum[FEW_WAVES];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    // (token n_tokens, behind the last, are the positions that give nothing)
    const uint32_t most = 1u << F.shift, t0 = blockIdx.x << F.shift,
                   range = min(most, F.n_tokens + 1 - t0);
    uint32_t first;
    (void)sum_below(threadIdx.x < blockIdx.x ? F.totals[threadIdx.x] : 0, wave_sum, &first);
    const uint32_t end = first + F.totals[blockIdx.x];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < FEW_WAVES * most; i += FEW_TPB) seen[i] = 0;
    __syncthreads();
    uint32_t *mine = seen + w * most;
    // a wave's positions, side by side
    const uint32_t each = ((end - first + FEW_TPB - 1) / FEW_TPB) * 64;
    const uint32_t i0 = first + w * each, i1 = min(i0 + each, end);
    for (uint32_t i = i0 + lane; i < i1; i += 8 * 64) {
        uint32_t key[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) key[j] = F.part_keys[min(i + 64 * j, i1 - 1)];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (i + 64 * j < i1) atomicAdd(&mine[key[j] - t0], 1u);
    }
    __syncthreads();
    uint32_t c[2] = {0, 0}, all;
    for (uint32_t j = 0; j < 2; j++)
        if (2 * threadIdx.x + j < range)
            for (uint32_t v = 0; v < FEW_WAVES; v++) c[j] += seen[v * most + 2 * threadIdx.x + j];
    uint32_t at = first + sum_below(c[0] + c[1], wave_sum, &all);
    for (uint32_t j = 0; j < 2; j++)
        if (2 * threadIdx.x + j < range) {
            uint32_t a = at;
            for (uint32_t v = 0; v < FEW_WAVES; v++) {
                uint32_t *p = &seen[v * most + 2 * threadIdx.x + j];
                const uint32_t m = *p;
                *p = a;
                a += m;
            }
            at += c[j];
        }
    __syncthreads();
    for (uint32_t i = i0; i < i1; i += 8 * 64) {
        uint32_t key[8], val[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            const uint32_t at = min(i + 64 * j + lane, i1 - 1);
            key[j] = F.part_keys[at];
            val[j] = F.part_vals[at];
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            if (i + 64 * j >= i1) break;  // (the same for all lanes)
            const bool in = i + 64 * j + lane < i1;
            const uint32_t off = key[j] - t0;
            const uint32_t to = take_places(&mine[off], in, same_digit(in, off, F.shift));
            if (in) {
                F.keys[to] = key[j];
                F.vals[to] = val[j];
            }
        }
    }
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

// Joins the parts of the runs that start in a chunk and go on behind it, in doubles: a run
// over many chunks ends at the error of its parts, not of their number.
constexpr uint32_t JOIN_TPB = 1024;
template <class T, int VEC>
__global__ __launch_bounds__(JOIN_TPB) void grad_join_kernel(Runs R, T *table) {
    __shared__ uint32_t longs[JOIN_TPB], n_longs;
    constexpr int H = VEC > 1 ? VEC / 2 : 1;  // cells that the groups join at a time
    __shared__ double sums[JOIN_TPB * H];
    const uint32_t lanes = 1u << R.lg_g, groups = JOIN_TPB >> R.lg_g;
    const uint32_t g = threadIdx.x >> R.lg_g, lane = threadIdx.x & (lanes - 1);
    const uint32_t piece = (blockIdx.y << R.lg_g) + lane;
    const bool live = piece < R.n_pieces;
    const uint32_t cell = live ? min(piece * VEC, R.dim - VEC) : 0;
    const uint32_t chunks = (uint32_t)(((uint64_t)R.n + R.chunk - 1) / R.chunk);
    if (threadIdx.x == 0) n_longs = 0;
    __syncthreads();

    // the number of chunks behind c, up to JOIN_SHORT, whose first position has this key
    const auto behind = [&](uint32_t c, uint32_t key) {
        uint32_t k[JOIN_SHORT], n = 0;
#pragma unroll
        for (uint32_t i = 0; i < JOIN_SHORT; i++)
            k[i] = R.keys[(uint64_t)min(c + 1 + i, chunks - 1) * R.chunk];
#pragma unroll
        for (uint32_t i = 0; i < JOIN_SHORT; i++)
            if (n == i && c + 1 + i < chunks && k[i] == key) n++;
        return n;
    };
    const auto write = [&](uint32_t key, const double *a) {
        Piece<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; i++) o.v[i] = (T)(float)(a[i] * R.s);
        store_piece<T, VEC>(table + (uint64_t)key * R.dim + cell, o);
    };

    const uint32_t c = blockIdx.x * groups + g;
    const uint64_t c0 = (uint64_t)c * R.chunk, c1 = c0 + R.chunk;
    if (c1 < R.n) {
        const uint32_t key = R.keys[c1 - 1];
        const bool starts = R.keys[c0] != key || c0 == 0 || R.keys[c0 - 1] != key;
        if (key < R.n_tokens && starts && R.keys[c1] == key) {
            const uint32_t n = behind(c, key);
            if (n == JOIN_SHORT) {
                if (lane == 0) longs[atomicAdd(&n_longs, 1u)] = c;
            } else if (live) {
                double a[VEC];
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
        // (sorted: the chunks that start with this key are the ones right behind)
        uint32_t n = JOIN_SHORT + 1;
        for (uint32_t some = JOIN_TPB; some == JOIN_TPB;) {
            const uint64_t at = (uint64_t)lc + n + threadIdx.x;
            some = __syncthreads_count(at < chunks && R.keys[at * R.chunk] == key);
            n += some;
        }
        double a[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) a[i] = 0.0;
        if (live)
            for (uint32_t k0 = g; k0 < n; k0 += 8 * groups) {
                Piece<float, VEC> p[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) {
                    const uint32_t k = min(k0 + j * groups, n - 1);
                    p[j] = load_piece<float, VEC>(
                        R.parts + (2ull * (lc + k) + (k ? 0 : 1)) * R.dim + cell);
                }
#pragma unroll
                for (uint32_t j = 0; j < 8; j++)
                    if (k0 + j * groups < n)
#pragma unroll
                        for (int i = 0; i < VEC; i++) a[i] += p[j].v[i];
            }
#pragma unroll
        for (int h = 0; h < VEC; h += H) {
#pragma unroll
            for (int i = 0; i < H; i++) sums[threadIdx.x * H + i] = a[h + i];
            __syncthreads();
            if (g == 0)
                for (uint32_t k = 1; k < groups; k++)
#pragma unroll
                    for (int i = 0; i < H; i++) a[h + i] += sums[((k << R.lg_g) + lane) * H + i];
            __syncthreads();
        }
        if (g == 0 && live) write(key, a);
    }
}

// ---- Many rows of columns with few ids each (a model's trees, categorical columns).
// Each column's part of the table is summed over chunks of rows: a workgroup sorts a
// chunk's ids of one column in LDS, sums the runs, and leaves a part of the table (with
// the counts of its tokens) that the last kernel adds up chunk by chunk. Nothing is
// sorted through memory, and where the chunks are a multiple of 8 the gradient rows that all
// columns of a chunk gather stay in one XCD's L2: workgroups of one chunk then have numbers
// equal modulo the 8 XCDs (column_plan prefers such numbers above 4). 100k rows of 100 trees, 64
// cells of bfloat16: 22 us for the ids (their hashes), 101 for the sums (1.15 GB gathered, 11.4
// TB/s; instructions half of it) and 18 for the last; sorted by token they took 596, and 16
// chunks instead of 8 take 12 and 8 us more.
constexpr uint32_t COL_TPB = 512;
constexpr uint32_t COL_WAVES = COL_TPB / 64;
constexpr uint32_t COL_ITEMS = 32;                       // rows of a thread at most
constexpr uint32_t COL_MOST_ROWS = COL_TPB * COL_ITEMS;  // of a chunk: list entries are 16-bit
constexpr uint32_t COL_MOST_IDS = 1024;
constexpr uint32_t COL_NONE = 0xFFFF;

// local[column][row]: the id inside its column, COL_NONE where the position gives
// nothing; rows up to `padded` are written. 64 x 64 positions through LDS.
template <int ID, bool DROP>
__global__ __launch_bounds__(256) void column_ids_kernel(Positions P, uint32_t most_ids,
                                                         uint64_t padded, uint16_t *local) {
    __shared__ uint16_t tile[64][66];
    const uint64_t row0 = (uint64_t)blockIdx.x * 64;
    const uint32_t col0 = blockIdx.y * 64, lane = threadIdx.x & 63, w = threadIdx.x / 64;
    const uint32_t column = col0 + lane;
    uint32_t id[16];
#pragma unroll
    for (uint32_t r = 0; r < 16; r++) {
        // (always a load, of the last position where there is none: a branch for each would
        // have them wait for one another)
        const uint64_t row = min(row0 + w + 4 * r, P.n_rows - 1);
        id[r] = load_id<ID>(P.ids, row * P.n_columns + min(column, P.n_columns - 1));
    }
    Part part = part_of(P, min(column, P.n_columns - 1));
    part.size = min(part.size, most_ids);
#pragma unroll
    for (uint32_t r = 0; r < 16; r += 2) {
        const uint64_t row = row0 + w + 4 * r;
        const uint64_t pos[2] = {row * P.n_columns + column, (row + 4) * P.n_columns + column};
        uint32_t bits[2] = {0, 0};
        bits_of_two<DROP>(P, pos, bits);
#pragma unroll
        for (uint32_t k = 0; k < 2; k++) {
            const bool some = token_of<DROP>(P, part, id[r + k], bits[k]) != NO_TOKEN &&
                              row + 4 * k < P.n_rows && column < P.n_columns;
            tile[w + 4 * (r + k)][lane] = some ? (uint16_t)id[r + k] : (uint16_t)COL_NONE;
        }
    }
    __syncthreads();
#pragma unroll 4
    for (uint32_t c = w; c < 64; c += 4)
        if (col0 + c < P.n_columns && row0 + lane < padded)
            local[(col0 + c) * padded + row0 + lane] = tile[lane][c];
}

struct Columns {
    const uint16_t *local;
    const uint32_t *first;   // NULL: one column, from row 0
    uint64_t n_rows, padded;
    uint32_t column0, n_columns;  // of a launch: its parts take the same workspace as the
                                  // launch's before
    uint32_t part_tokens;         // tokens that the parts have room for, from column0's on
    uint32_t n_tokens, most_ids;
    uint32_t chunk, chunks;  // rows of a chunk (a multiple of 64), chunks
    uint32_t per_row;        // gradient vectors of a row: 1 (pooled) or the columns
    uint32_t dim, n_pieces, lg_g;
    float s;
    float *parts;            // [chunk][token of the launch][dim]
    uint16_t *counts;        // [chunk][token of the launch]: positions in the chunk

    bool grouped;            // a launch has not all columns

    // The table rows of the launch's columns: the first, and the one behind the last.
    __device__ __forceinline__ uint32_t begin() const {
        return grouped ? min(first[column0], n_tokens) : 0;
    }
    __device__ __forceinline__ uint32_t end() const {
        return grouped ? min(first[column0 + n_columns], n_tokens) : n_tokens;
    }
};

// LDS of column_sums_kernel, in byte offsets: the waves' counters and later the ranges'
// open sums; the ids' first blocks; the rows by id, each id's in blocks of 8.
struct ColumnLds {
    uint32_t starts, list, bytes;
};
__host__ __device__ inline ColumnLds column_lds(uint32_t most_ids, uint32_t chunk, uint32_t vec) {
    ColumnLds l{};
    const uint32_t seen = (COL_WAVES * most_ids * 2 + 15) & ~15u, sums = COL_TPB * vec * 4;
    l.starts = seen > sums ? seen : sums;
    l.list = l.starts + (((most_ids + 1) * 2 + 15) & ~15u);
    l.bytes = l.list + (chunk + 8 * most_ids) * 2;
    return l;
}

// BUFFER: the chunk's gradient rows are read by buffer loads, and the entries that fill an
// id's last block (row `chunk`, behind the buffer) read as zeros.
template <class T, int VEC, bool BUFFER>
__global__ __launch_bounds__(COL_TPB) void column_sums_kernel(Columns C, const T *grad,
                                                              T *table) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t wave_sum[COL_WAVES];
    // (chunk group, column, chunk of the group): a group's chunks go to one XCD each
    const uint32_t per = min(C.chunks, 8u);
    const uint32_t chunk = blockIdx.x / (C.n_columns * per) * per + blockIdx.x % per;
    const uint32_t t = C.column0 + blockIdx.x / per % C.n_columns;
    if (chunk >= C.chunks) return;
    const ColumnLds L = column_lds(C.most_ids, C.chunk, VEC);
    uint16_t *seen = reinterpret_cast<uint16_t *>(lds);
    float *sums = reinterpret_cast<float *>(lds);
    uint16_t *starts = reinterpret_cast<uint16_t *>(lds + L.starts);
    uint16_t *list = reinterpret_cast<uint16_t *>(lds + L.list);
    const uint32_t base = C.first ? min(C.first[t], C.n_tokens) : 0;
    const uint32_t part_base = base - C.begin();
    const uint32_t ids = min(C.most_ids, C.first ? min(C.first[t + 1] - base, C.n_tokens - base)
                                                 : C.n_tokens);
    // (never, but for falling offsets or columns of more than most_ids ids, which the caller
    // has ruled out)
    if ((uint64_t)part_base + ids > C.part_tokens) return;
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x / 64;
    const uint64_t row0 = (uint64_t)chunk * C.chunk;
    const uint16_t *from = C.local + t * C.padded + row0;

    // ---- the chunk's rows by id. A wave takes `rounds` times 256 rows, a lane 4 of them
    // side by side; "before" is by wave, then by round and place in the four, then by
    // lane: any order that is always the same will do.
    for (uint32_t i = threadIdx.x; i < COL_WAVES * C.most_ids; i += COL_TPB) seen[i] = 0;
    const uint32_t fill = C.chunk | C.chunk << 16;
    for (uint32_t i = threadIdx.x; i < (C.chunk + 8 * C.most_ids) / 8; i += COL_TPB)
        reinterpret_cast<uint4 *>(list)[i] = make_uint4(fill, fill, fill, fill);
    __syncthreads();
    uint32_t key[COL_ITEMS / 2], rank[COL_ITEMS / 2];  // two rows a word
    const uint32_t rounds = (C.chunk + COL_WAVES * 256 - 1) / (COL_WAVES * 256);
#pragma unroll
    for (uint32_t r = 0; r < COL_ITEMS / 4; r++) {
        const uint32_t at = (w * rounds + r) * 256 + lane * 4;
        uint2 q = make_uint2(~0u, ~0u);
        if (r < rounds && at < C.chunk) q = *reinterpret_cast<const uint2 *>(from + at);
        key[2 * r] = q.x;
        key[2 * r + 1] = q.y;
    }
    const uint32_t bits = 32 - __clz(max(C.most_ids - 1, 1u));
    uint16_t *mine = seen + w * C.most_ids;
#pragma unroll
    for (uint32_t r = 0; r < COL_ITEMS / 4; r++)
        if (r < rounds)
#pragma unroll
            for (uint32_t i = 4 * r; i < 4 * r + 4; i++) {
                const uint32_t k = (key[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
                const bool in = k != COL_NONE;
                uint64_t same = __ballot(in);
                for (uint32_t b = 0; b < bits; b++) {
                    const bool one = (k >> b) & 1;
                    const uint64_t ones = __ballot(one);
                    same &= one ? ones : ~ones;
                }
                const uint32_t below = __popcll(same & ((1ull << lane) - 1));
                uint32_t before = 0;
                if (in) before = *(volatile uint16_t *)&mine[k];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (in && below == 0)
                    *(volatile uint16_t *)&mine[k] = (uint16_t)(before + __popcll(same));
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                const uint32_t at = before + below;
                rank[i / 2] = i & 1 ? rank[i / 2] | at << 16 : at;
            }
    __syncthreads();
    // starts[id]: the blocks of lower ids, two ids a thread
    {
        uint32_t c[2] = {0, 0};
        for (uint32_t j = 0; j < 2; j++) {
            const uint32_t id = 2 * threadIdx.x + j;
            if (id < C.most_ids)
                for (uint32_t v = 0; v < COL_WAVES; v++) c[j] += seen[v * C.most_ids + id];
        }
        const uint32_t b0 = (c[0] + 7) / 8, b1 = (c[1] + 7) / 8;
        uint32_t x = b0 + b1;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(x, d);
            if (lane >= (uint32_t)d) x += y;
        }
        if (lane == 63) wave_sum[w] = x;
        __syncthreads();
        uint32_t at = x - b0 - b1;
        for (uint32_t v = 0; v < w; v++) at += wave_sum[v];
        for (uint32_t j = 0; j < 2; j++) {
            const uint32_t id = 2 * threadIdx.x + j;
            if (id < C.most_ids) {
                starts[id] = (uint16_t)at;
                if (id < ids)
                    C.counts[(uint64_t)chunk * C.part_tokens + part_base + id] = (uint16_t)c[j];
                uint32_t a = 8 * at;
                for (uint32_t v = 0; v < COL_WAVES; v++) {
                    const uint32_t n = seen[v * C.most_ids + id];
                    seen[v * C.most_ids + id] = (uint16_t)a;
                    a += n;
                }
                at += j ? b1 : b0;
                if (id == C.most_ids - 1) starts[C.most_ids] = (uint16_t)at;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < COL_ITEMS; i++) {
        const uint32_t k = (key[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
        if (i / 4 < rounds && k != COL_NONE)
            list[mine[k] + ((rank[i / 2] >> (16 * (i & 1))) & 0xFFFFu)] =
                (uint16_t)((w * rounds + i / 4) * 256 + lane * 4 + (i & 3));
    }
    __syncthreads();

    // ---- sums: the blocks in equal ranges, 2^lg_g lanes a range. Runs inside a range go
    // to memory; a range leaves the sum of the run that it continues in LDS, and adds
    // those behind it to the run that starts in it and goes on.
    const uint32_t g = threadIdx.x >> C.lg_g, glane = threadIdx.x & ((1u << C.lg_g) - 1);
    const uint32_t groups = COL_TPB >> C.lg_g;
    const uint32_t piece = (blockIdx.y << C.lg_g) + glane;
    const bool live = piece < C.n_pieces;
    const uint32_t cell = live ? min(piece * VEC, C.dim - VEC) : 0;
    const uint32_t n = starts[C.most_ids];
    const uint32_t each = (n + groups - 1) / groups;
    const uint32_t i0 = min(g * each, n), i1 = min(i0 + each, n);
    const uint64_t pitch = (uint64_t)C.per_row * C.dim;
    const T *rows = grad + row0 * pitch + (C.per_row > 1 ? (uint64_t)t * C.dim : 0);
    const uint32_t row_bytes = (uint32_t)(pitch * sizeof(T)),
                   cell_bytes = cell * (uint32_t)sizeof(T);
    const auto rsrc = buffer_of(rows, BUFFER ? C.chunk * row_bytes : 0);
    const bool whole = C.chunks == 1;
    float a[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) a[i] = 0.0f;
    const auto write = [&](uint32_t id, const auto *sum) {
        if (whole) {
            const uint64_t at = (uint64_t)(base + id) * C.dim + cell;
            Piece<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = (T)(float)(sum[i] * C.s);
            store_piece<T, VEC>(table + at, o);
        } else {
            const uint64_t at = (uint64_t)chunk * C.part_tokens + (part_base + id);
            Piece<float, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = (float)sum[i];
            store_piece<float, VEC>(C.parts + at * C.dim + cell, o);
        }
    };
    const auto leave = [&] {
#pragma unroll
        for (int i = 0; i < VEC; i++) sums[threadIdx.x * VEC + i] = a[i];
    };
    uint32_t id = 0, end = 0;
    bool begun = false;  // the run starts in this range
    if (live && i0 < i1) {
        uint32_t lo = 0, hi = C.most_ids;  // the last id whose blocks start at or before i0
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (starts[mid] <= i0) lo = mid;
            else hi = mid;
        }
        id = lo;
        end = starts[id + 1];
        begun = starts[id] == i0;
        for (uint32_t b = i0; b < i1; b++) {
            const uint4 q = reinterpret_cast<const uint4 *>(list)[b];
            const uint32_t pair[4] = {q.x, q.y, q.z, q.w};
            Piece<T, VEC> p[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t row = (pair[j / 2] >> (16 * (j & 1))) & 0xFFFFu;
                if constexpr (BUFFER) p[j] = load_offset<T, VEC>(rsrc, row * row_bytes + cell_bytes);
                else p[j] = load_piece<T, VEC>(rows + (row < C.chunk ? row : 0) * pitch + cell);
            }
            // The block by itself first, in pairs: a range's sum of up to 3072 rows has an
            // eighth of the steps, at the same number of additions.
            const auto at = [&](int j, int i) {
                const bool none =
                    !BUFFER && ((pair[j / 2] >> (16 * (j & 1))) & 0xFFFFu) >= C.chunk;
                return none ? 0.0f : (float)p[j].v[i];
            };
#pragma unroll
            for (int i = 0; i < VEC; i++)
                a[i] += ((at(0, i) + at(1, i)) + (at(2, i) + at(3, i))) +
                        ((at(4, i) + at(5, i)) + (at(6, i) + at(7, i)));
            if (b + 1 == end) {
                if (begun) write(id, a);
                else leave();
                begun = true;
#pragma unroll
                for (int i = 0; i < VEC; i++) a[i] = 0.0f;
                if (b + 1 < i1) {
                    do id++, end = starts[id + 1];
                    while (end == b + 1);
                } else {
                    end = 0;  // nothing is open
                }
            }
        }
        if (end && !begun) {
            leave();
            end = 0;
        }
    }
    if (whole && live) {
        for (uint32_t k = g; k < ids; k += groups)
            if (starts[k] == starts[k + 1]) {
                const uint64_t at = (uint64_t)(base + k) * C.dim + cell;
                Piece<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; i++) o.v[i] = (T)0.0f;
                store_piece<T, VEC>(table + at, o);
            }
    }
    __syncthreads();
    if (end) {
        double b[VEC];  // (ranges are joined in doubles, as chunks are)
#pragma unroll
        for (int i = 0; i < VEC; i++) b[i] = a[i];
        for (uint32_t h = g + 1; h * each < end; h++)
#pragma unroll
            for (int i = 0; i < VEC; i++) b[i] += sums[((h << C.lg_g) + glane) * VEC + i];
        write(id, b);
    }
}

// table[token] = s * the sum of its parts, in chunk order and in doubles.
template <class T, int VEC>
__global__ __launch_bounds__(256) void column_join_kernel(Columns C, T *table) {
    const uint64_t i = blockIdx.x * 256ull + threadIdx.x;
    const uint64_t tok = i / C.n_pieces;  // of the launch
    const uint64_t begin = C.begin();
    if (tok >= C.part_tokens || begin + tok >= C.end()) return;
    const uint32_t cell = min((uint32_t)(i - tok * C.n_pieces) * VEC, C.dim - VEC);
    const float *part = C.parts + tok * C.dim + cell;
    double a[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) a[j] = 0.0;
    for (uint32_t c0 = 0; c0 < C.chunks; c0 += 8) {
        bool some[8];
        Piece<float, VEC> p[8];
        uint16_t count[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
            count[k] = C.counts[(uint64_t)min(c0 + k, C.chunks - 1) * C.part_tokens + tok];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            // (a chunk without the token has left nothing; the first part is read instead)
            some[k] = c0 + k < C.chunks && count[k] != 0;
            p[k] = load_piece<float, VEC>(
                some[k] ? part + (uint64_t)(c0 + k) * C.part_tokens * C.dim : C.parts);
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
            if (some[k])
#pragma unroll
                for (int j = 0; j < VEC; j++) a[j] += p[k].v[j];
    }
    Piece<T, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = (T)(float)(a[j] * C.s);
    store_piece<T, VEC>(table + (begin + tok) * C.dim + cell, o);
}

// ------------------------------------------------------------------- host side
uint32_t lg_at_least(uint64_t n) {
    uint32_t l = 0;
    while ((1ull << l) < n) l++;
    return l;
}

float scale_of(const fbh_embed *e) { return (float)((double)e->scale / (1.0 - e->drop)); }

void check_embed(const fbh_embed *e) {
    head_input(e, "null argument");
    head_input(e->dtype <= FBH_BF16, "unknown cell type");
    head_input(e->id_type <= FBH_ID_F32, "unknown id type");
    head_input(e->dim >= 1 && e->dim <= EMB_MAX_DIM, "dim must be in 1..=32768");
    head_input(e->n_columns >= 1, "no columns");
    // (the summing kernels step over a row's columns in 32 bits)
    head_input(!e->pooled || e->n_columns <= 0x7FFFFFFFu, "at most 2147483647 columns to sum");
    head_input(!e->first || e->n_columns <= EMB_MAX_COLUMNS,
               "at most 32768 columns with parts of their own");
    head_input(e->n_tokens >= 1 && e->n_tokens <= 0x7FFFFFFFu,
               "n_tokens must be in 1..=2147483647");
    head_input(e->ids || e->n_rows == 0, "null argument");
    head_input(e->n_rows <= (1ull << 40) / e->n_columns, "more than 2^40 positions");
    head_input(e->most_ids <= e->n_tokens, "most_ids is larger than the table");
    (void)drop_threshold(e->drop);
    // (what takes nothing is scaled like the rest, and zero times infinity is none)
    head_input(std::isfinite(scale_of(e)), "scale / (1 - drop) must be a finite float");
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

// Whether buffer loads reach rows of row_bytes from p on: their bytes, in words.
bool in_buffer(const void *p, uint64_t bytes, uint64_t row_bytes) {
    return bytes <= BUFFER_MOST && row_bytes % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 4 == 0;
}

template <class T, int VEC, int ID, bool DROP>
void launch_embed(const fbh_embed *e, const void *table, void *out, hipStream_t s) {
    const Positions P = positions_of(e);
    const uint32_t pieces = (e->dim + VEC - 1) / VEC;
    const auto *tab = static_cast<const T *>(table);
    auto *to = static_cast<T *>(out);
    const float sc = scale_of(e);
    if (!e->pooled) {
        const uint64_t n_pos = P.n_rows * P.n_columns, vector = e->dim * sizeof(T);
        const uint64_t id_bytes = ID == FBH_ID_I64 ? 8 : 4;
        const bool past = VEC * sizeof(T) == 16 && n_pos * vector >= STREAM_BYTES;
        // (workgroups' positions: parts of the call start at a workgroup's first piece)
        const uint64_t all = (n_pos * pieces + ROW_BLOCK - 1) / ROW_BLOCK;
        const uint64_t most = std::min<uint64_t>(
            past ? TOUCH_BYTES / id_bytes * pieces / ROW_BLOCK : ~0ull, 1u << 22);
        for (uint64_t b0 = 0; b0 < all; b0 += most) {
            const uint64_t blocks = std::min(all - b0, most);
            if (past) {
                const uint64_t first = b0 * ROW_BLOCK / pieces * id_bytes;
                const uint64_t end =
                    std::min((b0 + blocks) * ROW_BLOCK / pieces + 1, n_pos) * id_bytes;
                hipLaunchKernelGGL(touch_kernel, dim3(2048), dim3(256), 0, s,
                                   static_cast<const uint8_t *>(P.ids) + first, (end - first) / 16);
            }
            const auto go = [&](auto past_caches) {
                hipLaunchKernelGGL(
                    (embed_rows_kernel<T, VEC, ID, DROP, decltype(past_caches)::value>),
                    dim3((uint32_t)blocks), dim3(EMB_TPB), 0, s, P, tab, to, e->dim,
                    divisor(pieces), divisor(P.n_columns), sc, b0);
            };
            if constexpr (VEC * sizeof(T) == 16) {
                if (past) go(std::true_type{});
                else go(std::false_type{});
            } else go(std::false_type{});
        }
    } else if (P.n_rows * pieces < 64 * EMB_TPB) {
        const uint32_t lg_g = std::max(std::min(lg_at_least(pieces), 6u), 4u);
        hipLaunchKernelGGL((embed_sum_few_kernel<T, VEC, ID, DROP>),
                           dim3((uint32_t)P.n_rows, (pieces + (1u << lg_g) - 1) >> lg_g),
                           dim3(SUMS << lg_g), (size_t)(SUMS << lg_g) * VEC * sizeof(float), s, P, tab,
                           to, e->dim, pieces, lg_g, sc);
    } else {
        const uint32_t lg_g = std::min(lg_at_least(pieces), 6u), rows = EMB_TPB >> lg_g;
        const uint32_t lg_c =
            std::min(std::max(lg_at_least(P.n_columns), 3u), lg_at_least(4096 / rows));
        const uint64_t blocks = (P.n_rows + rows - 1) / rows;
        const uint32_t bx = (uint32_t)std::min<uint64_t>(blocks, 1u << 22);
        const uint64_t bz = (blocks + bx - 1) / bx;
        head_input(bz <= 65535, "too many rows");
        const auto go = [&](auto buffer) {
            hipLaunchKernelGGL((embed_sum_kernel<T, VEC, ID, DROP, decltype(buffer)::value>),
                               dim3(bx, (pieces + (1u << lg_g) - 1) >> lg_g, (uint32_t)bz),
                               dim3(EMB_TPB), (size_t)rows * ((1u << lg_c) + 4) * 4, s, P, tab,
                               to, e->dim, pieces, lg_g, lg_c, sc);
        };
        if constexpr (VEC * sizeof(T) >= 4) {
            if (in_buffer(table, (uint64_t)e->n_tokens * e->dim * sizeof(T), e->dim * sizeof(T)))
                go(std::true_type{});
            else go(std::false_type{});
        } else go(std::false_type{});
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

// The chunks of rows that columns of few ids are summed in; 0: they are sorted by token
// instead. One chunk, where a workgroup gets through its column's gradient rows in the
// time of a launch or two, takes two launches where sorting takes six (64 rows of 100
// trees, 16 cells of float32: 20 us sorted). Otherwise a chunk of a column has 8
// positions an id on average at least, so that the parts are written and read for less
// than the gradient rows take, and a call has 64k positions at least.
//
// Where the parts of all columns would take more than COL_PART_BYTES, the columns are taken in
// groups whose parts do not (a column's by itself may: it has an eighth of a position a row at
// most, in f32). A group still has some 500 workgroups: 2^28 cells of parts, at most 1024 ids
// and 512 cells each.
constexpr uint64_t COL_ONE_BYTES = 256 << 10;
constexpr uint64_t COL_PART_BYTES = 1ull << 30;
struct ColumnPlan {
    uint32_t chunk = 0, chunks = 0;
    uint32_t group = 0, part_tokens = 0;  // columns of a group, and the most tokens of one
    uint64_t padded = 0, local = 0, counts = 0, parts = 0, bytes = 0;
};

ColumnPlan column_plan(const fbh_embed *e) {
    ColumnPlan c;
    const uint64_t ids = e->first ? e->most_ids : e->n_tokens;
    const uint64_t columns = e->first ? e->n_columns : 1;
    const uint64_t rows = e->first ? e->n_rows : e->n_rows * e->n_columns;
    if (rows == 0 || ids == 0 || ids > COL_MOST_IDS || rows > 1u << 29 ||
        (!e->first && e->pooled && e->n_columns > 1))
        return c;
    const uint32_t vec = piece_cells(e->dim, e->dtype);
    const uint64_t cells = e->dtype == FBH_F32 ? 4 : 2;
    uint64_t chunks;
    if (rows <= COL_MOST_ROWS && rows * std::min<uint64_t>(e->dim * cells, 1024) <= COL_ONE_BYTES) {
        chunks = 1;
    } else {
        if (rows < 8 * ids || rows * columns < 65536) return c;
        const uint64_t blocks = columns * (((e->dim + vec - 1) / vec + 63) / 64);
        const uint64_t most = rows / (8 * ids);
        chunks = std::max((rows + COL_MOST_ROWS - 1) / COL_MOST_ROWS,
                          std::min(most, (1023 + blocks) / blocks));
        if (chunks > 4) {  // the same on every XCD
            const uint64_t up = (chunks + 7) / 8 * 8;
            chunks = up <= std::max<uint64_t>(most, 8) ? up : chunks;
        }
    }
    c.chunk = (uint32_t)(((rows + chunks - 1) / chunks + 63) / 64 * 64);
    c.chunks = (uint32_t)((rows + c.chunk - 1) / c.chunk);
    c.padded = (uint64_t)c.chunks * c.chunk;
    const auto take = [&](uint64_t bytes) {
        const uint64_t at = c.bytes;
        c.bytes = (at + bytes + 255) & ~255ull;
        return at;
    };
    c.group = (uint32_t)columns;
    c.part_tokens = e->n_tokens;
    if (c.chunks > 1 && 4ull * c.chunks * e->n_tokens * e->dim > COL_PART_BYTES) {
        c.group = (uint32_t)std::clamp<uint64_t>(
            COL_PART_BYTES / (4ull * c.chunks * ids * e->dim), 1, columns);
        c.part_tokens = (uint32_t)std::min<uint64_t>(e->n_tokens, c.group * ids);
    }
    c.local = take(2 * c.padded * columns);
    c.counts = take(2ull * c.chunks * c.part_tokens);
    c.parts = take(c.chunks > 1 ? 4ull * c.chunks * c.part_tokens * e->dim : 0);
    return c;
}

// The gradient's workspace: two lists of sorted positions, a pass' counts, runs' parts.
struct GradPlan {
    uint32_t n = 0, passes = 0, bits = 0, blocks = 0, vec = 0, pieces = 0, lg_g = 0, chunk = 0,
             chunks = 0;
    bool few = false;    // buckets of 2^shift tokens
    uint32_t shift = 0;
    uint64_t keys[2], vals[2], counts = 0, totals = 0, parts = 0, bytes = 0;
};

GradPlan grad_plan(const fbh_embed *e) {
    GradPlan G;
    const uint64_t n = e->n_rows * e->n_columns;
    G.n = (uint32_t)n;
    const uint32_t key_bits = lg_at_least((uint64_t)e->n_tokens + 1);  // n_tokens: nothing
    G.passes = (key_bits + 7) / 8;
    G.bits = (key_bits + G.passes - 1) / G.passes;
    G.blocks = (uint32_t)((n + SORT_TPB * SORT_ROUNDS - 1) / (SORT_TPB * SORT_ROUNDS));
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
    if (n <= FEW_MOST && key_bits <= FEW_RANGE_BITS + FEW_BUCKET_BITS) {
        G.few = true;
        G.passes = 1;
        G.bits = std::min(key_bits, FEW_BUCKET_BITS);
        G.shift = key_bits - G.bits;
        G.blocks = (uint32_t)((n + SORT_TPB - 1) / SORT_TPB);
    }
    for (int i = 0; i < 2; i++) {
        G.keys[i] = take(4 * n);
        G.vals[i] = take(4 * n);
    }
    G.counts = take(4ull * (1u << G.bits) * G.blocks);
    G.totals = take(4 * 256);
    G.parts = take(8ull * G.chunks * e->dim);
    return G;
}

uint64_t grad_bytes(const fbh_embed *e) {
    head_input(e->n_rows * e->n_columns <= 0x7FFFFFFFull,
               "a gradient takes at most 2^31 - 1 positions");
    const ColumnPlan c = column_plan(e);
    return c.chunks ? c.bytes : grad_plan(e).bytes;
}

void columns_grad(const fbh_embed *e, const ColumnPlan &G, const void *grad, void *table,
                  void *work, hipStream_t s) {
    Positions P{e->ids, e->first, e->n_rows, e->n_columns, e->n_tokens, drop_key(e->seed),
                drop_threshold(e->drop)};
    if (!e->first) {
        P.n_rows *= P.n_columns;
        P.n_columns = 1;
    }
    const uint32_t most_ids = e->first ? e->most_ids : e->n_tokens;
    auto *w = static_cast<uint8_t *>(work);
    auto *local = reinterpret_cast<uint16_t *>(w + G.local);
    with_ids(e->id_type, e->drop > 0.0, [&](auto id, auto drop) {
        hipLaunchKernelGGL((column_ids_kernel<decltype(id)::value, decltype(drop)::value>),
                           dim3((uint32_t)(G.padded / 64), (P.n_columns + 63) / 64), dim3(256), 0,
                           s, P, most_ids, G.padded, local);
    });
    head_check(hipGetLastError(), "column ids");
    const uint32_t v = piece_cells(e->dim, e->dtype), pieces = (e->dim + v - 1) / v;
    const uint32_t lg_g = std::min(lg_at_least(pieces), 6u);
    Columns C{local, e->first, P.n_rows, G.padded, 0, 0, G.part_tokens, e->n_tokens, most_ids,
              G.chunk, G.chunks, e->pooled ? 1 : P.n_columns, e->dim, pieces, lg_g, scale_of(e),
              reinterpret_cast<float *>(w + G.parts), reinterpret_cast<uint16_t *>(w + G.counts),
              G.group < P.n_columns};
    with_cells(e->dtype, v, [&](auto one, auto vec) {
        using T = decltype(one);
        constexpr int VEC = decltype(vec)::value;
        const uint32_t lds = column_lds(most_ids, G.chunk, VEC).bytes;
        const uint32_t per = std::min(G.chunks, 8u);
        const auto sums = [&](auto buffer) {
            const auto kernel = &column_sums_kernel<T, VEC, decltype(buffer)::value>;
            if (lds > 64 * 1024)
                head_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize,
                                               128 * 1024),
                           "column sums");
            hipLaunchKernelGGL(kernel,
                               dim3((G.chunks + per - 1) / per * per * C.n_columns,
                                    (pieces + (1u << lg_g) - 1) >> lg_g),
                               dim3(COL_TPB), lds, s, C, static_cast<const T *>(grad),
                               static_cast<T *>(table));
        };
        const uint64_t row_bytes = (uint64_t)C.per_row * e->dim * sizeof(T);
        for (uint32_t t = 0; t < P.n_columns; t += G.group) {
            C.column0 = t;
            C.n_columns = std::min(G.group, P.n_columns - t);
            if constexpr (VEC * sizeof(T) >= 4) {
                if (row_bytes <= BUFFER_MOST / COL_MOST_ROWS &&
                    in_buffer(grad, G.chunk * row_bytes, e->dim * sizeof(T)))
                    sums(std::true_type{});
                else sums(std::false_type{});
            } else sums(std::false_type{});
            head_check(hipGetLastError(), "column sums");
            if (G.chunks == 1) return;
            const uint64_t threads = (uint64_t)G.part_tokens * pieces;
            hipLaunchKernelGGL((column_join_kernel<T, VEC>),
                               dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, s, C,
                               static_cast<T *>(table));
            head_check(hipGetLastError(), "column sums");
        }
    });
}

void embed_grad(const fbh_embed *e, const void *grad, void *table, void *work, hipStream_t s) {
    if (const ColumnPlan G = column_plan(e); G.chunks) return columns_grad(e, G, grad, table, work, s);
    Positions P{e->ids, e->first, e->n_rows, e->n_columns, e->n_tokens, drop_key(e->seed),
                drop_threshold(e->drop)};
    if (!e->first) {
        P.n_rows *= P.n_columns;
        P.n_columns = 1;
    }
    const GradPlan G = grad_plan(e);
    auto *w = static_cast<uint8_t *>(work);
    const auto list = [&](uint64_t at) { return reinterpret_cast<uint32_t *>(w + at); };
    const uint64_t zero_bytes =
        (uint64_t)e->n_tokens * e->dim * (e->dtype == FBH_F32 ? 4 : 2);
    uint32_t *counts = list(G.counts), *totals = list(G.totals);
    for (uint32_t pass = 0; pass < G.passes; pass++) {
        const uint32_t to = pass & 1;
        const SortFrom S{list(G.keys[1 - to]), list(G.vals[1 - to]), G.n,
                         G.few ? G.shift : pass * G.bits, G.bits, e->pooled ? e->n_columns : 1,
                         G.blocks, static_cast<uint8_t *>(table), zero_bytes};
        const uint32_t more = pass == 0 ? ZERO_BLOCKS : 0;
        uint32_t *keys = list(G.keys[to]), *vals = list(G.vals[to]);
        const auto go = [&](auto id, auto drop, auto first, auto rounds) {
            constexpr int ID = decltype(id)::value;
            constexpr bool DROP = decltype(drop)::value, FIRST = decltype(first)::value;
            constexpr uint32_t ROUNDS = decltype(rounds)::value;
            hipLaunchKernelGGL((sort_count_kernel<ID, DROP, FIRST, ROUNDS>), dim3(G.blocks + more),
                               dim3(SORT_TPB), 0, s, P, S, counts);
            hipLaunchKernelGGL(sort_scan_kernel, dim3((1u << G.bits) + more), dim3(SORT_TPB), 0, s,
                               S, counts, totals);
            hipLaunchKernelGGL((sort_scatter_kernel<ID, DROP, FIRST, ROUNDS>), dim3(G.blocks + more),
                               dim3(SORT_TPB), 0, s, P, S, counts, totals, keys, vals);
        };
        if (pass == 0)
            with_ids(e->id_type, e->drop > 0.0, [&](auto id, auto drop) {
                if (G.few) go(id, drop, std::true_type{}, Int<1>{});
                else go(id, drop, std::true_type{}, Int<SORT_ROUNDS>{});
            });
        else go(Int<FBH_ID_I32>{}, std::false_type{}, std::false_type{}, Int<SORT_ROUNDS>{});
        head_check(hipGetLastError(), "token sort");
        if (G.n == 0) return;  // (the table's zeros were all)
    }
    if (G.few) {
        const Few F{e->n_tokens, G.shift, totals, list(G.keys[0]), list(G.vals[0]),
                    list(G.keys[1]), list(G.vals[1])};
        hipLaunchKernelGGL(few_sort_kernel, dim3((e->n_tokens >> G.shift) + 1), dim3(FEW_TPB),
                           (FEW_WAVES * 4) << G.shift, s, F);
        head_check(hipGetLastError(), "token sort");
    }
    const uint32_t at = G.few ? 1 : (G.passes - 1) & 1;
    const Runs R{list(G.keys[at]), list(G.vals[at]), G.n, G.chunk, e->n_tokens, e->dim, G.pieces,
                 G.lg_g, scale_of(e), reinterpret_cast<float *>(w + G.parts)};
    with_cells(e->dtype, G.vec, [&](auto one, auto vec) {
        using T = decltype(one);
        constexpr int VEC = decltype(vec)::value;
        const uint32_t groups = EMB_TPB >> G.lg_g, join = JOIN_TPB >> G.lg_g;
        const uint32_t y = (G.pieces + (1u << G.lg_g) - 1) >> G.lg_g;
        hipLaunchKernelGGL((grad_runs_kernel<T, VEC>), dim3((G.chunks + groups - 1) / groups, y),
                           dim3(EMB_TPB), 0, s, R, static_cast<const T *>(grad),
                           static_cast<T *>(table));
        hipLaunchKernelGGL((grad_join_kernel<T, VEC>), dim3((G.chunks + join - 1) / join, y),
                           dim3(JOIN_TPB), 0, s, R, static_cast<T *>(table));
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
        bytes = grad_bytes(e);
    });
    return bytes;
}

int fbh_embed_grad(int device, const fbh_embed *e, const void *grad, void *table, void *work,
                   uint64_t work_bytes, void *stream) {
    return head_guard([&] {
        check_embed(e);
        head_input(table && (grad || e->n_rows == 0), "null argument");
        const uint64_t need = grad_bytes(e);
        head_input(work_bytes >= need && (work || need == 0), "the workspace is too small");
        head_input(reinterpret_cast<uintptr_t>(work) % 16 == 0,
                   "the workspace is not aligned to 16 bytes");
        const OnDevice on(device);
        embed_grad(e, grad, table, work, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
