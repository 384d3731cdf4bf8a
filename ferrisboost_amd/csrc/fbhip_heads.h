// fbhip_heads.h -- what the kernels of the heads on a model's outputs share
// (fbhip_embed.hip, fbhip_dropout.hip, fbhip_sample.hip): cell types, 16-byte
// pieces, the counter-based generator, errors and the calling device.
#pragma once

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "../../include/fbhip.h"
#include "fbhip_internal.h"

namespace fbh {

struct HeadError : std::runtime_error {
    int code;
    HeadError(int c, const std::string &m) : std::runtime_error(m), code(c) {}
};

inline void head_check(hipError_t e, const char *what) {
    if (e != hipSuccess)
        throw HeadError(FBH_RUNTIME_ERROR, std::string(what) + ": " + hipGetErrorString(e));
}

inline void head_input(bool ok, const char *message) {
    if (!ok) throw HeadError(FBH_INPUT_ERROR, message);
}

template <class F>
int head_guard(F &&f) {
    try {
        f();
        return FBH_OK;
    } catch (const HeadError &e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return FBH_RUNTIME_ERROR;
    } catch (...) {
        set_last_error("unknown error");
        return FBH_RUNTIME_ERROR;
    }
}

// The call's device, and the caller's one again afterwards.
class OnDevice {
    int before_ = -1;

  public:
    explicit OnDevice(int device) {
        int now = 0;
        head_check(hipGetDevice(&now), "hipGetDevice");
        if (now == device) return;
        head_check(hipSetDevice(device), "hipSetDevice");
        before_ = now;
    }
    ~OnDevice() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
};

// N cells as they lie in memory, moved together whatever their alignment (global
// loads and stores of up to 16 bytes need none on this device).
template <class T, int N>
struct Piece {
    T v[N];
};
template <class T, int N>
__device__ __forceinline__ Piece<T, N> load_piece(const T *p) {
    Piece<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <class T, int N>
__device__ __forceinline__ void store_piece(T *p, const Piece<T, N> &r) {
    __builtin_memcpy(p, &r, sizeof(r));
}

// Outputs beyond what the caches keep for whoever reads them next are written past them:
// 1.28 GB of vectors of 32 bytes (2M x 20 ids) take 320 to 335 us so, and 428 through the
// caches, where lines wait for their eviction; of 128 bytes 228 and 291, of 256 as bfloat16
// 225 and 287 (ids and outputs of another pass before them in the caches). Smaller ones stay
// in the cache for the next kernel.
constexpr uint64_t STREAM_BYTES = 128ull << 20;
template <class T, int N>
__device__ __forceinline__ void stream_piece(T *p, const Piece<T, N> &r) {
    static_assert(sizeof(r) == 16, "whole pieces");
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    typedef Words Loose __attribute__((aligned(2)));
    Words w;
    __builtin_memcpy(&w, &r, 16);
    __builtin_nontemporal_store(w, reinterpret_cast<Loose *>(p));
}

// Buffer loads: 4-byte aligned pieces at byte offsets of up to 2^31 - 1 from an address
// that all lanes share. What lies at or behind `bytes` reads as zeros, so a position that
// gives nothing needs an offset (NO_OFFSET) and no select; and an offset takes one
// 32-bit operation where an address takes a 64-bit product and sum.
constexpr uint32_t NO_OFFSET = 0x80000000u;
constexpr uint64_t BUFFER_MOST = 0x7FF00000ull;  // bytes; cells of a row come on top
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000);
}
template <class T, int N>
__device__ __forceinline__ Piece<T, N> load_offset(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    Piece<T, N> p;
    if constexpr (sizeof(p) == 16) {
        const auto q = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
        __builtin_memcpy(&p, &q, 16);
    } else if constexpr (sizeof(p) == 8) {
        const auto q = __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0);
        __builtin_memcpy(&p, &q, 8);
    } else {
        static_assert(sizeof(p) == 4, "a piece of whole words");
        const auto q = __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
        __builtin_memcpy(&p, &q, 4);
    }
    return p;
}

// ---- The counter-based generator: element e takes half of the 64 bits that the
// SplitMix64 finaliser gives for a seed's key and e / 2, as row sampling takes a
// row's bits from seed and row. Nothing is stored: whoever knows seed and element
// has the same bits again.
constexpr uint64_t DROP_STEP = 0xD6E8FEB86659FD93ull;

__host__ __device__ inline uint64_t drop_mix(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
inline uint64_t drop_key(uint64_t seed) { return drop_mix(seed ^ 0x9E3779B97F4A7C15ull); }

__device__ __forceinline__ uint64_t drop_word(uint64_t key, uint64_t pair) {
    return drop_mix(key ^ (pair * DROP_STEP));
}
__device__ __forceinline__ uint32_t drop_bits(uint64_t key, uint64_t e) {
    const uint64_t w = drop_word(key, e >> 1);
    return (e & 1) ? (uint32_t)(w >> 32) : (uint32_t)w;
}

// The bits of two elements where the lanes 2j and 2j + 1 hold neighbours, an even one and
// the next, both times: each lane hashes one of the two pairs and takes the other lane's
// word for the other. (A hash is 12 multiplies at a quarter of the rate; one for every
// element was two thirds of the time that 10M ids took to decode.)
__device__ __forceinline__ void drop_bits_of_neighbours(uint64_t key, const uint64_t (&e)[2],
                                                        uint32_t (&bits)[2]) {
    const bool odd = threadIdx.x & 1;
    const uint64_t mine = drop_word(key, (odd ? e[1] : e[0]) >> 1);
    const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
    const uint32_t other_lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)lo, 0xB1, 0xF, 0xF, true);
    const uint32_t other_hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)hi, 0xB1, 0xF, 0xF, true);
    bits[0] = odd ? other_hi : lo;
    bits[1] = odd ? hi : other_lo;
}

// Elements whose 32 bits are below this are dropped.
inline uint32_t drop_threshold(double drop) {
    head_input(drop >= 0.0 && drop < 1.0, "drop must be in [0, 1)");
    const double t = __builtin_rint(drop * 4294967296.0);
    return t >= 4294967295.0 ? 4294967295u : (uint32_t)t;
}

}  // namespace fbh
