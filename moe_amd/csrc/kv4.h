// kv4.h — the paged 4-bit key/value cache's layout (moe_kv4 in moe_hip.h) for
// the kernels that write and read it.
//
// A tile is 32 positions of one kv head: the keys' codes, the values' codes,
// the keys' scales, the values' scales.  Codes are laid out as the operands of
// the 16x16x32 f16 matrix instruction read them, so that a wave's loads of a
// tile are whole 1 KiB runs and each lane unpacks its own operand:
//   keys    S^T = K Q^T: a lane holds one position and eight of a block's 32
//           dims, one word: dims 4g..4g+3 (low nibbles), 16+4g.. (high)
//   values  O^T = V^T P^T: a lane holds one dim and eight positions; two words
//           (positions 4g.. and 16+4g..) hold two dims, d (low), d + 16 (high)
// The contraction runs over the same index on both sides, so its order inside
// a lane is free; nibble pairs 16 bits apart unpack to f16 pairs in one
// instruction each.  Scales lie as the product's result wants them: a lane's
// four positions of both halves side by side.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "moe_internal.h"

namespace moe {

constexpr int kTile = 32;  // positions of a tile

// Byte offset of word w (2 block + half) of a lane in a region of nb blocks:
// chunks of four words a lane, the last of two where nb is odd.
__host__ __device__ inline int kv4_word(int nb, int w, int lane) {
    return (w >> 2) * 1024 + lane * ((w >> 2) < nb / 2 ? 16 : 8) + (w & 3) * 4;
}
// Byte of a tile's key region holding dims 32 s + j and + 16 of position p (j < 16).
__host__ __device__ inline int kv4_key_byte(int nb, int p, int s, int j) {
    return kv4_word(nb, 2 * s + (p >> 4), 16 * (j >> 2) + (p & 15)) + (j & 3);
}
// The same in the value region.
__host__ __device__ inline int kv4_value_byte(int nb, int p, int b, int j) {
    return kv4_word(nb, 2 * b + (p >> 4), 16 * ((p & 15) >> 2) + j) + (p & 3);
}
// Index among a region's scales of block s at position p.
__host__ __device__ inline int kv4_scale_at(int p, int s) { return s * 32 + ((p & 15) >> 2) * 8 + (p >> 4) * 4 + (p & 3); }

// One layer's cache as the kernels take it.
struct Kv4 {
    uint8_t *pool;
    const int32_t *table;
    __half *means;
    int n_seq, max_pages, n_pages, n_kv, qd, vd;
    int page_shift;  // log2 of the positions of a page
    int tile_bytes;
    __host__ __device__ int tiles() const { return 1 << (page_shift - 5); }
    // First tile of a page's kv head.
    __host__ __device__ uint8_t *head(int page, int kv) const {
        return pool + (((size_t)page * n_kv + kv) << (page_shift - 5)) * (size_t)tile_bytes;
    }
    __host__ __device__ int v_codes() const { return 16 * qd; }
    __host__ __device__ int k_scales() const { return 16 * (qd + vd); }
    __host__ __device__ int v_scales() const { return 18 * qd + 16 * vd; }
};

// A launch is at most 2^32 - 1 threads.
constexpr long long kMostThreads = 0xffffffffll;

// Checks a caller's cache and turns it into the kernels' form: 0 or a
// MOE_E* code with its message set.
int kv4_of(const char *what, const moe_kv4 *c, Kv4 *out);

}  // namespace moe
