// kv8.h — the paged 8-bit cache's layout (moe_kv8 in moe_hip.h) for the kernels
// that write and read it.
//
// A tile is 64 positions of one kv head, four blocks of 16 positions with a
// scale each for keys and values (int8.h).  Codes are the operands of the
// 16x16x64 integer instruction as they stand; its contraction runs over the
// same index on both sides, so its order inside a lane is free:
//   keys    S = K Q^T, a block's 16 positions by 64 dims: lane (position, g)
//           holds dims 64 c + 16 g ..  -> [block][dims / 16][position][16]
//   values  O^T = V^T P^T, 16 dims by the tile's 64 positions: the product
//           before it leaves lane (column, g) with positions 16 T + 4 g + i of
//           block T, so lane (dim, g) holds those -> [dims / 16][g][dim][T][i]
#pragma once
#include <hip/hip_runtime.h>

#include "moe_internal.h"

namespace moe {

constexpr int kTile8 = 64, kBlock8 = 16;  // positions of a tile, of a block

// One layer's cache as the kernels take it.
struct Kv8 {
    uint8_t *codes;
    float *scales;
    uint8_t *open;
    const int32_t *table;
    int n_seq, max_pages, n_pages, n_kv, qd, vd;
    int page_shift;  // log2 of the positions of a page
    __host__ __device__ int tile_bytes() const { return kTile8 * (qd + vd); }
    __host__ __device__ int values() const { return kTile8 * qd; }  // where a tile's values begin
    // Number of the tile holding a page's position `off`.
    __host__ __device__ int64_t tile(int page, int kv, int off) const {
        return (((int64_t)page * n_kv + kv) << (page_shift - 6)) + (off >> 6);
    }
    __host__ __device__ uint8_t *at(int64_t tile) const { return codes + tile * tile_bytes(); }
    __host__ __device__ float *scale_at(int64_t tile, bool key, int block) const { return scales + tile * 8 + (key ? 0 : 4) + block; }
    // The values of a sequence's blocks that are filling: see moe_kv8_store.
    __host__ __device__ int64_t open_bytes() const { return 2 * kBlock8 * 4 * (qd + vd) + 32; }
    __host__ __device__ uint8_t *open_at(int seq, int kv) const { return open + ((int64_t)seq * n_kv + kv) * open_bytes(); }
};

// Byte in a tile's keys or values of dim d of position p.
__host__ __device__ inline int kv8_key_byte(int qd, int p, int d) {
    return (p >> 4) * 16 * qd + (d >> 4) * 256 + (p & 15) * 16 + (d & 15);
}
__host__ __device__ inline int kv8_value_byte(int p, int d) {
    return (d >> 4) * 1024 + ((p & 15) >> 2) * 256 + (d & 15) * 16 + (p >> 4) * 4 + (p & 3);
}

int kv8_of(const char *what, const moe_kv8 *c, Kv8 *out);

}  // namespace moe
