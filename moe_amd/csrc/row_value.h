// row_value.h — single values of rows stored in a checkpoint's formats.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_internal.h"

namespace moe {

__device__ inline float half_at(const uint8_t *p) {
    return __half2float(__ushort_as_half((unsigned short)(p[0] | (p[1] << 8))));
}

// Value c of a stored row (src/quant.rs:177-227).
__device__ inline float row_value(const uint8_t *row, int dt, int c) {
    const int b = c >> 5, i = c & 31;
    switch (dt) {
    case MOE_DT_F32: {
        float v;
        __builtin_memcpy(&v, row + 4 * (size_t)c, 4);
        return v;
    }
    case MOE_DT_F16: return half_at(row + 2 * (size_t)c);
    case MOE_DT_BF16: {
        const uint32_t u = (uint32_t)(row[2 * (size_t)c] | (row[2 * (size_t)c + 1] << 8)) << 16;
        return __uint_as_float(u);
    }
    case MOE_DT_Q8_0: {
        const uint8_t *blk = row + 34 * (size_t)b;
        return half_at(blk) * (float)(int8_t)blk[2 + i];
    }
    case MOE_DT_Q4_0: {
        const uint8_t *blk = row + 18 * (size_t)b;
        const uint32_t v = blk[2 + (i & 15)];
        const int nib = i < 16 ? (int)(v & 15) : (int)(v >> 4);
        return half_at(blk) * (float)(nib - 8);
    }
    default: {  // Q5_0
        const uint8_t *blk = row + 22 * (size_t)b;
        const uint32_t v = blk[6 + (i & 15)];
        const int nib = i < 16 ? (int)(v & 15) : (int)(v >> 4);
        const int hb = (blk[2 + i / 8] >> (i % 8)) & 1;
        return half_at(blk) * (float)((nib | (hb << 4)) - 16);
    }
    }
}

}  // namespace moe
