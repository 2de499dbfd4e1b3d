// int8.h — how groups of values are held in 8 bits with one f32 scale (a row of
// an integer product's operands, a block of the 8-bit cache).
//
//   scale = max|v| / 127, code = round(v * (127 / max|v|)), halves to even,
// every step rounded to f32.  A group whose largest value is below 2^-100 is
// held as zeros (the reciprocal would leave f32's range); one with an infinity
// or a NaN has a NaN for its scale and so reads as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

// The largest magnitude of a group as bits: above 0x7f800000 for a NaN.
__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Int8Scale {
    float scale, inv;
    __device__ explicit Int8Scale(uint32_t top) {
        const float m = __uint_as_float(top);
        const bool finite = top < 0x7f800000u, some = finite && m >= 0x1p-100f;
        scale = some ? m / 127.0f : finite ? 0.0f : __uint_as_float(0x7fc00000u);
        inv = some ? 127.0f / m : 0.0f;
    }
    // (a value beside a NaN, which inv = 0 makes 0 or NaN, gets 0)
    __device__ int code(float v) const { return inv == 0.0f ? 0 : (int)rintf(v * inv); }
};

__device__ inline uint32_t pack4(int a, int b, int c, int d) {
    return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | (uint32_t)d << 24;
}

}  // namespace moe
