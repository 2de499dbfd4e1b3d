// rotate.h — one pair's rotation (src/model.rs:324-333), the same arithmetic
// wherever a kernel rotates.
#pragma once
#include <hip/hip_runtime.h>

namespace moe {

__device__ inline void rotate(float a, float b, float c, float s, float &x, float &y) {
    const float u = fmaf(a, c, -(b * s)), v = fmaf(a, s, b * c);
    x = u, y = v;
}

}  // namespace moe
