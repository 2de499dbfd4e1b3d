// int8_linear.hip — products in 8-bit integers with a scale for each token and
// each channel (moe_int8_*).
//
//   y[t][n] = (sum_k cx[t][k] cw[n][k]) * (sx[t] * sw[n])
// with rows of x and of the weights held as int8.h says; the sum is exact in 32
// bits.  Codes of both operands lie as the 16x16x64 integer instruction reads
// them: a tile is 16 rows by 64 values, 1 KiB, lane (row % 16, g) holding values
// 16 g .. 16 g + 15:
//   [row / 16][k / 64][lane][16]
// so that a wave's load of a tile is one contiguous KiB and goes into the
// product as it is.  Rows and values past the matrix are zeros.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "int8.h"
#include "moe_internal.h"
#include "row_value.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMostK = 131072;  // 127 * 127 * K stays below 2^31

__host__ __device__ inline int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
// Byte of a packed matrix (chunks of 64 values a row) at which 16 values lie.
__host__ __device__ inline int64_t group_at(int64_t row, int64_t k, int64_t chunks) {
    return ((row >> 4) * chunks + (k >> 6)) * 1024 + (k >> 4 & 3) * 256 + (row & 15) * 16;
}

__device__ inline uint32_t block_max(uint32_t v, uint32_t *red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}

// Row blockIdx.x of a matrix in a checkpoint's format, into row row0 + it.
__global__ __launch_bounds__(256) void int8_pack_kernel(const uint8_t *__restrict__ w, int dt, int64_t row_bytes, int k,
                                                        int row0, uint8_t *__restrict__ codes, float *__restrict__ scales) {
    __shared__ uint32_t red[4];
    const uint8_t *row = w + (int64_t)blockIdx.x * row_bytes;
    const int64_t chunks = up(k, 64) / 64, to = row0 + blockIdx.x;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < k; i += 256) top = max(top, magnitude(row_value(row, dt, i)));
    const Int8Scale s(block_max(top, red));
    for (int g = threadIdx.x; g < chunks * 4; g += 256) {
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int c[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 16 * g + 4 * j + e;
                c[e] = i < k ? s.code(row_value(row, dt, i)) : 0;
            }
            y[j] = pack4(c[0], c[1], c[2], c[3]);
        }
        gstore((u32x4 *)(codes + group_at(to, 16 * (int64_t)g, chunks)), u32x4{y[0], y[1], y[2], y[3]});
    }
    if (threadIdx.x == 0) scales[to] = s.scale;
}

// Rows of x, a block each; rows up to the next 16th are zeros.
__global__ __launch_bounds__(256) void int8_rows_kernel(const float *__restrict__ x, int64_t xs, int t, int k,
                                                        uint8_t *__restrict__ codes, float *__restrict__ scales) {
    __shared__ uint32_t red[4];
    const int64_t to = blockIdx.x, chunks = up(k, 64) / 64;
    const float *row = x + to * xs;
    uint32_t top = 0;
    if (to < t)
        for (int i = threadIdx.x; i < k; i += 256) top = max(top, magnitude(gload(row + i)));
    const Int8Scale s(block_max(top, red));
    for (int g = threadIdx.x; g < chunks * 4; g += 256) {
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int c[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 16 * g + 4 * j + e;
                c[e] = to < t && i < k ? s.code(gload(row + i)) : 0;
            }
            y[j] = pack4(c[0], c[1], c[2], c[3]);
        }
        gstore((u32x4 *)(codes + group_at(to, 16 * (int64_t)g, chunks)), u32x4{y[0], y[1], y[2], y[3]});
    }
    if (threadIdx.x == 0) scales[to] = s.scale;
}

struct Product {
    const uint8_t *w, *x;
    const float *sw, *sx;
    float *y, *residual;
    int64_t ys, rs;
    int n, t;
    int64_t chunks;
};

// A wave computes 16 channels of 16 tokens: lane (token, g) ends with channels
// 4 g .. 4 g + 3.
__global__ __launch_bounds__(256) void int8_product_kernel(const Product p) {
    const int lane = threadIdx.x & 63;
    const int64_t nt = blockIdx.x * 4 + (threadIdx.x >> 6), tt = blockIdx.y;
    if (nt * 16 >= p.n) return;
    const u32x4 *w = (const u32x4 *)(p.w + nt * p.chunks * 1024) + lane, *x = (const u32x4 *)(p.x + tt * p.chunks * 1024) + lane;
    i32x4 acc = {0, 0, 0, 0};
    for (int64_t c = 0; c < p.chunks; c++)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, gload(w + 64 * c)),
                                                    __builtin_bit_cast(i32x4, gload(x + 64 * c)), acc, 0, 0, 0);
    const int64_t t = tt * 16 + (lane & 15), n = nt * 16 + 4 * (lane >> 4);
    if (t >= p.t) return;
    const float sx = gload(p.sx + t);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (n + i >= p.n) continue;
        const float v = (float)acc[i] * (sx * gload(p.sw + n + i));
        gstore(p.y + t * p.ys + n + i, v);
        if (p.residual) p.residual[t * p.rs + n + i] += v;
    }
}

int sizes_ok(const char *what, int32_t n, int32_t k) {
    if (n <= 0 || k <= 0) return fail(MOE_EINVAL, "%s: %d channels of %d values", what, n, k);
    if (k > kMostK) return fail(MOE_EUNSUP, "%s: %d values a channel, up to %d (sums of 32 bits)", what, k, kMostK);
    if (n > (1 << 24)) return fail(MOE_EUNSUP, "%s: %d channels, up to %d", what, n, 1 << 24);
    return MOE_OK;
}
uint64_t codes_bytes(int64_t rows, int64_t k) { return (uint64_t)(up(rows, 16) * up(k, 64)); }
uint64_t packed_size(int64_t rows, int64_t k) { return codes_bytes(rows, k) + (uint64_t)up(rows, 16) * 4; }

int done(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_int8_pack_size(int32_t n, int32_t k, uint64_t *bytes) {
    if (const int rc = sizes_ok("moe_int8_pack_size", n, k)) return rc;
    if (!bytes) return fail(MOE_EINVAL, "moe_int8_pack_size: bad argument");
    *bytes = packed_size(n, k);
    return MOE_OK;
}

int moe_int8_pack(const void *w, int32_t dt, int64_t row_bytes, int32_t rows, int32_t row0, int32_t n, int32_t k,
                  void *packed, uint64_t packed_bytes, void *stream) {
    if (const int rc = sizes_ok("moe_int8_pack", n, k)) return rc;
    const uint64_t rb = moe_row_bytes(dt, (uint64_t)k);
    if (dt != MOE_DT_F32 && dt != MOE_DT_F16 && dt != MOE_DT_BF16 && dt != MOE_DT_Q8_0 && dt != MOE_DT_Q4_0 && dt != MOE_DT_Q5_0)
        return fail(MOE_EUNSUP, "moe_int8_pack: rows of format %d", dt);
    if (rows < 0 || row0 < 0 || row0 > n - rows || rb == 0 || (dt != MOE_DT_F32 && dt != MOE_DT_F16 && dt != MOE_DT_BF16 && k % 32) ||
        row_bytes < (int64_t)rb || (rows && (!w || !packed)) || (uintptr_t)packed % 256 || packed_bytes < packed_size(n, k))
        return fail(MOE_EINVAL, "moe_int8_pack: bad argument (rows %d to %d of %d, %d values of format %d)", row0, row0 + rows, n, k, dt);
    if (rows == 0) return MOE_OK;
    uint8_t *codes = static_cast<uint8_t *>(packed);
    hipLaunchKernelGGL(int8_pack_kernel, dim3(rows), dim3(256), 0, (hipStream_t)stream, static_cast<const uint8_t *>(w), dt,
                       row_bytes, k, row0, codes, reinterpret_cast<float *>(codes + codes_bytes(n, k)));
    return done("weight packing kernel");
}

int moe_int8_linear_workspace_size(int32_t n, int32_t k, int32_t t, uint64_t *bytes) {
    if (const int rc = sizes_ok("moe_int8_linear_workspace_size", n, k)) return rc;
    if (!bytes || t < 0) return fail(MOE_EINVAL, "moe_int8_linear_workspace_size: bad argument (%d tokens)", t);
    *bytes = packed_size(t, k);
    return MOE_OK;
}

int moe_int8_linear(const void *packed, int32_t n, int32_t k, const float *x, int64_t x_stride, int32_t t, float *y,
                    int64_t y_stride, float *residual, int64_t residual_stride, void *workspace, uint64_t workspace_bytes,
                    void *stream) {
    if (const int rc = sizes_ok("moe_int8_linear", n, k)) return rc;
    if (t < 0 || t > (1 << 20)) return fail(MOE_EINVAL, "moe_int8_linear: %d tokens, up to %d", t, 1 << 20);
    if (t == 0) return MOE_OK;
    if (!packed || (uintptr_t)packed % 256 || !x || !y) return fail(MOE_EINVAL, "moe_int8_linear: bad argument");
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < packed_size(t, k))
        return fail(MOE_EINVAL, "moe_int8_linear: workspace of %llu bytes (256-byte aligned), %llu needed",
                    (unsigned long long)workspace_bytes, (unsigned long long)packed_size(t, k));
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *w = static_cast<const uint8_t *>(packed);
    uint8_t *xc = static_cast<uint8_t *>(workspace);
    float *sx = reinterpret_cast<float *>(xc + codes_bytes(t, k));
    hipLaunchKernelGGL(int8_rows_kernel, dim3((unsigned)up(t, 16)), dim3(256), 0, s, x, x_stride, t, k, xc, sx);
    const Product p{w, xc, reinterpret_cast<const float *>(w + codes_bytes(n, k)), sx, y, residual, y_stride, residual_stride, n, t,
                    up(k, 64) / 64};
    hipLaunchKernelGGL(int8_product_kernel, dim3((unsigned)(up(n, 64) / 64), (unsigned)(up(t, 16) / 16)), dim3(256), 0, s, p);
    return done("8-bit product kernel");
}

}  // extern "C"
