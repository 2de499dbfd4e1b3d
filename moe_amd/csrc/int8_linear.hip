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
// product as it is.  Values past a row's last are zeros, and so are x's rows past
// its last (channels past the last are whatever is there: nothing reads their sums).
//
// Large products: 8191 x 6144 x 4096 in 175 us, 2357 TOP/s (the library's own takes
// 183), the rows' codes before it 40 (168 MB, 4.2 TB/s).  A step of the 256 x 256
// kernel takes the matrix pipe 1024 of its 2067 cycles, and the LDS port, with 12
// operand tiles a wave for 32 products and the DMA's writes, about as many; the two
// overlap little (pipe 50% busy at 2.05 GHz, waves waiting 44% of their time).  Few
// rows are bound by the weights' bytes: 32 rows of 6144 x 4096 6.8 us (3.8 TB/s) after
// 3.0 for the codes, one row of 4096 x 4096 5.0 in all (3.4 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "int8.h"
#include "lds_dma.h"
#include "moe_internal.h"
#include "row_value.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // at any float
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

// Block b's row: the rows of a tile, 16 in turn, go to one XCD, so that the
// bytes of a line that different rows write meet in one L2.
__device__ inline int64_t row_of(unsigned b) { return (int64_t)((b >> 7) * 8 + (b & 7)) * 16 + (b >> 3 & 15); }
unsigned row_blocks(int64_t rows) { return (unsigned)((rows + 127) / 128 * 128); }

// Rows of x, a block each, a thread 16 values at a time (kept in registers where
// a row has no more than kHeld of them); rows up to the next 16th are zeros.
constexpr int kHeld = 2;
__global__ __launch_bounds__(256) void int8_rows_kernel(const float *__restrict__ x, int64_t xs, int t, int k,
                                                        uint8_t *__restrict__ codes, float *__restrict__ scales) {
    __shared__ uint32_t red[4];
    const int64_t to = row_of(blockIdx.x), chunks = up(k, 64) / 64;
    if (to >= up(t, 16)) return;
    const float *row = x + to * xs;
    const int units = (int)chunks * 4, whole = to < t ? k / 16 : 0;
    auto values = [&](int u, float (&v)[16]) __attribute__((always_inline)) {
        if (u < whole) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u32x4_dw y = gload_x4((const uint32_t *)row + 16 * u + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * j + e] = __uint_as_float(y[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = to < t && 16 * u + e < k ? gload(row + 16 * u + e) : 0.0f;
        }
    };
    float held[kHeld][16];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
        const int u = threadIdx.x + 256 * j;
        if (u >= units) continue;
        values(u, held[j]);
#pragma unroll
        for (int e = 0; e < 16; e++) top = max(top, magnitude(held[j][e]));
    }
    for (int u = threadIdx.x + 256 * kHeld; u < units; u += 256) {
        float v[16];
        values(u, v);
#pragma unroll
        for (int e = 0; e < 16; e++) top = max(top, magnitude(v[e]));
    }
    const Int8Scale s(block_max(top, red));
    auto write = [&](int u, const float (&v)[16]) __attribute__((always_inline)) {
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = pack4(s.code(v[4 * j]), s.code(v[4 * j + 1]), s.code(v[4 * j + 2]), s.code(v[4 * j + 3]));
        gstore((u32x4 *)(codes + group_at(to, 16 * (int64_t)u, chunks)), u32x4{y[0], y[1], y[2], y[3]});
    };
#pragma unroll
    for (int j = 0; j < kHeld; j++)
        if (threadIdx.x + 256 * j < units) write(threadIdx.x + 256 * j, held[j]);
    for (int u = threadIdx.x + 256 * kHeld; u < units; u += 256) {
        float v[16];
        values(u, v);
        write(u, v);
    }
    if (threadIdx.x == 0) scales[to] = s.scale;
}

struct Product {
    const uint8_t *w, *x;
    const float *sw, *sx;
    float *y, *residual;
    int64_t ys, rs;
    int n, t, chunks;
    int nt, tt;  // tiles of 16 channels, of 16 tokens
};

// y and residual of one channel and token.
__device__ inline void finish(const Product &p, int64_t t, int64_t n, int sum, float sx, float sw) {
    const float v = (float)sum * (sx * sw);
    gstore(p.y + t * p.ys + n, v);
    if (p.residual) gstore(p.residual + t * p.rs + n, gload(p.residual + t * p.rs + n) + v);
}

// y and residual of channels n .. n + 3 (as many as there are) of one token.
__device__ inline void finish4(const Product &p, int64_t t, int64_t n, i32x4 sum, float sx, f32x4_dw sw) {
    if (n + 4 > p.n) {
        for (int e = 0; n + e < p.n; e++) finish(p, t, n + e, sum[e], sx, sw[e]);
        return;
    }
    f32x4_dw v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)sum[e] * (sx * sw[e]);
    *(__attribute__((address_space(1))) f32x4_dw *)(p.y + t * p.ys + n) = v;
    if (!p.residual) return;
    __attribute__((address_space(1))) f32x4_dw *r = (__attribute__((address_space(1))) f32x4_dw *)(p.residual + t * p.rs + n);
    f32x4_dw z = *r;
#pragma unroll
    for (int e = 0; e < 4; e++) z[e] += v[e];
    *r = z;
}

// MT x NT tiles of 16 tokens by 16 channels a block, operands straight from
// memory, the chunks of K dealt to W waves whose sums meet in LDS.
template <int MT, int NT, int W>
__global__ __launch_bounds__(W * 64) void int8_direct_kernel(const Product p) {
    __shared__ i32x4 sums[W > 1 ? (W - 1) * MT * NT * 64 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * NT, t0 = blockIdx.y * MT;
    const u32x4 *w[NT], *x[MT];
#pragma unroll
    for (int j = 0; j < NT; j++) w[j] = (const u32x4 *)(p.w + (int64_t)min(n0 + j, p.nt - 1) * p.chunks * 1024) + lane;
#pragma unroll
    for (int i = 0; i < MT; i++) x[i] = (const u32x4 *)(p.x + (int64_t)min(t0 + i, p.tt - 1) * p.chunks * 1024) + lane;
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    // U chunks' loads at a time; past the last chunk the last one again, whose
    // products are left out.
    constexpr int U = MT + NT <= 3 ? 8 : MT + NT <= 6 ? 4 : 2;
    for (int c0 = wave; c0 < p.chunks; c0 += W * U) {
        i32x4 a[U][MT], b[U][NT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = min(c0 + u * W, p.chunks - 1);
#pragma unroll
            for (int j = 0; j < NT; j++) b[u][j] = __builtin_bit_cast(i32x4, gload(w[j] + 64 * c));
#pragma unroll
            for (int i = 0; i < MT; i++) a[u][i] = __builtin_bit_cast(i32x4, gload(x[i] + 64 * c));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c0 + u * W >= p.chunks) continue;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][i], b[u][j], acc[i][j], 0, 0, 0);
        }
    }
    if (W > 1) {
        // Wave w ends with tiles w, w + W ...: the others' shares of them.
        // Slot of wave v's tile: in order, its own share left out.
        auto slot = [&](int v, int tile) { return (tile * (W - 1) + (v < tile % W ? v : v - 1)) * 64 + lane; };
#pragma unroll
        for (int q = 0; q < MT * NT; q++)
            if (q % W != wave) sums[slot(wave, q)] = acc[q / NT][q % NT];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < MT * NT; q++)
            if (q % W == wave)
#pragma unroll
                for (int v = 0; v < W - 1; v++) acc[q / NT][q % NT] += sums[(q * (W - 1) + v) * 64 + lane];
    }
#pragma unroll
    for (int q = 0; q < MT * NT; q++) {
        if (W > 1 && q % W != wave) continue;
        const int64_t n = (n0 + q % NT) * 16 + (lane & 15), t = (t0 + q / NT) * 16 + 4 * (lane >> 4);
        if (n >= p.n) continue;
        const float sw = gload(p.sw + n);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (t + e < p.t) finish(p, t + e, n, acc[q / NT][q % NT][e], gload(p.sx + t + e), sw);
    }
}

// (The 16x16x64 instruction throughout: on random codes with every CU at work the
// chip's power holds it to 3800 TOP/s, the 32x32x32 one to 2940, which made this
// kernel's 256 x 256 tiles 219 us instead of 175 for 8191 x 6144 x 4096.)

// Large products: WM x WN waves of I x J tiles of 16 tokens by 16 channels each;
// a ring of STAGES stages of 64 values of both operands in LDS, filled by DMA
// STAGES - 1 ahead.
template <int WM, int WN, int I, int J, int STAGES>
__global__ __launch_bounds__(WM *WN * 64, 2) void int8_ring_kernel(const Product p, int blocks_n, int blocks) {
    constexpr int W = WM * WN, TM = WM * I, TN = WN * J, ROWS = TM + TN, EACH = ROWS / W;  // (16-row tiles)
    static_assert(ROWS % W == 0 && I % 2 == 0, "whole tiles a wave");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES * ROWS * 1024];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    // Each XCD takes blocks that follow one another, a band of four channel
    // blocks at a time: those in flight share both operands in its L2.
    const int per = (blocks + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= blocks) return;
    constexpr int BAND = 4;
    const int blocks_m = blocks / blocks_n, band = id / (BAND * blocks_m), in = id - band * BAND * blocks_m;
    const int width = min(BAND, blocks_n - band * BAND);
    const int t0 = in / width * TM, n0 = (band * BAND + in % width) * TN;
    const uint8_t *src[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int r = wave * EACH + e;
        src[e] = r < TM ? p.x + (int64_t)min(t0 + r, p.tt - 1) * p.chunks * 1024
                        : p.w + (int64_t)min(n0 + r - TM, p.nt - 1) * p.chunks * 1024;
    }
    const uint32_t base = lds::lds_addr(ring);
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const uint32_t to = base + (c % STAGES) * (ROWS * 1024), from = (uint32_t)min(c, p.chunks - 1) * 1024 + lane * 16;
#pragma unroll
        for (int e = 0; e < EACH; e++) lds::dma16(src[e], from, to + (wave * EACH + e) * 1024);
    };
    const lds::lds_p mine = (lds::lds_p)(ring) + lane * 16;
    auto tile = [&](int c, int t) __attribute__((always_inline)) {
        return *(const __attribute__((address_space(3))) i32x4 *)(mine + ((c % STAGES) * ROWS + t) * 1024);
    };
    i32x4 acc[I][J];
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < J; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    // A step's second half of tokens loads while the first is multiplied, the
    // next step's first while the second is: that stage is whole when the step
    // begins, so nothing waits behind the barrier.
    i32x4 x0[I / 2], x1[I / 2], w[2][J];
    auto first = [&](int c, i32x4 (&ww)[J]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < J; j++) ww[j] = tile(c, TM + wn * J + j);
#pragma unroll
        for (int i = 0; i < I / 2; i++) x0[i] = tile(c, wm * I + i);
    };
    auto step = [&](int c, i32x4 (&now)[J], i32x4 (&later)[J]) __attribute__((always_inline)) {
        lds::wait_vm_barrier<(STAGES - 3) * EACH>();
        fetch(c + STAGES - 1);
#pragma unroll
        for (int i = 0; i < I / 2; i++) x1[i] = tile(c, wm * I + I / 2 + i);
#pragma unroll
        for (int i = 0; i < I / 2; i++)
#pragma unroll
            for (int j = 0; j < J; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[j], x0[i], acc[i][j], 0, 0, 0);
        first(c + 1, later);
#pragma unroll
        for (int i = 0; i < I / 2; i++)
#pragma unroll
            for (int j = 0; j < J; j++)
                acc[I / 2 + i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[j], x1[i], acc[I / 2 + i][j], 0, 0, 0);
    };
#pragma unroll
    for (int c = 0; c < STAGES - 1; c++) fetch(c);
    lds::wait_vm_barrier<(STAGES - 2) * EACH>();
    first(0, w[0]);
    int c = 0;
    for (; c + 2 <= p.chunks; c += 2) step(c, w[0], w[1]), step(c + 1, w[1], w[0]);
    if (c < p.chunks) step(c, w[0], w[1]);
    lds::wait_vm<0>();
    // Lane (token, g): channels 4 g .. 4 g + 3.
    float sx[I];
#pragma unroll
    for (int i = 0; i < I; i++) sx[i] = gload(p.sx + (int64_t)min(t0 + wm * I + i, p.tt - 1) * 16 + (lane & 15));
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int64_t n = (int64_t)(n0 + wn * J + j) * 16 + 4 * (lane >> 4);
        if (n >= p.n) continue;
        const f32x4_dw sw = *(const __attribute__((address_space(1))) f32x4_dw *)(p.sw + n);
#pragma unroll
        for (int i = 0; i < I; i++) {
            const int64_t t = (int64_t)(t0 + wm * I + i) * 16 + (lane & 15);
            if (t < p.t) finish4(p, t, n, acc[i][j], sx[i], sw);
        }
    }
}

template <int MT, int NT, int W>
void direct(const Product &p, hipStream_t s) {
    hipLaunchKernelGGL((int8_direct_kernel<MT, NT, W>), dim3((p.nt + NT - 1) / NT, (p.tt + MT - 1) / MT), dim3(W * 64), 0, s, p);
}
template <int WM, int WN, int I, int J, int STAGES>
void ring(const Product &p, hipStream_t s) {
    const int m = (p.tt + WM * I - 1) / (WM * I), n = (p.nt + WN * J - 1) / (WN * J);
    hipLaunchKernelGGL((int8_ring_kernel<WM, WN, I, J, STAGES>), dim3((unsigned)((m * n + 7) / 8 * 8)), dim3(WM * WN * 64), 0, s, p, n, m * n);
}

// A few rows (up to 16384 values in all): each block quantises them for itself,
// under its first loads of weights, into LDS as [row][values]; lanes of rows past
// the last hold zeros.  One row of 4096 x 4096 5.0 us (3.4 TB/s), against 6.6 with
// the rows in a launch of their own; of 28672 x 4096 20 (5.8 TB/s); four rows 7.3
// and 6.8, but a launch less to queue.
constexpr int kFewBytes = 16384, kFewRows = 4;
template <int W>
__global__ __launch_bounds__(W * 64) void int8_few_kernel(const Product p, const float *x, int64_t xs, int k) {
    __shared__ uint32_t codes[kFewBytes / 4], red[W];
    __shared__ i32x4 sums[(W - 1) * 64];
    __shared__ float scale[kFewRows];
    constexpr int U = 8, T = W * 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int width = p.chunks * 64, row = lane & 15, g = lane >> 4;
    const u32x4 *w = (const u32x4 *)(p.w + (int64_t)blockIdx.x * p.chunks * 1024) + lane;
    i32x4 b[U];
    auto load = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) b[u] = __builtin_bit_cast(i32x4, gload(w + 64 * min(c0 + u * W, p.chunks - 1)));
    };
    load(wave);
    for (int t = 0; t < p.t; t++) {
        const float *src = x + t * xs;
        float held[4][4];
        uint32_t top = 0;
        auto values = [&](int i, float (&v)[4]) __attribute__((always_inline)) {
            if (i + 4 <= k) {
                const u32x4_dw y = gload_x4((const uint32_t *)src + i);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __uint_as_float(y[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = i + e < k ? gload(src + i + e) : 0.0f;
            }
        };
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = 4 * (threadIdx.x + T * j);
            if (i < width) values(i, held[j]);
#pragma unroll
            for (int e = 0; e < 4; e++) top = i < width ? max(top, magnitude(held[j][e])) : top;
        }
        for (int i = 4 * (threadIdx.x + T * 4); i < width; i += 4 * T) {
            float v[4];
            values(i, v);
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, magnitude(v[e]));
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        __syncthreads();
        if (lane == 0) red[wave] = top;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < W; v++) top = max(top, red[v]);
        const Int8Scale s(top);
        if (threadIdx.x == 0) scale[t] = s.scale;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = 4 * (threadIdx.x + T * j);
            if (i < width) codes[(t * width + i) / 4] = pack4(s.code(held[j][0]), s.code(held[j][1]), s.code(held[j][2]), s.code(held[j][3]));
        }
        for (int i = 4 * (threadIdx.x + T * 4); i < width; i += 4 * T) {
            float v[4];
            values(i, v);
            codes[(t * width + i) / 4] = pack4(s.code(v[0]), s.code(v[1]), s.code(v[2]), s.code(v[3]));
        }
    }
    __syncthreads();
    i32x4 acc = {0, 0, 0, 0};
    for (int c0 = wave; c0 < p.chunks; c0 += W * U) {
        if (c0 != wave) load(c0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + u * W;
            if (c >= p.chunks) continue;
            const i32x4 y = *(const i32x4 *)&codes[(min(row, p.t - 1) * width + c * 64 + g * 16) / 4];
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u], row < p.t ? y : i32x4{0, 0, 0, 0}, acc, 0, 0, 0);
        }
    }
    if (wave) sums[(wave - 1) * 64 + lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int v = 0; v < W - 1; v++) acc += sums[v * 64 + lane];
    const int64_t n = (int64_t)blockIdx.x * 16 + 4 * g;
    if (row < p.t && n < p.n) finish4(p, row, n, acc, scale[row], *(const __attribute__((address_space(1))) f32x4_dw *)(p.sw + n));
}

// Blocks by what fills the chip (time of the product alone, us, K = 4096 or 2048
// where n = 1024):
//   direct, 16 x 16 (tokens x channels) for 16 rows; 32 x 32 up to 256 blocks,
//   then 32 x 64 up to 512 (48 x 6144: 7.5 and 6.5; 256 x 1024: 4.2 and 4.7;
//   160 x 6144: 16.4 and 10.6, ring of 64 x 128 15.9); 32 x 16 where half the CUs
//   would have no block and rows are long (with the rows' codes, 32 x 1024 of 4096
//   values 8.7 and 7.7, 24 x 4096 of 8192 13.7 and 12.3, but 48 x 2048 of 2048 7.0
//   and 7.3);
//   ring, 64 x 128 below 256 blocks of 128 x 128 (512 x 6144: 22.6 and 24.3, 32 x
//   64 27.8; 768 x 6144: 34.1 and 31.7);
//   ring, 256 x 256 where its rounds of 256 blocks are at least 5/6 full (2048 x
//   4096, half a round: 49.5 and 36.7 with 128 x 128; 4096 x 4096: 61 and 74; 8191
//   x 6144, three rounds: 175 and 208).
void launch_product(const Product &p, hipStream_t s) {
    auto blocks = [&](int64_t m, int64_t n) { return (p.tt + m - 1) / m * ((p.nt + n - 1) / n); };
    const int64_t large = blocks(16, 16), rounds = (large + 255) / 256;
    if (p.tt == 1) direct<1, 1, 8>(p, s);
    else if (blocks(2, 2) <= 128 && p.chunks >= 64) direct<2, 1, 8>(p, s);
    else if (blocks(2, 2) <= 256) direct<2, 2, 8>(p, s);
    else if (blocks(2, 4) <= 512) direct<2, 4, 8>(p, s);
    else if (large * 6 >= rounds * 256 * 5) ring<4, 2, 4, 8, 4>(p, s);
    else if (blocks(8, 8) >= 256) ring<2, 2, 4, 4, 5>(p, s);
    else ring<2, 2, 2, 4, 6>(p, s);
}

int sizes_ok(const char *what, int32_t n, int32_t k) {
    if (n <= 0 || k <= 0) return fail(MOE_EINVAL, "%s: %d channels of %d values", what, n, k);
    if (k > kMostK) return fail(MOE_EUNSUP, "%s: %d values a channel, up to %d (sums of 32 bits)", what, k, kMostK);
    if (n >= (1 << 24)) return fail(MOE_EUNSUP, "%s: %d channels, up to %d", what, n, (1 << 24) - 1);  // (256 threads each)
    return MOE_OK;
}
uint64_t codes_bytes(int64_t rows, int64_t k) { return (uint64_t)(up(rows, 16) * up(k, 64)); }
uint64_t packed_size(int64_t rows, int64_t k) { return codes_bytes(rows, k) + (uint64_t)up(rows, 16) * 4; }

// Whether rows of `width` floats may lie in memory of other rows.
bool meet(const float *a, int64_t a_stride, int64_t a_width, const float *b, int64_t b_stride, int64_t b_width, int rows) {
    auto low = [&](const float *p, int64_t s) { return (intptr_t)p + std::min<int64_t>(0, s * (rows - 1)) * 4; };
    auto high = [&](const float *p, int64_t s, int64_t w) { return (intptr_t)p + (std::max<int64_t>(0, s * (rows - 1)) + w) * 4; };
    return low(a, a_stride) < high(b, b_stride, b_width) && low(b, b_stride) < high(a, a_stride, a_width);
}

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
    // Blocks that read x for themselves need no workspace, but x as it was.
    const bool few = t <= kFewRows && t * up(k, 64) <= kFewBytes && !meet(x, x_stride, k, y, y_stride, n, t) &&
                     !(residual && meet(x, x_stride, k, residual, residual_stride, n, t));
    if (few) workspace = nullptr;
    else if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < packed_size(t, k))
        return fail(MOE_EINVAL, "moe_int8_linear: workspace of %llu bytes (256-byte aligned), %llu needed",
                    (unsigned long long)workspace_bytes, (unsigned long long)packed_size(t, k));
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *w = static_cast<const uint8_t *>(packed);
    uint8_t *xc = static_cast<uint8_t *>(workspace);
    float *sx = few ? nullptr : reinterpret_cast<float *>(xc + codes_bytes(t, k));
    // (blocks of 128 x 64 at least, 512 threads at most)
    if (up(t, 128) / 128 * (up(n, 64) / 64) * 512 > 0xffffffffll)
        return fail(MOE_EUNSUP, "moe_int8_linear: %d tokens of %d channels are too many blocks", t, n);
    const Product p{w, xc, reinterpret_cast<const float *>(w + codes_bytes(n, k)), sx, y, residual, y_stride, residual_stride, n, t,
                    (int)(up(k, 64) / 64), (n + 15) / 16, (t + 15) / 16};
    if (few) {
        hipLaunchKernelGGL((int8_few_kernel<8>), dim3(p.nt), dim3(512), 0, s, p, x, x_stride, k);
        return done("8-bit product kernel");
    }
    hipLaunchKernelGGL(int8_rows_kernel, dim3(row_blocks(t)), dim3(256), 0, s, x, x_stride, t, k, xc, sx);
    launch_product(p, s);
    return done("8-bit product kernel");
}

}  // extern "C"
