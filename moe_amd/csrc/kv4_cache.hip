// kv4_cache.hip — writing and reading rows of the paged 4-bit cache
// (moe_kv4_store, moe_kv4_load): layout in kv4.h, quantiser as
// moe_quantize_rows(Q4_0) (src/quant.rs:304-365).
//
// Both are streams of f32 rows, eight lanes a 32-value block: 16376 rows of 8 kv
// heads of 128 are written in 40.5 us (152 MB, 3.8 TB/s; the byte-wide stores of
// a value's lanes are what keeps it off the copy's 4.9) and read in 31.4 (4.8),
// their 255 full pages' mean keys taken in 10.8; 999 rows of 16 heads of 192/128
// 11.5, 8.4 and 9 (the mean keys' pages are few, so latency); 32 rows 3.0, 2.3
// and 5.1.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

int kv4_of(const char *what, const moe_kv4 *c, Kv4 *out) {
    if (!c || !c->pool || !c->table) return fail(MOE_EINVAL, "%s: a cache without a pool or a table", what);
    if (c->n_seq <= 0 || c->max_pages <= 0 || c->n_pages <= 0 || c->n_kv <= 0)
        return fail(MOE_EINVAL, "%s: %d sequences of %d pages, pool of %d, %d kv heads", what, c->n_seq, c->max_pages,
                    c->n_pages, c->n_kv);
    if (c->page < 32 || c->page > 4096 || (c->page & (c->page - 1)) || (int64_t)c->max_pages * c->page > INT32_MAX)
        return fail(MOE_EINVAL, "%s: pages of %d positions, %d a sequence (32, 64 ... 4096; fewer than 2^31 positions)",
                    what, c->page, c->max_pages);
    if (c->qd <= 0 || c->vd <= 0 || c->qd % 32 || c->vd % 32 || c->qd > 256 || c->vd > 256)
        return fail(MOE_EUNSUP, "%s: key width %d, value width %d (multiples of 32 up to 256)", what, c->qd, c->vd);
    if (c->n_kv > 65535) return fail(MOE_EUNSUP, "%s: %d kv heads (up to 65535)", what, c->n_kv);  // a grid's second size
    Kv4 k{};
    k.pool = static_cast<uint8_t *>(c->pool), k.table = c->table, k.means = static_cast<__half *>(c->means);
    k.n_seq = c->n_seq, k.max_pages = c->max_pages, k.n_pages = c->n_pages, k.n_kv = c->n_kv, k.qd = c->qd, k.vd = c->vd;
    k.page_shift = __builtin_ctz((unsigned)c->page);
    k.tile_bytes = 18 * (c->qd + c->vd);
    uint64_t need = 0;
    if (__builtin_mul_overflow((uint64_t)k.n_pages * (uint64_t)k.tiles(), (uint64_t)k.n_kv * k.tile_bytes, &need))
        return fail(MOE_EINVAL, "%s: the pool's size overflows", what);
    if ((uintptr_t)c->pool % 16 || (uintptr_t)c->means % 16 || c->pool_bytes < need)
        return fail(MOE_EINVAL, "%s: a pool of %llu bytes (16-byte aligned), %llu needed", what,
                    (unsigned long long)c->pool_bytes, (unsigned long long)need);
    *out = k;
    return MOE_OK;
}

namespace {

// f32 -> f16 as the quantiser rounds it (src/quant.rs:149-174): nearest even
// for normals, half up for subnormals, too large and NaN to infinity; v >= 0.
__device__ inline uint32_t half_bits(float f) {
    const uint32_t x = __float_as_uint(f);
    int e = (int)(x >> 23) - 112;
    const uint32_t m = x & 0x7fffffu;
    if (e >= 31) return 0x7c00u;
    if (e <= 0) return e < -10 ? 0u : (((m | 0x800000u) >> (1 - e)) + 0x1000u) >> 13;
    const uint32_t r = m + 0x0fffu + ((m >> 13) & 1u);
    if (r & 0x800000u) e++;
    return e >= 31 ? 0x7c00u : (uint32_t)e << 10 | (r & 0x7fffffu) >> 13;
}

// round() half away from zero, + 8, within 0..15; NaN 8.
__device__ inline uint32_t code_of(float v, float inv) {
    const float q = roundf(v * inv) + 8.0f;
    return q != q ? 8u : (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f);
}

__device__ inline bool slot_ok(const Kv4 &c, int64_t slot) {
    return slot >= 0 && slot < ((int64_t)c.n_pages << c.page_shift);
}
// The tile of a slot's kv head and its position in it.
__device__ inline uint8_t *tile_of(const Kv4 &c, int64_t slot, int kv, int &p) {
    const int off = (int)(slot & ((1 << c.page_shift) - 1));
    p = off & (kTile - 1);
    return c.head((int)(slot >> c.page_shift), kv) + (size_t)(off >> 5) * c.tile_bytes;
}

typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // at any float
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// First of the R rows of a block.  The rows of a tile, 32 in turn in a prompt,
// go to one XCD, so that the bytes of a line that different rows write meet in
// one L2 instead of being written back by several.
template <int R>
__device__ inline int first_row(unsigned block) {
    constexpr unsigned per = 32 / R;
    return (int)(((block >> 3) / per * 8 + (block & 7)) * per + (block >> 3) % per) * R;
}
template <int R>
unsigned row_blocks(int rows) {
    return ((unsigned)rows + 255) / 256 * (256 / R);
}

// Quantise and write one 32-value block, eight lanes, four values each, of N
// rows whose slots follow one another from `slot` on: of one row, or of four
// that begin at a slot divisible by four, whose values' bytes then make whole
// words and whose scales lie together.
template <int N>
__device__ inline void store_block(const Kv4 &c, const float *src, int64_t stride, int64_t slot, bool key, int kv, int s) {
    const int i = threadIdx.x & 7, nb = (key ? c.qd : c.vd) / 32;
    f32x4_dw x[N];
#pragma unroll
    for (int r = 0; r < N; r++) x[r] = *(const __attribute__((address_space(1))) f32x4_dw *)(src + r * stride + 4 * i);
    uint32_t w[N], h[N];
#pragma unroll
    for (int r = 0; r < N; r++) {
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[r][e]));  // fmaxf drops NaNs
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float d = top / 7.0f;
        h[r] = half_bits(d);
        const float inv = d > 0.0f ? 1.0f / __half2float(__ushort_as_half((unsigned short)h[r])) : 0.0f;
        w[r] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w[r] |= code_of(x[r][e], inv) << (8 * e);
        w[r] |= (uint32_t)__shfl_down((int)w[r], 4, 64) << 4;  // dims j + 16 into the high nibbles (lanes 0..3)
    }
    int p;
    uint8_t *tile = tile_of(c, slot, kv, p);
    if (i == 4) {
        uint16_t *dst = (uint16_t *)(tile + (key ? c.k_scales() : c.v_scales())) + kv4_scale_at(p, s);
        if (N == 4) gstore((u32x2 *)dst, u32x2{h[0] | h[N > 1 ? 1 : 0] << 16, h[N > 2 ? 2 : 0] | h[N > 3 ? 3 : 0] << 16});
        else gstore(dst, (uint16_t)h[0]);
    }
    if (i >= 4) return;
    if (key) {
#pragma unroll
        for (int r = 0; r < N; r++) gstore((uint32_t *)(tile + kv4_key_byte(nb, p + r, s, 4 * i)), w[r]);
        return;
    }
    uint8_t *dst = tile + c.v_codes() + kv4_value_byte(nb, p, s, 4 * i);
    const int step = kv4_value_byte(nb, 0, s, 1) - kv4_value_byte(nb, 0, s, 0);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (N == 4) {
            uint32_t y = 0;
#pragma unroll
            for (int r = 0; r < N; r++) y |= (w[r] >> (8 * e) & 255) << (8 * r);
            gstore((uint32_t *)(dst + e * step), y);
        } else {
            gstore(dst + e * step, (uint8_t)(w[0] >> (8 * e)));
        }
    }
}

// A block of threads takes 32 blocks of 32 values of R rows.  R = 4: four rows
// in turn whose slots are too, from one divisible by four on, are written by
// the block that has the first of them; other rows one by one.
template <int R>
__global__ __launch_bounds__(256) void kv4_store_kernel(const Kv4 c, const float *__restrict__ k, int64_t ks,
                                                        const float *__restrict__ v, int64_t vs, int rows,
                                                        const int64_t *__restrict__ slots) {
    const int r0 = first_row<R>(blockIdx.x);
    const int nk = c.qd / 32, nv = c.vd / 32;
    const int at = blockIdx.y * 32 + (threadIdx.x >> 3);
    if (r0 >= rows || at >= c.n_kv * (nk + nv)) return;
    const bool key = at < c.n_kv * nk;
    const int blk = key ? at : at - c.n_kv * nk, nb = key ? nk : nv, kv = blk / nb, s = blk % nb;
    const float *src = (key ? k : v) + (size_t)blk * 32;
    const int64_t stride = key ? ks : vs;
    if (R == 1) {
        const int64_t slot = gload(slots + r0);
        if (slot_ok(c, slot)) store_block<1>(c, src + (int64_t)r0 * stride, stride, slot, key, kv, s);
        return;
    }
    // Slots of rows r0 - 3 .. r0 + 6, and which of them begin such a four.
    int64_t sl[10];
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const int r = r0 - 3 + i;
        sl[i] = r >= 0 && r < rows ? gload(slots + r) : -1;
    }
    bool four[7];
#pragma unroll
    for (int i = 0; i < 7; i++)
        four[i] = slot_ok(c, sl[i]) && (sl[i] & 3) == 0 && sl[i + 1] == sl[i] + 1 && sl[i + 2] == sl[i] + 2 &&
                  sl[i + 3] == sl[i] + 3;
#pragma unroll
    for (int i = 3; i < 7; i++) {
        const int64_t row = r0 - 3 + i;
        if (four[i]) store_block<4>(c, src + row * stride, stride, sl[i], key, kv, s);
        else if (!(four[i - 1] || four[i - 2] || four[i - 3]) && slot_ok(c, sl[i]))
            store_block<1>(c, src + row * stride, stride, sl[i], key, kv, s);
    }
}

// The mean keys of pages whose last position is among the rows: a block looks
// at 64 rows for one kv head, its waves take the dims' blocks of 32.  A word of
// the keys' region is eight dims of a position, so a lane sums eight dims over
// its positions and 16 lanes are added up.  In 64 bits the sums are exact for
// scales within 2^30 of each other, whatever their order.
__global__ __launch_bounds__(256) void kv4_means_kernel(const Kv4 c, const int64_t *__restrict__ slots, int rows) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kv = blockIdx.y;
    const int64_t last = (1 << c.page_shift) - 1, row = (int64_t)blockIdx.x * 64 + lane;
    const int64_t mine = row < rows ? gload(slots + row) : -1;
    const int nq = c.qd / 32, g = lane >> 4, col = lane & 15;
    for (unsigned long long full = __ballot(slot_ok(c, mine) && (mine & last) == last); full; full &= full - 1) {
        const int page = (int)(__shfl(mine, __builtin_ctzll(full), 64) >> c.page_shift);
        const uint8_t *head = c.head(page, kv);
        for (int s = wave; s < nq; s += 4) {
            double sum[8] = {};
#pragma unroll 4
            for (int t = 0; t < 2 * c.tiles(); t++) {
                const uint8_t *tile = head + (size_t)(t >> 1) * c.tile_bytes;
                const int half = t & 1;
                const uint32_t w = gload((const uint32_t *)(tile + kv4_word(nq, 2 * s + half, lane)));
                const uint16_t hb = gload((const uint16_t *)(tile + c.k_scales()) + kv4_scale_at(16 * half + col, s));
                const float d = __half2float(__ushort_as_half(hb));
#pragma unroll
                for (int e = 0; e < 8; e++)  // bytes' low nibbles: dims 4 g + e; high: 16 + 4 g + e - 4
                    sum[e] += (double)(d * (float)((int)(w >> (8 * (e & 3) + (e & 4)) & 15) - 8));
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] += __shfl_xor(sum[e], o, 64);
            if (col == 0)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float m = (float)(sum[e] / (double)(last + 1));
                    m = m > 65504.0f ? 65504.0f : m < -65504.0f ? -65504.0f : m;
                    c.means[((size_t)page * c.n_kv + kv) * c.qd + 32 * s + (e & 4) * 4 + 4 * g + (e & 3)] = __float2half_rn(m);
                }
        }
    }
}

// As the write: eight lanes per block of 32, four values each.
__global__ __launch_bounds__(256) void kv4_load_kernel(const Kv4 c, const int64_t *__restrict__ slots, int rows,
                                                       float *__restrict__ k, int64_t ks, float *__restrict__ v,
                                                       int64_t vs) {
    const int row = first_row<1>(blockIdx.x);
    if (row >= rows) return;
    const int64_t slot = gload(slots + row);
    const int nk = k ? c.qd / 32 : 0, nv = v ? c.vd / 32 : 0, i = threadIdx.x & 7;
    const int at = blockIdx.y * 32 + (threadIdx.x >> 3);
    if (!slot_ok(c, slot) || at >= c.n_kv * (nk + nv)) return;
    const bool key = at < c.n_kv * nk;
    const int blk = key ? at : at - c.n_kv * nk, nb = key ? nk : nv, kv = blk / nb, s = blk % nb;
    int p;
    const uint8_t *tile = tile_of(c, slot, kv, p);
    const uint16_t hb = gload((const uint16_t *)(tile + (key ? c.k_scales() : c.v_scales())) + kv4_scale_at(p, s));
    uint32_t w = 0;
    if (key) {
        w = gload((const uint32_t *)(tile + kv4_key_byte(nk, p, s, 4 * (i & 3))));
    } else {
        const uint8_t *src = tile + c.v_codes() + kv4_value_byte(nv, p, s, 4 * (i & 3));
        const int step = kv4_value_byte(nv, 0, s, 1) - kv4_value_byte(nv, 0, s, 0);
#pragma unroll
        for (int e = 0; e < 4; e++) w |= (uint32_t)gload(src + e * step) << (8 * e);
    }
    const float d = __half2float(__ushort_as_half(hb));
    f32x4_dw x;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = d * (float)((int)(w >> (8 * e + (i & 4)) & 15) - 8);
    float *dst = (key ? k + (size_t)row * ks : v + (size_t)row * vs) + (size_t)blk * 32 + 4 * i;
    *(__attribute__((address_space(1))) f32x4_dw *)dst = x;
}

constexpr int kMostRows = (1 << 24) - 256;  // a block of 256 threads a row

int rc_of(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_pool_size(const moe_kv4 *c, uint64_t *bytes) {
    Kv4 k;
    if (!c || !bytes) return fail(MOE_EINVAL, "moe_kv4_pool_size: bad argument");
    moe_kv4 any = *c;  // the sizes alone count
    any.pool = reinterpret_cast<void *>(16), any.pool_bytes = UINT64_MAX, any.means = nullptr;
    any.table = reinterpret_cast<const int32_t *>(16);
    any.n_seq = any.max_pages = 1;
    const int rc = kv4_of("moe_kv4_pool_size", &any, &k);
    if (rc) return rc;
    *bytes = (uint64_t)k.n_pages * (uint64_t)k.tiles() * (uint64_t)k.n_kv * (uint64_t)k.tile_bytes;
    return MOE_OK;
}

int moe_kv4_store(const moe_kv4 *c, const float *k, int64_t k_stride, const float *v, int64_t v_stride, int32_t rows,
                  const int64_t *slots, void *stream) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_store", c, &a)) return rc;
    if (rows < 0 || (rows > 0 && (!k || !v || !slots)))
        return fail(MOE_EINVAL, "moe_kv4_store: bad argument (%d rows)", rows);
    if (rows > kMostRows) return fail(MOE_EUNSUP, "moe_kv4_store: %d rows, up to %d at once", rows, kMostRows);
    if (rows == 0) return MOE_OK;
    hipStream_t s = (hipStream_t)stream;
    const int blocks = a.n_kv * (a.qd + a.vd) / 32;
    // Word stores of four rows pay where there are prompts, one row a block where
    // a few rows are latency (32 rows of 8 heads of 128: 5.7 -> 3.0 us).  One row
    // and four, back to back: 4096 rows of 8 heads of 128 14.4 and 11.2 us, of 16
    // of 192/128 29.3 and 22.9, of 2 of 64 5.7 and 6.3; 16376 rows 49.5 and 33.4,
    // 120 and 90.5, 10.2 and 8.8.  At 2048 rows it is 8.7 and 7.8, 16.2 and 13.4,
    // 5.7 and 6.1, at 1024 5.9 and 6.4, 9.2 and 8.4, 5.7 and 6.4.
    const unsigned y = (unsigned)(blocks + 31) / 32;
    if (rows >= 4096)
        hipLaunchKernelGGL((kv4_store_kernel<4>), dim3(row_blocks<4>(rows), y), dim3(256), 0, s, a, k, k_stride, v, v_stride,
                           rows, slots);
    else
        hipLaunchKernelGGL((kv4_store_kernel<1>), dim3(row_blocks<1>(rows), y), dim3(256), 0, s, a, k, k_stride, v, v_stride,
                           rows, slots);
    if (a.means) hipLaunchKernelGGL(kv4_means_kernel, dim3((rows + 63) / 64, a.n_kv), dim3(256), 0, s, a, slots, rows);
    return rc_of("cache write kernel");
}

int moe_kv4_load(const moe_kv4 *c, const int64_t *slots, int32_t rows, float *k, int64_t k_stride, float *v,
                 int64_t v_stride, void *stream) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_load", c, &a)) return rc;
    if (rows < 0 || (rows > 0 && !slots)) return fail(MOE_EINVAL, "moe_kv4_load: bad argument (%d rows)", rows);
    if (rows > kMostRows) return fail(MOE_EUNSUP, "moe_kv4_load: %d rows, up to %d at once", rows, kMostRows);
    if (rows == 0 || (!k && !v)) return MOE_OK;
    const int blocks = a.n_kv * ((k ? a.qd : 0) + (v ? a.vd : 0)) / 32;
    hipLaunchKernelGGL(kv4_load_kernel, dim3(row_blocks<1>(rows), (blocks + 31) / 32), dim3(256), 0, (hipStream_t)stream, a,
                       slots, rows, k, k_stride, v, v_stride);
    return rc_of("cache read kernel");
}

}  // extern "C"
