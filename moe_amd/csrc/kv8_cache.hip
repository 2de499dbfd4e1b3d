// kv8_cache.hip — writing and reading rows of the paged 8-bit cache
// (moe_kv8_store, moe_kv8_load): layout in kv8.h, quantiser in int8.h.
//
// A block's scale is its largest value's, so a row that joins a block may change
// all of its codes.  A wave takes what a step writes of one block's keys or
// values, of one kv head: the rows of this step, and before them those of
// earlier steps, whose values `open` keeps while their block is filling.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "int8.h"
#include "kv8.h"

namespace moe {
int fail(int code, const char *fmt, ...);

int kv8_of(const char *what, const moe_kv8 *c, Kv8 *out) {
    if (!c || !c->codes || !c->scales || !c->open || !c->table)
        return fail(MOE_EINVAL, "%s: a cache without codes, scales, open blocks or a table", what);
    if (c->n_seq <= 0 || c->max_pages <= 0 || c->n_pages <= 0 || c->n_kv <= 0)
        return fail(MOE_EINVAL, "%s: %d sequences of %d pages, pool of %d, %d kv heads", what, c->n_seq, c->max_pages,
                    c->n_pages, c->n_kv);
    if (c->page < 64 || c->page > 4096 || (c->page & (c->page - 1)) || (int64_t)c->max_pages * c->page > INT32_MAX)
        return fail(MOE_EINVAL, "%s: pages of %d positions, %d a sequence (64, 128 ... 4096; fewer than 2^31 positions)",
                    what, c->page, c->max_pages);
    if (c->qd <= 0 || c->vd <= 0 || c->qd % 32 || c->vd % 32 || c->qd > 256 || c->vd > 256)
        return fail(MOE_EUNSUP, "%s: key width %d, value width %d (multiples of 32 up to 256)", what, c->qd, c->vd);
    if (c->n_kv > 65535) return fail(MOE_EUNSUP, "%s: %d kv heads (up to 65535)", what, c->n_kv);  // a grid's second size
    Kv8 k{};
    k.codes = static_cast<uint8_t *>(c->codes), k.scales = c->scales, k.open = static_cast<uint8_t *>(c->open), k.table = c->table;
    k.n_seq = c->n_seq, k.max_pages = c->max_pages, k.n_pages = c->n_pages, k.n_kv = c->n_kv, k.qd = c->qd, k.vd = c->vd;
    k.page_shift = __builtin_ctz((unsigned)c->page);
    const uint64_t tiles = (uint64_t)k.n_pages * (uint64_t)(c->page / kTile8) * (uint64_t)k.n_kv;  // (below 2^31 * 2^6 * 2^16)
    uint64_t codes = 0;
    if (__builtin_mul_overflow(tiles, (uint64_t)k.tile_bytes(), &codes) || codes > INT64_MAX)
        return fail(MOE_EINVAL, "%s: the pool's size overflows", what);
    const uint64_t open = (uint64_t)k.n_seq * (uint64_t)k.n_kv * (uint64_t)k.open_bytes();
    if ((uintptr_t)c->codes % 16 || (uintptr_t)c->scales % 16 || (uintptr_t)c->open % 16 || c->codes_bytes < codes ||
        c->scales_bytes < tiles * 32 || c->open_bytes < open)
        return fail(MOE_EINVAL, "%s: %llu, %llu and %llu bytes (16-byte aligned), %llu, %llu and %llu needed", what,
                    (unsigned long long)c->codes_bytes, (unsigned long long)c->scales_bytes, (unsigned long long)c->open_bytes,
                    (unsigned long long)codes, (unsigned long long)tiles * 32, (unsigned long long)open);
    *out = k;
    return MOE_OK;
}

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // at any float

struct Store {
    Kv8 c;
    const float *k, *v;
    int64_t ks, vs;
    const int32_t *row_start, *seq, *pos;
    const int64_t *slots;
    int rows;
};

__device__ inline bool slot_ok(const Kv8 &c, int64_t slot) {
    return slot >= 0 && slot < ((int64_t)c.n_pages << c.page_shift);
}

// What `open` says of a sequence's kv head: for keys (values: [2], [3]) in each
// of two halves the block whose values it holds, plus 1, and how many of them.
struct Half {
    int block1, count;
};

// Where a block's values come from: `before` of them from earlier steps (out of
// `held` where that is not null, else as the codes read), then n of this step's
// rows from `row` on.
struct Block {
    const float *held, *row;
    int64_t stride;
    int before, n, d, T;
    const uint8_t *tile;  // its keys or values
    float scale;          // the codes' so far
    bool key;
    __device__ int code_byte(int p, int i) const { return key ? kv8_key_byte(d, 16 * T + p, i) : kv8_value_byte(16 * T + p, i); }
};

template <int N>
__device__ inline void take(const Block &b, int p, int i, float (&x)[N]) {
    if (p >= b.before) {
        const bool there = p < b.before + b.n;
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = there ? gload(b.row + (int64_t)(p - b.before) * b.stride + i + e) : 0.0f;
    } else if (b.held) {
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = gload(b.held + p * b.d + i + e);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = b.scale * (float)(int8_t)gload(b.tile + b.code_byte(p, i + e));
    }
}

__device__ inline uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// One row a block, the first wave its keys, the second its values; the row that
// is its block's last in this step writes the block.
__global__ __launch_bounds__(128) void kv8_store_kernel(const Store a) {
    const Kv8 &c = a.c;
    const int r = blockIdx.x, kv = blockIdx.y, lane = threadIdx.x & 63;
    const bool key = threadIdx.x < 64;
    const int64_t slot = gload(a.slots + r);
    const int s = gload(a.seq + r), p = gload(a.pos + r);
    if (!slot_ok(c, slot) || (unsigned)s >= (unsigned)c.n_seq || p < 0) return;
    const int r0 = max(0, min(r, gload(a.row_start + s))), r1 = max(r + 1, min(a.rows, gload(a.row_start + s + 1)));
    const int T = p >> 4 & 3, in = p & 15;
    if (in != 15 && r + 1 < r1) return;
    Block b;
    b.key = key, b.T = T, b.d = key ? c.qd : c.vd;
    const int p0 = p - (r - r0);  // the sequence's first row's
    b.n = min(in + 1, r - r0 + 1), b.before = in + 1 - b.n;
    b.stride = key ? a.ks : a.vs;
    b.row = (key ? a.k : a.v) + (int64_t)(r - b.n + 1) * b.stride + (int64_t)kv * b.d;
    const int64_t tile = c.tile((int)(slot >> c.page_shift), kv, (int)(slot & ((1 << c.page_shift) - 1)));
    uint8_t *codes = c.at(tile) + (key ? 0 : c.values());
    float *scale = c.scale_at(tile, key, T);
    b.tile = codes, b.scale = b.before ? gload(scale) : 0.0f;

    // The half that holds the values of the block that was filling.
    uint8_t *open = c.open_at(s, kv);
    Half *tags = (Half *)(open + 2 * kBlock8 * 4 * (c.qd + c.vd)) + (key ? 0 : 2);
    float *halves = (float *)open + (key ? 0 : 2 * kBlock8 * c.qd);
    const int was = p0 >> 4, had = p0 & 15;
    int half = -1;
    if (had)
        for (int i = 0; i < 2; i++)
            if (tags[i].block1 == was + 1 && tags[i].count >= had) half = i;
    b.held = half < 0 ? nullptr : halves + half * kBlock8 * b.d;

    uint32_t top = 0;
    const int nu = b.d / 16;
    if (key) {
        for (int u = lane >> 4; u < nu; u += 4) {
            float x[16];
            take(b, lane & 15, 16 * u, x);
            for (int e = 0; e < 16; e++) top = max(top, magnitude(x[e]));
        }
    } else {
        for (int u = 0; u < nu; u++)
            for (int i = 0; i < 4; i++) {
                float x[1];
                take(b, 4 * (lane >> 4) + i, 16 * u + (lane & 15), x);
                top = max(top, magnitude(x[0]));
            }
    }
    const Int8Scale q(wave_max(top));
    // The step's last block of the sequence: what it holds so far is kept where
    // the block before is not (another wave may be reading that one, and a step
    // that is made again finds it).
    if (r + 1 == r1) {
        const bool same = (p >> 4) == was, full = in == 15;
        const int to = half < 0 ? 0 : same ? half : 1 - half;
        const int from = half >= 0 && same ? b.before : 0;  // (those before lie there)
        float *dst = halves + to * kBlock8 * b.d;
        for (int i = from * b.d + lane; !full && i < (in + 1) * b.d; i += 64) {
            float x[1];
            take(b, i / b.d, i % b.d, x);
            dst[i] = x[0];
        }
        if (lane == 0) {
            if (!full) tags[to] = Half{(p >> 4) + 1, in + 1};
            // Nothing that an earlier block or sequence left stays, but the half
            // that this step has read.
            for (int i = 0; i < 2; i++)
                if (i != half && (full || i != to)) tags[i] = Half{0, 0};
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // codes are read above, by lanes other than their writers
    }
    // (a lane reads the bytes that it writes, and no other's)
    if (key) {
        for (int u = lane >> 4; u < nu; u += 4) {
            float x[16];
            take(b, lane & 15, 16 * u, x);
            uint32_t y[4];
            for (int j = 0; j < 4; j++)
                y[j] = pack4(q.code(x[4 * j]), q.code(x[4 * j + 1]), q.code(x[4 * j + 2]), q.code(x[4 * j + 3]));
            gstore((u32x4 *)(codes + kv8_key_byte(c.qd, 16 * T + (lane & 15), 16 * u)), u32x4{y[0], y[1], y[2], y[3]});
        }
    } else {
        for (int u = 0; u < nu; u++) {
            int y[4];
            for (int i = 0; i < 4; i++) {
                float x[1];
                take(b, 4 * (lane >> 4) + i, 16 * u + (lane & 15), x);
                y[i] = q.code(x[0]);
            }
            gstore((uint32_t *)(codes + kv8_value_byte(16 * T + 4 * (lane >> 4), 16 * u + (lane & 15))), pack4(y[0], y[1], y[2], y[3]));
        }
    }
    if (lane == 0) gstore(scale, q.scale);
}

// A block of 256 threads takes a row and 256 values of it.
__global__ __launch_bounds__(256) void kv8_load_kernel(const Kv8 c, const int64_t *__restrict__ slots, float *__restrict__ k,
                                                       int64_t ks, float *__restrict__ v, int64_t vs) {
    const int64_t row = blockIdx.x, slot = gload(slots + row);
    const int nk = k ? c.n_kv * c.qd : 0, at = blockIdx.y * 256 + threadIdx.x;
    if (!slot_ok(c, slot) || at >= nk + (v ? c.n_kv * c.vd : 0)) return;
    const bool key = at < nk;
    const int i = key ? at : at - nk, d = key ? c.qd : c.vd, kv = i / d;
    const int off = (int)(slot & ((1 << c.page_shift) - 1)), p = off & 63;
    const int64_t tile = c.tile((int)(slot >> c.page_shift), kv, off);
    const uint8_t *src = c.at(tile) + (key ? kv8_key_byte(d, p, i % d) : c.values() + kv8_value_byte(p, i % d));
    const float x = gload(c.scale_at(tile, key, p >> 4)) * (float)(int8_t)gload(src);
    gstore((key ? k + row * ks : v + row * vs) + i, x);
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

int moe_kv8_sizes(const moe_kv8 *c, uint64_t *codes, uint64_t *scales, uint64_t *open) {
    Kv8 k;
    if (!c || !codes || !scales || !open) return fail(MOE_EINVAL, "moe_kv8_sizes: bad argument");
    moe_kv8 any = *c;  // the sizes alone count
    any.codes = any.open = reinterpret_cast<void *>(16), any.scales = reinterpret_cast<float *>(16);
    any.codes_bytes = any.scales_bytes = any.open_bytes = UINT64_MAX;
    any.table = reinterpret_cast<const int32_t *>(16);
    any.max_pages = 1;
    if (const int rc = kv8_of("moe_kv8_sizes", &any, &k)) return rc;
    const uint64_t tiles = (uint64_t)k.n_pages * (uint64_t)(c->page / kTile8) * (uint64_t)k.n_kv;
    *codes = tiles * (uint64_t)k.tile_bytes(), *scales = tiles * 32;
    *open = (uint64_t)k.n_seq * (uint64_t)k.n_kv * (uint64_t)k.open_bytes();
    return MOE_OK;
}

int moe_kv8_store(const moe_kv8 *c, const float *k, int64_t k_stride, const float *v, int64_t v_stride, int32_t rows,
                  const int32_t *row_start, const int32_t *seq, const int32_t *pos, const int64_t *slots, void *stream) {
    Store a{};
    if (const int rc = kv8_of("moe_kv8_store", c, &a.c)) return rc;
    if (rows < 0 || (rows > 0 && (!k || !v || !row_start || !seq || !pos || !slots)))
        return fail(MOE_EINVAL, "moe_kv8_store: bad argument (%d rows)", rows);
    if (rows > kMostRows) return fail(MOE_EUNSUP, "moe_kv8_store: %d rows, up to %d at once", rows, kMostRows);
    if (rows == 0) return MOE_OK;
    a.k = k, a.v = v, a.ks = k_stride, a.vs = v_stride, a.rows = rows;
    a.row_start = row_start, a.seq = seq, a.pos = pos, a.slots = slots;
    hipLaunchKernelGGL(kv8_store_kernel, dim3(rows, a.c.n_kv), dim3(128), 0, (hipStream_t)stream, a);
    return rc_of("8-bit cache write kernel");
}

int moe_kv8_load(const moe_kv8 *c, const int64_t *slots, int32_t rows, float *k, int64_t k_stride, float *v,
                 int64_t v_stride, void *stream) {
    Kv8 a;
    if (const int rc = kv8_of("moe_kv8_load", c, &a)) return rc;
    if (rows < 0 || (rows > 0 && !slots)) return fail(MOE_EINVAL, "moe_kv8_load: bad argument (%d rows)", rows);
    if (rows > kMostRows) return fail(MOE_EUNSUP, "moe_kv8_load: %d rows, up to %d at once", rows, kMostRows);
    if (rows == 0 || (!k && !v)) return MOE_OK;
    const int values = a.n_kv * ((k ? a.qd : 0) + (v ? a.vd : 0));
    hipLaunchKernelGGL(kv8_load_kernel, dim3(rows, (values + 255) / 256), dim3(256), 0, (hipStream_t)stream, a, slots, k,
                       k_stride, v, v_stride);
    return rc_of("8-bit cache read kernel");
}

}  // extern "C"
