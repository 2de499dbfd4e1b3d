// kv8_cache.hip — writing and reading rows of the paged 8-bit cache
// (moe_kv8_store, moe_kv8_load): layout in kv8.h, quantiser in int8.h.
//
// A block's scale is its largest value's, so a row that joins a block may change
// all of its codes.  A block of threads takes what a step writes of one tile of one
// kv head, a wave its blocks' keys or values each: the rows of this step, and before
// them those of earlier steps, whose values `open` keeps while their block is
// filling.  Both kernels are streams: 16376 rows of 8 kv heads of 128 are written in
// 44 us (168 MB, 3.9 TB/s; 46 to 50 where nothing is cached) and read in 43 (33 where
// the codes are cached); 32 rows in 7.6 (three dependent loads: the row's place, its
// sequence's, the values) and 3.9.
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
// of two halves the block whose values it holds, plus 1, and how many of them, the
// block's first, are the sequence's.
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

__device__ inline uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// Bytes 0..3 of the words of lanes 0..3 of a quad, transposed.
__device__ inline uint32_t quad_transpose(uint32_t x) {
    const int i = threadIdx.x & 3;
    uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false);  // the lane 1 away
    x = i & 1 ? __builtin_amdgcn_perm(x, y, 0x07030501u) : __builtin_amdgcn_perm(y, x, 0x06020400u);
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false);  // 2 away
    return i & 2 ? __builtin_amdgcn_perm(x, y, 0x07060302u) : __builtin_amdgcn_perm(y, x, 0x05040100u);
}

// The row that is its tile's last in this step writes what the step has of the
// tile, for one kv head, with eight waves: four blocks' keys, four blocks' values
// (whose bytes meet in LDS).  A block of threads looks at `window` rows.  A lane
// takes four dims of one position at a time.
// NU: units of 16 dims there may be.  Up to 8, three blocks a CU: 16376 rows of 8
// heads of 128 52 -> 45 us, 256 decoding sequences 27 -> 22.
template <int NU>
__global__ __launch_bounds__(512, NU <= 8 ? 6 : 4) void kv8_store_kernel(const Store a, int window, int windows) {
    __shared__ uint32_t words[NU * 64 * 4];  // [dims / 16][lane][block]
    __shared__ f32x4_dw earlier[2][NU * 64];  // of the first block, [values, keys][dims / 16][lane]
    const Kv8 &c = a.c;
    const int kv = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int T = wave & 3;
    const bool key = wave < 4;
    // Each XCD takes windows that follow one another: those with a tile's last row,
    // every so many-th in a prompt, would otherwise meet on a few.
    const int per = (windows + 7) / 8, which = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (which >= windows) return;
    // What each row of the window is, a lane each.
    const int mine = which * window + min(lane, window - 1), from = min(mine, a.rows - 1);
    const int64_t my_slot = gload(a.slots + from);
    const int my_seq = gload(a.seq + from), my_pos = gload(a.pos + from);
    // Rows that are to be skipped may lie anywhere among a sequence's, so whose row
    // each is, or -1: of the window, the one behind it and the 64 before it (a tile's
    // last row and all others of the tile).
    auto row_of = [&](int j) {
        const int64_t slot = gload(a.slots + j);
        const int s = gload(a.seq + j), p = gload(a.pos + j);
        return slot_ok(c, slot) && p >= 0 ? s : -1;
    };
    const int start = which * window, next_of = row_of(min(mine + 1, a.rows - 1)), past = start - 64 + lane;
    const int past_row = row_of(max(past, 0)), past_of = past >= 0 ? past_row : -1;
    const bool good = lane < window && mine < a.rows && slot_ok(c, my_slot) && (unsigned)my_seq < (unsigned)c.n_seq && my_pos >= 0;
    const int my_r0 = good ? max(0, min(mine, gload(a.row_start + my_seq))) : 0;
    const int my_r1 = good ? max(mine + 1, min(a.rows, gload(a.row_start + my_seq + 1))) : 0;
    const u32x4 my_tags = good ? gload((const u32x4 *)(c.open_at(my_seq, kv) + 2 * kBlock8 * 4 * (c.qd + c.vd) + (key ? 0 : 16)))
                               : u32x4{0, 0, 0, 0};
    const bool followed = good && mine + 1 < my_r1 && next_of == my_seq;
    bool ends = good && ((my_pos & 63) == 63 || !followed);
    if (__builtin_expect(ends && !followed && mine + 2 < my_r1 && (my_pos & 63) < 62, 0))
        for (int j = mine + 2, of_tile = min(my_r1, mine + 64 - (my_pos & 63)); ends && j < of_tile; j++) ends = row_of(j) != my_seq;
    const unsigned long long follow = __ballot(followed);
    unsigned long long last = __ballot(ends);
    for (; last; last &= last - 1) {
        const int at = __builtin_ctzll(last), r = which * window + at;
        const int64_t slot = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(my_slot >> 32), at) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)my_slot, at));
        const int s = __builtin_amdgcn_readlane(my_seq, at), p = __builtin_amdgcn_readlane(my_pos, at);
        const int r0 = __builtin_amdgcn_readlane(my_r0, at), r1 = __builtin_amdgcn_readlane(my_r1, at);
        // Rows r - 63 .. r that are the sequence's and written; those of the tile, by
        // its positions; whether any lies before the tile.
        const int t0 = r - (p & 63);
        const unsigned long long late = __ballot(good && my_seq == s && mine >= r0), early = __ballot(past_of == s && past >= r0);
        const unsigned long long rows = late << (63 - at) | (at < 63 ? early >> (at + 1) : 0), there = rows >> (63 - (p & 63));
        // The sequence's first row from j on, before row `end` (or -1).
        auto first_row = [&](int j, int end) {
            for (; j < end; j += 64) {
                const unsigned long long some = __ballot(j + lane < end && row_of(min(j + lane, end - 1)) == s);
                if (some) return j + __builtin_ctzll(some);
            }
            return -1;
        };
        bool behind = t0 > r0;
        if (behind) {
            const int j = t0 - 1 - start;  // (-64 at least)
            behind = (j >= 0 ? late >> j : early >> (j + 64)) & 1 || first_row(r0, t0) >= 0;
        }
        const bool ends_here = !(follow >> at & 1) && (r + 2 >= r1 || first_row(r + 2, r1) < 0);
        // The position of the first row in the tile.
        const int p0 = behind ? p & ~63 : (p & ~63) + __builtin_ctzll(there);
        auto of_block = [&](int k) { return (uint32_t)(there >> (16 * k)) & 0xffffu; };
        const int final = p >> 4 & 3;
        const int64_t tile = c.tile((int)(slot >> c.page_shift), kv, (int)(slot & ((1 << c.page_shift) - 1)));
        uint8_t *codes = c.at(tile) + (key ? 0 : c.values());
        if (of_block(T)) {
            const int start = (p & ~63) + 16 * T, end = min(p, start + 15), in = end & 15;
            Block b;
            b.key = key, b.T = T, b.d = key ? c.qd : c.vd;
            b.n = end - max(start, p0) + 1, b.before = in + 1 - b.n;
            b.stride = key ? a.ks : a.vs;
            b.row = (key ? a.k : a.v) + (int64_t)(r - (p - max(start, p0))) * b.stride + (int64_t)kv * b.d;
            float *scale = c.scale_at(tile, key, T);
            b.tile = codes;
            // The half that holds the values of the block that was filling.
            uint8_t *open = c.open_at(s, kv);
            Half *tags = (Half *)(open + 2 * kBlock8 * 4 * (c.qd + c.vd)) + (key ? 0 : 2);
            float *halves = (float *)open + (key ? 0 : 2 * kBlock8 * c.qd);
            const bool keeps = T == final && ends_here;
            int was = 0, had = 0, half = -1;
            auto went_on = [&](int first) {  // from position `first` on
                was = first >> 4, had = first & 15;
                if (had)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (__builtin_amdgcn_readlane((int)my_tags[2 * h], at) == was + 1 &&
                            __builtin_amdgcn_readlane((int)my_tags[2 * h + 1], at) >= had)
                            half = h;
            };
            if (!behind) went_on(p0);
            b.held = half < 0 ? nullptr : halves + half * kBlock8 * b.d;
            b.scale = half < 0 && b.before ? gload(scale) : 0.0f;

            const int nu = b.d / 16;
            const int t = key ? lane >> 2 : (lane >> 4) * 4 + (lane & 3), i = key ? 4 * (lane & 3) : lane & 12;
            // Loads are unconditional (units past the last read it again), so that
            // they are in flight together.
            const bool now = t >= b.before, some = !now || (of_block(T) >> t & 1);
            const float *src = (!now && b.held ? b.held + t * b.d : b.row + (int64_t)(now && some ? t - b.before : 0) * b.stride) + i;
            f32x4_dw x[NU];
#pragma unroll
            for (int u = 0; u < NU; u++) x[u] = *(const __attribute__((address_space(1))) f32x4_dw *)(src + 16 * min(u, nu - 1));
            if (b.before && !b.held) {  // (through LDS: in registers the loop took 50 more)
                f32x4_dw *as_read = earlier[key] + lane;
#pragma unroll 1
                for (int u = 0; u < (now ? 0 : nu); u++) {
                    f32x4_dw y;
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = b.scale * (float)(int8_t)gload(b.tile + b.code_byte(t, 16 * u + i + e));
                    as_read[u * 64] = y;
                }
#pragma unroll
                for (int u = 0; u < NU; u++) x[u] = now || u >= nu ? x[u] : as_read[u * 64];
            }
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[u][e] = some && u < nu ? x[u][e] : 0.0f;
                    top = max(top, magnitude(x[u][e]));
                }
            // Kept: of the block that the step goes on in the values before it (which
            // may be what its codes read as), so that the step made again, or another
            // from there, finds them whatever this one makes of the codes; of the last
            // block, while it is filling, all of them, in the other half if it is
            // another block (that one's wave may be reading).  A half's count is how
            // many of its values are still the sequence's, so the first's goes back to
            // `had`, and nothing stays of earlier steps and sequences.
            const bool full = in == 15, on = !behind && had && (p >> 6) * 4 + T == was;
            if (on || keeps) {
                if (behind) went_on(max(0, p - (r - first_row(r0, t0))));
                const int near = half < 0 ? 0 : half;  // the first block's, from now on
                const bool all = keeps && !full;
                const int to = on || !had ? near : 1 - near, lo = on && half >= 0 ? b.before : 0, hi = all ? in + 1 : on ? had : 0;
                float *dst = halves + to * kBlock8 * b.d;
                if (t >= lo && t < hi)
#pragma unroll
                    for (int u = 0; u < NU; u++)
                        if (u < nu) *(__attribute__((address_space(1))) f32x4_dw *)(dst + t * b.d + 16 * u + i) = x[u];
                if (lane == 0) {
                    tags[to] = all ? Half{(p >> 4) + 1, in + 1} : on ? Half{was + 1, had} : Half{0, 0};
                    if (keeps && (on || !had)) tags[1 - to] = Half{0, 0};
                }
            }
            const Int8Scale q(wave_max(top));
#pragma unroll
            for (int u = 0; u < NU; u++)
                if (u < nu) {
                    const uint32_t w = pack4(q.code(x[u][0]), q.code(x[u][1]), q.code(x[u][2]), q.code(x[u][3]));
                    if (key) gstore((uint32_t *)(codes + T * 16 * c.qd + u * 256 + lane * 4), w);
                    else words[(u * 64 + lane) * 4 + T] = quad_transpose(w);
                }
            if (lane == 0) gstore(scale, q.scale);
        }
        __syncthreads();
        // The values' words: position by position inside, block by block.
        uint8_t *values = c.at(tile) + c.values();
        for (int w = threadIdx.x; w < c.vd * 4; w += 512) {
            if (of_block(0) && of_block(1) && of_block(2) && of_block(3)) {
                gstore((u32x4 *)(values + w * 16), *(const u32x4 *)&words[w * 4]);
                continue;
            }
            for (int k = 0; k < 4; k++)
                if (of_block(k)) gstore((uint32_t *)(values + w * 16 + k * 4), words[w * 4 + k]);
        }
        __syncthreads();
    }
}

// A thread takes four dims of R rows.  64 rows in turn, a tile's in a prompt, go to
// one XCD: they read the same lines of its values, four positions of a dim to a word.
template <int R>
__global__ __launch_bounds__(256) void kv8_load_kernel(const Kv8 c, const int64_t *__restrict__ slots, int rows,
                                                       float *__restrict__ k, int64_t ks, float *__restrict__ v, int64_t vs) {
    constexpr unsigned kGroups = 64 / R;  // of rows in 64
    const int64_t row = (int64_t)((blockIdx.x / (8 * kGroups) * 8 + (blockIdx.x & 7)) * 64 + (blockIdx.x >> 3 & (kGroups - 1)) * R);
    const int nk = k ? c.n_kv * c.qd : 0, at = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (row >= rows || at >= nk + (v ? c.n_kv * c.vd : 0)) return;
    const bool key = at < nk;
    const int i = key ? at : at - nk, d = key ? c.qd : c.vd, kv = i / d, dim = i - kv * d;
    int64_t slot[R], tile[R];
    bool ok[R];
    float scale[R];
    uint32_t w[R];
#pragma unroll
    for (int j = 0; j < R; j++) slot[j] = row + j < rows ? gload(slots + row + j) : -1;
#pragma unroll
    for (int j = 0; j < R; j++) {
        ok[j] = slot_ok(c, slot[j]);
        if (!ok[j]) slot[j] = 0;  // read, not written
        const int off = (int)(slot[j] & ((1 << c.page_shift) - 1));
        tile[j] = c.tile((int)(slot[j] >> c.page_shift), kv, off);
        scale[j] = gload(c.scale_at(tile[j], key, (off & 63) >> 4));
    }
    if (key) {
#pragma unroll
        for (int j = 0; j < R; j++) w[j] = gload((const uint32_t *)(c.at(tile[j]) + kv8_key_byte(c.qd, (int)(slot[j] & 63), dim)));
    } else {
        auto words = [&](int j, uint32_t (&y)[4]) {
            const uint8_t *src = c.at(tile[j]) + c.values() + kv8_value_byte((int)(slot[j] & 60), dim);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = gload((const uint32_t *)(src + 16 * e));
        };
        // Rows of a prompt find their words among the first's and the last's.
        uint32_t first[4], last[4];
        words(0, first);
        if (R > 1) words(R - 1, last);
#pragma unroll
        for (int j = 0; j < R; j++) {
            uint32_t y[4];
            const bool a = slot[j] >> 2 == slot[0] >> 2;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = R == 1 || a ? first[e] : last[e];
            if (R > 2 && !a && slot[j] >> 2 != slot[R - 1] >> 2) words(j, y);
            const uint32_t by = (uint32_t)(slot[j] & 3);
            const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], by | (by + 4) << 8 | 0x0c0c0000u);
            w[j] = lo | __builtin_amdgcn_perm(y[3], y[2], by << 16 | (by + 4) << 24 | 0x0c0cu);
        }
    }
#pragma unroll
    for (int j = 0; j < R; j++) {
        f32x4_dw x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = scale[j] * (float)(int8_t)(w[j] >> (8 * e));
        if (ok[j]) *(__attribute__((address_space(1))) f32x4_dw *)((key ? k + (row + j) * ks : v + (row + j) * vs) + i) = x;
    }
}

template <int NU>
void launch_store(const Store &a, int window, int windows, hipStream_t s) {
    hipLaunchKernelGGL((kv8_store_kernel<NU>), dim3((windows + 7) / 8 * 8, a.c.n_kv), dim3(512), 0, s, a, window, windows);
}

constexpr int kMostRows = (1 << 24) - 512;  // a block of 256 threads a row, 512 rows at a time

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
    // Rows that are their tile's last lie `apart` rows from each other on average: a
    // window of about as many leaves few blocks without one and few with several.
    // Where all rows' blocks are resident at once (three a CU) each takes one row; where
    // there are very many, blocks of 16 rows and more start faster than they wait.  us
    // with one row a block and as here: 1000 rows of one sequence, 8 heads of 128, 17.8
    // and 7.0; 20 sequences of 100 34 and 10.3; 64 of 40 20.5 and 17.9; 4000 of 1 273
    // and 237; 8 of 40, 2 heads of 64 (640 blocks) 6.0 and 7.5 without the first rule.
    const double each = (double)rows / a.c.n_seq, apart = 1.25 * each / (1.0 + each / kTile8);
    const int64_t blocks = (int64_t)rows * a.c.n_kv;
    int window = blocks > 16384 ? 16 : 1;
    if (blocks > 768)
        while (window < 64 && 2 * window <= apart) window *= 2;
    const int windows = (rows + window - 1) / window;
    const int units = std::max(a.c.qd, a.c.vd) / 16;
    if (units <= 4) launch_store<4>(a, window, windows, (hipStream_t)stream);
    else if (units <= 8) launch_store<8>(a, window, windows, (hipStream_t)stream);
    else if (units <= 12) launch_store<12>(a, window, windows, (hipStream_t)stream);
    else launch_store<16>(a, window, windows, (hipStream_t)stream);
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
    auto go = [&](auto load, unsigned each) {
        hipLaunchKernelGGL(load, dim3(((unsigned)rows + 511) / 512 * (512 / each), (values + 1023) / 1024), dim3(256), 0,
                           (hipStream_t)stream, a, slots, rows, k, k_stride, v, v_stride);
    };
    // us with a row and with four a thread: 16440 rows of 8 heads of 128 60 and 44, 1000
    // 6.1 and 5.7, 300 (614400 values) 4.4 and 4.8; 300 of 16 heads of 192/128 6.6 and
    // 6.1; 4000 of 2 heads of 64 (1.0e6) 4.5 and 4.7.
    if ((int64_t)rows * values >= 5 << 18) go(kv8_load_kernel<4>, 4);
    else go(kv8_load_kernel<1>, 1);
    return rc_of("8-bit cache read kernel");
}

}  // extern "C"
