// kv8_attention.hip — causal attention over the paged 8-bit cache
// (moe_kv8_attention), layout in kv8.h.
//
// Rows find their sequence and position on the device, so one kernel serves
// decode steps, prompts and chunks.  A block takes a group of consecutive rows
// and one kv head, splits the group into runs of one sequence and makes each
// run's (row, query head) pairs the columns of its products on the 8-bit integer
// matrix cores, 16 a wave.
//
// Codes are the products' operands as they lie in memory; queries and weights
// meet them as whole numbers of 24 bits in three signed bytes,
//   q scale = Q 2^(e - 22),  Q = 65536 d2 + 256 d1 + d0,  |Q| <= 2^22
// (2^e above the head's largest), so a block's scores are
//   s = s_k 2^(e - 22) (256 (256 K d2 + K d1) + K d0),
// sums of whole numbers, exact, then three roundings of 2^-24 (none below 2^24).
// The result's layout (lane = column, positions 4 g + i of each block) is the
// second operand of the values' product.  There the weights p = 2^(s - m) meet the values' scales first:
//   W = p s_v C 2^-r,  r the largest s - m + log2 s_v of the step,  C = 2^23 - ..
// so W below 2^23 keeps each block's product of weight and scale to 2^-23 of the
// step's largest.  A step takes blocks whose value scales lie within 2^5 of each
// other and goes over its tiles once more for others, so that what is small in some
// of a head's dims keeps its precision beside what is large in others (in the same
// pass a block 2^-16 of its neighbours kept 7 bits).  Multiplied and added to 2^23 +
// 0x8080 in one instruction, a weight's bits are its three digits (the two low ones
// with 128 added).  A step's sums are whole numbers too; they join
// the f32 sums O, which are multiples of 2^(m + e) (the weights' sum's of 2^m).
// Everything is in differences from m, and m and e are whole numbers, so that no
// step's scores, however large, round what earlier steps left: one position whose
// score is 1e20 above the others gives its value to 2^-23.
// Sums that stayed whole numbers over many steps would need references
// with room above them: three bits of it cost a digit's eighth (1e-5 of the output
// against 1e-6) and still had to move for one wave of a block in every second step.
//
// Decode reads the cache once and is bound by that: 64 sequences of 6000 to 12000
// positions, 8 kv heads of 128, 235 us (5.0 TB/s of codes), one of 100001 in 128
// parts 40 with the joining launch, 32 of up to 1500 19 (4.0 TB/s: one block a CU
// with 12 to 24 tiles, then a merge).  Prompts are bound by the issue of vector
// instructions beside the products: 4001 rows of 32 heads of 128 271 us (484
// TFLOP/s of the attention's own operations), 8000 rows 955 (549), of which the
// matrix pipe is busy in 29% and vector instructions issue in 71% (25 to a
// score: joining three sums 4, the exponential 2, the weight and its digits 4, a
// step's sums into O 5 for every two).  Two tiles' products a step halve that last
// part; three and four waves a SIMD, at one tile a step, were no faster.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "gmem.h"
#include "kv8.h"
#include "lds_dma.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // at any float
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    Kv8 c;
    const float *q;
    const int32_t *seq, *pos;
    float *out, *part, *part_ml;  // part [row][head][ps][vd], part_ml [row][head][ps][m, l, e]
    int64_t q_stride, out_stride;
    int rows, heads, rep, window;
    float scale;
    int tt, groups;  // rows of a group, groups
    int rc, chunks;  // query heads of a block, blocks that share a kv head's
    int split;       // blocks that share a group's runs
    int ps;          // blocks that share a run's tiles
};

constexpr float kNone = -3e38f;          // below every score: where nothing has been seen
constexpr float kMost = 8355000.0f;      // largest weight (C): its digits' room is 8355711, what exp2 errs by taken off
constexpr float kLeastLog = -100.0f;     // log2 of a value scale, where it is smaller or 0

__device__ inline i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// The largest of a column's four lanes (16 apart), in each of them.
__device__ inline float column_max(float x) {
    const uint32_t u = __float_as_uint(x);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A product's sums of the three digits begin at the bits of 3 x 2^22: an integer
// below 2^22 added to those is the float 3 x 2^22 + it, so nothing is converted
// (127 x 128 of up to 256 products stay below).
constexpr int kZero = 0x4b400000;

// 65536 d2 + 256 d1 + d0 of such sums: the constants cancel inside the two
// multiply-adds, each of which, and the second subtraction, rounds once (2^-24;
// not at all up to 2^24).
__device__ inline float joined(int d2, int d1, int d0) {
    const float u = fmaf(__int_as_float(d2) - (12582912.0f + 49152.0f), 256.0f, __int_as_float(d1));
    return fmaf(u - 49152.0f, 256.0f, __int_as_float(d0));
}

// Four weights' digits, by digit: 2 (highest), 1, 0.
struct Digits {
    uint32_t d2, d1, d0;
};
__device__ inline Digits digits_of(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
    const uint32_t a = __builtin_amdgcn_perm(w1, w0, 0x05010400u), b = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
    Digits d;
    d.d0 = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
    d.d1 = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u;
    d.d2 = __builtin_amdgcn_perm(w1, w0, 0x0c0c0602u) | __builtin_amdgcn_perm(w3, w2, 0x06020c0cu);
    return d;
}

// A wave's 16 columns.  Lane (column, g) of o[D] holds dims 16 D + 4 g + i.
template <int NV>
struct Columns {
    f32x4 o[NV];
    float m, e, l;      // whole numbers, see above; this lane's positions' weights
    float qs;           // 2^(e - 22) |scale| log2(e)
    int pos, lo;        // what a column sees: positions lo .. pos
    int first, last;    // of all columns: everything in first .. last is seen by every one
};

// One step of NT tiles over their blocks `todo` (a bit each), or those of them whose
// value scales are near the largest; returns which are left.  k(b, c) and v(D, t)
// give operands, base[t] the tiles' first positions (negative: no such tile).  read()
// is called when the keys are done with.  Lane 8 t + b holds the scale of tile t's
// block b of keys, lane 8 t + 4 + b that of its values (0 where there is no tile):
// uniform values go through scalar registers.
template <int NQ, int NV, int NT, bool EX, class K, class V, class F>
__device__ __attribute__((always_inline)) inline int step(Columns<NV> &x, const i32x4 (&q)[3][NQ], K k, V v, F read, float scale,
                                                          const int (&base)[NT], int nv, int g, int todo) {
    f32x4 s[4 * NT];
#pragma unroll
    for (int b = 0; b < 4 * NT; b++) {
        const i32x4 zero = {kZero, kZero, kZero, kZero};
        i32x4 d[3] = {zero, zero, zero};
#pragma unroll
        for (int c = 0; c < NQ; c++) {
            const i32x4 kk = k(b, c);
#pragma unroll
            for (int p = 0; p < 3; p++) d[p] = mfma(kk, q[p][c], d[p]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[b][i] = joined(d[0][i], d[1][i], d[2][i]);
    }
    read();
    const int lane = threadIdx.x & 63;
    auto exponent = [&](float y) { return (int)(__float_as_uint(y) >> 23); };
    // Value scales' exponents within 2 of the first's are within 2^5 of each other
    // (0: zeros, anyone's).
    int now = todo, first = x.first;
    const int about = __builtin_amdgcn_readlane(exponent(scale), 4) - 2;
    if (__builtin_expect(__ballot(!(fabsf(scale) < INFINITY)) |
                             (__ballot(scale != 0.0f && (unsigned)(exponent(scale) - about) > 4) & (NT > 1 ? 0xf0f0 : 0xf0)), 0)) {
        for (int b = 0; b < 4 * NT; b++) {  // a block that reads as NaN: so are the columns that see it
            const int at = b / 4 * 8 + b % 4;
            if (fabsf(__shfl(scale, at, 64)) < INFINITY && fabsf(__shfl(scale, at + 4, 64)) < INFINITY) continue;
            const int p = (b < 4 ? base[0] : base[NT - 1]) + 16 * (b % 4);
            if (p <= x.pos && p + 15 >= x.lo) x.l = __uint_as_float(0x7fc00000u);
            if (lane == at || lane == at + 4) scale = 0.0f;
        }
        // Blocks of the largest scales, 2^5 down at most; `first`: a step that is not whole.
        const int mine = lane & 4 && todo >> ((lane >> 1 & 4) + (lane & 3)) & 1 ? exponent(scale) : -1;
        int largest = max(mine, __shfl_xor(mine, 1, 64));
        largest = max(largest, __shfl_xor(largest, 2, 64));
        largest = max(largest, __shfl_xor(largest, 8, 64));
        const uint32_t near = (uint32_t)__ballot(mine == 0 || mine >= largest - 4);
        now = todo & ((near >> 4 & 15) | (near >> 12 & 15) << 4);
        if (now != (1 << 4 * NT) - 1) first = 0x7fffffff;
    }
    const float log_ = fmaxf(__builtin_amdgcn_logf(scale), kLeastLog);
    auto of = [&](float y, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(y), i)); };
    float sc[4 * NT];
#pragma unroll
    for (int b = 0; b < 4 * NT; b++) sc[b] = of(scale, b / 4 * 8 + b % 4) * x.qs;
    bool whole = true;
#pragma unroll
    for (int t = 0; t < NT; t++) whole = whole && base[t] >= first && base[t] + 63 <= x.last;
    if (!whole) {
#pragma unroll
        for (int b = 0; b < 4 * NT; b++) {
            const int p = base[b / 4] + 16 * (b % 4) + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[b][i] = (now >> b & 1) && base[b / 4] >= 0 && p + i >= x.lo && p + i <= x.pos ? s[b][i] * sc[b] : -INFINITY;
            sc[b] = 1.0f;
        }
    }
    float most[4 * NT], top = kNone;
#pragma unroll
    for (int b = 0; b < 4 * NT; b++) {
        most[b] = fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3]));
        top = fmaxf(top, most[b] * sc[b]);
    }
    top = column_max(top);
    // Scores whose rounding is more than the weights' range bears: all are rounded,
    // as the largest is (where not all positions are seen they have been).
    if (__builtin_expect(whole && __any(fabsf(top) > 4194304.0f), 0)) {
#pragma unroll
        for (int b = 0; b < 4 * NT; b++) {
#pragma unroll
            for (int i = 0; i < 4; i++) s[b][i] *= sc[b];
            most[b] *= sc[b], sc[b] = 1.0f;
        }
    }
    top = __builtin_ceilf(top);
    float ref = kLeastLog - 2.0f;  // (where nothing is seen)
#pragma unroll
    for (int b = 0; b < 4 * NT; b++) ref = fmaxf(ref, fmaf(most[b], sc[b], -top) + of(log_, b / 4 * 8 + 4 + b % 4));
    ref = column_max(ref);
    const float f = __builtin_amdgcn_exp2f(-ref) * kMost;
    float sum = 0.0f;
    i32x4 w[NT][3];
#pragma unroll
    for (int b = 0; b < 4 * NT; b++) {
        const float scaled = fminf(of(scale, b / 4 * 8 + 4 + b % 4) * f, 3e38f);  // (p is 0 where it would be more)
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[b][i], sc[b], -top));
            sum += p;
            y[i] = __float_as_uint(fmaf(p, scaled, 8388608.0f + 32896.0f));
        }
        const Digits d = digits_of(y[0], y[1], y[2], y[3]);
        w[b / 4][0][b % 4] = (int)d.d2, w[b / 4][1][b % 4] = (int)d.d1, w[b / 4][2][b % 4] = (int)d.d0;
    }
    const float m = fmaxf(x.m, top), was = x.e + (x.m - m), here = ref + (top - m), e = fmaxf(was, __builtin_ceilf(here));
    x.l = x.l * __builtin_amdgcn_exp2f(x.m - m) + sum * __builtin_amdgcn_exp2f(top - m);
    if (__any(e > was)) {
        const float keep = __builtin_amdgcn_exp2f(was - e);
#pragma unroll
        for (int D = 0; D < NV; D++)
#pragma unroll
            for (int i = 0; i < 4; i++) x.o[D][i] *= keep;
    }
    const float in0 = __builtin_amdgcn_exp2f(here - e) * (1.0f / kMost);
    x.m = m, x.e = e;
#pragma unroll
    for (int D = 0; D < NV; D++) {
        if (!EX && D >= nv) continue;
        const i32x4 zero = {kZero, kZero, kZero, kZero};
        i32x4 d[3] = {zero, zero, zero};
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const i32x4 vv = v(D, t);
#pragma unroll
            for (int p = 0; p < 3; p++) d[p] = mfma(vv, w[t][p], d[p]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            x.o[D][i] = fmaf(joined(d[0][i], d[1][i], d[2][i]), in0, x.o[D][i]);
    }
    return todo & ~now;
}

// Lanes of my_seq and my_pos that begin a run of one sequence's rows or are
// none; the runs' first lanes.
struct Runs {
    unsigned long long cuts, starts, valid;
};
__device__ inline Runs runs_of(const Kv8 &c, int my_seq, int my_pos, int nr) {
    const int lane = threadIdx.x & 63;
    const bool valid = lane < nr && my_pos >= 0 && (unsigned)my_seq < (unsigned)c.n_seq;
    const int before = __shfl_up(my_seq, 1, 64);
    const bool before_ok = __shfl_up((int)valid, 1, 64);
    Runs r;
    r.valid = __ballot(valid);
    r.cuts = __ballot(!valid || lane == 0 || my_seq != before || !before_ok);
    r.starts = r.cuts & r.valid;
    return r;
}

// One run of a group: rows first .. end - 1 of it, and what they see.
struct Run {
    int first, end, seq, lo, hi;
};
__device__ inline bool next_run(const Runs &r, unsigned long long &starts, int nr, int my_seq, int my_pos, int window, Run &x) {
    if (!starts) return false;
    const int lane = threadIdx.x & 63;
    x.first = __builtin_ctzll(starts);
    starts &= starts - 1;
    const unsigned long long after = x.first < 63 ? r.cuts >> (x.first + 1) : 0;
    x.end = min(nr, after ? x.first + 1 + __builtin_ctzll(after) : 64);
    const bool mine = lane >= x.first && lane < x.end;
    int hi = mine ? my_pos : -1, lo = mine ? (window > 0 ? max(0, my_pos + 1 - window) : 0) : 0x7fffffff;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        hi = max(hi, __shfl_xor(hi, o, 64));
        lo = min(lo, __shfl_xor(lo, o, 64));
    }
    x.hi = __builtin_amdgcn_readfirstlane(hi), x.lo = __builtin_amdgcn_readfirstlane(lo);
    x.seq = __builtin_amdgcn_readlane(my_seq, x.first);
    return true;
}

// Pages of a run, 64 at a time, one a lane: where the kv head's tiles are (as a
// tile's number; negative: no such page).
struct Pages {
    int b0 = -64;
    uint32_t lo = 0;
    int hi = -1;
    __device__ int64_t tile(const Kv8 &c, const int32_t *table, int kv, int t) {  // of the sequence's tile t
        const int shift = c.page_shift - 6, i = t >> shift;
        if (i < b0 || i >= b0 + 64) {
            b0 = i;
            const int page = b0 + (threadIdx.x & 63), pid = page < c.max_pages ? gload(table + page) : -1;
            const int64_t at = (unsigned)pid < (unsigned)c.n_pages ? c.tile(pid, kv, 0) : -1;
            lo = (uint32_t)at, hi = (int)(at >> 32);
            asm volatile("" : "+v"(lo), "+v"(hi));  // waited for here, not at every tile
        }
        const int h = __builtin_amdgcn_readlane(hi, i - b0);
        const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)lo, i - b0);
        return h < 0 ? -1 : ((int64_t)h << 32 | l) + (t & ((1 << shift) - 1));
    }
};

// Queries' digits into LDS as the product reads them, [digit][chunk][lane], for
// COLS columns; a column's factor 2^(e - 22) |scale| log2(e), NaN where the query
// is not finite.  16 threads a column, 16 dims each.
template <int NQ, int COLS>
__device__ inline void stage_queries(const Args &a, u32x4 *sq, float *sk, int r0, int h0, int hn, int c0, int c1) {
    const int u = threadIdx.x & 15, nu = a.c.qd / 16;
    for (int col = threadIdx.x >> 4; col < COLS; col += blockDim.x >> 4) {
        const int cc = c0 + col;
        float x[16];
        const bool there = cc < c1 && u < nu;
        const float *src = a.q + (int64_t)(r0 + (there ? cc : c0) / hn) * a.q_stride + (int64_t)(h0 + (there ? cc : c0) % hn) * a.c.qd +
                           (there ? 16 * u : 0);
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const f32x4 y = __builtin_bit_cast(f32x4, gload_x4((const uint32_t *)src + 4 * j));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[4 * j + e] = there ? y[e] : 0.0f;
                top = max(top, __float_as_uint(x[4 * j + e]) & 0x7fffffffu);
            }
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const bool finite = top < 0x7f800000u;
        // 2^e above the largest (of a subnormal one, 2^-126)
        const int e = max((int)(top >> 23) - 126, -126);
        uint32_t d[3][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = finite ? rintf(ldexpf(x[4 * j + i], 22 - e)) : 0.0f;
                w[i] = (uint32_t)((int)(a.scale < 0.0f ? -v : v) + 0x808080);
            }
            const Digits z = digits_of(w[0], w[1], w[2], w[3]);
            d[0][j] = z.d2 ^ 0x80808080u, d[1][j] = z.d1, d[2][j] = z.d0;
        }
        if (u < 4 * NQ)
#pragma unroll
            for (int p = 0; p < 3; p++)
                sq[((col >> 4) * 3 + p) * NQ * 64 + (u >> 2) * 64 + (u & 3) * 16 + (col & 15)] = u32x4{d[p][0], d[p][1], d[p][2], d[p][3]};
        if (u == 0) sk[col] = finite ? ldexpf(fabsf(a.scale) * 1.44269504088896341f, e - 22) : __uint_as_float(0x7fc00000u);
    }
}

// A wave's columns at the start of a run; `row`: the lane's column's row in the group.
template <int NQ, int NV>
__device__ inline void begin(Columns<NV> &x, i32x4 (&q)[3][NQ], const u32x4 *sq, const float *sk, int my_pos, int window, int row) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < 3; p++)
#pragma unroll
        for (int c = 0; c < NQ; c++) q[p][c] = __builtin_bit_cast(i32x4, sq[(p * NQ + c) * 64 + lane]);
#pragma unroll
    for (int D = 0; D < NV; D++) x.o[D] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float k = sk[lane & 15];
    x.qs = k != k ? 0.0f : k;
    x.m = kNone, x.e = 0.0f;
    x.l = k != k ? k : 0.0f;
    x.pos = __shfl(my_pos, row, 64);
    x.lo = window > 0 ? max(0, x.pos + 1 - window) : 0;
    int first = x.lo, last = x.pos;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        first = max(first, __shfl_xor(first, o, 64));
        last = min(last, __shfl_xor(last, o, 64));
    }
    x.first = __builtin_amdgcn_readfirstlane(first), x.last = __builtin_amdgcn_readfirstlane(last);
}

// What a block of 16 columns shares.
template <int NQ, int NV>
struct Narrow {
    u32x4 sq[3 * NQ * 64];
    f32x4 so[4 * NV * 64];  // O of the waves: [wave][D][lane]
    float sk[16], sm[4][16], sl[4][16], se[4][16];
};

typedef const __attribute__((address_space(1))) uint8_t *gbytes;
__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const void *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00020000);
}

// 16 columns, four waves sharing the positions: rows r0 .. r0 + nr - 1 (whose
// sequences and positions the lanes hold), heads h0 .. h0 + hn - 1; every
// split-th run from `sub` on, of its tiles the part-th part.
template <int NQ, int NV, bool EX>
__device__ __attribute__((always_inline)) inline void narrow(const Args &a, Narrow<NQ, NV> &lds, int kv, int part, int r0, int nr, int h0,
                                                             int hn, int my_seq, int my_pos, int sub, int split) {
    const Kv8 &c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int nv = EX ? NV : c.vd / 16, qd = EX ? 64 * NQ : c.qd;
    stage_queries<NQ, 16>(a, lds.sq, lds.sk, r0, h0, hn, 0, nr * hn);
    __syncthreads();
    const Runs runs = runs_of(c, my_seq, my_pos, nr);
    unsigned long long starts = runs.starts;
    Run run;
    for (int n = 0; next_run(runs, starts, nr, my_seq, my_pos, a.window, run); n++) {
        if (n % split != sub) continue;
        const int c0 = run.first * hn, ncol = run.end * hn - c0;
        Columns<NV> x;
        i32x4 q[3][NQ];
        // (columns of other runs do as this run's first or last)
        begin<NQ, NV>(x, q, lds.sq, lds.sk, my_pos, a.window, min(max(col, c0), c0 + ncol - 1) / hn);
        const int32_t *table = c.table + (int64_t)run.seq * c.max_pages;
        const int t0 = run.lo >> 6, nt = (run.hi >> 6) - t0 + 1;
        const int parts = a.ps * 4, me = part * 4 + wave;
        int t = t0 + (int)((long long)nt * me / parts);
        const int t1 = t0 + (int)((long long)nt * (me + 1) / parts);
        Pages pages;
        i32x4 k[4][NQ], v[NV];
        float scale;
        int base[1];
        __amdgpu_buffer_rsrc_t buf;
        // A tile's values are asked for when its keys are done with, the next one's
        // keys behind its values: in flight over the softmax and the other waves'
        // work (a tile earlier took 18 to 30 more registers; 300 sequences of 9 rows
        // at 200 positions 107 -> 103 us, 32 that decode 20.2 -> 19.9).  Where there
        // is no tile the loads read nothing (0).
        auto load_keys = [&](int at) __attribute__((always_inline)) {
            const int64_t tile = at < t1 ? pages.tile(c, table, kv, at) : -1;
            base[0] = tile < 0 ? -64 : at * 64;
            buf = buffer_of(tile < 0 ? c.codes : c.at(tile), tile < 0 ? 0 : c.tile_bytes());
            const __amdgpu_buffer_rsrc_t sb = buffer_of(tile < 0 ? (const void *)c.scales : c.scales + tile * 8, tile < 0 ? 0 : 32);
            scale = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sb, 4 * (lane & 7), 0, 0));
#pragma unroll
            for (int T = 0; T < 4; T++)
#pragma unroll
                for (int cc = 0; cc < NQ; cc++)
                    k[T][cc] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, 16 * lane, T * 16 * qd + cc * 1024, 0));
        };
        auto load_values = [&] __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int D = 0; D < NV; D++)
                v[D] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, 16 * lane, 64 * qd + D * 1024, 0));
            __builtin_amdgcn_sched_barrier(0);
        };
        if (t < t1) load_keys(t);
        for (int todo = 15; t < t1;) {
            if (base[0] >= 0)
                todo = step<NQ, NV, 1, EX>(x, q, [&](int b, int cc) { return k[b][cc]; }, [&](int D, int) { return v[D]; }, load_values,
                                           scale, base, nv, g, todo);
            else todo = 0;
            __builtin_amdgcn_sched_barrier(0);
            if (todo == 0) t++, todo = 15;  // (else the same tile's once more)
            load_keys(t);
        }

        // Merge the waves: sums as they are and their references through LDS,
        // then every wave takes a share of the output's dims.
        x.l += __shfl_xor(x.l, 16, 64);
        x.l += __shfl_xor(x.l, 32, 64);
        if (g == 0) lds.sm[wave][col] = x.m, lds.sl[wave][col] = x.l, lds.se[wave][col] = x.e;
#pragma unroll
        for (int D = 0; D < NV; D++) lds.so[(wave * NV + D) * 64 + lane] = x.o[D];
        __syncthreads();
        float m = kNone, e = -INFINITY, l = 0.0f, f[4];
#pragma unroll
        for (int w = 0; w < 4; w++) m = fmaxf(m, lds.sm[w][col]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = lds.se[w][col] + (lds.sm[w][col] - m), e = fmaxf(e, f[w]);
            l += lds.sl[w][col] * __builtin_amdgcn_exp2f(lds.sm[w][col] - m);
        }
#pragma unroll
        for (int w = 0; w < 4; w++) f[w] = __builtin_amdgcn_exp2f(f[w] - e);
        if (col >= c0 && col < c0 + ncol) {
            const int64_t row = r0 + col / hn, head = h0 + col % hn;
            float *dst = a.out + row * a.out_stride + head * c.vd;
            float by = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(e) / l;
            if (a.ps > 1) {
                const int64_t at = (row * a.heads + head) * a.ps + part;
                dst = a.part + at * c.vd, by = 1.0f;
                if (g == 0 && wave == 0) a.part_ml[3 * at] = m, a.part_ml[3 * at + 1] = l, a.part_ml[3 * at + 2] = e;
            }
#pragma unroll
            for (int i = 0; i < (NV + 3) / 4; i++) {
                const int D = 4 * i + wave;
                if (D >= nv) continue;
                f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const f32x4 y = lds.so[(w * NV + D) * 64 + lane];
#pragma unroll
                    for (int k = 0; k < 4; k++) z[k] = fmaf(y[k], f[w], z[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) z[k] *= by;
                *(__attribute__((address_space(1))) f32x4_dw *)(dst + 16 * D + 4 * g) = __builtin_bit_cast(f32x4_dw, z);
            }
        }
        __syncthreads();
    }
}

// What a block of 64 columns shares: two steps of NT tiles (the queries' digits
// before the first).
template <int NQ, int NV, int NT>
struct Wide {
    static constexpr int kTile = 64 * (64 * NQ + 16 * NV);
    union {
        uint8_t tiles[2][NT * kTile];
        u32x4 sq[4 * 3 * NQ * 64];
    };
    float scales[2][NT * 8], sk[64];
};

// 64 columns of one run, 16 a wave; every wave goes over all tiles, which come
// through LDS by DMA, a step ahead.
template <int NQ, int NV, int NT>
__device__ __attribute__((always_inline)) inline void wide(const Args &a, Wide<NQ, NV, NT> &lds_, int kv, int r0, int nr, int h0, int hn,
                                                           int my_seq, int my_pos, const Runs &runs) {
    const Kv8 &c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    constexpr int qd = 64 * NQ, bytes = Wide<NQ, NV, NT>::kTile;
    unsigned long long starts = runs.starts;
    Run run;
    next_run(runs, starts, nr, my_seq, my_pos, a.window, run);
    const int c0 = run.first * hn, ncol = (run.end - run.first) * hn;
    stage_queries<NQ, 64>(a, lds_.sq, lds_.sk, r0, h0, hn, c0, c0 + ncol);
    __syncthreads();
    Columns<NV> x;
    i32x4 q[3][NQ];
    const int mine = wave * 16 + col, own = c0 + min(mine, ncol - 1);
    begin<NQ, NV>(x, q, lds_.sq + wave * 3 * NQ * 64, lds_.sk + wave * 16, my_pos, a.window, own / hn);
    // What any column of the wave sees.
    int lo = x.lo, hi = x.pos;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    const int32_t *table = c.table + (int64_t)run.seq * c.max_pages;
    const int t0 = run.lo >> 6, t1 = (run.hi >> 6) + 1;
    Pages pages;
    const uint32_t to = lds::lds_addr(lds_.tiles[0]), to_scales = lds::lds_addr(lds_.scales[0]);
    // Queue a step's loads; which of its tiles there are.
    auto fetch = [&](int t, int buffer) __attribute__((always_inline)) {
        int there = 0;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int64_t tile = t + i < t1 ? pages.tile(c, table, kv, t + i) : -1;
            if (tile < 0) continue;
            there |= 1 << i;
            const uint8_t *src = c.at(tile);
            const uint32_t dst = to + buffer * (uint32_t)sizeof(lds_.tiles[0]) + i * bytes;
            for (int k = wave; k < bytes / 1024; k += 4) lds::dma16(src + k * 1024, lane * 16, dst + k * 1024);
            if (wave == i % 4 && lane < 8) lds::dma4(c.scales + tile * 8, lane * 4, to_scales + buffer * (uint32_t)sizeof(lds_.scales[0]) + i * 32);
        }
        return there;
    };
    __syncthreads();  // the queries are read
    int now = fetch(t0, 0);
    for (int t = t0, buffer = 0; t < t1; t += NT, buffer ^= 1) {
        lds::wait_vm_barrier<0>();
        const int later = t + NT < t1 ? fetch(t + NT, buffer ^ 1) : 0;
        if (t <= hi >> 6 && t + NT > lo >> 6) {
            auto go = [&](int tt, lds::lds_p at, float scale, int todo) __attribute__((always_inline)) {
                int base[NT];
#pragma unroll
                for (int i = 0; i < NT; i++) base[i] = now >> i & 1 ? (tt + i) * 64 : -64;
                return step<NQ, NV, NT, true>(
                    x, q,
                    [&](int b, int cc) __attribute__((always_inline)) {
                        return *(const __attribute__((address_space(3))) i32x4 *)(at + (b >> 2) * bytes + (b & 3) * 16 * qd + cc * 1024);
                    },
                    [&](int D, int i) __attribute__((always_inline)) {
                        return *(const __attribute__((address_space(3))) i32x4 *)(at + i * bytes + 64 * qd + D * 1024);
                    },
                    [] {}, scale, base, NV, g, todo);
            };
            auto scale_of = [&] { return now >> (lane >> 3 & (NT - 1)) & 1 ? lds_.scales[buffer][lane & (8 * NT - 1)] : 0.0f; };
            // (A loop around one copy of the step took 8 us more for a prompt's 267; above,
            // for 16 columns, two copies took 0 to 4% more.)
            int todo = go(t, (lds::lds_p)lds_.tiles[buffer] + lane * 16, scale_of(), (1 << 4 * NT) - 1);
            while (__builtin_expect(todo, 0)) {
                int tt = t;
                lds::lds_p at = (lds::lds_p)lds_.tiles[buffer] + lane * 16;
                asm volatile("" : "+s"(tt), "+v"(at)::"memory");  // (operands are read again, not kept)
                todo = go(tt, at, scale_of(), todo);
            }
        }
        now = later;
    }
    x.l += __shfl_xor(x.l, 16, 64);
    x.l += __shfl_xor(x.l, 32, 64);
    if (mine >= ncol) return;
    const float by = x.l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x.e) / x.l;
    float *dst = a.out + (int64_t)(r0 + own / hn) * a.out_stride + (int64_t)(h0 + own % hn) * c.vd + 4 * g;
#pragma unroll
    for (int D = 0; D < NV; D++) {
        f32x4_dw z;
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = x.o[D][e] * by;
        *(__attribute__((address_space(1))) f32x4_dw *)(dst + 16 * D) = z;
    }
}

// NT tiles a step for groups of 64 columns; 0: groups of 16 only.  Blocks of 64
// columns pay where one run fills them: a group with several runs (sequences that
// decode, ends of prompts), or with no more than 16 columns, is dealt to its blocks
// in groups of 16 instead.
// Waves a SIMD: heads wider than 128 take the registers of two (at two a SIMD 95
// were spilled, 32 sequences of 16 heads over 8 of 256 at 2000 positions 65 -> 44
// us); heads of 64 fit three (16000 rows of 8 heads over 2 676 -> 608, 1000
// sequences of 9 rows at 300 positions 86 -> 66).
template <int NQ, int NV, bool EX, int NT>
__global__ __launch_bounds__(256, NV > 8 ? 1 : NV > 4 ? 2 : 3) void kv8_attention_kernel(const Args a) {
    static_assert(NT == 0 || EX, "widths of their own");
    union Both {
        Narrow<NQ, NV> narrow;
        Wide<NQ, NV, NT ? NT : 1> wide;
    };
    __shared__ std::conditional_t<NT != 0, Both, Narrow<NQ, NV>> lds;
    const Kv8 &c = a.c;
    const int lane = threadIdx.x & 63;
    // Kv heads next to each other go to the XCDs in turn, so that one head's
    // blocks find its tiles in their L2.  Later rows of a prompt see more
    // positions: the last groups go first.  A group's blocks that find no run of
    // their own leave at once, so the first ones come together.
    int id = blockIdx.x;
    const int kv = id % c.n_kv;
    id /= c.n_kv;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int part = id % a.ps;
    id /= a.ps;
    const int sub = id / a.groups;
    const int r0 = (a.groups - 1 - id % a.groups) * a.tt;
    const int nr = min(a.tt, a.rows - r0);
    const int h0 = kv * a.rep + chunk * a.rc, hn = min(a.rc, a.rep - chunk * a.rc);
    const int my_seq = gload(a.seq + r0 + min(lane, nr - 1)), my_pos = gload(a.pos + r0 + min(lane, nr - 1));
    if constexpr (NT == 0) {
        narrow<NQ, NV, EX>(a, lds, kv, part, r0, nr, h0, hn, my_seq, my_pos, sub, a.split);
    } else {
        const Runs runs = runs_of(c, my_seq, my_pos, nr);
        if (__popcll(runs.starts) == 1 && __popcll(runs.valid) * hn > 16) {
            if (sub == 0) wide<NQ, NV, NT>(a, lds.wide, kv, r0, nr, h0, hn, my_seq, my_pos, runs);
            return;
        }
        const int chunks = (hn + 15) / 16, rc = min(hn, 16), tt = 16 / rc;
        const int r1 = sub / chunks * tt, h1 = sub % chunks * 16;
        if (r1 >= nr) return;
        const int n1 = min(tt, nr - r1), from = r1 + min(lane, n1 - 1);
        narrow<NQ, NV, EX>(a, lds.narrow, kv, 0, r0 + r1, n1, h0 + h1, min(rc, hn - h1), __shfl(my_seq, from, 64), __shfl(my_pos, from, 64),
                           0, 1);
    }
}

// The parts of rows whose tiles several blocks shared: a block of T threads
// per (row, head), each group of vd / 4 of them every so many-th part; the
// groups' sums in order.
template <int T>
__global__ __launch_bounds__(T) void kv8_join_kernel(const Args a) {
    __shared__ float w[256], red;
    __shared__ f32x4 sums[T];
    const int vd = a.c.vd, row = blockIdx.x / a.heads, head = blockIdx.x % a.heads, i = threadIdx.x;
    if (a.pos[row] < 0 || (unsigned)a.seq[row] >= (unsigned)a.c.n_seq) return;
    const float *ml = a.part_ml + (int64_t)blockIdx.x * a.ps * 3, *part = a.part + (int64_t)blockIdx.x * a.ps * vd;
    if (i < 64) {
        float m = kNone, e = -INFINITY, l = 0.0f, pm[4], pl[4], pe[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int p = i + 64 * k;
            pm[k] = p < a.ps ? gload(ml + 3 * p) : kNone, pl[k] = p < a.ps ? gload(ml + 3 * p + 1) : 0.0f;
            pe[k] = p < a.ps ? gload(ml + 3 * p + 2) : 0.0f;
            m = fmaxf(m, pm[k]);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
        for (int k = 0; k < 4; k++) {
            pe[k] += pm[k] - m, e = fmaxf(e, pe[k]);
            l += pl[k] * __builtin_amdgcn_exp2f(pm[k] - m);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) e = fmaxf(e, __shfl_xor(e, o, 64)), l += __shfl_xor(l, o, 64);
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i + 64 * k < a.ps) w[i + 64 * k] = __builtin_amdgcn_exp2f(pe[k] - e);
        if (i == 0) red = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(e) / l;
    }
    __syncthreads();
    const int n = vd / 4, groups = T / n, g = i / n, at = i % n;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (g < groups)
        for (int p = g; p < a.ps; p += groups) {
            const f32x4 x = gload((const f32x4 *)(part + (int64_t)p * vd) + at);
#pragma unroll
            for (int k = 0; k < 4; k++) acc[k] = fmaf(x[k], w[p], acc[k]);
        }
    sums[i] = acc;
    __syncthreads();
    if (i >= n) return;
    for (int k = 1; k < groups; k++) acc += sums[k * n + i];
    float *dst = a.out + (int64_t)row * a.out_stride + (int64_t)head * vd + 4 * i;
#pragma unroll
    for (int k = 0; k < 4; k++) dst[k] = acc[k] * red;
}

// How a call is cut up: see Args.
struct Plan {
    int cols, rc, chunks, tt, groups, split, ps;  // cols: columns of a block
    uint64_t bytes;
};

Plan plan_of(const Kv8 &c, int rows, int heads, int max_pos, int window) {
    Plan p{};
    const int rep = heads / c.n_kv;
    const long long wide = ((long long)rows * rep + 63) / 64 * c.n_kv;
    // Blocks of 64 columns share what they load, but are a quarter as many (us with
    // 16 columns and with 64): 32 heads over 8 of 128, 450 rows (225 blocks of 64)
    // 17.4 and 20.2, 600 (300) 25.3 and 24.0, 850 35.3 and 31.3, 1000 40.6 and 34.4;
    // 16 of 192/128, one tile a step, 2100 rows (528) 69 and 75, 2600 (656) 92 and 89,
    // 3200 126 and 119; 8 over 2 of 64, 6000 (750) 115 and 119, 8000 (1000) 190 and
    // 182.  Widths that count their operands at run time lose (96 dims, 12000 rows of
    // 6 heads over 2 511 and 558).
    const int from = c.qd == 128 && c.vd == 128 ? 280 : c.qd == 192 && c.vd == 128 ? 640 : c.qd == 64 && c.vd == 64 ? 900 : 0;
    p.cols = from && wide >= from ? 64 : 16;
    p.rc = std::min(rep, p.cols);
    p.chunks = (rep + p.rc - 1) / p.rc;
    p.tt = p.cols / p.rc;
    p.groups = (int)(((long long)rows + p.tt - 1) / p.tt);
    const long long base = (long long)p.groups * p.chunks * c.n_kv;
    const int narrow = std::min(p.rc, 16);  // query heads of a group of 16 columns
    p.split = p.cols == 64 ? (p.tt + 16 / narrow - 1) / (16 / narrow) * ((p.rc + 15) / 16)
                           : (int)std::max<long long>(1, std::min<long long>(p.tt, 1024 / base));
    const long long tiles = (window > 0 ? std::min((long long)window + p.tt, (long long)max_pos + 1) : max_pos + 1LL) / 64 + 1;
    const long long units = base * p.split;
    const long long ps = p.cols == 64   ? 1
                         : units >= 256 ? std::min((512 + units - 1) / units, tiles / 32)
                         : tiles < 24   ? 1
                                        : std::min<long long>({(1024 + units - 1) / units, tiles / 6, 256});
    p.ps = (int)std::max<long long>(1, ps);
    p.bytes = p.ps > 1 ? (uint64_t)rows * heads * p.ps * (c.vd + 3) * 4 : 0;
    return p;
}

constexpr long long kMostThreads = 0xffffffffll;  // of a launch

template <int NQ, int NV, bool EX, int NT>
void launch(const Args &a, hipStream_t s) {
    const long long blocks = (long long)a.groups * a.split * a.ps * a.chunks * a.c.n_kv;
    hipLaunchKernelGGL((kv8_attention_kernel<NQ, NV, EX, NT>), dim3((unsigned)blocks), dim3(256), 0, s, a);
}
template <int NQ, int NV, bool EX, int NT>
void launch(const Args &a, bool wide, hipStream_t s) {
    wide ? launch<NQ, NV, EX, NT>(a, s) : launch<NQ, NV, EX, 0>(a, s);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv8_attention_workspace_size(const moe_kv8 *c, int32_t rows, int32_t heads, int32_t max_pos, int32_t window,
                                     uint64_t *bytes) {
    Kv8 a;
    if (const int rc = kv8_of("moe_kv8_attention_workspace_size", c, &a)) return rc;
    if (!bytes || rows < 0 || heads <= 0 || heads % a.n_kv || max_pos < 0 || max_pos >= (int64_t)a.max_pages << a.page_shift)
        return fail(MOE_EINVAL, "moe_kv8_attention_workspace_size: bad argument (%d rows, %d heads over %d, max position %d"
                    " of %lld)", rows, heads, a.n_kv, max_pos, (long long)a.max_pages << a.page_shift);
    *bytes = rows ? plan_of(a, rows, heads, max_pos, window).bytes : 0;
    return MOE_OK;
}

int moe_kv8_attention(const moe_kv8 *c, const float *q, int64_t q_stride, int32_t rows, int32_t heads, float scale,
                      const int32_t *seq, const int32_t *pos, int32_t max_pos, int32_t window, float *out,
                      int64_t out_stride, void *workspace, uint64_t workspace_bytes, void *stream) {
    Args a{};
    if (const int rc = kv8_of("moe_kv8_attention", c, &a.c)) return rc;
    if ((rows > 0 && (!q || !seq || !pos || !out)) || rows < 0 || heads <= 0 || heads % a.c.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.c.max_pages << a.c.page_shift)
        return fail(MOE_EINVAL, "moe_kv8_attention: bad argument (%d rows, %d heads over %d, max position %d of %lld)", rows,
                    heads, a.c.n_kv, max_pos, (long long)a.c.max_pages << a.c.page_shift);
    if (rows == 0) return MOE_OK;
    const Plan p = plan_of(a.c, rows, heads, max_pos, window);
    if (p.bytes && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < p.bytes))
        return fail(MOE_EINVAL, "moe_kv8_attention: workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)p.bytes);
    a.q = q, a.seq = seq, a.pos = pos, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.rows = rows, a.heads = heads, a.rep = heads / a.c.n_kv, a.window = window, a.scale = scale;
    a.tt = p.tt, a.groups = p.groups, a.rc = p.rc, a.chunks = p.chunks, a.split = p.split, a.ps = p.ps;
    a.part = static_cast<float *>(workspace);
    a.part_ml = a.part + (size_t)rows * heads * p.ps * a.c.vd;
    if ((long long)a.groups * a.split * a.ps * a.chunks * a.c.n_kv > kMostThreads / 256)
        return fail(MOE_EUNSUP, "moe_kv8_attention: %d rows of %d heads are too many blocks", rows, heads);
    hipStream_t s = (hipStream_t)stream;
    const int qd = a.c.qd, vd = a.c.vd;
    // Widths of their own: a power-of-two head and the latent cache's 192/128;
    // the others count their operands at run time.
    const bool wide = p.cols == 64;
    if (qd == 64 && vd == 64) launch<1, 4, true, 2>(a, wide, s);
    else if (qd == 128 && vd == 128) launch<2, 8, true, 2>(a, wide, s);
    else if (qd == 192 && vd == 128) launch<3, 8, true, 1>(a, wide, s);
    else if (qd <= 192 && vd <= 128) launch<3, 8, false, 0>(a, s);
    else if (qd == 256 && vd == 256) launch<4, 16, true, 0>(a, s);
    else launch<4, 16, false, 0>(a, s);
    if (a.ps > 16) hipLaunchKernelGGL((kv8_join_kernel<256>), dim3((unsigned)rows * heads), dim3(256), 0, s, a);
    else if (a.ps > 1) hipLaunchKernelGGL((kv8_join_kernel<64>), dim3((unsigned)rows * heads), dim3(64), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "8-bit attention kernel: %s", hipGetErrorString(e));
}

}  // extern "C"
