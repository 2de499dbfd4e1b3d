// kv4_attention.hip — causal attention over the paged 4-bit cache
// (moe_kv4_attention), layout in kv4.h.
//
// Rows find their sequence and position on the device, so one kernel serves
// decode steps, prompts and chunks.  A block takes a group of consecutive rows
// and one kv head, splits the group into runs of one sequence and makes each
// run's (row, query head) pairs the 16 or 64 columns of its products on the
// f16 matrix cores; its waves (and, where there are few rows, several blocks)
// split the run's tiles of 32 positions and merge at the end.
//
// A code minus 8 is exact in f16, and a block of 32 dims is one step of the
// 16x16x32 instruction, so nothing is dequantised: per block of a key
//   S^T += d_k (C Q_hi^T + C Q_lo^T)
// with q scale log2(e) 2^k in two f16 pieces (22 bits of the row's largest
// value) and the block's scale applied to the f32 sum.  The result's layout
// (lane = column, positions 4g.. of both halves) is the B operand of the
// second product, whose sum runs over positions with a scale each:
//   O^T += C (P d_v)_hi + C (P d_v)_lo
// The weights P = 2^(s - ref) are kept so large that two f16 pieces hold
// their products with the scales to 2^-34 of the largest: ref = m + E - 9 with
// m a running maximum (it moves when a score exceeds it by 6) and 2^E above
// every value scale seen, so P d_v stays below 2^15 and mostly above 2^-10.
// Sums are f32; the two pieces' rounding is 2^-22, as f32 dot products' own.
// Where all value scales of a wave's tiles lie within 2^8 of each other, the
// position of weight 2^9 and more alone makes every block's sum 2 or more, of
// which what the pieces leave is less than 2^-22 (2^-25 a product).  Where they
// do not (a block of small values beside large ones, a far larger value that
// hardly weighs, a 0 that takes all weight), the wave goes over its tiles once
// more with the references it has found and four pieces: a block's precision
// is then its own down to 2^-70 of the largest product.  (One block of four
// 2^-12 of the others: 32-sequence decode 28 -> 53 us, 64 x 12000 164 -> 354,
// prompt of 2000 rows 134 -> 299, one row at 100001 37 -> 66.)
//
// Decode reads the cache once and is bound by it: 64 sequences of 6000 to 12000
// positions, 8 kv heads of 128, 152 us (4.4 TB/s of tiles); 32 sequences of up to
// 1200 with 16 heads of 192/128 28 (3 TB/s: all blocks resident at once, two a
// CU, with 19 to 38 tiles, so the longest sets the time; beside them a start, in
// which each block of a group loads and stages the group's 16 queries, and a
// merge); one sequence of 100001 positions in 256 parts 32 + 5.5 for the joining
// launch.  Prompts are bound by nothing alone: a wave issues in 45% of its time,
// waits for loads and LDS in 29% and to be issued in 26%, at 1.5 waves a SIMD
// (256 registers, 35 spilled); vector instructions, 9.4 to a product (scaling
// block by block, exponentials, the weights' two pieces), are issued in 52% of
// the cycles, the matrix pipe is busy in 19%.  2000 rows of 32 heads of 128 113 us
// in a loop, 130 alone (290 and 252 TFLOP/s of the attention's own operations),
// 8000 rows 390 TFLOP/s, against 1200 of a large f16 product.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_dw __attribute__((ext_vector_type(4), aligned(4)));  // at any float
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

struct Args {
    Kv4 c;
    const float *q;
    const int32_t *seq, *pos, *lists;
    float *out, *part, *part_ml;  // part [row][head][ps][vd], part_ml [row][head][ps][2]
    int64_t q_stride, out_stride;
    int rows, heads, rep, window, n_sel;
    float scale;
    int tt, groups;  // rows of a group, groups
    int rc, chunks;  // query heads of a block, blocks that share a kv head's
    int split;       // blocks that share a group's runs (of 64 columns: its groups of 16)
    int ps;          // blocks that share a run's tiles
};

__device__ inline half2v as_h2(uint32_t v) { return __builtin_bit_cast(half2v, v); }

// Constants the compiler may not fold: (w & mask) | one is then one
// instruction (v_and_or_b32 takes no literal, and one scalar register).
struct Nibbles {
    uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, lo1 = 0x64006400u, hi1 = 0x54005400u;
    __device__ Nibbles() { asm("" : "+s"(lo), "+s"(hi), "+v"(lo1), "+v"(hi1)); }
};

// Codes minus 8 as f16 pairs, from the low or high nibbles of bytes 0 and 2: a
// nibble becomes the low mantissa bits of 1024 (or, four bits up, of 64); the
// subtraction is exact.
__device__ inline half2v low_pair(uint32_t w, const Nibbles &n) {
    return as_h2((w & n.lo) | n.lo1) - half2v{(_Float16)1032.0f, (_Float16)1032.0f};
}
__device__ inline half2v high_pair(uint32_t w, const Nibbles &n) {
    return as_h2((w & n.hi) | n.hi1) - half2v{(_Float16)72.0f, (_Float16)72.0f};
}
__device__ inline half8 join8(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// f16 operands of f32 multiply-adds are read as they lie in half a register
// (v_fma_mix_f32), which the compiler chooses for fmaf of a widened f16; so a
// product is written as a multiply-add of 0 and a difference as one of -1,
// the -1 hidden from it.
__device__ inline float minus_one() {
    float m = -1.0f;
    asm("" : "+s"(m));
    return m;
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ inline half2v pack_half(float a, float b) { return __builtin_convertvector((f32x2{a, b}), half2v); }

// Lanes of a wave hand each other values through LDS: its LDS operations run in
// order, so only the compiler has to keep them so.
__device__ inline void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A tile's words of a lane.
template <int QC, int VC>
struct Tile {
    static constexpr int NS = (QC + VC + 3) / 4;
    uint32_t k[2 * QC], v[2 * VC], s[NS];
    int base;  // position of its first row
    int ok;    // whether there is such a tile
};

// Loads of a tile go through a buffer descriptor: its base is the wave's, in
// scalar registers, and a lane's offset the same for every tile, so that a
// tile's loads need no vector address (temporaries of which made the loop wait
// for loads in flight).  Reads past `bytes` give 0.
__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, bytes, 0x00020000);
}

template <int NB, bool EX>
__device__ inline void load_words(uint32_t (&w)[2 * NB], __amdgpu_buffer_rsrc_t buf, int at, int nb, int lane) {
#pragma unroll
    for (int c = 0; c < (NB + 1) / 2; c++) {
        if (EX ? 2 * c + 2 <= NB : 2 * c + 2 <= nb) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(buf, 16 * lane, at + 1024 * c, 0);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * c + i < 2 * NB) w[4 * c + i] = x[i];
        } else if (EX || 2 * c < nb) {
            const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(buf, 8 * lane, at + 1024 * c, 0);
            w[4 * c] = x[0], w[4 * c + 1] = x[1];
        }
    }
}

// What a block shares.
template <int QC, int VC, int C, int S, int W>
struct Lds {
    u32x4 sq_[S * C * QC * 2 * 64];  // Q operands: [column tile][block][hi, lo][lane]
    f32x4 smo[W * VC * 2 * 64];      // O of the waves: [wave][block][half][lane]
    uint32_t ssc[W][Tile<QC, VC>::NS * 64];
    float sm_r[W][C * 16], sm_l[W][C * 16], sm_k[S * C * 16];
};

// Lanes of my_seq and my_pos that begin a run of one sequence's rows or are
// none; the runs' first lanes.
struct Runs {
    unsigned long long cuts, starts, valid;
};
__device__ inline Runs runs_of(const Kv4 &c, int my_seq, int my_pos, int nr) {
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

// A block's work: rows r0 .. r0 + nr - 1 (whose sequences and positions the
// lanes hold), heads h0 .. h0 + hn - 1; of the rows' runs every split-th from
// `sub` on, of their tiles the part-th part.
// QC, VC: blocks of a key and a value (EX) or the most there may be.  C:
// 16-column tiles of a wave.  W waves: S sets of columns, W / S parts of the
// positions.
template <int QC, int VC, bool EX, int C, int S, int W>
__device__ __attribute__((always_inline)) inline void attend(const Args &a, Lds<QC, VC, C, S, W> &lds, int kv, int part, int r0,
                                                             int nr, int h0, int hn, int my_seq, int my_pos, int sub,
                                                             int split) {
    typedef Tile<QC, VC> T;
    constexpr int P = W / S;
    auto &sq_ = lds.sq_;
    auto &smo = lds.smo;
    auto &ssc = lds.ssc;
    auto &sm_r = lds.sm_r, &sm_l = lds.sm_l;
    auto &sm_k = lds.sm_k;
    const Kv4 &kc = a.c;
    const Nibbles nib;
    const float less = minus_one();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, set = wave % S, share = wave / S;
    const int nq = EX ? QC : kc.qd / 32, nv = EX ? VC : kc.vd / 32;
    // Column cc of the block is query head h0 + cc % hn of row r0 + cc / hn,
    // whatever run it is in: queries load while sequences and tables do.  16
    // threads a column, four values each at a time.
    constexpr int kPer = (QC + 1) / 2, kCols = S * C * 16 / (W * 4);
    f32x4 qv[kCols][kPer];
    const int qi = threadIdx.x & 15;
#pragma unroll
    for (int k = 0; k < kCols; k++) {
        const int cc = min((int)(threadIdx.x >> 4) + k * W * 4, nr * hn - 1);
        const float *row = a.q + (size_t)(r0 + cc / hn) * a.q_stride + (size_t)(h0 + cc % hn) * kc.qd;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int d = min(4 * qi + 64 * j, kc.qd - 4);
            qv[k][j] = __builtin_bit_cast(f32x4, gload_x4((const uint32_t *)(row + d)));
        }
    }
    const Runs runs = runs_of(kc, my_seq, my_pos, nr);
    const unsigned long long cuts = runs.cuts;
    unsigned long long starts = runs.starts;
    const int tshift = kc.page_shift - 5;
    bool staged = false;

    for (int run = 0; starts; run++) {
        const int first = __builtin_ctzll(starts);
        starts &= starts - 1;
        if (run % split != sub) continue;
        const unsigned long long after = first < 63 ? cuts >> (first + 1) : 0;
        const int end = min(nr, after ? first + 1 + __builtin_ctzll(after) : 64);
        const bool mine = lane >= first && lane < end;
        int hi = mine ? my_pos : -1;
        int lo = mine ? (a.window > 0 ? max(0, my_pos + 1 - a.window) : 0) : 0x7fffffff;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            hi = max(hi, __shfl_xor(hi, o, 64));
            lo = min(lo, __shfl_xor(lo, o, 64));
        }
        hi = __builtin_amdgcn_readfirstlane(hi);
        lo = __builtin_amdgcn_readfirstlane(lo);
        const int sq = __builtin_amdgcn_readlane(my_seq, first);
        // The run's columns, and what each sees.  A run of few columns has them
        // several times over, one copy for each block of a value: see `second`.
        const int c0 = first * hn, ncol = end * hn - c0;
        const int wide = ncol > 1 ? 32 - __builtin_clz(ncol - 1) : 0;  // log2 of the columns' room
        const bool copies = C == 1 && nv << wide <= 16;
        int cc[C], cp[C], cl[C];
        bool cv[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int x = copies ? col & ((1 << wide) - 1) : (set * C + c) * 16 + col - c0;
            cv[c] = x >= 0 && x < ncol;
            cc[c] = c0 + (cv[c] ? x : 0);
            cp[c] = __shfl(my_pos, cc[c] / hn, 64);
            cl[c] = a.window > 0 ? max(0, cp[c] + 1 - a.window) : 0;
        }
        const int copy = copies ? min(col >> wide, nv - 1) : 0;

        // This wave's tiles: v0 .. v1 - 1 of the run's (of the lists' pages).
        const int t0 = a.lists ? 0 : lo >> 5;
        const int nt = a.lists ? a.n_sel << tshift : (hi >> 5) - t0 + 1;
        const int parts = a.ps * P, me = part * P + share;
        const int v0 = (int)((long long)nt * me / parts);
        int v = v0;
        const int v1 = (int)((long long)nt * (me + 1) / parts);
        const int32_t *list = a.lists ? a.lists + ((size_t)(r0 + first) * kc.n_kv + kv) * a.n_sel : nullptr;
        const int32_t *table = kc.table + (size_t)sq * kc.max_pages;
        // Pages b0 .. b0 + 63 of the run, one a lane: first position (-1: no
        // such page) and where the kv head's tiles are.
        int b0 = -64, my_base = -1;
        uint32_t my_at[2] = {0, 0};
        const uint8_t *at = kc.pool;
        // Find tile v, and queue its loads.  Control and addresses are the wave's,
        // and the loads unconditional (where there is no such tile, those of the
        // one before again), so that waiting for one tile leaves the next in
        // flight.
        auto find = [&](T &x) __attribute__((always_inline)) {
            x.ok = 0;
            if (v < v1) {
                const int t = t0 + v, i = t >> tshift;
                if (i >= b0 + 64 || i < b0) {
                    b0 = i;
                    const int j = b0 + lane;
                    int page = j;
                    bool there = true;
                    if (list) {
                        page = j < a.n_sel ? gload(list + j) : -1;
                        const int prev = j > 0 && j <= a.n_sel ? gload(list + j - 1) : -1;
                        there = page > prev;
                    }
                    there = there && page >= 0 && page < kc.max_pages;
                    const int pid = there ? gload(table + page) : -1;
                    there = (unsigned)pid < (unsigned)kc.n_pages;
                    my_base = there ? page << kc.page_shift : -1;
                    const uint64_t p = (uint64_t)kc.head(there ? pid : 0, kv);
                    my_at[0] = (uint32_t)p, my_at[1] = (uint32_t)(p >> 32);
                    asm volatile("" : "+v"(my_base), "+v"(my_at[0]), "+v"(my_at[1]));  // waited for here, not at every tile
                }
                const int in = t & ((1 << tshift) - 1), page = __builtin_amdgcn_readlane(my_base, i - b0);
                x.base = page + in * kTile;
                if (page >= 0 && x.base <= hi && x.base + kTile > lo) {
                    x.ok = 1;
                    const uint64_t p = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(my_at[1], i - b0) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane(my_at[0], i - b0);
                    at = (const uint8_t *)p + (uint32_t)(in * kc.tile_bytes);
                }
            }
            v++;
        };
        auto load_keys = [&](T &x) __attribute__((always_inline)) {
            const __amdgpu_buffer_rsrc_t buf = buffer_of(at, kc.tile_bytes);
#pragma unroll
            for (int e = 0; e < T::NS; e++)
                x.s[e] = __builtin_amdgcn_raw_buffer_load_b32(buf, 4 * lane, kc.k_scales() + 256 * e, 0);
            load_words<QC, EX>(x.k, buf, 0, nq, lane);
        };
        auto load_values = [&](T &x) __attribute__((always_inline)) {
            load_words<VC, EX>(x.v, buffer_of(at, kc.tile_bytes), kc.v_codes(), nv, lane);
        };
        auto load = [&](T &x) __attribute__((always_inline)) {
            find(x);
            load_keys(x);
            load_values(x);
        };
        T x, y;
        const bool any = v < v1;
        if (any) load(x);

        // Q into LDS, once: a column's values times scale log2(e), by a power of
        // two that brings its largest into [2^14, 2^15), in two f16 pieces.
        if (!staged) {
            staged = true;
            const float f = a.scale * 1.44269504f;
#pragma unroll
            for (int k = 0; k < kCols; k++) {
                const int cc = (threadIdx.x >> 4) + k * W * 4;
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < kPer; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) qv[k][j][e] *= f, top = fmaxf(top, fabsf(qv[k][j][e]));
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
                // 2^(14 - exponent of top), within what both it and its inverse can be.
                const int ex = min(max(127 + 14 - ((int)(__float_as_uint(top) >> 23) - 127), 1), 253);
                const float up = __uint_as_float((uint32_t)ex << 23);
                if (qi == 0) sm_k[cc] = __uint_as_float((uint32_t)(254 - ex) << 23);
#pragma unroll
                for (int j = 0; j < kPer; j++) {
                    const int d = 4 * qi + 64 * j;
                    if (d >= kc.qd) continue;
                    // Dims 32 s + 16 h + 4 g + 0, 2, 1, 3 are elements 4 h.. of lane (g, column).
                    const f32x4 z = qv[k][j] * up;
                    const half2v h0 = pack_half(z[0], z[2]), h1 = pack_half(z[1], z[3]);
                    const half2v l0 = pack_half(z[0] - (float)h0[0], z[2] - (float)h0[1]);
                    const half2v l1 = pack_half(z[1] - (float)h1[0], z[3] - (float)h1[1]);
                    u32x2 *dst = (u32x2 *)(sq_ + ((cc >> 4) * QC + (d >> 5)) * 2 * 64 + (d >> 2 & 3) * 16 + (cc & 15)) + (d >> 4 & 1);
                    dst[0] = u32x2{__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)};
                    dst[128] = u32x2{__builtin_bit_cast(uint32_t, l0), __builtin_bit_cast(uint32_t, l1)};
                }
            }
            __syncthreads();
        }
        float ck[C];
#pragma unroll
        for (int c = 0; c < C; c++) ck[c] = sm_k[C == 1 ? cc[0] : (set * C + c) * 16 + col];
        const int ql_at = C == 1 ? g * 16 + cc[0] : lane;

        f32x4 o[C][VC][2];
        float ref[C], lim[C], l[C];
        int E = -24;
        int low = 0x7c00;  // the smallest value scale seen (f16 bits), of this lane's
#pragma unroll
        for (int c = 0; c < C; c++) {
            ref[c] = 0.0f, lim[c] = -INFINITY, l[c] = 0.0f;
#pragma unroll
            for (int b = 0; b < VC; b++) o[c][b][0] = o[c][b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // O^T += the tile's values times the weights p.  A block of a value has
        // its own scales, so its own products of weights and scales: 24
        // instructions a column tile.  With `once` copy k of the columns takes
        // block k's scales, all blocks' products are made at once, and of what
        // comes out only copy b's columns of block b are read.
        auto second = [&](const T &x, const f32x4 (&p)[C][2], auto once) __attribute__((always_inline)) {
            const u32x4 *sc = (const u32x4 *)ssc[wave];
            half8 h8[C], l8[C], w0, w1;
            // Weights times scales in the codes' order, bytes 0, 2, 1, 3 of
            // each half; both pieces.
            auto scaled = [&](const u32x4 &ds) __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < C; c++) {
                    half2v ph[4], pl[4];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const half2v d0 = as_h2(ds[2 * h]), d1 = as_h2(ds[2 * h + 1]);
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float u = fmaf((float)d0[e], p[c][h][e], 0.0f), w = fmaf((float)d1[e], p[c][h][2 + e], 0.0f);
                            const half2v z = pack_half(u, w);
                            ph[2 * h + e] = z;
                            pl[2 * h + e] = pack_half(fmaf((float)z[0], less, u), fmaf((float)z[1], less, w));
                        }
                    }
                    h8[c] = join8(ph[0], ph[1], ph[2], ph[3]), l8[c] = join8(pl[0], pl[1], pl[2], pl[3]);
                }
            };
            auto unpack = [&](int b) __attribute__((always_inline)) {
                const uint32_t y0 = x.v[2 * b], y1 = x.v[2 * b + 1];
                w0 = join8(low_pair(y0, nib), low_pair(y0 >> 8, nib), low_pair(y1, nib), low_pair(y1 >> 8, nib));
                w1 = join8(high_pair(y0, nib), high_pair(y0 >> 8, nib), high_pair(y1, nib), high_pair(y1 >> 8, nib));
            };
            scaled(sc[(nq + (once ? copy : 0)) * 4 + g]);
            u32x4 ds = sc[(nq + min(1, nv - 1)) * 4 + g];  // the next block's, read one ahead
            unpack(0);
#pragma unroll
            for (int b = 0; b < VC; b++) {
                if (!EX && b >= nv) continue;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    o[c][b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w0, h8[c], o[c][b][0], 0, 0, 0);
                    o[c][b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w1, h8[c], o[c][b][1], 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < C; c++) {
                    o[c][b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w0, l8[c], o[c][b][0], 0, 0, 0);
                    o[c][b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w1, l8[c], o[c][b][1], 0, 0, 0);
                }
                // The next block's operands while these products run.
                if (b + 1 < VC && (EX || b + 1 < nv)) {
                    unpack(b + 1);
                    if (!once) {
                        const u32x4 y = ds;
                        if (b + 2 < VC && (EX || b + 2 < nv)) ds = sc[(nq + b + 2) * 4 + g];
                        scaled(y);
                    }
                }
                if (C > 1) __builtin_amdgcn_sched_barrier(0);
            }
        };
        // O^T += what second()'s two pieces leave of products below 1: steps of
        // 2^-24 are all that f16 has there.  In two pieces again, 2^39 times as
        // large, and through sums of their own.
        auto rest = [&](const T &x, const f32x4 (&p)[C][2], auto once) __attribute__((always_inline)) {
            const u32x4 *sc = (const u32x4 *)ssc[wave];
#pragma unroll
            for (int c = 0; c < C; c++) {
                half8 h8, l8;
#pragma unroll
                for (int b = 0; b < VC; b++) {
                    if (!EX && b >= nv) continue;
                    if (!once || b == 0) {
                        const u32x4 ds = sc[(nq + (once ? copy : b)) * 4 + g];
                        half2v ph[4], pl[4];
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                // (as second() has them)
                                const float u0 = fmaf((float)as_h2(ds[2 * h])[e], p[c][h][e], 0.0f);
                                const float u1 = fmaf((float)as_h2(ds[2 * h + 1])[e], p[c][h][2 + e], 0.0f);
                                const half2v a = pack_half(u0, u1);
                                const float v0 = u0 - (float)a[0], v1 = u1 - (float)a[1];
                                const half2v b = pack_half(v0, v1);
                                const float r0 = fabsf(u0) < 1.0f ? (v0 - (float)b[0]) * 0x1p39f : 0.0f;
                                const float r1 = fabsf(u1) < 1.0f ? (v1 - (float)b[1]) * 0x1p39f : 0.0f;
                                const half2v z = pack_half(r0, r1);
                                ph[2 * h + e] = z;
                                pl[2 * h + e] = pack_half(r0 - (float)z[0], r1 - (float)z[1]);
                            }
                        h8 = join8(ph[0], ph[1], ph[2], ph[3]), l8 = join8(pl[0], pl[1], pl[2], pl[3]);
                    }
                    const uint32_t y0 = x.v[2 * b], y1 = x.v[2 * b + 1];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const half8 w = h ? join8(high_pair(y0, nib), high_pair(y0 >> 8, nib), high_pair(y1, nib), high_pair(y1 >> 8, nib))
                                          : join8(low_pair(y0, nib), low_pair(y0 >> 8, nib), low_pair(y1, nib), low_pair(y1 >> 8, nib));
                        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
                        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, h8, r, 0, 0, 0);
                        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, l8, r, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; i++) o[c][b][h][i] = fmaf(r[i], 0x1p-39f, o[c][b][h][i]);
                    }
                }
            }
        };
        // between(): what to do when the keys' words have been read.  again: with
        // the references that a walk before has found.
        auto step = [&](const T &x, int base, auto once, auto again, auto between) __attribute__((always_inline)) {
            // Scales through LDS (the wave's own: in order, no barrier): every
            // lane reads its four positions of both halves, 16 bytes.
            lds_order();  // the reads of the tile before
            u16x2 top = {0, 0}, least = {0x7fff, 0x7fff};  // of the lane's value scales, f16 bits
#pragma unroll
            for (int e = 0; e < T::NS; e++) {
                ssc[wave][lane + 64 * e] = x.s[e];
                const int at = lane + 64 * e;
                const bool value = at >= nq * 16 && at < (nq + nv) * 16;
                const uint32_t y = x.s[e] & 0x7fff7fffu;
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, value ? y : 0u));
                least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, value ? y : 0x7fff7fffu));
            }
            const bool inf = __any(max(top[0], top[1]) >= 0x7c00);
            if (__builtin_expect(inf || base < lo || base + kTile - 1 > hi, 0)) {
                // Finite ones of positions that the run sees: what lies in a
                // page's rest or before the window must not set the weights'
                // power of two.  A lane's pair of scales is the same two positions
                // in every block.
                const int w = 2 * col, p = base + 4 * (w >> 3) + 16 * (w >> 2 & 1) + (w & 3);
                top = u16x2{0, 0}, least = u16x2{0x7fff, 0x7fff};
#pragma unroll
                for (int e = 0; e < T::NS; e++) {
                    const int at = lane + 64 * e;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint16_t y = x.s[e] >> (16 * k) & 0x7fff;
                        if (at < nq * 16 || at >= (nq + nv) * 16 || y >= 0x7c00 || p + k < lo || p + k > hi) continue;
                        top[k] = max(top[k], y), least[k] = min(least[k], y);
                    }
                }
            }
            const int most = max(top[0], top[1]);
            low = min(low, (int)min(least[0], least[1]));
            lds_order();
            const u32x4 *sc = (const u32x4 *)ssc[wave];
            f32x4 s[C][2];
#pragma unroll
            for (int c = 0; c < C; c++) s[c][0] = s[c][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            // A block's sums are scaled while the next block's products run.
            half8 dp;
            f32x4 rp[C][2];
            auto scale = [&] __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s[c][0][i] = fmaf((float)dp[i], rp[c][0][i], s[c][0][i]);
                        s[c][1][i] = fmaf((float)dp[4 + i], rp[c][1][i], s[c][1][i]);
                    }
            };
            // (reads of LDS one block ahead)
            u32x4 qn[C][2], dn;
            auto operands = [&](int b) __attribute__((always_inline)) {
                dn = sc[b * 4 + g];
#pragma unroll
                for (int c = 0; c < C; c++) {
                    qn[c][0] = sq_[(((set * C + c) * QC + b) * 2 + 1) * 64 + ql_at];
                    qn[c][1] = sq_[(((set * C + c) * QC + b) * 2) * 64 + ql_at];
                }
            };
            operands(0);
#pragma unroll
            for (int b = 0; b < QC; b++) {
                if (!EX && b >= nq) continue;
                const half8 d = __builtin_bit_cast(half8, dn);
                u32x4 q[C][2];
#pragma unroll
                for (int c = 0; c < C; c++) q[c][0] = qn[c][0], q[c][1] = qn[c][1];
                if (b + 1 < QC && (EX || b + 1 < nq)) operands(b + 1);
                const uint32_t w0 = x.k[2 * b], w1 = x.k[2 * b + 1];
                const half8 k0 = join8(low_pair(w0, nib), low_pair(w0 >> 8, nib), high_pair(w0, nib), high_pair(w0 >> 8, nib));
                const half8 k1 = join8(low_pair(w1, nib), low_pair(w1 >> 8, nib), high_pair(w1, nib), high_pair(w1 >> 8, nib));
                f32x4 r[C][2];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        const half8 qq = __builtin_bit_cast(half8, q[c][i]);
                        const f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                        r[c][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qq, i ? r[c][0] : z, 0, 0, 0);
                        r[c][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qq, i ? r[c][1] : z, 0, 0, 0);
                    }
                if (b > 0) scale();
                dp = d;
#pragma unroll
                for (int c = 0; c < C; c++) rp[c][0] = r[c][0], rp[c][1] = r[c][1];
                if (C > 1) __builtin_amdgcn_sched_barrier(0);
            }
            scale();
            between();
            // Positions a column does not see.
            bool some = false;
#pragma unroll
            for (int c = 0; c < C; c++) some |= cv[c] && (base < cl[c] || base + kTile - 1 > cp[c]);
            if (__any(some)) {
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int at = base + (i >> 2) * 16 + 4 * g + (i & 3);
                        if (at < cl[c] || at > cp[c]) s[c][i >> 2][i & 3] = -INFINITY;
                    }
            }
            // The references move: a score too far above, or a larger scale.
            float mx[C];
            bool move = false;
#pragma unroll
            for (int c = 0; c < C; c++) {
                mx[c] = s[c][0][0];
#pragma unroll
                for (int i = 1; i < 8; i++) mx[c] = fmaxf(mx[c], s[c][i >> 2][i & 3]);
                mx[c] *= ck[c];
                move |= mx[c] > lim[c];
            }
            const bool grow = (most >> 10) - 14 > E;  // not below 2^E
            if (!again && __any(move || grow)) {
                int ne = (most >> 10) - 14;
#pragma unroll
                for (int w = 32; w >= 1; w >>= 1) ne = max(ne, __shfl_xor(ne, w, 64));
                ne = max(ne, E);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    float y = fmaxf(mx[c], __shfl_xor(mx[c], 16, 64));
                    y = fmaxf(y, __shfl_xor(y, 32, 64));
                    const float m = lim[c] - 6.0f;
                    const float mn = y > lim[c] ? y : m;
                    const float nref = mn == -INFINITY ? 0.0f : mn + (float)(ne - 9);
                    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref[c] - nref);
                    lim[c] = mn + 6.0f, ref[c] = nref;
                    l[c] *= f;
#pragma unroll
                    for (int b = 0; b < VC; b++) o[c][b][0] *= f, o[c][b][1] *= f;
                }
                E = __builtin_amdgcn_readfirstlane(ne);
            }
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[c][i >> 2][i & 3], ck[c], -ref[c]));
                    s[c][i >> 2][i & 3] = p;
                    l[c] += p;
                }
            // Scales that are infinite or NaN (rare): positions of weight 0 may
            // hold them, so they become 0, and what a column does see of them
            // makes the block's 32 values NaN.
            if (__builtin_expect(inf, 0)) {
#pragma unroll
                for (int b = 0; b < VC; b++) {
                    if (!EX && b >= nv) continue;
                    const u32x4 y = sc[(nq + (once ? copy : b)) * 4 + g];
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        int bad = 0;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            bad |= (y[i >> 1] >> (16 * (i & 1)) & 0x7c00u) == 0x7c00u && s[c][i >> 2][i & 3] != 0.0f;
                        bad |= __shfl_xor(bad, 16, 64);
                        bad |= __shfl_xor(bad, 32, 64);
                        const float nan = bad ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; i++) o[c][b][0][i] += nan, o[c][b][1][i] += nan;
                    }
                }
                lds_order();
#pragma unroll
                for (int e = 0; e < T::NS; e++) {
                    uint32_t y = ssc[wave][lane + 64 * e];
                    if ((y & 0x7c00u) == 0x7c00u) y &= 0xffff0000u;
                    if ((y & 0x7c000000u) == 0x7c000000u) y &= 0xffffu;
                    if (lane + 64 * e >= nq * 16) ssc[wave][lane + 64 * e] = y;
                }
                lds_order();
            }
            second(x, s, once);
            if (again) rest(x, s, once);
        };
        auto none = [] {};
        auto walk = [&](auto once) __attribute__((always_inline)) {
            // One column tile: two sets of words, a whole tile ahead.  Two, whose
            // sums need the registers: one set, the next tile's keys queued when
            // this one's have been read, its values at the end.
            while (C == 1 && any) {
                load(y);
                if (x.ok) step(x, x.base, once, std::false_type{}, none);
                if (v > v1) break;
                load(x);
                if (y.ok) step(y, y.base, once, std::false_type{}, none);
                if (v > v1) break;
            }
            while (C > 1 && any) {
                // (a tile that is none: behind the last position there can be)
                const int base = x.ok ? x.base : 0x7fffffff - (kTile - 1);
                find(x);
                step(x, base, once, std::false_type{}, [&] { load_keys(x); });
                load_values(x);
                if (v > v1) break;
            }
            // Scales 2^-8 of the largest and less (or subnormal ones, or 0): what
            // they scale may be all that has weight in a block of a value, below
            // what two pieces under one power of two hold.  The same tiles again,
            // with what those leave.
            if (__builtin_expect(!__any(low < max((E + 6) << 10, 0x400)), 1)) return;
#pragma unroll
            for (int c = 0; c < C; c++) {
                l[c] = 0.0f;
#pragma unroll
                for (int b = 0; b < VC; b++) o[c][b][0] = o[c][b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            for (v = v0; v < v1;) {
                load(x);
                if (x.ok) step(x, x.base, once, std::true_type{}, none);
            }
        };
        if (C == 1 && copies) walk(std::integral_constant<bool, C == 1>{});
        else walk(std::false_type{});

        // Merge the waves, a column tile at a time: sums as they are and their
        // references through LDS, then every wave takes a share of the output's
        // dims and brings the parts to the largest reference.
#pragma unroll
        for (int c = 0; c < C; c++) {
            l[c] += __shfl_xor(l[c], 16, 64);
            l[c] += __shfl_xor(l[c], 32, 64);
            if (lim[c] == -INFINITY && l[c] == 0.0f) ref[c] = -INFINITY;  // saw nothing
            if (g == 0) sm_r[wave][c * 16 + col] = ref[c], sm_l[wave][c * 16 + col] = l[c];
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
#pragma unroll
            for (int b = 0; b < VC * 2; b++) smo[(wave * VC * 2 + b) * 64 + lane] = o[c][b >> 1][b & 1];
            __syncthreads();
            float rr = -INFINITY, ll = 0.0f, fw[P];
#pragma unroll
            for (int w = 0; w < P; w++) rr = fmaxf(rr, sm_r[w * S + set][c * 16 + col]);
#pragma unroll
            for (int w = 0; w < P; w++) {
                const float rw = sm_r[w * S + set][c * 16 + col];
                fw[w] = rw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rw - rr);
                ll += rw == -INFINITY ? 0.0f : sm_l[w * S + set][c * 16 + col] * fw[w];
            }
            if (cv[c]) {
                const size_t row = r0 + cc[c] / hn, head = h0 + cc[c] % hn;
                float *dst = a.out + row * a.out_stride + head * kc.vd;
                float f = ll == 0.0f ? 0.0f : 1.0f / ll;
                if (a.ps > 1) {
                    const size_t where = (row * a.heads + head) * a.ps + part;
                    dst = a.part + where * kc.vd;
                    if (g == 0 && share == 0 && (!copies || col >> wide == 0)) a.part_ml[2 * where] = rr, a.part_ml[2 * where + 1] = ll;
                    f = 1.0f;
                }
                // Lane (column, g) of [block][half] holds dims 32 b + 16 h + 4 g + i.
#pragma unroll
                for (int bh = 0; bh < VC * 2; bh += P) {
                    const int b = (bh + share) >> 1;
                    if (b >= nv || (copies && col >> wide != b)) continue;
                    f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < P; w++) {
                        const f32x4 ow = smo[((w * S + set) * VC * 2 + bh + share) * 64 + lane];
#pragma unroll
                        for (int i = 0; i < 4; i++) z[i] = fw[w] == 0.0f ? z[i] : fmaf(ow[i], fw[w], z[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) z[i] *= f;
                    *(__attribute__((address_space(1))) f32x4_dw *)(dst + 16 * (bh + share) + 4 * g) = __builtin_bit_cast(f32x4_dw, z);
                }
            }
            __syncthreads();
        }
    }
}

// C tiles of 16 columns a wave and S sets of them pay where one run fills them:
// a group of 64 columns with several runs (sequences that decode, ends of
// prompts), or with no more than 16 columns, is dealt to its blocks in groups of
// 16 instead.  (1024 sequences of 32 heads over 8 that decode at 500 positions:
// 499 us with 64 columns a block, 191 with 16; a prompt of 2000 rows 124 and 144;
// that prompt beside 512 that decode 1402 and 387.)
template <int QC, int VC, bool EX, int C, int S, int W>
__global__ __launch_bounds__(W * 64, 2) void kv4_attention_kernel(const Args a) {
    union Both {
        Lds<QC, VC, C, S, W> wide;
        Lds<QC, VC, 1, 1, W> narrow;
    };
    __shared__ Both lds;
    const Kv4 &kc = a.c;
    const int lane = threadIdx.x & 63;
    // Kv heads next to each other go to the XCDs in turn, so that one head's
    // blocks find its tiles in their L2.  Later rows of a prompt see more
    // positions: the last groups go first.  A group's blocks that find no run
    // of their own leave at once, so the first ones come together.
    int id = blockIdx.x;
    const int kv = id % kc.n_kv;
    id /= kc.n_kv;
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int part = id % a.ps;
    id /= a.ps;
    const int sub = id / a.groups;
    const int r0 = (a.groups - 1 - id % a.groups) * a.tt;
    const int nr = min(a.tt, a.rows - r0);
    const int h0 = kv * a.rep + chunk * a.rc, hn = min(a.rc, a.rep - chunk * a.rc);
    const int my_seq = gload(a.seq + r0 + min(lane, nr - 1)), my_pos = gload(a.pos + r0 + min(lane, nr - 1));
    if (C == 1) {
        attend<QC, VC, EX, 1, 1, W>(a, lds.narrow, kv, part, r0, nr, h0, hn, my_seq, my_pos, sub, a.split);
        return;
    }
    const Runs runs = runs_of(kc, my_seq, my_pos, nr);
    if (__popcll(runs.starts) == 1 && __popcll(runs.valid) * hn > 16) {
        if (sub == 0) attend<QC, VC, EX, C, S, W>(a, lds.wide, kv, 0, r0, nr, h0, hn, my_seq, my_pos, 0, 1);
        return;
    }
    const int chunks = (hn + 15) / 16, rc = min(hn, 16), tt = 16 / rc;
    const int r1 = sub / chunks * tt, h1 = sub % chunks * 16;
    if (r1 >= nr) return;
    const int n1 = min(tt, nr - r1), from = r1 + min(lane, n1 - 1);
    attend<QC, VC, EX, 1, 1, W>(a, lds.narrow, kv, 0, r0 + r1, n1, h0 + h1, min(rc, hn - h1), __shfl(my_seq, from, 64),
                                __shfl(my_pos, from, 64), 0, 1);
}

// The parts of rows whose tiles several blocks shared: a block of T threads
// per (row, head), each group of vd / 4 of them every so many-th part; the
// groups' sums in order.
template <int T>
__global__ __launch_bounds__(T) void kv4_join_kernel(const Args a) {
    __shared__ float w[256], red[2];
    __shared__ f32x4 sums[T];
    const int vd = a.c.vd, row = blockIdx.x / a.heads, head = blockIdx.x % a.heads, i = threadIdx.x;
    if (a.pos[row] < 0 || (unsigned)a.seq[row] >= (unsigned)a.c.n_seq) return;
    const float *ml = a.part_ml + (size_t)blockIdx.x * a.ps * 2, *part = a.part + (size_t)blockIdx.x * a.ps * vd;
    if (i < 64) {
        float ref[4], l = 0.0f, rr = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int p = i + 64 * k;
            ref[k] = p < a.ps ? ml[2 * p] : -INFINITY;
            rr = fmaxf(rr, ref[k]);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) rr = fmaxf(rr, __shfl_xor(rr, o, 64));
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int p = i + 64 * k;
            if (p >= a.ps) continue;
            const float f = ref[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref[k] - rr);
            w[p] = f;
            l += ref[k] == -INFINITY ? 0.0f : ml[2 * p + 1] * f;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
        if (i == 0) red[0] = l == 0.0f ? 0.0f : 1.0f / l;
    }
    __syncthreads();
    const int n = vd / 4, groups = T / n, g = i / n, at = i % n;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (g < groups)
        for (int p = g; p < a.ps; p += groups) {
            const f32x4 x = gload((const f32x4 *)(part + (size_t)p * vd) + at);
            const float f = w[p];
#pragma unroll
            for (int k = 0; k < 4; k++) acc[k] = f == 0.0f ? acc[k] : fmaf(x[k], f, acc[k]);
        }
    sums[i] = acc;
    __syncthreads();
    if (i >= n) return;
    for (int k = 1; k < groups; k++) acc += sums[k * n + i];
    float *dst = a.out + (int64_t)row * a.out_stride + (int64_t)head * vd + 4 * i;
#pragma unroll
    for (int k = 0; k < 4; k++) dst[k] = acc[k] * red[0];
}

// How a call is cut up: see Args.
struct Plan {
    int C, cols, rc, chunks, tt, groups, split, ps;  // cols: columns of a block
    uint64_t bytes;
};

Plan plan_of(const Kv4 &c, int rows, int heads, int max_pos, int window, int n_sel) {
    Plan p{};
    const int rep = heads / c.n_kv;
    // Two column tiles a wave halve the unpacking, and two sets of them a block
    // halve what comes before the first tile and after the last, where rows come
    // in runs; but blocks of 64 columns are a quarter as many.  At 128 dims they
    // pay from about two such blocks a CU on (blocks of 16 columns and of 64: 520
    // rows of 32 heads over 8 26.1 and 29.4 us, 700 33.5 and 34.5, 1000 52.8 and
    // 48.5, 1200 68.6 and 59.2, 2000 149 and 122, 8000 1715 and 1355).  Wider heads
    // lose a wave of every SIMD to the registers (4000 rows of 16 heads of 192/128
    // 298 and 359), 96 dims gain nothing (4000 rows of 6 heads 194 and 222), nor do
    // 64 below 16000 rows.
    const long long wide = ((long long)rows * rep + 63) / 64 * c.n_kv;
    p.C = n_sel == 0 && c.qd == 128 && c.vd == 128 && wide >= 512 ? 2 : 1;
    p.cols = p.C == 2 ? 64 : 16;
    p.rc = std::min(rep, p.cols);
    p.chunks = (rep + p.rc - 1) / p.rc;
    // Rows with lists of their own share nothing.
    p.tt = n_sel ? 1 : p.cols / p.rc;
    p.groups = (int)(((long long)rows + p.tt - 1) / p.tt);
    const long long base = (long long)p.groups * p.chunks * c.n_kv;
    const int narrow = std::min(p.rc, 16);  // query heads of a group of 16 columns
    p.split = p.C == 2 ? (p.tt + 16 / narrow - 1) / (16 / narrow) * ((p.rc + 15) / 16)
                       : (int)std::max<long long>(1, std::min<long long>(p.tt, 1024 / base));
    const long long tiles = n_sel ? (long long)n_sel * c.tiles()
                                  : (window > 0 ? std::min((long long)window + p.tt, (long long)max_pos + 1) : max_pos + 1LL) / 32 + 1;
    const long long units = base * p.split;
    // Parts of a run's tiles.  A block costs about as much as 8 tiles of a wave
    // before its first and after its last, and parts a launch that joins them
    // (5 us): with a block for every CU they pay for long runs only, below that
    // from 12 tiles a wave on.  (Kernel + join: 512 blocks of 19 to 38 tiles
    // 28.2 us, in two parts 34 + 4.6; 488 of 64 tiles 34.5, 39.4 + 4.8; 512 of
    // 190 to 375 152.6, 152.3 + 4.8; 8 of 3126 tiles in 64, 128, 256 parts 60.8 +
    // 5.7, 36.8 + 5.0, 32.4 + 5.6.)
    const long long ps = p.C == 2       ? 1  // (512 blocks and more: nothing to share)
                         : units >= 256 ? std::min((512 + units - 1) / units, tiles / 64)
                         : tiles < 48 ? 1
                                      : std::min<long long>({(2048 + units - 1) / units, tiles / 12, 256});
    p.ps = (int)std::max<long long>(1, ps);
    p.bytes = p.ps > 1 ? (uint64_t)rows * heads * p.ps * (c.vd + 2) * 4 : 0;
    return p;
}

template <int QC, int VC, bool EX, int C>
void launch(const Args &a, hipStream_t s) {
    constexpr int W = 4;
    const long long blocks = (long long)a.groups * a.split * a.ps * a.chunks * a.c.n_kv;
    hipLaunchKernelGGL((kv4_attention_kernel<QC, VC, EX, C, C, W>), dim3((unsigned)blocks), dim3(W * 64), 0, s, a);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_attention_workspace_size(const moe_kv4 *c, int32_t rows, int32_t heads, int32_t max_pos, int32_t window,
                                     int32_t n_sel, uint64_t *bytes) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_attention_workspace_size", c, &a)) return rc;
    if (!bytes || rows < 0 || heads <= 0 || heads % a.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.max_pages << a.page_shift || n_sel < 0 || (int64_t)n_sel << a.page_shift > INT32_MAX)
        return fail(MOE_EINVAL, "moe_kv4_attention_workspace_size: bad argument (%d rows, %d heads over %d, max position %d"
                    " of %lld)", rows, heads, a.n_kv, max_pos, (long long)a.max_pages << a.page_shift);
    *bytes = rows ? plan_of(a, rows, heads, max_pos, window, n_sel).bytes : 0;
    return MOE_OK;
}

int moe_kv4_attention(const moe_kv4 *c, const float *q, int64_t q_stride, int32_t rows, int32_t heads, float scale,
                      const int32_t *seq, const int32_t *pos, int32_t max_pos, int32_t window, const int32_t *lists,
                      int32_t n_sel, float *out, int64_t out_stride, void *workspace, uint64_t workspace_bytes,
                      void *stream) {
    Args a{};
    if (const int rc = kv4_of("moe_kv4_attention", c, &a.c)) return rc;
    if ((rows > 0 && (!q || !seq || !pos || !out)) || rows < 0 || heads <= 0 || heads % a.c.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.c.max_pages << a.c.page_shift ||
        (lists && (n_sel <= 0 || (int64_t)n_sel << a.c.page_shift > INT32_MAX)))
        return fail(MOE_EINVAL, "moe_kv4_attention: bad argument (%d rows, %d heads over %d, max position %d of %lld, %d pages)",
                    rows, heads, a.c.n_kv, max_pos, (long long)a.c.max_pages << a.c.page_shift, n_sel);
    if (rows == 0) return MOE_OK;
    const Plan p = plan_of(a.c, rows, heads, max_pos, window, lists ? n_sel : 0);
    if (p.bytes && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < p.bytes))
        return fail(MOE_EINVAL, "moe_kv4_attention: workspace of %llu bytes, %llu needed",
                    (unsigned long long)workspace_bytes, (unsigned long long)p.bytes);
    a.q = q, a.seq = seq, a.pos = pos, a.lists = lists, a.out = out;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.rows = rows, a.heads = heads, a.rep = heads / a.c.n_kv, a.window = window, a.n_sel = lists ? n_sel : 0;
    a.scale = scale;
    a.tt = p.tt, a.groups = p.groups, a.rc = p.rc, a.chunks = p.chunks, a.split = p.split, a.ps = p.ps;
    a.part = static_cast<float *>(workspace);
    a.part_ml = a.part + (size_t)rows * heads * p.ps * a.c.vd;
    if ((long long)a.groups * a.split * a.ps * a.chunks * a.c.n_kv > kMostThreads / 256)
        return fail(MOE_EUNSUP, "moe_kv4_attention: %d rows of %d heads are too many blocks", rows, heads);
    hipStream_t s = (hipStream_t)stream;
    const int qc = a.c.qd / 32, vc = a.c.vd / 32;
    // Widths of their own: a power-of-two head and the latent cache's 192/128;
    // the others count their blocks at run time.
    if (qc == 2 && vc == 2) launch<2, 2, true, 1>(a, s);
    else if (qc == 4 && vc == 4) p.C == 2 ? launch<4, 4, true, 2>(a, s) : launch<4, 4, true, 1>(a, s);
    else if (qc == 6 && vc == 4) launch<6, 4, true, 1>(a, s);
    else if (qc <= 6 && vc <= 4) launch<6, 4, false, 1>(a, s);
    else if (qc == 8 && vc == 8) launch<8, 8, true, 1>(a, s);
    else launch<8, 8, false, 1>(a, s);
    if (a.ps > 16) hipLaunchKernelGGL((kv4_join_kernel<256>), dim3((unsigned)rows * heads), dim3(256), 0, s, a);
    else if (a.ps > 1) hipLaunchKernelGGL((kv4_join_kernel<64>), dim3((unsigned)rows * heads), dim3(64), 0, s, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "4-bit attention kernel: %s", hipGetErrorString(e));
}

}  // extern "C"
