// kv4_select.hip — the pages a query's sparse attention reads (moe_kv4_select).
//
// A page's score is the largest of q . mean key over the kv head's query
// heads, in 64 bits: which of two near pages wins does not hang on the order
// of a sum.  Scoring every page so was bound by f64 conversions and fused
// multiply-adds and by LDS reads of the queries, so the f16 matrix cores bound
// the scores first (bound_pages: f32 sums and a margin above all their errors),
// an order statistic of the bounds settles most pages, and the few that it
// leaves in doubt are scored in 64 bits (settle).  The choice is the exact one,
// ties to the lower page, the same every time; where more pages are in doubt
// than fit (many equal scores, infinities), all are scored in 64 bits and the
// n_sel-th largest found digit by digit (score_pages, pick).
//
// A block per (row, kv head).  32 rows of 500 pages, 8 kv heads of 4 query heads
// of 128 dims 17.5 -> 14.7 us (the means' 33 MB: 6.7 at the copy's rate), 61 rows
// of 1100 pages 52.9 -> 32.4 (several rows of one sequence read its means from
// L2 again; what is left is the order statistic, a chain of passes and barriers,
// about 9 us, and two dependent loads), 4 kv heads of 16 38 -> 16, one of 40
// heads of 64 dims, 40 rows of 600 pages, 45 -> 20.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 512;
constexpr int kHeads = 4;        // query heads scored at once
constexpr int kLdsPages = 4096;  // scores a block keeps in LDS (32 KiB)

struct Args {
    Kv4 c;
    const float *q;
    const int32_t *seq, *pos;
    int32_t *lists;
    uint64_t *keys;  // workspace [row][kv head][n], where the scores are another launch's
    int64_t q_stride;
    int rep, n_kv, sinks, recent, n_sel, n;
};

// A score's place in the order of doubles as unsigned integers, 1 ... 2^64 - 2:
// NaN below every number, 0 for pages there are not, 2^64 - 1 for forced.
__device__ inline uint64_t order_of(double s) {
    if (s != s) return 1;
    const int64_t b = __double_as_longlong(s);
    return b < 0 ? ~(uint64_t)b : (uint64_t)b | 0x8000000000000000ull;
}

// Exact keys of all of the row's pages by the block.  cur: the row's own page.
// qs: LDS of kHeads * qd doubles.
__device__ inline void score_pages(const Args &a, int row, int kv, int sid, int cur, double *qs, uint64_t *out) {
    const Kv4 &c = a.c;
    const int nq = c.qd / 32, e = threadIdx.x & 3, n = cur + 1;
    const int32_t *table = c.table + (size_t)sid * c.max_pages;
    for (int h0 = 0; h0 < a.rep; h0 += kHeads) {
        const int hn = min(kHeads, a.rep - h0);
        __syncthreads();  // the reads of the heads before
        for (int i = threadIdx.x; i < kHeads * c.qd; i += kThreads) {
            const int h = min(i / c.qd, hn - 1), d = i % c.qd;  // past the last head: the last again
            qs[i] = (double)gload(a.q + (size_t)row * a.q_stride + (size_t)(kv * a.rep + h0 + h) * c.qd + d);
        }
        __syncthreads();
        for (int t = threadIdx.x >> 2; t < (n + 15) / 16 * 16; t += kThreads / 4) {  // (a wave's 16 pages together)
            const int id = t >= a.sinks && t <= cur - a.recent ? gload(table + t) : -1;
            const bool has = (unsigned)id < (unsigned)c.n_pages;
            const __half *mean = c.means + ((size_t)(has ? id : 0) * c.n_kv + kv) * c.qd + 8 * e;
            double acc[kHeads];
#pragma unroll
            for (int h = 0; h < kHeads; h++) acc[h] = 0.0;
#pragma unroll 2
            for (int s = 0; s < nq; s++) {
                const half8 m = gload((const half8 *)(mean + 32 * s));
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const double x0 = (double)(float)m[i], x1 = (double)(float)m[i + 1];
#pragma unroll
                    for (int h = 0; h < kHeads; h++) {
                        const f64x2 y = *(const f64x2 *)(qs + h * c.qd + 32 * s + 8 * e + i);
                        acc[h] = fma(y[1], x1, fma(y[0], x0, acc[h]));
                    }
                }
            }
            uint64_t best = 1;
#pragma unroll
            for (int h = 0; h < kHeads; h++) {
                double v = acc[h];
                v += __shfl_xor(v, 1, 64);
                v += __shfl_xor(v, 2, 64);
                best = max(best, order_of(v));
            }
            if (e == 0 && t < n) {
                uint64_t k = has ? best : 1;
                if (h0 > 0) k = max(k, out[t]);
                if (t < a.sinks || t > cur - a.recent) k = ~0ull;
                out[t] = k;
            }
        }
    }
    __syncthreads();
}

// Exact keys of n pages (LDS) that are not forced, into LDS: eight lanes a page
// and query head.
__device__ inline void score_list(const Args &a, int row, int kv, int sid, const int *list, int n, unsigned long long *out) {
    const Kv4 &c = a.c;
    const int nq = c.qd / 32, e = threadIdx.x & 7;
    const int32_t *table = c.table + (size_t)sid * c.max_pages;
    for (int i = threadIdx.x; i < n; i += kThreads) out[i] = 1;
    __syncthreads();
    const int items = n * a.rep;
    for (int t = threadIdx.x >> 3; t < (items + 7) / 8 * 8; t += kThreads / 8) {  // (a wave's eight together)
        const int i = min(t, items - 1) / a.rep, h = min(t, items - 1) % a.rep, id = gload(table + list[i]);
        const bool has = (unsigned)id < (unsigned)c.n_pages;
        const __half *mean = c.means + ((size_t)(has ? id : 0) * c.n_kv + kv) * c.qd + 4 * e;
        const float *q = a.q + (size_t)row * a.q_stride + (size_t)(kv * a.rep + h) * c.qd + 4 * e;
        double v = 0.0;
#pragma unroll 4
        for (int s = 0; s < nq; s++) {
            const u32x4 x = gload_x4((const uint32_t *)(q + 32 * s));
            const half4 m = gload((const half4 *)(mean + 32 * s));
#pragma unroll
            for (int k = 0; k < 4; k++) v = fma((double)__uint_as_float(x[k]), (double)(float)m[k], v);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) v += __shfl_xor(v, o, 64);
        if (e == 0 && has) atomicMax(out + i, (unsigned long long)order_of(v));
    }
    __syncthreads();
}

// The order of floats as unsigned integers: 2^23 ... 2^32 - 2^23 - 1 for finite ones.
__device__ inline uint32_t order32(float f) {
    const uint32_t b = __float_as_uint(f);
    return b >> 31 ? ~b : b | 0x80000000u;
}

// Bounds of the scores of pages [j0, j1) by the block into out[j - j0], lower
// one << 32 | upper one, as order32: both 1 for pages that are not in the pool,
// 2^32 - 1 for forced ones, 0 and 2^32 - 2 where nothing is known.
//
// Rows of the matrix product are query heads, columns pages.  A query, by a
// power of two that brings its largest value into [2^14, 2^15), goes in two f16
// pieces, a mean key is f16.  With A the sum of |mean| no partial sum is above
// 2^15 A; 64 QC f32 sums are off by 2^-23 of that each, the pieces by 2^-22 of
// a value, or 2^-14 where a small one counts as 0: less than (QC + 2) 2^-17 2^15 A
// together, and the true score lies within.
template <int QC>
__device__ inline void bound_pages(const Args &a, int row, int kv, int sid, int cur, int j0, int j1, uint64_t *out) {
    const Kv4 &c = a.c;
    const int nq = c.qd / 32, lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = threadIdx.x >> 6;
    const int32_t *table = c.table + (size_t)sid * c.max_pages;
    for (int h0 = 0; h0 < a.rep; h0 += 16) {
        // P tiles of 16 pages a wave; the means of the next load while these are
        // multiplied, the table's entries of those after them before.  One tile
        // keeps four waves a SIMD, two blocks a CU, at 128 dims (61 rows of 1100
        // pages: 40.5 us with two tiles and two waves).
        constexpr int P = QC <= 2 ? 2 : 1, kStep = kThreads / 64 * 16 * P;
        int id[P];
        u32x4 mn[P][QC];
        bool hasn[P];
        auto load_ids = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                const int j = base + 16 * p + col;
                id[p] = j < j1 && j >= a.sinks && j <= cur - a.recent ? gload(table + j) : -1;
            }
        };
        auto load_means = [&] __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                hasn[p] = (unsigned)id[p] < (unsigned)c.n_pages;
                const __half *mean = c.means + ((size_t)(hasn[p] ? id[p] : 0) * c.n_kv + kv) * c.qd;
#pragma unroll
                for (int s = 0; s < QC; s++)
                    if (s < nq) mn[p][s] = gload((const u32x4 *)(mean + 32 * s + 8 * g));
            }
        };
        load_ids(j0 + wave * 16 * P);
        // Head h0 + col (past the last: the last again), dims 32 s + 8 g ...
        float top = 0.0f;
        u32x4 x[QC][2];
        const float *q = a.q + (size_t)row * a.q_stride + (size_t)(kv * a.rep + min(h0 + col, a.rep - 1)) * c.qd;
#pragma unroll
        for (int s = 0; s < QC; s++) {
            if (s >= nq) break;
            x[s][0] = gload_x4((const uint32_t *)(q + 32 * s + 8 * g));
            x[s][1] = gload_x4((const uint32_t *)(q + 32 * s + 8 * g + 4));
        }
        load_means();
        load_ids(j0 + wave * 16 * P + kStep);
#pragma unroll
        for (int s = 0; s < QC; s++) {
            if (s >= nq) break;
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(__uint_as_float(x[s][i >> 2][i & 3])));
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const int ex = min(max(127 + 14 - ((int)(__float_as_uint(top) >> 23) - 127), 1), 253);
        const float up = __uint_as_float((uint32_t)ex << 23), down = __uint_as_float((uint32_t)(254 - ex) << 23);
        half8 hi[QC], lo[QC];
#pragma unroll
        for (int s = 0; s < QC; s++) {
            if (s >= nq) break;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float z = __uint_as_float(x[s][i >> 2][i & 3]) * up;
                hi[s][i] = (_Float16)z;
                lo[s][i] = (_Float16)(z - (float)hi[s][i]);
            }
        }
        const _Float16 one = (_Float16)1.0f;
        const half8 ones = {one, one, one, one, one, one, one, one};
        float back[4];  // a result's row is head h0 + 4 g + i
#pragma unroll
        for (int i = 0; i < 4; i++) back[i] = __shfl(down, 4 * g + i, 64);
        for (int base = j0 + wave * 16 * P; base < j1; base += kStep) {
            u32x4 m[P][QC];
            bool has[P];
#pragma unroll
            for (int p = 0; p < P; p++) {
                has[p] = hasn[p];
#pragma unroll
                for (int s = 0; s < QC; s++) m[p][s] = mn[p][s];
            }
            load_means();
            load_ids(base + 2 * kStep);
            f32x4 sum[P], most[P];
#pragma unroll
            for (int p = 0; p < P; p++) sum[p] = most[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < QC; s++) {
                if (s >= nq) break;
#pragma unroll
                for (int p = 0; p < P; p++) {
                    const half8 v = __builtin_bit_cast(half8, m[p][s]);
                    const half8 w = __builtin_bit_cast(half8, m[p][s] & 0x7fff7fffu);
                    sum[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[s], v, sum[p], 0, 0, 0);
                    most[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w, most[p], 0, 0, 0);
                    sum[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[s], v, sum[p], 0, 0, 0);
                }
            }
#pragma unroll
            for (int p = 0; p < P; p++) {
                float l = -INFINITY, u = -INFINITY;
                bool known = true;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // (1e-37: what a number too small for f32 loses)
                    const float v = sum[p][i] * back[i], e = fmaf(most[p][i] * back[i], (QC + 2) * 0x1p-2f, 1e-37f);
                    l = fmaxf(l, v - e), u = fmaxf(u, v + e);
                    known = known && fabsf(v) + e <= 3e38f;
                }
                l = fmaxf(l, __shfl_xor(l, 16, 64)), u = fmaxf(u, __shfl_xor(u, 16, 64));
                l = fmaxf(l, __shfl_xor(l, 32, 64)), u = fmaxf(u, __shfl_xor(u, 32, 64));
                const unsigned long long k = __ballot(known);
                known = (k >> col & k >> (col + 16) & k >> (col + 32) & k >> (col + 48) & 1) != 0;
                const int j = base + 16 * p + col;
                if (g == 0 && j < j1) {
                    uint32_t kl = known ? order32(l) : 0, ku = known ? order32(u) : ~1u;
                    if (!has[p]) kl = ku = 1;
                    if (h0 > 0) {
                        const uint64_t o = out[j - j0];
                        const uint32_t ol = (uint32_t)(o >> 32);
                        ku = max(ku, (uint32_t)o), kl = kl == 0 || ol == 0 ? 0 : max(kl, ol);
                    }
                    if (j < a.sinks || j > cur - a.recent) kl = ku = ~0u;
                    out[j - j0] = (uint64_t)kl << 32 | ku;
                }
            }
        }
    }
    __syncthreads();
}

// The n_sel-th largest of n keys, digit by digit of the bits from `last` on:
// every key with (key & mask) >= prefix is among the first n_sel or (all false)
// equal to the n_sel-th in those bits, `want` of which are.
struct Cut {
    uint64_t prefix, mask;
    int want;
    bool all;
};
__device__ inline Cut cut_of(const uint64_t *keys, int n, int n_sel, int last) {
    __shared__ int hist[256];
    __shared__ int s_digit, s_above, s_here;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t prefix = 0, mask = 0;
    int want = n_sel;  // how many of those that agree with prefix
    bool all = false;  // every one that does
    for (int shift = 56; shift >= last && !all; shift -= 8) {
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kThreads) {
            const uint64_t k = keys[j];
            if (k != 0 && (k & mask) == prefix) atomicAdd(hist + (int)(k >> shift & 255), 1);
        }
        __syncthreads();
        if (wave == 0) {
            // Sums from the top: lane l holds digits 255 - 4 l downwards.
            int h[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = hist[255 - 4 * lane - i], sum += h[i];
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(upto, o, 64);
                if (lane >= o) upto += y;
            }
            int above = upto - sum;
            const unsigned long long there = __ballot(upto >= want);
            if (there == 0) {
                if (lane == 0) s_digit = -1;  // fewer than wanted: all of them
            } else if (lane == __builtin_ctzll(there)) {
                int i = 0;
#pragma unroll
                for (int t = 0; t < 3; t++)
                    if (i == t && above + h[t] < want) above += h[t], i = t + 1;
                s_digit = 255 - 4 * lane - i, s_above = above;
                s_here = i == 0 ? h[0] : i == 1 ? h[1] : i == 2 ? h[2] : h[3];
            }
        }
        __syncthreads();
        if (s_digit < 0) {
            all = true;  // prefix and mask stay: every key there is
        } else {
            want -= s_above;
            prefix |= (uint64_t)s_digit << shift, mask |= 255ull << shift;
            all = s_here == want;
        }
    }
    return Cut{prefix, mask, want, all};
}

// The pages of `in` keys, ascending, into list.
template <class In>
__device__ inline void write_list(int n, int n_sel, int32_t *list, In in_of) {
    __shared__ int found[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;
    for (int base = 0; base < n; base += kThreads) {
        const int j = base + threadIdx.x;
        const bool in = in_of(j);
        const unsigned long long b = __ballot(in);
        __syncthreads();
        if (lane == 0) found[wave] = __popcll(b);
        __syncthreads();
        int at = before + __popcll(b & ((1ull << lane) - 1));
        for (int w = 0; w < wave; w++) at += found[w];
        if (in && at < n_sel) list[at] = j;
        for (int w = 0; w < kThreads / 64; w++) before += found[w];
    }
    for (int i = before + (int)threadIdx.x; i < n_sel; i += kThreads) list[i] = -1;
}

// The first n_sel of n exact keys in their order, equal ones by index.
__device__ inline void pick(const uint64_t *keys, int n, int n_sel, int32_t *list) {
    __shared__ int found[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Cut t = cut_of(keys, n, n_sel, 0);
    int ties = 0;  // pages equal to the last one, so far
    write_list(n, n_sel, list, [&](int j) {
        const uint64_t k = j < n ? keys[j] : 0;
        const bool edge = k != 0 && (k & t.mask) == t.prefix;
        const bool in = k != 0 && (k & t.mask) > t.prefix;
        if (t.all) return in || edge;
        const unsigned long long b = __ballot(edge);
        __syncthreads();
        if (lane == 0) found[wave] = __popcll(b);
        __syncthreads();
        int at = ties + __popcll(b & ((1ull << lane) - 1));
        for (int w = 0; w < wave; w++) at += found[w];
        for (int w = 0; w < kThreads / 64; w++) ties += found[w];
        return in || (edge && at < t.want);
    });
}

constexpr int kDoubt = 256;  // pages in doubt that are scored apart

// The first n_sel of n pages in the order of their exact scores, of which
// `keys` holds bounds (and is overwritten).  With C the n_sel pages of the
// largest lower bounds (those above the n_sel-th where it is shared), T the
// n_sel-th lower bound and M the largest upper bound outside C: a page whose
// lower bound is above M is among the first n_sel, one whose upper bound is
// below T is not, and the others are scored exactly.
__device__ inline void settle(const Args &a, int row, int kv, int sid, int cur, uint64_t *keys, double *qs, int32_t *list) {
    __shared__ int doubt[kDoubt], sure, doubts;
    __shared__ unsigned long long exact[kDoubt];
    __shared__ uint32_t s_low, s_most;
    const int n = cur + 1;
    if (threadIdx.x == 0) sure = doubts = 0, s_low = ~0u, s_most = 0;
    const Cut t = cut_of(keys, n, a.n_sel, 32);
    uint32_t low = ~0u, most = 0;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        const uint64_t k = keys[j];
        const bool in = t.all ? (k & t.mask) >= t.prefix : (k & t.mask) > t.prefix;
        if (in) low = min(low, (uint32_t)(k >> 32));
        else most = max(most, (uint32_t)k);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        low = min(low, (uint32_t)__shfl_xor((int)low, o, 64));
        most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    }
    if ((threadIdx.x & 63) == 0) atomicMin(&s_low, low), atomicMax(&s_most, most);
    __syncthreads();
    const uint32_t T = t.all ? s_low : (uint32_t)(t.prefix >> 32), M = s_most;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        const uint32_t l = (uint32_t)(keys[j] >> 32), u = (uint32_t)keys[j];
        if (l > M) {
            atomicAdd(&sure, 1);
        } else if (u >= T) {
            const int at = atomicAdd(&doubts, 1);
            if (at < kDoubt) doubt[at] = j;
        }
    }
    __syncthreads();
    const int nd = doubts, want = a.n_sel - sure;
    if (nd > want && nd > kDoubt) {
        score_pages(a, row, kv, sid, cur, qs, keys);
        pick(keys, n, a.n_sel, list);
        return;
    }
    if (nd > want) {
        // A page's place among them, whatever order they were noted in.
        score_list(a, row, kv, sid, doubt, nd, exact);
        if ((int)threadIdx.x < nd) {
            const uint64_t k = exact[threadIdx.x];
            const int j = doubt[threadIdx.x];
            int place = 0;
            for (int i = 0; i < nd; i++) place += exact[i] > k || (exact[i] == k && doubt[i] < j);
            keys[j] = place < want ? ~0ull : 0;
        }
        __syncthreads();
        write_list(n, a.n_sel, list, [&](int j) { return j < n && (keys[min(j, n - 1)] >> 32) > M; });
    } else {
        write_list(n, a.n_sel, list, [&](int j) {
            const uint64_t k = keys[min(j, n - 1)];
            return j < n && ((k >> 32) > M || (uint32_t)k >= T);
        });
    }
}

// FUSED: bounds and choice; otherwise the choice from the workspace's bounds.
template <int QC, bool FUSED>
__global__ __launch_bounds__(kThreads, QC <= 4 ? 4 : 2) void kv4_select_kernel(const Args a) {
    __shared__ uint64_t lds[FUSED ? kLdsPages : 1];
    __shared__ double qs[kHeads * QC * 32];
    const int row = blockIdx.x / a.n_kv, kv = blockIdx.x % a.n_kv;
    int32_t *list = a.lists + (size_t)blockIdx.x * a.n_sel;
    const int sid = gload(a.seq + row), top = gload(a.pos + row);
    if (top < 0 || (unsigned)sid >= (unsigned)a.c.n_seq) {
        for (int i = threadIdx.x; i < a.n_sel; i += kThreads) list[i] = -1;
        return;
    }
    const int cur = min(top >> a.c.page_shift, a.n - 1);
    if (cur < a.n_sel) {  // every page
        for (int i = threadIdx.x; i < a.n_sel; i += kThreads) list[i] = i <= cur ? i : -1;
        return;
    }
    if (FUSED) {
        bound_pages<QC>(a, row, kv, sid, cur, 0, cur + 1, lds);
        settle(a, row, kv, sid, cur, lds, qs, list);
    } else {
        settle(a, row, kv, sid, cur, a.keys + (size_t)blockIdx.x * a.n, qs, list);
    }
}

constexpr int kScorePages = 256;  // pages of a block of kv4_bound_kernel
template <int QC>
__global__ __launch_bounds__(kThreads, QC <= 4 ? 4 : 2) void kv4_bound_kernel(const Args a) {
    const int row = blockIdx.x / a.n_kv, kv = blockIdx.x % a.n_kv;
    const int sid = gload(a.seq + row), top = gload(a.pos + row);
    if (top < 0 || (unsigned)sid >= (unsigned)a.c.n_seq) return;
    const int cur = min(top >> a.c.page_shift, a.n - 1), j0 = blockIdx.y * kScorePages;
    if (cur < a.n_sel || j0 > cur) return;
    bound_pages<QC>(a, row, kv, sid, cur, j0, min(cur + 1, j0 + kScorePages), a.keys + (size_t)blockIdx.x * a.n + j0);
}

// Bounds of a launch of their own: more pages than LDS holds, or so few blocks
// that each would go over many pages alone (8 pairs of 4000 pages 45.8 -> 25.8
// us, 64 of 1500 24.6 -> 23.6, 112 of 3000 38.7 -> 47.2).
bool apart(int64_t pairs, int n) { return n > kLdsPages || (pairs <= 64 && n > 2 * kScorePages); }

template <int QC>
void launch(const Args &a, int rows, hipStream_t s) {
    const unsigned pairs = (unsigned)rows * a.n_kv;
    if (apart(pairs, a.n)) {
        hipLaunchKernelGGL((kv4_bound_kernel<QC>), dim3(pairs, (a.n + kScorePages - 1) / kScorePages), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL((kv4_select_kernel<QC, false>), dim3(pairs), dim3(kThreads), 0, s, a);
    } else {
        hipLaunchKernelGGL((kv4_select_kernel<QC, true>), dim3(pairs), dim3(kThreads), 0, s, a);
    }
}

uint64_t workspace_of(const Kv4 &c, int rows, int max_pos) {
    const int n = (max_pos >> c.page_shift) + 1;
    return apart((int64_t)rows * c.n_kv, n) ? 8 * (uint64_t)rows * c.n_kv * n : 0;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_select_workspace_size(const moe_kv4 *c, int32_t rows, int32_t max_pos, uint64_t *bytes) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_select_workspace_size", c, &a)) return rc;
    if (!bytes || rows < 0 || max_pos < 0 || max_pos >= (int64_t)a.max_pages << a.page_shift)
        return fail(MOE_EINVAL, "moe_kv4_select_workspace_size: bad argument (%d rows, max position %d of %lld)", rows, max_pos,
                    (long long)a.max_pages << a.page_shift);
    *bytes = workspace_of(a, rows, max_pos);
    return MOE_OK;
}

int moe_kv4_select(const moe_kv4 *c, const float *q, int64_t q_stride, int32_t rows, int32_t heads, const int32_t *seq,
                   const int32_t *pos, int32_t max_pos, int32_t sinks, int32_t recent, int32_t n_sel, int32_t *lists,
                   void *workspace, uint64_t workspace_bytes, void *stream) {
    Args a{};
    if (const int rc = kv4_of("moe_kv4_select", c, &a.c)) return rc;
    if (!a.c.means) return fail(MOE_EINVAL, "moe_kv4_select: the cache keeps no mean keys");
    if ((rows > 0 && (!q || !seq || !pos || !lists)) || rows < 0 || heads <= 0 || heads % a.c.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.c.max_pages << a.c.page_shift)
        return fail(MOE_EINVAL, "moe_kv4_select: bad argument (%d rows, %d heads over %d, max position %d of %lld)", rows,
                    heads, a.c.n_kv, max_pos, (long long)a.c.max_pages << a.c.page_shift);
    if (sinks < 0 || recent < 1 || n_sel < 1 || (int64_t)n_sel << a.c.page_shift > INT32_MAX || (int64_t)sinks + recent > n_sel)
        return fail(MOE_EINVAL, "moe_kv4_select: %d first and %d last pages of %d", sinks, recent, n_sel);
    if (rows == 0) return MOE_OK;
    const int64_t pages = (max_pos >> a.c.page_shift) + 1;
    if ((int64_t)rows * a.c.n_kv * kThreads > kMostThreads || pages > 65535ll * kScorePages)
        return fail(MOE_EUNSUP, "moe_kv4_select: %d rows of %d kv heads and %lld pages are too many blocks", rows, a.c.n_kv,
                    (long long)pages);
    const uint64_t need = workspace_of(a.c, rows, max_pos);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
        return fail(MOE_EINVAL, "moe_kv4_select: workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)need);
    a.q = q, a.seq = seq, a.pos = pos, a.lists = lists, a.keys = static_cast<uint64_t *>(workspace);
    a.q_stride = q_stride, a.rep = heads / a.c.n_kv, a.n_kv = a.c.n_kv;
    a.sinks = sinks, a.recent = recent, a.n_sel = n_sel, a.n = (max_pos >> a.c.page_shift) + 1;
    hipStream_t s = (hipStream_t)stream;
    if (a.c.qd <= 64) launch<2>(a, rows, s);
    else if (a.c.qd <= 128) launch<4>(a, rows, s);
    else if (a.c.qd <= 192) launch<6>(a, rows, s);
    else launch<8>(a, rows, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "page selection: %s", hipGetErrorString(e));
}

}  // extern "C"
