// kv4_select.hip — the pages a query's sparse attention reads (moe_kv4_select).
//
// A page's score is the largest of q . mean key over the kv head's query
// heads, in 64 bits: which of two near pages wins does not hang on the order
// of a sum.  A score becomes an integer of the same order, and the n_sel-th
// largest is found digit by digit from a histogram (equal ones: the lower page
// first), so the choice is exact and the same every time.
//
// kv4_select_kernel: a block per (row, kv head).  Queries sit in LDS in 64
// bits; four lanes share a page (contiguous 64-byte pieces of its mean key) and
// take two pages at once, since an LDS read of two queries feeds two fused
// multiply-adds a page and LDS, not f64, is the tighter pipe.  Scores stay in
// LDS.  Where there are few rows, or more pages than LDS holds, kv4_score_kernel
// spreads the pages over blocks and leaves the scores in the workspace.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
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

// The keys of pages [j0, j1) of a (row, kv head) by the block into out[j -
// j0].  cur: the row's own page.  qs: LDS of kHeads * qd doubles.
template <int QC>
__device__ inline void score_pages(const Args &a, int row, int kv, int sid, int cur, int j0, int j1, double *qs,
                                   uint64_t *out) {
    const Kv4 &c = a.c;
    const int nq = c.qd / 32, lane = threadIdx.x & 63, e = lane & 3, wave = threadIdx.x >> 6;
    const int32_t *table = c.table + (size_t)sid * c.max_pages;
    for (int h0 = 0; h0 < a.rep; h0 += kHeads) {
        const int hn = min(kHeads, a.rep - h0);
        __syncthreads();  // the reads of the heads before
        for (int i = threadIdx.x; i < kHeads * c.qd; i += kThreads) {
            const int h = min(i / c.qd, hn - 1), d = i % c.qd;  // past the last head: the last again
            qs[i] = (double)gload(a.q + (size_t)row * a.q_stride + (size_t)(kv * a.rep + h0 + h) * c.qd + d);
        }
        __syncthreads();
        // 16 pages a wave, twice.  The means of the next 32 load while these are
        // scored, the table's entries of those after them before.
        constexpr int kStep = kThreads / 64 * 32;
        int id[2];
        half8 m[2][QC], mn[2][QC];
        bool has[2], hasn[2];
        auto load_ids = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const int j = base + 16 * p + (lane >> 2);
                id[p] = j < j1 && j >= a.sinks && j <= cur - a.recent ? gload(table + j) : -1;
            }
        };
        auto load_means = [&](half8 (&m)[2][QC], bool (&has)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                has[p] = (unsigned)id[p] < (unsigned)c.n_pages;
                const __half *mean = c.means + ((size_t)(has[p] ? id[p] : 0) * c.n_kv + kv) * c.qd;
#pragma unroll
                for (int s = 0; s < QC; s++)
                    if (s < nq) m[p][s] = gload((const half8 *)(mean + 32 * s + 8 * e));
            }
        };
        load_ids(j0 + wave * 32);
        load_means(mn, hasn);
        load_ids(j0 + wave * 32 + kStep);
        for (int base = j0 + wave * 32; base < j1; base += kStep) {
            const int j[2] = {base + (lane >> 2), base + 16 + (lane >> 2)};
#pragma unroll
            for (int p = 0; p < 2; p++) {
                has[p] = hasn[p];
#pragma unroll
                for (int s = 0; s < QC; s++) m[p][s] = mn[p][s];
            }
            load_means(mn, hasn);
            load_ids(base + 2 * kStep);
            double acc[2][kHeads];
#pragma unroll
            for (int h = 0; h < kHeads; h++) acc[0][h] = acc[1][h] = 0.0;
#pragma unroll
            for (int s = 0; s < QC; s++) {
                if (s >= nq) break;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    double x[2][2];
#pragma unroll
                    for (int p = 0; p < 2; p++) x[p][0] = (double)(float)m[p][s][i], x[p][1] = (double)(float)m[p][s][i + 1];
#pragma unroll
                    for (int h = 0; h < kHeads; h++) {
                        const f64x2 y = *(const f64x2 *)(qs + h * c.qd + 32 * s + 8 * e + i);
#pragma unroll
                        for (int p = 0; p < 2; p++) acc[p][h] = fma(y[1], x[p][1], fma(y[0], x[p][0], acc[p][h]));
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < 2; p++) {
                uint64_t best = 1;
#pragma unroll
                for (int h = 0; h < kHeads; h++) {
                    double s = acc[p][h];
                    s += __shfl_xor(s, 1, 64);
                    s += __shfl_xor(s, 2, 64);
                    best = max(best, order_of(s));
                }
                if (e == 0 && j[p] < j1) {
                    uint64_t k = has[p] ? best : 1;
                    if (h0 > 0) k = max(k, out[j[p] - j0]);
                    if (j[p] > cur) k = 0;
                    else if (j[p] < a.sinks || j[p] > cur - a.recent) k = ~0ull;
                    out[j[p] - j0] = k;
                }
            }
        }
    }
    __syncthreads();
}

// The first n_sel of n keys in their order, equal ones by index, as ascending
// indices into list.
__device__ inline void pick(const uint64_t *keys, int n, int n_sel, int32_t *list) {
    __shared__ int hist[256], found[kThreads / 64];
    __shared__ int s_digit, s_above, s_here;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t prefix = 0, mask = 0;
    int want = n_sel;  // how many of those that agree with prefix
    bool all = false;  // every one that does
    for (int shift = 56; shift >= 0 && !all; shift -= 8) {
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
    int before = 0, ties = 0;  // chosen pages and those equal to the last one, so far
    for (int base = 0; base < n; base += kThreads) {
        const int j = base + threadIdx.x;
        const uint64_t k = j < n ? keys[j] : 0;
        const bool edge = k != 0 && (k & mask) == prefix;
        bool in = k != 0 && (k & mask) > prefix;
        if (all) {
            in |= edge;
        } else {
            const unsigned long long b = __ballot(edge);
            __syncthreads();
            if (lane == 0) found[wave] = __popcll(b);
            __syncthreads();
            int at = ties + __popcll(b & ((1ull << lane) - 1));
            for (int w = 0; w < wave; w++) at += found[w];
            in |= edge && at < want;
            for (int w = 0; w < kThreads / 64; w++) ties += found[w];
        }
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

// FUSED: score and pick; otherwise pick from the workspace's keys.
template <int QC, bool FUSED>
__global__ __launch_bounds__(kThreads) void kv4_select_kernel(const Args a) {
    __shared__ uint64_t keys[FUSED ? kLdsPages : 1];
    __shared__ double qs[FUSED ? kHeads * QC * 32 : 1];
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
        score_pages<QC>(a, row, kv, sid, cur, 0, cur + 1, qs, keys);
        pick(keys, cur + 1, a.n_sel, list);
    } else {
        pick(a.keys + (size_t)blockIdx.x * a.n, cur + 1, a.n_sel, list);
    }
}

constexpr int kScorePages = 256;  // pages of a block of kv4_score_kernel
template <int QC>
__global__ __launch_bounds__(kThreads) void kv4_score_kernel(const Args a) {
    __shared__ double qs[kHeads * QC * 32];
    const int row = blockIdx.x / a.n_kv, kv = blockIdx.x % a.n_kv;
    const int sid = gload(a.seq + row), top = gload(a.pos + row);
    if (top < 0 || (unsigned)sid >= (unsigned)a.c.n_seq) return;
    const int cur = min(top >> a.c.page_shift, a.n - 1), j0 = blockIdx.y * kScorePages;
    if (cur < a.n_sel || j0 > cur) return;
    score_pages<QC>(a, row, kv, sid, cur, j0, min(cur + 1, j0 + kScorePages), qs, a.keys + (size_t)blockIdx.x * a.n + j0);
}

// Scores of a launch of their own: more pages than LDS holds, or so few
// blocks that each would score many pages alone.
bool apart(int64_t pairs, int n) { return n > kLdsPages || (pairs < 128 && n > 2 * kScorePages); }

template <int QC>
void launch(const Args &a, int rows, hipStream_t s) {
    const unsigned pairs = (unsigned)rows * a.n_kv;
    if (apart(pairs, a.n)) {
        hipLaunchKernelGGL((kv4_score_kernel<QC>), dim3(pairs, (a.n + kScorePages - 1) / kScorePages), dim3(kThreads), 0, s, a);
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
