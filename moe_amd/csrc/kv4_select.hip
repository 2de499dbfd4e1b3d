// kv4_select.hip — the pages a query's sparse attention reads (moe_kv4_select).
//
// kv4_score_kernel: a thread per (row, kv head, page), the largest of the
// group's products with the page's mean key in 64 bits (so that which of two
// near pages wins does not hang on the order of a sum), as an integer whose
// order is the score's.  kv4_pick_kernel: a block per (row, kv head); a page's
// rank is the number of pages before it, the first n_sel are written in order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

// A score's place in the order of doubles as unsigned integers, 1 ... 2^64 - 2:
// NaN below every number, 0 free for pages there are not, 2^64 - 1 for forced.
__device__ inline uint64_t order_of(double s) {
    if (s != s) return 1;
    const int64_t b = __double_as_longlong(s);
    return b < 0 ? ~(uint64_t)b : (uint64_t)b | 0x8000000000000000ull;
}

__global__ __launch_bounds__(256) void kv4_score_kernel(const Kv4 c, const float *__restrict__ q, int64_t qs, int heads,
                                                        const int32_t *__restrict__ seq, const int32_t *__restrict__ pos,
                                                        int sinks, int recent, int n, uint64_t *__restrict__ key) {
    const int r = blockIdx.x, kv = blockIdx.y, j = blockIdx.z * 256 + threadIdx.x, rep = heads / c.n_kv;
    if (j >= n) return;
    const int sid = seq[r], top = pos[r];
    uint64_t *dst = key + ((size_t)r * c.n_kv + kv) * n + j;
    const int cur = top >> c.page_shift;
    if (top < 0 || sid < 0 || sid >= c.n_seq || j > cur) {
        *dst = 0;
        return;
    }
    if (j < sinks || j > cur - recent) {
        *dst = ~0ull;
        return;
    }
    const int id = c.table[(size_t)sid * c.max_pages + j];
    uint64_t best = 1;
    if ((unsigned)id < (unsigned)c.n_pages) {
        const __half *mean = c.means + ((size_t)id * c.n_kv + kv) * c.qd;
        for (int h = 0; h < rep; h++) {
            const float *row = q + (size_t)r * qs + (size_t)(kv * rep + h) * c.qd;
            double s = 0.0;
            for (int d = 0; d < c.qd; d++) s = fma((double)row[d], (double)__half2float(mean[d]), s);
            best = max(best, order_of(s));
        }
    }
    *dst = best;
}

__global__ __launch_bounds__(256) void kv4_pick_kernel(const uint64_t *__restrict__ key, int n, int n_sel,
                                                       int32_t *__restrict__ lists) {
    __shared__ int found;
    const uint64_t *k = key + (size_t)blockIdx.x * n;
    int32_t *out = lists + (size_t)blockIdx.x * n_sel;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    for (int base = 0; base < n; base += 256) {
        const int j = base + threadIdx.x;
        bool in = j < n && k[j] != 0;
        if (in) {
            int rank = 0;
            for (int i = 0; i < n; i++) rank += k[i] > k[j] || (k[i] == k[j] && i < j);
            in = rank < n_sel;
        }
        // Chosen pages of these 256 in order.
        const unsigned long long b = __ballot(in);
        __shared__ int waves[4];
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        if (lane == 0) waves[wave] = __popcll(b);
        __syncthreads();
        int at = found + __popcll(b & ((1ull << lane) - 1));
        for (int w = 0; w < wave; w++) at += waves[w];
        if (in && at < n_sel) out[at] = j;
        __syncthreads();
        if (threadIdx.x == 0) found += waves[0] + waves[1] + waves[2] + waves[3];
        __syncthreads();
    }
    for (int i = found + (int)threadIdx.x; i < n_sel; i += 256) out[i] = -1;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_select_workspace_size(const moe_kv4 *c, int32_t rows, int32_t max_pos, uint64_t *bytes) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_select_workspace_size", c, &a)) return rc;
    if (!bytes || rows < 0 || max_pos < 0 || max_pos >= (int64_t)a.max_pages << a.page_shift)
        return fail(MOE_EINVAL, "moe_kv4_select_workspace_size: bad argument");
    *bytes = 8 * (uint64_t)rows * a.n_kv * ((max_pos >> a.page_shift) + 1);
    return MOE_OK;
}

int moe_kv4_select(const moe_kv4 *c, const float *q, int64_t q_stride, int32_t rows, int32_t heads, const int32_t *seq,
                   const int32_t *pos, int32_t max_pos, int32_t sinks, int32_t recent, int32_t n_sel, int32_t *lists,
                   void *workspace, uint64_t workspace_bytes, void *stream) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_select", c, &a)) return rc;
    if (!a.means) return fail(MOE_EINVAL, "moe_kv4_select: the cache keeps no mean keys");
    if ((rows > 0 && (!q || !seq || !pos || !lists)) || rows < 0 || heads <= 0 || heads % a.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.max_pages << a.page_shift)
        return fail(MOE_EINVAL, "moe_kv4_select: bad argument (%d rows, %d heads over %d, max position %d of %lld)", rows,
                    heads, a.n_kv, max_pos, (long long)a.max_pages << a.page_shift);
    if (sinks < 0 || recent < 1 || n_sel < 1 || (int64_t)sinks + recent > n_sel)
        return fail(MOE_EINVAL, "moe_kv4_select: %d first and %d last pages of %d", sinks, recent, n_sel);
    if (rows == 0) return MOE_OK;
    const int n = (max_pos >> a.page_shift) + 1;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < 8 * (uint64_t)rows * a.n_kv * n)
        return fail(MOE_EINVAL, "moe_kv4_select: workspace of %llu bytes", (unsigned long long)workspace_bytes);
    hipStream_t s = (hipStream_t)stream;
    uint64_t *key = static_cast<uint64_t *>(workspace);
    hipLaunchKernelGGL(kv4_score_kernel, dim3(rows, a.n_kv, (n + 255) / 256), dim3(256), 0, s, a, q, q_stride, heads, seq,
                       pos, sinks, recent, n, key);
    hipLaunchKernelGGL(kv4_pick_kernel, dim3((unsigned)rows * a.n_kv), dim3(256), 0, s, key, n, n_sel, lists);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "page selection: %s", hipGetErrorString(e));
}

}  // extern "C"
