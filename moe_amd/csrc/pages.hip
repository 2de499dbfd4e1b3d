// pages.hip — block tables and slot maps from request lengths, on the device
// (moe_pages_advance).
//
// pages_plan_kernel, one block: sequences in chunks of a thread each; three
// running sums over them (rows wanted, pages wanted, then rows, pages given
// back and pages taken of those not refused) settle what every sequence gets.
// Rows and pages are refused by their running sums with the refused ones
// counted, so those that are given pages are the first of those that want any
// and their offsets from the ring's head are the sums themselves.
// pages_rows_kernel: a thread per row finds its sequence among the starts and
// writes position and slot; the row that opens a page enters it in the table.
// A block per sequence that ended appends its pages to the ring: what is
// taken lies before head + count, what is given back behind it, so the two do
// not meet.
//
// Latency bound: a few integers per sequence and row.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "moe_internal.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

struct Pages {
    const int32_t *length, *add, *state;
    int32_t *length_out, *table, *ring, *state_out, *row_start, *seq, *pos, *status;
    int64_t *slot;
    int32_t *take, *give;  // workspace: first page taken, first given back [n_seq]; length before [n_seq]
    int32_t *before;
    int32_t *sums;  // workspace: rows, head, count
    int n_seq, max_pages, shift, n_pages, max_rows;
};

// Exclusive sum over the block's 1024 threads; `total` receives the whole.
__device__ inline int64_t block_scan(int64_t v, int64_t *red, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int64_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        const int64_t s = red[w];
        if (w < wave) base += s;
        all += s;
    }
    __syncthreads();
    total = all;
    return base + x - v;
}

__device__ inline int ceil_pages(int64_t n, int shift) { return (int)((n + (1 << shift) - 1) >> shift); }

__global__ __launch_bounds__(1024) void pages_plan_kernel(const Pages a) {
    __shared__ int64_t red[16];
    const int64_t cap = (int64_t)a.max_pages << a.shift;
    const int h = a.state[0] % a.n_pages, head = h < 0 ? h + a.n_pages : h;
    const int count = min(max(a.state[1], 0), a.n_pages);
    int64_t rows1 = 0, wanted = 0, rows = 0, given = 0, taken = 0;
    for (int base = 0; base < a.n_seq; base += 1024) {
        const int i = base + threadIdx.x;
        const bool in = i < a.n_seq;
        const int64_t len = in ? min(max((int64_t)a.length[i], (int64_t)0), cap) : 0;
        const int64_t add = in ? a.add[i] : 0;
        const bool gone = add < 0;
        int status = 0;
        bool ok = in && !gone;
        if (ok && len + add > cap) ok = false, status = 2;
        int64_t total;
        const int64_t r = ok ? add : 0;
        const int64_t r_end = rows1 + block_scan(r, red, total) + r;
        rows1 += total;
        if (ok && r > 0 && r_end > a.max_rows) ok = false, status = 3;
        const int old = ceil_pages(len, a.shift);
        const int64_t need = ok ? ceil_pages(len + add, a.shift) - old : 0;
        const int64_t first = wanted + block_scan(need, red, total);
        wanted += total;
        if (ok && need > 0 && first + need > count) ok = false, status = 1;
        const int64_t start = rows + block_scan(ok ? add : 0, red, total);
        rows += total;
        const int64_t back = given + block_scan(gone ? old : 0, red, total);
        given += total;
        block_scan(ok ? need : 0, red, total);
        taken += total;
        if (in) {
            a.row_start[i] = (int)start;
            a.status[i] = status;
            a.take[i] = (int)first;
            a.give[i] = gone ? (int)back : -1;
            a.before[i] = (int)len;
            a.length_out[i] = gone ? 0 : (int)(ok ? len + add : len);
        }
    }
    if (threadIdx.x == 0) {
        a.row_start[a.n_seq] = (int)rows;
        a.sums[0] = (int)rows;
        a.sums[1] = head;
        a.sums[2] = count;
        a.state_out[0] = (int)(((int64_t)head + taken) % a.n_pages);
        a.state_out[1] = (int)(count - taken + given);
    }
}

__global__ __launch_bounds__(256) void pages_rows_kernel(const Pages a, int row_blocks) {
    const int rows = a.sums[0], head = a.sums[1], count = a.sums[2];
    if ((int)blockIdx.x >= row_blocks) {
        const int i = blockIdx.x - row_blocks;
        const int at = a.give[i];
        if (at < 0) return;
        const int n = ceil_pages(a.before[i], a.shift);
        for (int j = threadIdx.x; j < n; j += 256)
            a.ring[((int64_t)head + count + at + j) % a.n_pages] = a.table[(size_t)i * a.max_pages + j];
        return;
    }
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= a.max_rows) return;
    if (r >= rows) {
        a.seq[r] = a.pos[r] = -1;
        a.slot[r] = -1;
        return;
    }
    // The last sequence that starts at or before r: it has rows.
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_start[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int len = a.before[lo], p = len + r - a.row_start[lo];
    const int page = p >> a.shift, old = ceil_pages(len, a.shift);
    int32_t *entry = a.table + (size_t)lo * a.max_pages + page;
    int id;
    if (page < old) {
        id = *entry;
    } else {
        id = a.ring[((int64_t)head + a.take[lo] + page - old) % a.n_pages];
        if ((p & ((1 << a.shift) - 1)) == 0) *entry = id;
    }
    a.seq[r] = lo;
    a.pos[r] = p;
    a.slot[r] = ((int64_t)id << a.shift) + (p & ((1 << a.shift) - 1));
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_pages_workspace_size(int32_t n_seq, uint64_t *bytes) {
    if (n_seq <= 0 || !bytes) return fail(MOE_EINVAL, "moe_pages_workspace_size: bad argument");
    *bytes = 12 * (uint64_t)n_seq + 16;
    return MOE_OK;
}

int moe_pages_advance(int32_t n_seq, const int32_t *length, const int32_t *add, int32_t *length_out, int32_t *table,
                      int32_t max_pages, int32_t page, int32_t *ring, int32_t n_pages, const int32_t *state,
                      int32_t *state_out, int32_t max_rows, int32_t *row_start, int32_t *seq, int32_t *pos,
                      int64_t *slot, int32_t *status, void *workspace, uint64_t workspace_bytes, void *stream) {
    if (!length || !add || !length_out || !table || !ring || !state || !state_out || !row_start || !status ||
        (max_rows > 0 && (!seq || !pos || !slot)) || n_seq <= 0 || max_pages <= 0 || n_pages <= 0 || max_rows < 0)
        return fail(MOE_EINVAL, "moe_pages_advance: bad argument (%d sequences of %d pages, pool of %d, %d rows)", n_seq,
                    max_pages, n_pages, max_rows);
    if (page < 32 || page > 4096 || (page & (page - 1)) || (int64_t)max_pages * page > INT32_MAX)
        return fail(MOE_EINVAL, "moe_pages_advance: pages of %d positions, %d of them", page, max_pages);
    if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < 12 * (uint64_t)n_seq + 16)
        return fail(MOE_EINVAL, "moe_pages_advance: workspace of %llu bytes", (unsigned long long)workspace_bytes);
    Pages a{};
    a.length = length, a.add = add, a.state = state, a.length_out = length_out, a.table = table, a.ring = ring;
    a.state_out = state_out, a.row_start = row_start, a.seq = seq, a.pos = pos, a.status = status, a.slot = slot;
    a.sums = (int32_t *)workspace;
    a.take = a.sums + 4, a.give = a.take + n_seq, a.before = a.give + n_seq;
    a.n_seq = n_seq, a.max_pages = max_pages, a.shift = __builtin_ctz(page), a.n_pages = n_pages, a.max_rows = max_rows;
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, s, a);
    const int row_blocks = (int)(((int64_t)max_rows + 255) / 256);
    hipLaunchKernelGGL(pages_rows_kernel, dim3((unsigned)row_blocks + n_seq), dim3(256), 0, s, a, row_blocks);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "page tables: %s", hipGetErrorString(e));
}

}  // extern "C"
