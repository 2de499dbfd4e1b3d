// pages.hip — block tables and slot maps from request lengths, on the device
// (moe_pages_advance).
//
// plan_pages, one block, four sequences a thread: five running sums over
// them (rows wanted; pages wanted; then rows, pages given back and pages taken
// of those not refused) settle what every sequence gets.  Rows and pages are
// refused by their running sums with the refused ones counted, so those that
// are given pages are the first of those that want any, and their offsets from
// the ring's head are the sums themselves.  Sums saturate (2^30), which keeps
// them associative and above every bound they are compared with.
// put_row: a row finds its sequence among the starts, writes position and slot,
// and enters the page that it opens in the table.  give_back: the pages of a
// sequence that ended, appended to the ring: what is taken lies before head +
// count, what is given back behind it, so the two do not meet.
//
// Latency bound (a few integers per sequence and row), so a step of up to
// 1024 sequences and rows is one launch of one block: 32 sequences 5.4 us (two
// launches, a 1024-thread block and 64-bit sums: 21.5).  Beyond that the rows
// are a launch of their own: 4096 sequences and 100000 rows 14.3 + 6.2 us, the
// first one's five scans, one after the other, and their barriers on one CU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "moe_internal.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

constexpr int kMost = 1 << 30;
constexpr int kMostSeq = 1 << 24;  // blocks of the second launch: 2^22 for them and for the rows

struct Pages {
    const int32_t *length, *add, *state;
    int32_t *length_out, *table, *ring, *state_out, *row_start, *seq, *pos, *status;
    int64_t *slot;
    int32_t *take, *give, *before;  // workspace [n_seq]: first page taken, first given back (or -1), length before
    int32_t *sums;                  // workspace: rows, head, count
    int n_seq, max_pages, shift, n_pages, max_rows;
};

__device__ inline int sat(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kMost); }
__device__ inline int ceil_pages(int n, int shift) { return (int)(((int64_t)n + (1 << shift) - 1) >> shift); }

// Exclusive saturating sums of four values a thread over the block, in place;
// `total` receives the whole.  red: T / 64 ints a call may use until the next
// barrier but one.
template <int T>
__device__ inline void block_scan(int (&v)[4], int *red, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = sat(sat(v[0], v[1]), sat(v[2], v[3]));
    int x = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x = sat(x, y);
    }
    int before = __shfl_up(x, 1, 64);
    before = lane == 0 ? 0 : before;
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        const int s = red[w];
        if (w < wave) before = sat(before, s);
        all = sat(all, s);
    }
    total = all;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int s = v[k];
        v[k] = before;
        before = sat(before, s);
    }
}

// What every sequence gets; start, take, give, before: where the rows' part
// reads it from (memory or LDS).  Returns the rows, the ring's head and count
// as they were.
template <int T>
__device__ inline int plan_pages(const Pages &a, int *red, int *start, int *take, int *give, int *before, int &head,
                                 int &count) {
    const int64_t cap = (int64_t)a.max_pages << a.shift;
    const int h = gload(a.state) % a.n_pages;
    head = h < 0 ? h + a.n_pages : h;
    count = min(max(gload(a.state + 1), 0), a.n_pages);
    int rows1 = 0, wanted = 0, rows = 0, given = 0, taken = 0;  // of the sequences before
    for (int base = 0; base < a.n_seq; base += 4 * T) {
        int len[4], add[4], status[4], old[4], need[4], v[4], total;
        bool ok[4], gone[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = base + 4 * threadIdx.x + k;
            const bool in = i < a.n_seq;
            len[k] = in ? gload(a.length + i) : 0;
            add[k] = in ? gload(a.add + i) : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            len[k] = (int)min((int64_t)max(len[k], 0), cap);
            gone[k] = add[k] < 0;
            ok[k] = !gone[k] && (int64_t)len[k] + add[k] <= cap;
            status[k] = ok[k] || gone[k] ? 0 : 2;
            old[k] = ceil_pages(len[k], a.shift);
            v[k] = ok[k] ? min(add[k], kMost) : 0;
        }
        block_scan<T>(v, red, total);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (ok[k] && add[k] > 0 && sat(rows1, sat(v[k], min(add[k], kMost))) > a.max_rows) ok[k] = false, status[k] = 3;
            need[k] = ok[k] ? ceil_pages(len[k] + add[k], a.shift) - old[k] : 0;
            v[k] = need[k];
        }
        rows1 = sat(rows1, total);
        block_scan<T>(v, red + 16, total);
        int first[4], back[4], took[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            first[k] = sat(wanted, v[k]);
            if (ok[k] && need[k] > 0 && sat(first[k], need[k]) > count) ok[k] = false, status[k] = 1;
            v[k] = ok[k] ? add[k] : 0;
            back[k] = gone[k] ? old[k] : 0;
            took[k] = ok[k] ? need[k] : 0;
        }
        wanted = sat(wanted, total);
        block_scan<T>(v, red + 32, total);
        const int rows0 = rows, given0 = given;
        rows = sat(rows, total);
        block_scan<T>(back, red, total);  // two barriers after its last use
        given = sat(given, total);
        block_scan<T>(took, red + 16, total);
        taken = sat(taken, total);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = base + 4 * threadIdx.x + k;
            if (i >= a.n_seq) continue;
            start[i] = rows0 + v[k];
            take[i] = first[k];
            give[i] = gone[k] ? given0 + back[k] : -1;
            before[i] = len[k];
            a.status[i] = status[k];
            a.length_out[i] = gone[k] ? 0 : ok[k] ? len[k] + add[k] : len[k];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        start[a.n_seq] = rows;
        a.state_out[0] = (int)(((int64_t)head + taken) % a.n_pages);
        a.state_out[1] = min(sat(count - taken, given), a.n_pages);
    }
    return rows;
}

__device__ inline void put_row(const Pages &a, int r, int rows, int head, const int *start, const int *take,
                               const int *before) {
    if (r >= rows) {
        a.seq[r] = a.pos[r] = -1;
        a.slot[r] = -1;
        return;
    }
    // The last sequence that starts at or before r: it has rows.
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int len = before[lo], p = len + r - start[lo];
    const int page = p >> a.shift, old = ceil_pages(len, a.shift), in = p & ((1 << a.shift) - 1);
    int32_t *entry = a.table + (size_t)lo * a.max_pages + page;
    int id;
    if (page < old) {
        id = gload(entry);
    } else {
        id = gload(a.ring + ((int64_t)head + take[lo] + page - old) % a.n_pages);
        if (in == 0) gstore(entry, id);
    }
    a.seq[r] = lo;
    a.pos[r] = p;
    a.slot[r] = ((int64_t)id << a.shift) + in;
}

// `threads` of them together.
__device__ inline void give_back(const Pages &a, int i, int at, int len, int head, int count, int thread, int threads) {
    const int n = ceil_pages(len, a.shift);
    for (int j = thread; j < n; j += threads)
        a.ring[((int64_t)head + count + at + j) % a.n_pages] = gload(a.table + (size_t)i * a.max_pages + j);
}

constexpr int kOneBlock = 1024;  // sequences and rows of a step in one launch

__global__ __launch_bounds__(256) void pages_step_kernel(const Pages a) {
    __shared__ int red[48], start[kOneBlock + 1], take[kOneBlock], give[kOneBlock], before[kOneBlock];
    int head, count;
    const int rows = plan_pages<256>(a, red, start, take, give, before, head, count);
    __syncthreads();
    for (int r = threadIdx.x; r < a.max_rows; r += 256) put_row(a, r, rows, head, start, take, before);
    for (int i = threadIdx.x; i <= a.n_seq; i += 256) a.row_start[i] = start[i];
    // A wave looks at 64 sequences, then copies the pages of those that ended.
    const int lane = threadIdx.x & 63;
    for (int base = threadIdx.x & ~63; base < a.n_seq; base += 256) {
        unsigned long long ended = __ballot(base + lane < a.n_seq && give[min(base + lane, a.n_seq - 1)] >= 0);
        for (; ended; ended &= ended - 1) {
            const int i = base + __builtin_ctzll(ended);
            give_back(a, i, give[i], before[i], head, count, lane, 64);
        }
    }
}

__global__ __launch_bounds__(1024) void pages_plan_kernel(const Pages a) {
    __shared__ int red[48];
    int head, count;
    const int rows = plan_pages<1024>(a, red, a.row_start, a.take, a.give, a.before, head, count);
    if (threadIdx.x == 0) a.sums[0] = rows, a.sums[1] = head, a.sums[2] = count;
}

__global__ __launch_bounds__(256) void pages_rows_kernel(const Pages a, int row_blocks) {
    const int rows = a.sums[0], head = a.sums[1], count = a.sums[2];
    if ((int)blockIdx.x < row_blocks) {
        const int r = blockIdx.x * 256 + threadIdx.x;
        if (r < a.max_rows) put_row(a, r, rows, head, a.row_start, a.take, a.before);
    } else {
        // A wave per sequence.
        const int i = (blockIdx.x - row_blocks) * 4 + (threadIdx.x >> 6);
        if (i < a.n_seq && a.give[i] >= 0) give_back(a, i, a.give[i], a.before[i], head, count, threadIdx.x & 63, 64);
    }
}

uint64_t workspace_of(int n_seq) { return 12 * (uint64_t)n_seq + 16; }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_pages_workspace_size(int32_t n_seq, uint64_t *bytes) {
    if (n_seq <= 0 || !bytes) return fail(MOE_EINVAL, "moe_pages_workspace_size: bad argument");
    *bytes = workspace_of(n_seq);
    return MOE_OK;
}

int moe_pages_advance(int32_t n_seq, const int32_t *length, const int32_t *add, int32_t *length_out, int32_t *table,
                      int32_t max_pages, int32_t page, int32_t *ring, int32_t n_pages, const int32_t *state,
                      int32_t *state_out, int32_t max_rows, int32_t *row_start, int32_t *seq, int32_t *pos,
                      int64_t *slot, int32_t *status, void *workspace, uint64_t workspace_bytes, void *stream) {
    if (!length || !add || !length_out || !table || !ring || !state || !state_out || !row_start || !status ||
        (max_rows > 0 && (!seq || !pos || !slot)) || n_seq <= 0 || max_pages <= 0 || n_pages <= 0 || max_rows < 0 ||
        n_seq > kMostSeq || n_pages > kMost || max_rows >= kMost)
        return fail(MOE_EINVAL, "moe_pages_advance: bad argument (%d sequences of %d pages, pool of %d, %d rows)", n_seq,
                    max_pages, n_pages, max_rows);
    if (page < 32 || page > 4096 || (page & (page - 1)) || (int64_t)max_pages * page > INT32_MAX)
        return fail(MOE_EINVAL, "moe_pages_advance: pages of %d positions, %d of them", page, max_pages);
    if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < workspace_of(n_seq))
        return fail(MOE_EINVAL, "moe_pages_advance: workspace of %llu bytes", (unsigned long long)workspace_bytes);
    Pages a{};
    a.length = length, a.add = add, a.state = state, a.length_out = length_out, a.table = table, a.ring = ring;
    a.state_out = state_out, a.row_start = row_start, a.seq = seq, a.pos = pos, a.status = status, a.slot = slot;
    a.sums = (int32_t *)workspace;
    a.take = a.sums + 4, a.give = a.take + n_seq, a.before = a.give + n_seq;
    a.n_seq = n_seq, a.max_pages = max_pages, a.shift = __builtin_ctz(page), a.n_pages = n_pages, a.max_rows = max_rows;
    hipStream_t s = (hipStream_t)stream;
    if (n_seq <= kOneBlock && max_rows <= kOneBlock) {
        hipLaunchKernelGGL(pages_step_kernel, dim3(1), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, s, a);
        const int row_blocks = (int)(((int64_t)max_rows + 255) / 256), seq_blocks = (int)(((int64_t)n_seq + 3) / 4);
        hipLaunchKernelGGL(pages_rows_kernel, dim3((unsigned)row_blocks + seq_blocks), dim3(256), 0, s, a, row_blocks);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "page tables: %s", hipGetErrorString(e));
}

}  // extern "C"
