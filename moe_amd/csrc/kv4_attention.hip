// kv4_attention.hip — causal attention over the paged 4-bit cache
// (moe_kv4_attention).
//
// One wavefront per (row, query head): a tile's 32 positions at a time, two
// lanes a position for the scores (half of the dims each), a running maximum
// and sum, then each lane its value columns.  All in f32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv4.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

__global__ __launch_bounds__(64) void kv4_attention_kernel(const Kv4 c, const float *__restrict__ q, int64_t qs, int heads,
                                                           float scale, const int32_t *__restrict__ seq,
                                                           const int32_t *__restrict__ pos, int window,
                                                           const int32_t *__restrict__ lists, int n_sel,
                                                           float *__restrict__ out, int64_t os) {
    __shared__ float sq[256], sp[32];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, rep = heads / c.n_kv, kv = h / rep;
    const int sid = seq[r], top = pos[r];
    if (top < 0 || sid < 0 || sid >= c.n_seq) return;
    const int lo = window > 0 ? max(0, top + 1 - window) : 0;
    for (int i = lane; i < c.qd; i += 64) sq[i] = q[(size_t)r * qs + (size_t)h * c.qd + i];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int first = lists ? 0 : lo >> c.page_shift, n = lists ? n_sel : (top >> c.page_shift) + 1;
    int before = -1;
    for (int i = first; i < n; i++) {
        int page = i;
        if (lists) {
            page = lists[((size_t)r * c.n_kv + kv) * n_sel + i];
            const bool skip = page <= before;
            before = page;
            if (skip) continue;
        }
        if (page >= c.max_pages) continue;
        const int id = c.table[(size_t)sid * c.max_pages + page];
        if ((unsigned)id >= (unsigned)c.n_pages) continue;
        for (int t = 0; t < c.tiles(); t++) {
            const int base = (page << c.page_shift) + t * kTile;
            if (base > top || base + kTile <= lo) continue;
            const uint8_t *tile = c.head(id, kv) + (size_t)t * c.tile_bytes;
            const int p = lane & 31, half = lane >> 5, at = base + p;
            float s = 0.0f;
            for (int b = 0; b < c.qd / 32; b++) {
                float sum = 0.0f;
                for (int j = 0; j < 16; j++) {
                    const uint8_t byte = tile[kv4_key_byte(c.qd / 32, p, b, j)];
                    sum = fmaf((float)((int)(half ? byte >> 4 : byte & 15) - 8), sq[32 * b + 16 * half + j], sum);
                }
                s = fmaf(__half2float(((const __half *)(tile + c.k_scales()))[kv4_scale_at(p, b)]), sum, s);
            }
            s = (s + __shfl_xor(s, 32, 64)) * scale;
            const bool seen = at >= lo && at <= top;
            if (!seen) s = -INFINITY;
            float x = s;
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) x = fmaxf(x, __shfl_xor(x, w, 64));
            const float mn = fmaxf(m, x), f = mn == -INFINITY ? 1.0f : expf(m - mn);
            const float e = seen ? expf(s - (mn == -INFINITY ? 0.0f : mn)) : 0.0f;
            m = mn;
            float sum = e;
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor(sum, w, 64);
            l = l * f + sum;
            if (half == 0) sp[p] = e;
            __syncthreads();
            for (int k = 0; k < 4; k++) {
                const int d = lane + 64 * k;
                if (d >= c.vd) continue;
                float acc = 0.0f;  // a tile's sum first: fewer roundings of the long sum
                for (int j = 0; j < 32; j++) {
                    if (base + j < lo || base + j > top) continue;
                    const uint8_t byte = tile[c.v_codes() + kv4_value_byte(c.vd / 32, j, d >> 5, d & 15)];
                    const float dv = __half2float(((const __half *)(tile + c.v_scales()))[kv4_scale_at(j, d >> 5)]);
                    acc = fmaf(sp[j], dv * (float)((int)(d & 16 ? byte >> 4 : byte & 15) - 8), acc);
                }
                o[k] = fmaf(o[k], f, acc);
            }
            __syncthreads();
        }
    }
    for (int k = 0; k < 4; k++) {
        const int d = lane + 64 * k;
        if (d < c.vd) out[(size_t)r * os + (size_t)h * c.vd + d] = l == 0.0f ? 0.0f : o[k] / l;
    }
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_attention_workspace_size(const moe_kv4 *c, int32_t rows, int32_t heads, int32_t max_pos, int32_t window,
                                     int32_t n_sel, uint64_t *bytes) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_attention_workspace_size", c, &a)) return rc;
    if (!bytes || rows < 0 || heads <= 0 || heads % a.n_kv || max_pos < 0 || n_sel < 0)
        return fail(MOE_EINVAL, "moe_kv4_attention_workspace_size: bad argument");
    *bytes = 0;
    return MOE_OK;
}

int moe_kv4_attention(const moe_kv4 *c, const float *q, int64_t q_stride, int32_t rows, int32_t heads, float scale,
                      const int32_t *seq, const int32_t *pos, int32_t max_pos, int32_t window, const int32_t *lists,
                      int32_t n_sel, float *out, int64_t out_stride, void *workspace, uint64_t workspace_bytes,
                      void *stream) {
    Kv4 a;
    if (const int rc = kv4_of("moe_kv4_attention", c, &a)) return rc;
    if ((rows > 0 && (!q || !seq || !pos || !out)) || rows < 0 || heads <= 0 || heads % a.n_kv || max_pos < 0 ||
        max_pos >= (int64_t)a.max_pages << a.page_shift || (lists && n_sel <= 0))
        return fail(MOE_EINVAL, "moe_kv4_attention: bad argument (%d rows, %d heads over %d, max position %d of %lld)",
                    rows, heads, a.n_kv, max_pos, (long long)a.max_pages << a.page_shift);
    if (rows == 0) return MOE_OK;
    hipLaunchKernelGGL(kv4_attention_kernel, dim3(rows, heads), dim3(64), 0, (hipStream_t)stream, a, q, q_stride, heads,
                       scale, seq, pos, window, lists, n_sel, out, out_stride);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "4-bit attention kernel: %s", hipGetErrorString(e));
}

}  // extern "C"
