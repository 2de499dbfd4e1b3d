// kv8_attention.hip — causal attention over the paged 8-bit cache
// (moe_kv8_attention), layout in kv8.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "kv8.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

struct Args {
    Kv8 c;
    const float *q;
    const int32_t *seq, *pos;
    float *out;
    int64_t q_stride, out_stride;
    int rows, heads, rep, window;
    float scale;
};

// A block takes one row's head, a tile at a time: four threads a position for
// the scores, a thread a dim for the values.
__global__ __launch_bounds__(256) void kv8_attention_kernel(const Args a) {
    __shared__ float sq[256], sp[64], part[4][64];
    const Kv8 &c = a.c;
    const int row = blockIdx.x, head = blockIdx.y, kv = head / a.rep, i = threadIdx.x, p = i & 63, share = i >> 6;
    const int pos = gload(a.pos + row), seq = gload(a.seq + row);
    if (pos < 0 || (unsigned)seq >= (unsigned)c.n_seq) return;
    const float mine = i < c.qd ? gload(a.q + row * a.q_stride + (int64_t)head * c.qd + i) : 0.0f;
    sq[i] = mine;
    const bool lost = __syncthreads_or(!(fabsf(mine) < INFINITY));  // a query that is not finite
    const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int t0 = lo & ~63; t0 <= pos; t0 += 64) {
        const int page = t0 >> c.page_shift, id = page < c.max_pages ? gload(c.table + (int64_t)seq * c.max_pages + page) : -1;
        if ((unsigned)id >= (unsigned)c.n_pages) continue;
        const int64_t tile = c.tile(id, kv, t0 & ((1 << c.page_shift) - 1));
        const uint8_t *codes = c.at(tile);
        __syncthreads();
        float s = 0.0f;
        for (int d = share; d < c.qd; d += 4) s = fmaf(sq[d], (float)(int8_t)gload(codes + kv8_key_byte(c.qd, p, d)), s);
        part[share][p] = s;
        __syncthreads();
        const bool seen = t0 + p >= lo && t0 + p <= pos;
        s = seen ? (((part[0][p] + part[1][p]) + (part[2][p] + part[3][p])) * gload(c.scale_at(tile, true, p >> 4))) * a.scale : -INFINITY;
        float top = s;
        bool bad = lost || s != s || (seen && gload(c.scale_at(tile, false, p >> 4)) != gload(c.scale_at(tile, false, p >> 4)));
        for (int x = 32; x >= 1; x >>= 1) {
            top = fmaxf(top, __shfl_xor(top, x, 64));
            bad |= (bool)__shfl_xor((int)bad, x, 64);
        }
        if (bad) top = __uint_as_float(0x7fc00000u);
        const float m1 = bad || m != m ? __uint_as_float(0x7fc00000u) : fmaxf(m, top);
        const float w = m1 == -INFINITY ? 0.0f : expf(s - m1), f = m1 == -INFINITY ? 1.0f : expf(m - m1);
        m = m1;
        if (share == 0) sp[p] = w;
        float sum = w;
        for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x, 64);
        l = l * f + sum;
        __syncthreads();
        if (i < c.vd) {
            o *= f;
            for (int t = 0; t < 64; t++) {
                if (t0 + t < lo || t0 + t > pos) continue;
                const float v = gload(c.scale_at(tile, false, t >> 4)) * (float)(int8_t)gload(codes + c.values() + kv8_value_byte(t, i));
                o = fmaf(sp[t], v, o);
            }
        }
    }
    if (i < c.vd) gstore(a.out + row * a.out_stride + (int64_t)head * c.vd + i, l == 0.0f ? 0.0f : o / l);
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
    *bytes = 0;
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
    if (heads > 65535 || rows > (1 << 24) - 256) return fail(MOE_EUNSUP, "moe_kv8_attention: %d rows of %d heads", rows, heads);
    a.q = q, a.seq = seq, a.pos = pos, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.rows = rows, a.heads = heads, a.rep = heads / a.c.n_kv, a.window = window, a.scale = scale;
    hipLaunchKernelGGL(kv8_attention_kernel, dim3(rows, heads), dim3(256), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "8-bit attention kernel: %s", hipGetErrorString(e));
}

}  // extern "C"
