// head_rope.hip — biases, norms and rotation of a step's queries and keys in
// one pass (moe_head_rope_rows).
//
// The reference's attention does this in steps (src/model.rs:707-730): add the
// projections' biases, norm each head (or the whole projection), rotate.  Each
// is a read and a write of every value; here a value is read and written once.
// The arithmetic is that of moe_add_bias, moe_rmsnorm and moe_rope, operation
// by operation and sum by sum, so the results are theirs bit for bit.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gmem.h"
#include "moe_internal.h"
#include "rotate.h"

namespace moe {
int fail(int code, const char *fmt, ...);

namespace {

struct Part {  // the queries, the keys or the values of a call
    const float *x, *bias, *norm;
    float *out;
    int64_t xs, os;
    int heads, span;  // span: heads of a norm
};
struct Args {
    Part part[3];
    const int32_t *pos;
    const float *inv;
    int width, offset, dim, n_inv;
    float eps;
};

// A block of 256 threads takes what one norm spans of a row.  Pairs are read
// and written by one thread each, so rows may be rotated in place.
__global__ __launch_bounds__(256) void head_rope_kernel(const Args a) {
    __shared__ float red[4];
    int s = blockIdx.y, k = 0;
    for (; k < 2 && s >= a.part[k].heads / a.part[k].span; k++) s -= a.part[k].heads / a.part[k].span;
    const Part &p = a.part[k];
    const int64_t row = blockIdx.x;
    const int n = p.span * a.width, at = s * n;
    const float *x = p.x + row * p.xs + at, *bias = p.bias ? p.bias + at : nullptr;
    float *out = p.out + row * p.os + at;
    const float *w = p.norm;
    auto value = [&](int i) { return bias ? x[i] + bias[i] : x[i]; };
    float scale = 1.0f;
    if (w) {
        float ss = 0.0f;
        for (int i = threadIdx.x; i < n; i += 256) {
            const float v = value(i);
            ss = fmaf(v, v, ss);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = (red[0] + red[1]) + (red[2] + red[3]);
        scale = 1.0f / sqrtf(ss / (float)n + a.eps);
    }
    auto normed = [&](int i) { return w ? (value(i) * scale) * w[i] : value(i); };
    const int half = a.dim / 2, turned = k < 2 ? min(half, a.n_inv) : 0;
    const float where = (float)a.pos[row];
    for (int i = threadIdx.x; i < n; i += 256) {
        const int h = i / a.width, d = i - h * a.width - a.offset;
        const bool second = d >= half && d < half + turned;
        if (second) continue;
        const float v = normed(i);
        if (d < 0 || d >= turned) {
            out[i] = v;
            continue;
        }
        const float ang = where * a.inv[d];
        rotate(v, normed(i + half), cosf(ang), sinf(ang), out[i], out[i + half]);
    }
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_head_rope_rows(const moe_head_rope *h, const float *q, int64_t q_stride, const float *k, int64_t k_stride,
                                  const float *v, int64_t v_stride, int32_t rows, const int32_t *pos, float *q_out,
                                  int64_t q_out_stride, float *k_out, int64_t k_out_stride, float *v_out,
                                  int64_t v_out_stride, void *stream) {
    if (!h || h->heads <= 0 || h->n_kv <= 0 || h->width <= 0 || h->offset < 0 || h->dim < 0 || h->dim % 2 || h->n_inv < 0 ||
        (int64_t)h->offset + h->dim > h->width || (h->dim && h->n_inv && !h->inv_freq) || rows < 0 ||
        (int64_t)h->heads * h->width > INT32_MAX / 2 || (int64_t)h->n_kv * h->width > INT32_MAX / 2 ||
        (h->q_span != 1 && h->q_span != h->heads) || (h->k_span != 1 && h->k_span != h->n_kv) ||
        (v && (h->v_width <= 0 || h->v_width > INT32_MAX / 2)))
        return fail(MOE_EINVAL, "moe_head_rope_rows: bad argument (%d rows)", rows);
    if (rows == 0) return MOE_OK;
    if (!q || !k || !pos || !q_out || !k_out || (v && !v_out)) return fail(MOE_EINVAL, "moe_head_rope_rows: bad argument");
    if (h->heads > 30000 || h->n_kv > 30000)  // a grid's second size
        return fail(MOE_EUNSUP, "moe_head_rope_rows: %d heads over %d (up to 30000)", h->heads, h->n_kv);
    if (rows > (1 << 24) - 1) return fail(MOE_EUNSUP, "moe_head_rope_rows: %d rows, up to %d at once", rows, (1 << 24) - 1);
    Args a{};
    a.pos = pos, a.inv = h->inv_freq, a.width = h->width, a.offset = h->offset, a.dim = h->dim, a.n_inv = h->n_inv, a.eps = h->eps;
    a.part[0] = Part{q, h->q_bias, h->q_norm, q_out, q_stride, q_out_stride, h->heads, h->q_norm ? h->q_span : 1};
    a.part[1] = Part{k, h->k_bias, h->k_norm, k_out, k_stride, k_out_stride, h->n_kv, h->k_norm ? h->k_span : 1};
    const int spans = a.part[0].heads / a.part[0].span + a.part[1].heads / a.part[1].span;
    hipLaunchKernelGGL(head_rope_kernel, dim3(rows, spans), dim3(256), 0, (hipStream_t)stream, a);
    if (v) {
        Args b{};
        b.pos = pos, b.inv = nullptr, b.width = h->v_width;
        b.part[0] = b.part[1] = Part{nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 1};
        b.part[2] = Part{v, h->v_bias, nullptr, v_out, v_stride, v_out_stride, 1, 1};
        hipLaunchKernelGGL(head_rope_kernel, dim3(rows, 1), dim3(256), 0, (hipStream_t)stream, b);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "head norm and rotation kernel: %s", hipGetErrorString(e));
}
