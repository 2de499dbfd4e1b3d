// head_rope.hip — biases, norms and rotation of a step's queries and keys in
// one pass (moe_head_rope_rows).
//
// The reference's attention does this in steps (src/model.rs:707-730): add the
// projections' biases, norm each head (or the whole projection), rotate.  Each
// is a read and a write of every value; here a value is read and written once:
// 16376 rows of 32 query and 8 key heads of 128 with norms 169 us (671 MB, 4.0
// TB/s of the copy's 4.7), where the steps took four launches, 32 rows 3.4.  What
// bounds it is the stream; the sines (accurate far beyond 2 pi, so long) are shared
// by a wave's heads.
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

// Heads of up to 256 values whose norms span one head: a wave takes a few heads
// of a row, lane l the values l, l + 64 ... of each.
struct Heads {
    Part part[3];
    const int32_t *pos;
    const float *inv;
    int64_t items;
    int rows, width, offset, half, turned, each, chunks, heads;  // each: heads of a wave; heads: of all parts
    float eps;
};

template <int ROW, int BANKS>
__device__ inline float dpp(float old, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), ROW, 0xf, BANKS, false));
}
// The sum over a wave, lanes 32 apart first, then 16, 8, 4, 2, 1: __shfl_xor's
// order without its trips through LDS.
__device__ inline float wave_sum(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    x += dpp<0x128, 0xf>(x, x);                       // row_ror:8
    x += dpp<0x114, 0xa>(dpp<0x104, 0x5>(x, x), x);   // row_shl:4 for the even fours, row_shr:4 for the odd ones
    x += dpp<0x4e, 0xf>(x, x);                        // quad_perm 2 3 0 1
    x += dpp<0xb1, 0xf>(x, x);                        // quad_perm 1 0 3 2
    return x;
}

// NJ: values of a lane.  PH: a pair's values are 64 PH apart, from 0 on, so that
// one lane has both; 0: anywhere, the pair's other value comes through LDS.
template <int NJ, int PH>
__global__ __launch_bounds__(256) void head_rope_wave_kernel(const Heads a) {
    __shared__ float rows[PH ? 1 : 4][PH ? 1 : 64 * NJ];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    if (item >= a.items) return;
    const int64_t row = item / a.chunks;
    const int h0 = (int)(item - row * a.chunks) * a.each, h1 = min(h0 + a.each, a.heads);
    const int turned_heads = a.part[0].heads + a.part[1].heads;
    float c[NJ], s[NJ], w[2][NJ];
    const float where = (float)gload(a.pos + row);
    bool first[NJ], second[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int e = lane + 64 * j, d = e - a.offset;
        first[j] = d >= 0 && d < a.turned, second[j] = d >= a.half && d < a.half + a.turned;
        c[j] = s[j] = 0.0f;
        if (h0 < turned_heads && (first[j] || (!PH && second[j]))) {
            const float ang = where * gload(a.inv + (first[j] ? d : d - a.half));
            s[j] = sinf(ang), c[j] = cosf(ang);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) w[k][j] = a.part[k].norm && e < a.width ? gload(a.part[k].norm + e) : 1.0f;
    }
    struct At {
        int k;
        int64_t in, out, bias;
    };
    auto find = [&](int h) {
        At x;
        x.k = h < a.part[0].heads ? 0 : h < turned_heads ? 1 : 2;
        const Part &p = a.part[x.k];
        const int64_t n = (int64_t)(h - (x.k == 0 ? 0 : x.k == 1 ? a.part[0].heads : turned_heads)) * a.width;
        x.in = row * p.xs + n, x.out = row * p.os + n, x.bias = n;
        return x;
    };
    auto load = [&](int h, float (&v)[NJ], float (&b)[NJ]) __attribute__((always_inline)) {
        const At x = find(h);
        const Part &p = a.part[x.k];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int e = min(lane + 64 * j, a.width - 1);
            v[j] = gload(p.x + x.in + e);
            b[j] = p.bias ? gload(p.bias + x.bias + e) : 0.0f;
        }
    };
    auto one = [&](int h, float (&v)[NJ], const float (&b)[NJ]) __attribute__((always_inline)) {
        const At x = find(h);
        const Part &p = a.part[x.k];
        if (p.bias)
#pragma unroll
            for (int j = 0; j < NJ; j++) v[j] += b[j];
        if (p.norm) {
            float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NJ; j++) r[j] = wave_sum(lane + 64 * j < a.width ? v[j] * v[j] : 0.0f);
            const float scale = 1.0f / sqrtf(((r[0] + r[1]) + (r[2] + r[3])) / (float)a.width + a.eps);
#pragma unroll
            for (int j = 0; j < NJ; j++) v[j] = (v[j] * scale) * (x.k ? w[1][j] : w[0][j]);
        }
        if (x.k < 2 && a.turned > 0) {
            if (PH) {
#pragma unroll
                for (int j = 0; j + PH < NJ; j++) {
                    if (j >= PH) continue;
                    float y, z;
                    rotate(v[j], v[j + PH], c[j], s[j], y, z);
                    v[j] = first[j] ? y : v[j], v[j + PH] = first[j] ? z : v[j + PH];
                }
            } else {
#pragma unroll
                for (int j = 0; j < NJ; j++) rows[wave][lane + 64 * j] = v[j];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const int e = lane + 64 * j, o = first[j] ? e + a.half : second[j] ? e - a.half : e;
                    const float other = rows[wave][o];
                    float y, z;
                    rotate(first[j] ? v[j] : other, first[j] ? other : v[j], c[j], s[j], y, z);
                    v[j] = first[j] ? y : second[j] ? z : v[j];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++)
            if (lane + 64 * j < a.width) gstore(p.out + x.out + lane + 64 * j, v[j]);
    };
    // Two heads' values in flight beside the one at work.
    float v[3][NJ], b[3][NJ];
    load(h0, v[0], b[0]);
    load(min(h0 + 1, h1 - 1), v[1], b[1]);
    for (int h = h0; h < h1; h += 3) {
#pragma unroll
        for (int u = 0; u < 3; u++) {
            if (h + u >= h1) continue;
            load(min(h + u + 2, h1 - 1), v[(u + 2) % 3], b[(u + 2) % 3]);
            one(h + u, v[u], b[u]);
        }
    }
}

template <int NJ>
void launch_waves(const Heads &a, hipStream_t s) {
    const dim3 grid((unsigned)((a.items + 3) / 4));
    if (a.offset == 0 && a.half == 64 && NJ >= 2) hipLaunchKernelGGL((head_rope_wave_kernel<NJ, NJ >= 2 ? 1 : 0>), grid, dim3(256), 0, s, a);
    else if (a.offset == 0 && a.half == 128 && NJ == 4) hipLaunchKernelGGL((head_rope_wave_kernel<NJ, NJ == 4 ? 2 : 0>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((head_rope_wave_kernel<NJ, 0>), grid, dim3(256), 0, s, a);
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
    hipStream_t st = (hipStream_t)stream;
    const Part parts[3] = {Part{q, h->q_bias, h->q_norm, q_out, q_stride, q_out_stride, h->heads, h->q_norm ? h->q_span : 1},
                           Part{k, h->k_bias, h->k_norm, k_out, k_stride, k_out_stride, h->n_kv, h->k_norm ? h->k_span : 1},
                           Part{v, h->v_bias, nullptr, v_out, v_stride, v_out_stride, 1, 1}};
    const bool waves = h->width <= 256 && parts[0].span == 1 && parts[1].span == 1;
    const bool values = v && waves && h->v_width % h->width == 0 && h->v_width / h->width <= 30000;  // as more heads
    if (waves) {
        Heads a{};
        a.pos = pos, a.inv = h->inv_freq, a.rows = rows, a.width = h->width, a.offset = h->offset, a.half = h->dim / 2;
        a.turned = std::min(a.half, h->n_inv), a.eps = h->eps;
        for (int i = 0; i < 3; i++) a.part[i] = parts[i];
        a.part[2].heads = values ? h->v_width / h->width : 0;
        a.heads = h->heads + h->n_kv + a.part[2].heads;
        // Sines and cosines are a wave's, for all its heads, so it takes up to 48 of
        // them; where there are fewer than 4096 waves, fewer (us at 12, 20, 40 heads
        // a wave: 16376 rows of 32 + 8 heads of 128 183, 172, 169; 4096 rows 41.5,
        // 39.9, 40.1).
        a.each = (int)std::min<int64_t>(48, std::max<int64_t>(1, (int64_t)rows * a.heads / 4096));
        a.chunks = (a.heads + a.each - 1) / a.each;
        a.each = (a.heads + a.chunks - 1) / a.chunks;
        a.items = (int64_t)rows * a.chunks;
        if ((a.items + 3) / 4 > 0xffffff) return fail(MOE_EUNSUP, "moe_head_rope_rows: %d rows of %d heads", rows, a.heads);
        if (h->width <= 64) launch_waves<1>(a, st);
        else if (h->width <= 128) launch_waves<2>(a, st);
        else launch_waves<4>(a, st);
    } else {
        Args a{};
        a.pos = pos, a.inv = h->inv_freq, a.width = h->width, a.offset = h->offset, a.dim = h->dim, a.n_inv = h->n_inv, a.eps = h->eps;
        a.part[0] = parts[0], a.part[1] = parts[1];
        const int spans = parts[0].heads / parts[0].span + parts[1].heads / parts[1].span;
        hipLaunchKernelGGL(head_rope_kernel, dim3(rows, spans), dim3(256), 0, st, a);
    }
    if (v && !values) {
        Args b{};
        b.pos = pos, b.width = h->v_width;
        b.part[0] = b.part[1] = Part{nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 1};
        b.part[2] = parts[2];
        hipLaunchKernelGGL(head_rope_kernel, dim3(rows, 1), dim3(256), 0, st, b);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MOE_OK : fail(MOE_EHIP, "head norm and rotation kernel: %s", hipGetErrorString(e));
}
