// attn_paged.cuh -- attention of one token per sequence over the paged int8
// KV cache of kv_append.cuh.
//
// For sequence s with n = length[s] keys, query head h of the group of KV
// head g, key i in page P(i) with codes kq, vq and scales ks, vs:
//   z_i = scale * ks[P(i)] * (q . kq_i),    m = max_i z_i
//   out = (sum_i exp(z_i - m) * vs[P(i)] * vq_i) / (sum_i exp(z_i - m)),
// zeros where n = 0.  Keys at and behind n take no part: their codes are
// finite whatever they hold, and a page without a key below n is not read.
#pragma once

#include <cstdint>

#include "kv_append.cuh"

namespace wl {

struct AttnDecodeParams {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    uint32_t n_pages, page_size, n_kv, head_dim;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const int32_t *length, *page_table;
    uint32_t type, out_type;  // 0 f32, 1 f16, 2 bf16
    uint32_t n_seqs, group, max_pages;
    float scale;
    uint32_t *status;
};

__device__ __forceinline__ float load_typed(const void *base, uint32_t type, size_t at) {
    if (type == 0u) return static_cast<const float *>(base)[at];
    if (type == 1u) return __half2float(static_cast<const __half *>(base)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(base)[at]);
}
__device__ __forceinline__ void store_typed(void *base, uint32_t type, size_t at, float x) {
    if (type == 0u)
        static_cast<float *>(base)[at] = x;
    else if (type == 1u)
        static_cast<__half *>(base)[at] = __float2half_rn(x);
    else
        static_cast<__nv_bfloat16 *>(base)[at] = __float2bfloat16_rn(x);
}

constexpr int PAGED_THREADS = 128;

// One CTA per (query head, sequence); 128 keys a step, one thread a key for
// the scores, one thread a dimension for the values.
__global__ void __launch_bounds__(PAGED_THREADS) attn_decode_i8_kernel(const AttnDecodeParams p) {
    __shared__ float q[128], z[PAGED_THREADS], w[PAGED_THREADS];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, head = blockIdx.x, seq = blockIdx.y, D = p.head_dim;
    const uint32_t h = head / p.group, P = p.page_size;
    int64_t n = __ldg(p.length + seq);
    if (n < 0 || n > (int64_t)p.max_pages * P) {
        if (tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        n = 0;
    }
    if (tid < D) q[tid] = load_typed(p.q, p.type, seq * p.q_stride + (size_t)head * D + tid);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t i0 = 0; i0 < n; i0 += PAGED_THREADS) {
        const int64_t i = i0 + tid;
        float s = -INFINITY, vscale = 0.0f;
        if (i < n) {
            const int32_t page = __ldg(p.page_table + (size_t)seq * p.max_pages + i / P);
            if (page < 0 || (uint32_t)page >= p.n_pages) {
                atomicOr(p.status, WL_DEV_ERR_INDEX);
            } else {
                const size_t block = (size_t)page * p.n_kv + h;
                const int8_t *k = p.kc + (block * P + i % P) * D;
                float d = 0.0f;
                for (uint32_t e = 0; e < D; e += 4) {
                    const char4 c = *reinterpret_cast<const char4 *>(k + e);
                    d = fmaf(q[e], (float)c.x, d);
                    d = fmaf(q[e + 1], (float)c.y, d);
                    d = fmaf(q[e + 2], (float)c.z, d);
                    d = fmaf(q[e + 3], (float)c.w, d);
                }
                s = d * (p.scale * p.ks[block]);
                vscale = p.vs[block];
            }
        }
        z[tid] = s;
        __syncthreads();
        float top = m;
        bool nan = false;
        for (int t = 0; t < PAGED_THREADS; ++t) {
            top = fmaxf(top, z[t]);
            nan |= z[t] != z[t];
        }
        if (nan) top = NAN;
        const float base = top == -INFINITY ? 0.0f : top;
        const float e = __expf(s - base);
        w[tid] = e * vscale;
        const float shrink = __expf(m - base);
        __syncthreads();
        z[tid] = e;
        __syncthreads();
        l *= shrink;
        acc *= shrink;
        for (int t = 0; t < PAGED_THREADS; ++t) l += z[t];
        m = top;
        if (tid < D) {
            for (int t = 0; t < PAGED_THREADS && i0 + t < n; ++t) {
                const int32_t page = __ldg(p.page_table + (size_t)seq * p.max_pages + (i0 + t) / P);
                if (page < 0 || (uint32_t)page >= p.n_pages) continue;
                const size_t block = (size_t)page * p.n_kv + h;
                acc = fmaf(w[t], (float)p.vc[(block * P + (i0 + t) % P) * D + tid], acc);
            }
        }
        __syncthreads();
    }
    if (tid < D)
        store_typed(p.out, p.out_type, seq * p.out_stride + (size_t)head * D + tid,
                    l == 0.0f ? 0.0f : acc / l);
}

}  // namespace wl
