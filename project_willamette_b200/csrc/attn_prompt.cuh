// attn_prompt.cuh -- causal attention of packed whole prompts, grouped heads.
//
// Tokens of sequence s are rows [seq_start[s], seq_start[s + 1]) of q, k, v.
// For row i of it and query head h in the group of KV head g:
//   z_j = scale * (q_i . k_j),  j = 0 .. i (rows of the same sequence),
//   out_i = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  m = max_j z_j.
// Rows outside every sequence are left as they were.
#pragma once

#include <cstdint>

#include "attn_paged.cuh"

namespace wl {

struct AttnPromptParams {
    const void *q, *k, *v;
    void *out;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    const int32_t *seq_start;
    uint32_t out_type;  // 0 f32, 1 f16, 2 bf16
    uint32_t n_tokens, n_seqs, group, n_kv;
    float scale;
    uint32_t *status;
};

// One row of the output by one warp: 32 keys a step, a lane a key for the
// scores, D / 32 dimensions a lane for the values.  The rows that the mask
// leaves out are not read, so whatever they hold has no effect.
template <typename T, int D>
__device__ __forceinline__ void prompt_row(const AttnPromptParams &p, int64_t begin, int64_t row,
                                           uint32_t head, uint32_t lane) {
    const uint32_t h = head / p.group;
    const T *q = static_cast<const T *>(p.q) + row * p.q_stride + (size_t)head * D;
    const T *kb = static_cast<const T *>(p.k) + (size_t)h * D;
    const T *vb = static_cast<const T *>(p.v) + (size_t)h * D;
    float m = -INFINITY, l = 0.0f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
    for (int64_t j0 = begin; j0 <= row; j0 += 32) {
        const int64_t j = j0 + lane;
        float z = -INFINITY;
        if (j <= row) {
            float d = 0.0f;
            const T *k = kb + j * p.k_stride;
#pragma unroll
            for (int e = 0; e < D; e += 8) {
                float a[8], b[8];
                load8(q + e, true, a);
                load8(k + e, true, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) d = fmaf(a[i], b[i], d);
            }
            z = d * p.scale;
        }
        float top = z;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, m);
        if (__any_sync(0xffffffffu, z != z)) top = NAN;
        const float base = top == -INFINITY ? 0.0f : top;
        const float shrink = __expf(m - base);
        const float w = __expf(z - base);
        m = top;
        l *= shrink;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= shrink;
        const int count = (int)min((int64_t)32, row - j0 + 1);
        for (int t = 0; t < count; ++t) {
            const float wt = __shfl_sync(0xffffffffu, w, t);
            const T *v = vb + (j0 + t) * p.v_stride;
            l += wt;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(wt, to_f32(v[lane + 32 * i]), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        store_typed(p.out, p.out_type, row * p.out_stride + (size_t)head * D + lane + 32 * i,
                    acc[i] / l);
}

// One warp per (row, head).
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_prompt_rows_kernel(const AttnPromptParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32u;
    if (row >= p.n_tokens) return;
    const uint32_t seq = find_seq(p.seq_start, p.n_seqs, 1u, 0u, (uint32_t)row, lane);
    const int64_t begin = __ldg(p.seq_start + seq), end = __ldg(p.seq_start + seq + 1);
    if (begin < 0 || end < begin || end > (int64_t)p.n_tokens) {
        if (lane == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        return;
    }
    if (row < begin || row >= end) return;
    prompt_row<T, D>(p, begin, row, blockIdx.y, lane);
}

}  // namespace wl
