// kv_append.cuh -- appending keys and values to a paged int8 KV cache, with the
// rotation to their positions applied on the way.
//
// For token t of a sequence, at position p, and a head's row x[0 .. D):
//   rotation, over the first n_rot elements, (c_j, s_j) = rope[p][j]:
//     a' = a c_j - b s_j,   b' = a s_j + b c_j,   each product and sum rounded
//     to f32, pairs (a, b) = (x_j, x_{j + n_rot/2}) or (x_{2j}, x_{2j+1});
//   the page's scale (one for each page and KV head, of K and of V apart):
//     need = (largest |x| of the call's new rows in the page) / 127
//     s    = need                       where the call begins the page
//          = s_old                      where need <= s_old
//          = need                       where s_old = 0
//          = s_old * 2^k                else, k the smallest with s >= need;
//     the codes in front of the new ones become rint(code / 2^k);
//   codes  rint(x / s) in [-127, 127], 0 where s is 0 or NaN.
// A scale grows by whole doublings because the codes that are there already
// are rounded again each time it grows: after doublings k1, k2, ... their
// error is at most (1/2 + 1/4 + 1/8 + ...) steps of the last scale, below one
// step however many tokens come one by one (growing to the exact maximum
// each time would add half a step with every new maximum).  A NaN or an
// infinity among the new rows makes the page's scale NaN, so that whatever
// reads the page shows it, and the codes 0.
//
// One CTA for each (page that the call writes, KV head): half of its threads
// hold the K rows and half the V rows in registers (8 elements a thread and
// row), so the largest |x| and the codes come from one pass over the inputs;
// the group's query heads of the same tokens are rotated by the same CTA.
// Bound by memory: inputs and outputs are read and written once.  Which
// sequence and page a CTA has follows from seq_start alone: sequence s owns
// the CTAs [seq_start[s] / P + 2 s, seq_start[s + 1] / P + 2 (s + 1)), at
// least as many as n tokens can touch pages (n / P + 2); the rest leave.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "wl_ptx.cuh"

namespace wl {

// Device status bit: a page id, a position, a length or a sequence's extent
// read on the device lay outside its range; the access was left out.
constexpr uint32_t WL_DEV_ERR_INDEX = 4u;

struct KvAppendParams {
    int8_t *kc, *vc;
    float *ks, *vs;
    uint32_t n_pages, page_size, n_kv, head_dim;
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    const int32_t *seq_start, *position, *page_table;
    const float2 *rope;
    void *q_out, *k_out, *v_out;
    uint32_t out_type;  // 0 f32, 1 f16, 2 bf16
    uint32_t n_tokens, n_seqs, group, max_pages, n_rot, rope_len, rope_pairs;
    uint32_t *status;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Eight consecutive elements as f32; src 16-byte aligned when `vec`.
template <typename T>
__device__ __forceinline__ void load8(const T *src, bool vec, float (&x)[8]) {
    if (vec) {
        uint4 raw[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            raw[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(src[i]);
    }
}

// Eight consecutive elements of a dense output row, rounded once to its type.
__device__ __forceinline__ void store8(void *base, uint32_t type, size_t at, const float (&x)[8]) {
    if (type == 0u) {
        float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    uint4 w;
    uint32_t *p = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == 1u) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            p[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + at) = w;
}

// Elements e .. e+7 of a row, rotated with the position's table row `cs`.
template <typename T>
__device__ __forceinline__ void load_rotated8(const T *row, uint32_t e, const float2 *cs,
                                              uint32_t n_rot, uint32_t pairs, float (&x)[8]) {
    load8(row + e, true, x);
    if (e >= n_rot) return;
    const uint32_t half = n_rot / 2u;
    if (pairs) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (e + i < n_rot) {
                const float2 t = __ldg(cs + (e + i) / 2u);
                const float a = x[i], b = x[i + 1];
                x[i] = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
                x[i + 1] = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
            }
        }
        return;
    }
    if (e + 8u <= half || (e >= half && e + 8u <= n_rot)) {  // all eight on one side
        const bool lo = e < half;
        const uint32_t j = lo ? e : e - half, partner = lo ? e + half : e - half;
        float y[8];
        load8(row + partner, (half & 7u) == 0u, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 t = __ldg(cs + j + i);
            x[i] = lo ? __fsub_rn(__fmul_rn(x[i], t.x), __fmul_rn(y[i], t.y))
                      : __fadd_rn(__fmul_rn(y[i], t.y), __fmul_rn(x[i], t.x));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t m = e + i;
        if (m < n_rot) {
            const bool lo = m < half;
            const float2 t = __ldg(cs + (lo ? m : m - half));
            const float y = to_f32(row[lo ? m + half : m - half]);
            x[i] = lo ? __fsub_rn(__fmul_rn(x[i], t.x), __fmul_rn(y, t.y))
                      : __fadd_rn(__fmul_rn(y, t.y), __fmul_rn(x[i], t.x));
        }
    }
}

// The unit (block of `size` tokens, with `extra` units to spare a sequence)
// u's sequence: the last s with seq_start[s] / size + extra * s <= u.  A warp
// probes 32 borders a step.  The borders ascend strictly when seq_start
// does not descend, which the caller checks for the sequence it gets.
__device__ __forceinline__ uint32_t find_seq(const int32_t *seq_start, uint32_t n_seqs,
                                             uint32_t size, uint32_t extra, uint32_t u,
                                             uint32_t lane) {
    uint32_t lo = 0, n = n_seqs;  // the answer is in [lo, lo + n)
    while (n > 1u) {
        const uint32_t step = (n + 31u) / 32u, s = lo + lane * step;
        bool below = lane * step < n;
        if (below) {
            const int32_t a = __ldg(seq_start + s);
            below = a >= 0 && (uint64_t)((uint32_t)a / size) + (uint64_t)extra * s <= u;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, below) | 1u;
        const uint32_t last = 31u - __clz(m);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

// Named barrier of one half of the CTA.
__device__ __forceinline__ void bar_named(uint32_t id, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// RT threads for K and RT for V, each with ITS rows' pieces of 8 elements:
// RT * ITS * 8 = page_size * head_dim at least.
template <typename T, int ITS, int RT>
__global__ void __launch_bounds__(2 * RT) kv_append_kernel(const KvAppendParams p) {
    __shared__ uint32_t s_top[2];
    __shared__ float s_scale[2];
    __shared__ int s_grow[2];
    __shared__ uint32_t s_seq;
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    pdl_launch_dependents();
    pdl_wait();
    if (tid < 32u) {
        const uint32_t s = find_seq(p.seq_start, p.n_seqs, p.page_size, 2u, blockIdx.x, lane);
        if (lane == 0) s_seq = s;
    }
    if (tid < 2u) s_top[tid] = 0u;
    __syncthreads();
    const uint32_t seq = s_seq, h = blockIdx.y, D = p.head_dim, P = p.page_size;
    const int64_t t_begin = __ldg(p.seq_start + seq), t_end = __ldg(p.seq_start + seq + 1);
    const int64_t p0 = __ldg(p.position + seq);
    if (t_begin == t_end) return;
    const int64_t n = t_end - t_begin;
    if (t_begin < 0 || n < 0 || t_end > (int64_t)p.n_tokens || p0 < 0 ||
        p0 + n > (int64_t)p.max_pages * P || (p.n_rot && p0 + n > (int64_t)p.rope_len)) {
        if (tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        return;
    }
    const int64_t u0 = t_begin / P + 2 * (int64_t)seq;
    if ((int64_t)blockIdx.x < u0) return;
    const int64_t j = p0 / P + ((int64_t)blockIdx.x - u0);  // the page's index in the sequence
    if (j * P >= p0 + n) return;
    // the call's tokens in this page: positions [a, b)
    const int64_t a = max(p0, j * P), b = min(p0 + n, (j + 1) * P);
    const uint32_t first = (uint32_t)(a - j * P), rows = (uint32_t)(b - a);
    const int64_t t0 = t_begin + (a - p0);
    const uint32_t half = p.n_rot / 2u;
    const uint32_t tpr = D / 8u;  // threads a row

    // the group's query heads of these tokens; they start at the second warp,
    // so that a single token's K row (first warp) does not wait behind them
    if (p.q_out) {
        const uint32_t items = rows * p.group * tpr;
        for (uint32_t i = (tid + 2u * RT - 32u) % (2u * RT); i < items; i += 2u * RT) {
            const uint32_t e = i % tpr * 8u, r = i / tpr, g = r % p.group, row = r / p.group;
            const uint32_t head = h * p.group + g;
            const int64_t t = t0 + row;
            float x[8];
            load_rotated8(static_cast<const T *>(p.q) + t * p.q_stride + (size_t)head * D, e,
                          p.rope + (size_t)(a + row) * half, p.n_rot, p.rope_pairs, x);
            store8(p.q_out, p.out_type, ((size_t)t * p.n_kv * p.group + head) * D + e, x);
        }
    }

    const uint32_t role = tid / RT, rt = tid % RT;  // 0: K, 1: V
    const T *src = static_cast<const T *>(role ? p.v : p.k);
    const uint64_t stride = role ? p.v_stride : p.k_stride;
    void *copy = role ? p.v_out : p.k_out;
    const uint32_t e = rt % tpr * 8u, r0 = rt / tpr, rstep = RT / tpr;
    float x[ITS][8];
    uint32_t top = 0u;
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
        const uint32_t row = r0 + it * rstep;
        if (row < rows) {
            const T *base = src + (t0 + row) * stride + (size_t)h * D;
            if (role == 0u)
                load_rotated8(base, e, p.rope + (size_t)(a + row) * half, p.n_rot, p.rope_pairs,
                              x[it]);
            else
                load8(base + e, true, x[it]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[it][i]) & 0x7FFFFFFFu);
            if (copy)
                store8(copy, p.out_type, ((size_t)(t0 + row) * p.n_kv + h) * D + e, x[it]);
        }
    }
    const int32_t page = __ldg(p.page_table + (size_t)seq * p.max_pages + j);
    if (page < 0 || (uint32_t)page >= p.n_pages) {  // the same for every thread
        if (tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        return;
    }
    const size_t block = (size_t)page * p.n_kv + h;
    float *scale = (role ? p.vs : p.ks) + block;
    int8_t *codes = (role ? p.vc : p.kc) + block * P * D;
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && top) atomicMax(&s_top[role], top);
    bar_named(1u + role, RT);
    if (rt == 0) {
        // bit patterns of |x| order as the values do, infinities and NaN above
        const uint32_t m = s_top[role];
        float need = __fdiv_rn(__uint_as_float(m), 127.0f), s = need;
        int k = 0;
        if (m >= 0x7F800000u) need = s = __uint_as_float(0x7FC00000u);
        if (first != 0u) {
            const float old = *scale;
            if (!(need == need) || !(old == old)) {
                s = __uint_as_float(0x7FC00000u);
            } else if (need <= old) {
                s = old;
            } else if (old != 0.0f) {
                s = old;
                while (s < need) {  // at most 2^8 + 2^5 doublings between two floats
                    s *= 2.0f;
                    ++k;
                }
            }
        }
        *scale = s;
        s_scale[role] = s;
        s_grow[role] = k;
    }
    bar_named(1u + role, RT);
    const float s = s_scale[role];
    const int grow = s_grow[role];
    if (grow) {  // the codes in front of the new ones
        const float f = ldexpf(1.0f, -min(grow, 100));
        for (uint32_t i = rt; i < first * tpr; i += RT) {
            uint2 *at = reinterpret_cast<uint2 *>(codes + (size_t)i * 8u);
            uint2 w = *at;
            int8_t *c = reinterpret_cast<int8_t *>(&w);
#pragma unroll
            for (int m = 0; m < 8; ++m) c[m] = (int8_t)__float2int_rn((float)c[m] * f);
            *at = w;
        }
    }
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
        const uint32_t row = r0 + it * rstep;
        if (row < rows) {
            uint2 w = make_uint2(0u, 0u);
            if (s > 0.0f) {
                int q[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    q[i] = max(-127, min(127, __float2int_rn(__fdiv_rn(x[it][i], s))));
                w = make_uint2(pack_i8x4(q[0], q[1], q[2], q[3]), pack_i8x4(q[4], q[5], q[6], q[7]));
            }
            *reinterpret_cast<uint2 *>(codes + (size_t)(first + row) * D + e) = w;
        }
    }
}

}  // namespace wl
