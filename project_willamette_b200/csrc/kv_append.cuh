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
//          = s_old                      where need <= |s_old|
//          = need                       where s_old = 0
//          = s_old * 2^k                else, k the smallest with |s| >= need;
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
// Bound by memory: inputs and outputs are read and written once.  For each (page that the
// call writes, KV head) as many threads hold the K rows as the V rows in registers (pieces of 8 elements), so the largest |x| and the codes come
// from one pass over the inputs; a thread takes elements j .. j+3 and their partners
// j + n_rot/2 .. of the half layout, so that nothing is loaded twice.  The queries are
// rotated by CTAs of their own in front of those.  Which sequence and page a CTA has
// follows from seq_start alone: sequence s owns the page CTAs [seq_start[s] / P + 2 s,
// seq_start[s + 1] / P + 2 (s + 1)), at least as many as n tokens can touch pages
// (n / P + 2); the rest leave.
// Measured (median call in a captured chain): 64 single tokens, 20 / 5 heads of 128 in f32,
// 4.4 us, of 32 with 9 / 3 heads of 64 3.7 us (a launch and its dependent loads); 512
// tokens with f16 copies 10.7 us; 14,845 bf16 tokens, 32 / 8 heads of 128, pages of 16,
// with copies, 98 us = 4.02 TB/s of inputs and outputs (0.61 of a plain copy; through DRAM
// 3.5, the last outputs stay in L2).  64 % of the issue slots are taken: conversions,
// addresses, and the spills of this instance (104 bytes stored and 156 loaded a thread).
// Queries in the page CTAs and one head a CTA took 141 us; a query warp's pieces share one
// table piece, and 64 registers (four CTAs of 256) beat 80 or 120 with more loads in flight
// (98 against 109 and 217).  At 512 tokens 40 page CTAs with work stand behind 512 of
// queries that hold one token each.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "kv_scale.h"
#include "wl_ptx.cuh"

namespace wl {

// Device status bit: a page id, a position, a length or a sequence's extent
// read on the device lay outside its range; the access was left out.
constexpr uint32_t WL_DEV_ERR_INDEX = 4u;

constexpr uint32_t KV_APPEND_MAX_Q_BLOCK = 64;

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
    uint32_t q_block, q_ctas;  // tokens of a query CTA, and those CTAs (0: no queries)
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

// Four consecutive elements as they lie in memory, src aligned to them, and as f32.
template <typename T>
struct Raw4 {
    using Word = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
    Word w;
    __device__ __forceinline__ void load(const T *src) { w = __ldg(reinterpret_cast<const Word *>(src)); }
    __device__ __forceinline__ void to(float *x) const {
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = to_f32(e[i]);
    }
};
__device__ __forceinline__ void store4(void *base, uint32_t type, size_t at, const float *x) {
    if (type == 0u) {
        *reinterpret_cast<float4 *>(static_cast<float *>(base) + at) = make_float4(x[0], x[1], x[2], x[3]);
        return;
    }
    uint2 w;
    if (type == 1u) {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + at) = w;
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

// Which elements piece i of a row holds: [a, a + 4) and [b, b + 4).  WHOLE: n_rot is a
// multiple of 8, so no piece ends inside the rotated part or inside a half.
template <bool WHOLE>
struct RopePlan {
    uint32_t n_rot, half, pairs;
    __device__ __forceinline__ bool split(uint32_t i) const { return WHOLE && !pairs && i < n_rot / 8u; }
    __device__ __forceinline__ uint32_t a(uint32_t i) const { return split(i) ? 4u * i : 8u * i; }
    __device__ __forceinline__ uint32_t b(uint32_t i) const { return split(i) ? half + 4u * i : 8u * i + 4u; }
};

// The four pairs' (cos, sin) of piece i (WHOLE), from the position's table row `cs`.
struct RopeTerms {
    float c[4], s[4];
    __device__ __forceinline__ void load(const float2 *cs, uint32_t i) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(cs + 4u * i));
        const float4 b = __ldg(reinterpret_cast<const float4 *>(cs + 4u * i) + 1);
        c[0] = a.x, s[0] = a.y, c[1] = a.z, s[1] = a.w;
        c[2] = b.x, s[2] = b.y, c[3] = b.z, s[3] = b.w;
    }
    __device__ __forceinline__ void turn(float &a, float &b, int k) const {
        const float a0 = a;
        a = __fsub_rn(__fmul_rn(a0, c[k]), __fmul_rn(b, s[k]));
        b = __fadd_rn(__fmul_rn(a0, s[k]), __fmul_rn(b, c[k]));
    }
    __device__ __forceinline__ void turn8(float (&x)[8], uint32_t pairs) const {
        if (pairs) {
#pragma unroll
            for (int k = 0; k < 4; ++k) turn(x[2 * k], x[2 * k + 1], k);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) turn(x[k], x[k + 4], k);
        }
    }
};

// Piece i of a row, rotated with the position's table row `cs`.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_piece(const T *row, uint32_t i, const float2 *cs, const RopePlan<WHOLE> &r,
                                           float (&x)[8]) {
    if constexpr (!WHOLE) {
        load_rotated8(row, 8u * i, cs, r.n_rot, r.pairs, x);
    } else {
        Raw4<T> a, b;
        a.load(row + r.a(i));
        b.load(row + r.b(i));
        RopeTerms t;
        const bool turned = i < r.n_rot / 8u;
        if (turned) t.load(cs, i);
        a.to(x);
        b.to(x + 4);
        if (turned) t.turn8(x, r.pairs);
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

// As find_seq, with the sequence's first and last token and (position not NULL) the tokens
// before it.
struct SeqExtent {
    uint32_t seq;
    int32_t begin, end, before;
};
__device__ __forceinline__ SeqExtent find_extent(const int32_t *seq_start, const int32_t *position, uint32_t n_seqs,
                                                 uint32_t size, uint32_t extra, uint32_t u, uint32_t lane) {
    uint32_t lo = 0, n = n_seqs;
    SeqExtent e = {0u, 0, 0, 0};
    if (n == 1u) e = {0u, __ldg(seq_start), __ldg(seq_start + 1), position ? __ldg(position) : 0};
    while (n > 1u) {
        const uint32_t step = (n + 31u) / 32u, s = lo + lane * step;
        bool below = lane * step < n;
        int32_t a = 0, b = 0, before = 0;
        if (below) {
            a = __ldg(seq_start + s);
            if (step == 1u) {  // the last step: what the lane that it ends at needs is loaded beside
                b = __ldg(seq_start + s + 1u);
                if (position) before = __ldg(position + s);
            }
            below = a >= 0 && (uint64_t)((uint32_t)a / size) + (uint64_t)extra * s <= u;
        }
        const uint32_t last = 31u - __clz(__ballot_sync(0xffffffffu, below) | 1u);
        n = min(step, n - last * step);
        lo += last * step;
        if (step == 1u)
            e = {lo, __shfl_sync(0xffffffffu, a, last), __shfl_sync(0xffffffffu, b, last),
                 __shfl_sync(0xffffffffu, before, last)};
        else if (n == 1u)
            e = {lo, __ldg(seq_start + lo), __ldg(seq_start + lo + 1u), position ? __ldg(position + lo) : 0};
    }
    return e;
}

// Named barrier of one half of the CTA.
__device__ __forceinline__ void bar_named(uint32_t id, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Whether a sequence's extent, read on the device, lies within the call's buffers.
__device__ __forceinline__ bool append_extent_ok(const KvAppendParams &p, int64_t begin, int64_t end, int64_t p0) {
    const int64_t n = end - begin;
    return begin >= 0 && n >= 0 && end <= (int64_t)p.n_tokens && p0 >= 0 &&
           p0 + n <= (int64_t)p.max_pages * p.page_size && (!p.n_rot || p0 + n <= (int64_t)p.rope_len);
}

// The rotated queries of `q_block` tokens.
template <typename T, bool WHOLE>
__device__ __forceinline__ void rotate_queries(const KvAppendParams &p, uint32_t block, int32_t *s_pos) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, D = p.head_dim, heads = p.n_kv * p.group;
    const uint32_t t0 = block * p.q_block, count = min(p.q_block, p.n_tokens - t0);
    if (tid < 32u) {
        uint32_t s = find_seq(p.seq_start, p.n_seqs, 1u, 0u, t0, lane);
        for (uint32_t i = lane; i < count; i += 32u) {  // a token's position, -1 where no sequence has it
            while (s + 1u < p.n_seqs && __ldg(p.seq_start + s + 1u) <= (int32_t)(t0 + i)) ++s;
            const int64_t begin = __ldg(p.seq_start + s), end = __ldg(p.seq_start + s + 1u);
            const int64_t p0 = __ldg(p.position + s);
            const bool inside = begin <= (int64_t)(t0 + i) && (int64_t)(t0 + i) < end;
            s_pos[i] = inside && append_extent_ok(p, begin, end, p0) ? (int32_t)(p0 + (t0 + i - begin)) : -1;
        }
    }
    __syncthreads();
    // a warp takes 32 * U pieces of a token at a time
    const RopePlan<WHOLE> r = {p.n_rot, p.n_rot / 2u, p.rope_pairs};
    const uint32_t tshift = D == 128u ? 4u : 3u, row = heads << tshift;
    constexpr int U = 4;  // pieces of a lane in flight
    const uint32_t e = lane & ((1u << tshift) - 1u);  // a lane's pieces are the same one of every head
    const uint32_t runs = (row + 32u * U - 1u) / (32u * U);
    for (uint32_t w = tid >> 5; w < count * runs; w += blockDim.x >> 5) {
        const uint32_t t = w / runs, i0 = (w - t * runs) * 32u * U + lane;
        const int32_t pos = s_pos[t];
        if (pos < 0) continue;
        const T *src = static_cast<const T *>(p.q) + (t0 + t) * p.q_stride;
        const float2 *cs = p.rope + (size_t)pos * r.half;
        const size_t to = (size_t)(t0 + t) * heads * D;
        if constexpr (WHOLE) {
            RopeTerms terms;
            const bool turned = e < r.n_rot / 8u;
            if (turned) terms.load(cs, e);
            Raw4<T> a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = i0 + 32u * u, at = (i >> tshift) * D;
                if (i < row) {
                    a[u].load(src + at + r.a(e));
                    b[u].load(src + at + r.b(e));
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = i0 + 32u * u, at = (i >> tshift) * D;
                if (i < row) {
                    float x[8];
                    a[u].to(x);
                    b[u].to(x + 4);
                    if (turned) terms.turn8(x, r.pairs);
                    store4(p.q_out, p.out_type, to + at + r.a(e), x);
                    store4(p.q_out, p.out_type, to + at + r.b(e), x + 4);
                }
            }
        } else {
            for (uint32_t i = i0; i < min(row, i0 + 32u * U); i += 32u) {
                const uint32_t at = (i >> tshift) * D + 8u * e;
                float x[8];
                load_piece(src + (i >> tshift) * D, e, cs, r, x);
                store4(p.q_out, p.out_type, to + at, x);
                store4(p.q_out, p.out_type, to + at + 4u, x + 4);
            }
        }
    }
}

// rint(x / s) in [-127, 127] of eight values, x / s rounded to f32 first, as two words
// of codes.  x * (1 / s) is within 2^-15 of the quotient for quotients to 128, so it
// rounds to the same whole number unless its fraction is near a half; those pieces, and
// steps whose reciprocal is not a number, divide.
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float s, float inv) {
    constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: v + MAGIC holds rint(v) in its low bits
    float v[8], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = x[i] * inv;
        const float d = fabsf(v[i] - ((v[i] + MAGIC) - MAGIC));
        far = d <= far ? far : d;  // an infinite `inv` makes all eight NaN, the last one too
    }
    if (!(far < 0.4999f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(__fdiv_rn(x[i], s), -127.0f), 127.0f);
    }
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __float_as_uint(v[i] + MAGIC);
    return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
}

// HB KV heads a CTA; of each RT threads for K and RT for V, each with ITS pieces in
// registers.  A page's rows beyond RT * ITS pieces are read twice: for the largest |x|,
// then for the codes.
template <typename T, int ITS, int RT, int HB, bool WHOLE>
__global__ void __launch_bounds__(2 * RT * HB, 1024 / (2 * RT * HB)) kv_append_kernel(const KvAppendParams p) {
    __shared__ uint32_t s_top[2 * HB];
    __shared__ float s_scale[2 * HB];
    __shared__ int s_grow[2 * HB];
    __shared__ SeqExtent s_extent;
    __shared__ int32_t s_pos[KV_APPEND_MAX_Q_BLOCK];
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x < p.q_ctas) {
        rotate_queries<T, WHOLE>(p, blockIdx.x, s_pos);
        return;
    }
    const uint32_t head_ctas = (p.n_kv + HB - 1) / HB;
    const uint32_t unit = (blockIdx.x - p.q_ctas) / head_ctas;
    const uint32_t part = tid / RT, rt = tid % RT, role = part & 1u;  // role 0: K, 1: V
    const uint32_t h = (blockIdx.x - p.q_ctas) % head_ctas * HB + (part >> 1);
    if (tid < 32u) {
        const SeqExtent e = find_extent(p.seq_start, p.position, p.n_seqs, p.page_size, 2u, unit, lane);
        if (lane == 0) s_extent = e;
    }
    if (tid < 2u * HB) s_top[tid] = 0u;
    __syncthreads();
    const uint32_t seq = s_extent.seq, D = p.head_dim, P = p.page_size;
    const int64_t t_begin = s_extent.begin, t_end = s_extent.end, p0 = s_extent.before;
    if (t_begin == t_end || h >= p.n_kv) return;  // the barriers below are each of one part
    if (!append_extent_ok(p, t_begin, t_end, p0)) {
        if (tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        return;
    }
    const int64_t n = t_end - t_begin, u0 = t_begin / P + 2 * (int64_t)seq;
    if ((int64_t)unit < u0) return;
    const int64_t j = p0 / P + ((int64_t)unit - u0);  // the page's index in the sequence
    if (j * P >= p0 + n) return;
    const int32_t page = __ldg(p.page_table + (size_t)seq * p.max_pages + j);
    // the call's tokens in this page: positions [a, b)
    const int64_t a = max(p0, j * P), b = min(p0 + n, (j + 1) * P);
    const uint32_t first = (uint32_t)(a - j * P), rows = (uint32_t)(b - a);
    const int64_t t0 = t_begin + (a - p0);
    const RopePlan<WHOLE> plan = {p.n_rot, p.n_rot / 2u, p.rope_pairs};
    const T *src = static_cast<const T *>(role ? p.v : p.k) + (size_t)h * D;
    const uint64_t stride = role ? p.v_stride : p.k_stride;
    void *copy = role ? p.v_out : p.k_out;
    const uint32_t tpr = D / 8u, i8 = rt % tpr, r0 = rt / tpr, rstep = RT / tpr;  // threads a row
    const uint32_t ea = role ? 8u * i8 : plan.a(i8), eb = role ? 8u * i8 + 4u : plan.b(i8);
    float x[ITS][8];
    auto load_rows = [&](uint32_t from) {
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
            const uint32_t row = from + r0 + it * rstep;
            if (row < rows) {
                const T *base = src + (t0 + row) * stride;
                if (role == 0u)
                    load_piece(base, i8, p.rope + (size_t)(a + row) * plan.half, plan, x[it]);
                else
                    load8(base + 8u * i8, true, x[it]);
            }
        }
    };
    const uint32_t chunk = ITS * rstep;  // rows in registers at a time
    uint32_t top = 0u;
    for (uint32_t from = 0; from < rows; from += chunk) {
        load_rows(from);
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
            const uint32_t row = from + r0 + it * rstep;
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[it][i]) & 0x7FFFFFFFu);
                if (copy) {
                    const size_t to = ((size_t)(t0 + row) * p.n_kv + h) * D;
                    store4(copy, p.out_type, to + ea, x[it]);
                    store4(copy, p.out_type, to + eb, x[it] + 4);
                }
            }
        }
    }
    if (page < 0 || (uint32_t)page >= p.n_pages) {  // the same for every thread
        if (tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
        return;
    }
    const size_t block = (size_t)page * p.n_kv + h;
    float *scale = (role ? p.vs : p.ks) + block;
    int8_t *codes = (role ? p.vc : p.kc) + block * P * D;
    const float old = rt == 0 && first != 0u ? *scale : 0.0f;
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && top) atomicMax(&s_top[part], top);
    bar_named(1u + part, RT);
    if (rt == 0) {
        // bit patterns of |x| order as the values do, infinities and NaN above
        const uint32_t m = s_top[part];
        const float nan = __uint_as_float(0x7FC00000u);
        const float need = m >= 0x7F800000u ? nan : __fdiv_rn(__uint_as_float(m), 127.0f);
        PageScale g = {need, 0};
        if (first != 0u) g = grown_scale(old, need);
        *scale = g.scale;
        s_scale[part] = g.scale;
        s_grow[part] = g.doublings;
    }
    bar_named(1u + part, RT);
    const float s = s_scale[part];
    const float inv = 1.0f / s;
    const int grow = s_grow[part];
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
    for (uint32_t from = 0; from < rows; from += chunk) {
        if (rows > chunk) load_rows(from);
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
            const uint32_t row = from + r0 + it * rstep;
            if (row < rows) {
                const uint2 w = fabsf(s) > 0.0f ? quantise8(x[it], s, inv) : make_uint2(0u, 0u);
                int8_t *to = codes + (size_t)(first + row) * D;
                *reinterpret_cast<uint32_t *>(to + ea) = w.x;
                *reinterpret_cast<uint32_t *>(to + eb) = w.y;
            }
        }
    }
}

}  // namespace wl
