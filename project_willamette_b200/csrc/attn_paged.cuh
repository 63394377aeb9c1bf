// attn_paged.cuh -- attention of one token per sequence over the paged int8
// KV cache of kv_append.cuh.
//
// For sequence s with n = length[s] keys, query head h of the group of KV
// head g, key i in page P(i) with codes kq, vq and scales ks, vs:
//   z_i = scale * ks[P(i)] * (q . kq_i),    m = max_i z_i
//   out = (sum_i exp(z_i - m) * vs[P(i)] * vq_i) / (sum_i exp(z_i - m)),
// zeros where n = 0.  Keys at and behind n take no part: their codes are
// finite whatever they hold, and a page without a key below n is not read.
//
// Arithmetic.  A warp takes 32 keys at a time on m16n8k16 tiles (f16 x f16 -> f32).
// A code is exact in f16 (its byte under the exponent of 1024, minus 1152).  q, scaled by
// a power of two, and the weights exp(z - m) * 2^14 are each split into two f16 numbers,
// hi in tile rows 0-7 and lo in rows 8-15, so that a tile's 16 rows serve 8 query heads
// with 22 bits and the f32 sums of hi and lo land in the same lane.  exp is 2^x by
// the hardware's approximation (2^-22) of scores in log2 units.  The values' scale
// enters the weights relative to the largest scale so far, as the scores enter
// relative to their maximum.  Groups of more than 8 heads take several passes.
//
// Work.  Units of 128 keys of all (sequence, KV head, pass) items, plus one for each
// item's beginning, are cut into equal contiguous shares, one for each of two CTAs an SM
// (fewer where the page table has no room for as many places), from the lengths on the
// device: no share waits for a long sequence and a captured graph stays balanced as
// lengths grow.  Every warp copies its tiles (8 KB of K and V at D = 128) by TMA into a
// ring of its own, across its segments.  An item cut between CTAs is joined by the last
// CTA to arrive, in CTA order, so results repeat.
//
// Bound by HBM: 2 bytes a key, head and dimension, 4 G flops each.  Over growing lengths the
// time rises at 5.8 TB/s (64 equal sequences of 1024 to 16384 keys, 5 KV heads of 128: 28.0,
// 43.0, 71.3, 128.5, 246.4 us; 4 of 12,500 to 200,000, 4 KV heads: 24.1 to 155.6), 0.88 of a
// plain copy's 6.55: no pipe is full, a warp's chain for one tile and the borders between
// segments hold it.  The rest is a call's beginning and end, 13 to 15 us of such calls and
// 9 of a small one.  Measured (median call in a captured chain; in ordinary launches back to
// back in brackets): 64 sequences to 8192 keys, 5 KV heads of 128, 65.8 us (68.4) = 4.42
// TB/s; 4 sequences to 100,000 keys, 4 KV heads, 74.3 us (79.0) = 4.67 TB/s; 32 sequences to
// 1024 keys, 3 KV heads of 64, 9.8 us; one of 640 keys, 5 heads of 128, 9.0 us.  Three CTAs an
// SM at 168 registers (spilling) instead of two at 212: 64.8, 75.2, 10.1 and 10.7; rings of 24
// KB a warp instead of 16 at D = 128: 67.6, 76.9; rings of 16 KB instead of 24 at D = 64:
// 10.3 for 9.8; CTAs without a place not launched: 9.25 to 9.0.  Steps on the way at 64 x
// 8192: one CTA a (query head, sequence) on the CUDA cores 6169 us; tiles from registers
// 160; TMA rings 95; vector query loads and joins by whole warps 75; three CTAs an SM 71;
// beginnings counted in the shares 64.7; two CTAs again, as above.  Not kept: scores as
// exact s8 products of three query digits (m16n8k32; 71.2: the conversions it saves are
// not what bounds it, and it spills), the joining as a kernel of its own (89.8: a chain of
// calls then waits twice).
#pragma once

#include <cuda.h>

#include <cstdint>

#include "i2s_gemm.cuh"
#include "kv_append.cuh"

namespace wl {

struct AttnDecodeParams {
    const float *ks, *vs;
    uint32_t n_pages, page_shift, n_kv;  // 2^page_shift keys a page
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const int32_t *length, *page_table;
    uint32_t type, out_type;  // 0 f32, 1 f16, 2 bf16
    uint32_t n_seqs, group, max_pages;
    float scale;
    void *workspace;
    uint32_t *status;
};

__device__ __forceinline__ void store_typed(void *base, uint32_t type, size_t at, float x) {
    if (type == 0u)
        static_cast<float *>(base)[at] = x;
    else if (type == 1u)
        static_cast<__half *>(base)[at] = __float2half_rn(x);
    else
        static_cast<__nv_bfloat16 *>(base)[at] = __float2bfloat16_rn(x);
}

constexpr int PAGED_THREADS = 128;
constexpr int PAGED_WARPS = PAGED_THREADS / 32;
constexpr int PAGED_TILE = 32;                           // keys of a warp's step
constexpr int PAGED_UNIT = PAGED_TILE * PAGED_WARPS;     // keys of a CTA's step: the unit of work
constexpr int PAGED_CTAS_PER_SM = 2;
constexpr int PAGED_MAX_CTAS = 148 * PAGED_CTAS_PER_SM;
constexpr int PAGED_JOIN = 16;                          // parts of a row read at once when joined
constexpr int PAGED_ROWS = 8;                            // query heads of one pass over the keys

// Caller's workspace: one arrival counter a CTA (zero between calls), then two partial
// results a CTA (max and sum of each row, unnormalised output rows).
__host__ __device__ constexpr size_t paged_ml_offset() { return (PAGED_MAX_CTAS * 4u + 255u) & ~255u; }
__host__ __device__ constexpr size_t paged_o_offset() {
    return paged_ml_offset() + (size_t)PAGED_MAX_CTAS * 2u * PAGED_ROWS * 8u;
}
__host__ __device__ constexpr size_t paged_workspace_bytes(uint32_t head_dim) {
    return paged_o_offset() + (size_t)PAGED_MAX_CTAS * 2u * PAGED_ROWS * head_dim * 4u;
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two biased codes u = code + 128 in bytes 0 and 2 under the exponent byte of
// 1024: the half is 1024 + u, and minus 1152 the code, both exact.
__device__ __forceinline__ uint32_t unbias(uint32_t h) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(h), "r"(0x64806480u));
    return d;
}
constexpr uint32_t EXP1024 = 0x64646464u;

// v = hi + lo in two f16 with 22 bits between them.
__device__ __forceinline__ void split_f16(float v0, float v1, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(v0, v1);
    const __half2 l = __floats2half2_rn(__fsub_rn(v0, __low2float(h)), __fsub_rn(v1, __high2float(h)));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

template <int D>
struct PagedSmem {
    static constexpr uint32_t STAGES = D == 128 ? 2 : 6;
    static constexpr uint32_t HALF = PAGED_TILE * D;   // a tile's keys; its values follow
    static constexpr uint32_t STAGE = 2u * HALF;
    static constexpr uint32_t WARP = STAGES * STAGE;
    static constexpr size_t DYN = PAGED_WARPS * WARP + 1024;  // + alignment slack
    static_assert(PAGED_ROWS * (D + 8) * 4 <= STAGE, "a warp's output rows fit a stage");
};

struct AttnDecodeMaps {
    CUtensorMap k, v;  // all pages as rows of D bytes; box {D, min(32, page_size)}, swizzle of D bytes
};

// A contiguous run of one item's units, of one CTA.
struct PagedSegment {
    uint32_t seq, h, head, rows;  // sequence, KV head, the pass's first query head and their number
    uint32_t n, u0, u1, n_units;  // keys; units [u0, u1) of the item's n_units
    uint32_t valid;               // 0: the share is used up
    uint64_t item0;               // the item's place: one for its beginning, then one a unit
};

__device__ __forceinline__ uint64_t div_fast(uint64_t a, uint32_t b) {
    return a >> 32 ? a / b : (uint64_t)((uint32_t)a / b);
}

// W consecutive elements, as they lie in memory (16-bit types fill half of raw)
// and, once they are there, as f32.
template <int W>
__device__ __forceinline__ void load_row_part(const void *base, uint32_t type, size_t at, uint4 (&raw)[W / 4]) {
    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(base) + at * (type == 0u ? 4u : 2u));
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
        if (i < W / 8 || type == 0u) raw[i] = __ldg(src + i);
}
template <int W>
__device__ __forceinline__ void prefetch_row_part(const void *base, uint32_t type, size_t at) {
    const uint32_t size = type == 0u ? 4u : 2u;
    asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const uint8_t *>(base) + at * size));
    asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const uint8_t *>(base) + (at + W - 1) * size));
}
template <int W>
__device__ __forceinline__ void row_part_f32(const uint4 (&raw)[W / 4], uint32_t type, float (&x)[W]) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (type == 0u) {
                x[4 * i + k] = __uint_as_float(u[k]);
            } else if (i < W / 8) {
                const float2 f = type == 1u ? __half22float2(*reinterpret_cast<const __half2 *>(&u[k]))
                                            : make_float2(__uint_as_float(u[k] << 16),
                                                          __uint_as_float(u[k] & 0xFFFF0000u));
                x[8 * i + 2 * k] = f.x;
                x[8 * i + 2 * k + 1] = f.y;
            }
        }
    }
}

// A row's output from its sums.  A lane holds values k = lane * D / 32 + i, which
// stand for dimensions (k % 8) * D / 8 + k / 8.
template <int D>
__device__ __forceinline__ void write_output_row(void *out, uint32_t out_type, size_t at,
                                                 const float (&acc)[D / 32], float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const uint32_t k = (threadIdx.x & 31u) * (D / 32) + i;
        store_typed(out, out_type, at + (k & 7u) * (D / 8) + (k >> 3), sum == 0.0f ? 0.0f : acc[i] * inv);
    }
}

// One row of an item from its parts, of CTAs first, first + 1, ..., in that order; by a warp.
template <int D>
__device__ __forceinline__ void join_row(const void *workspace, uint32_t first, uint32_t count, uint32_t r, void *out,
                                         uint32_t out_type, size_t at) {
    constexpr int OV = D / 32, B = PAGED_JOIN;  // values a lane, parts in flight
    const uint32_t lane = threadIdx.x & 31u;
    const auto *ml = reinterpret_cast<const float2 *>(static_cast<const uint8_t *>(workspace) + paged_ml_offset());
    const auto *po = reinterpret_cast<const float *>(static_cast<const uint8_t *>(workspace) + paged_o_offset());
    auto part = [&](uint32_t x) { return ((first + x) * 2u + (x == 0u)) * PAGED_ROWS + r; };
    float mx = -INFINITY, sum = 0.0f, acc[OV];
#pragma unroll
    for (int i = 0; i < OV; ++i) acc[i] = 0.0f;
#pragma unroll 1
    for (uint32_t x0 = 0; x0 < count; x0 += B) {
        float v[B][OV];
        float2 e = make_float2(-INFINITY, 0.0f);
        if (lane < B && x0 + lane < count) e = __ldcg(&ml[part(x0 + lane)]);
#pragma unroll
        for (int x = 0; x < B; ++x) {
            const float *src = po + part(min(x0 + x, count - 1u)) * D + lane * OV;
            if constexpr (OV == 4)
                *reinterpret_cast<float4 *>(v[x]) = __ldcg(reinterpret_cast<const float4 *>(src));
            else
                *reinterpret_cast<float2 *>(v[x]) = __ldcg(reinterpret_cast<const float2 *>(src));
        }
        float top = e.x;
#pragma unroll
        for (int q = B / 2; q; q >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
        top = fmaxf(__shfl_sync(0xffffffffu, top, 0), mx);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float shrink = ex2_approx(mx - ref), f = ex2_approx(e.x - ref);
        mx = top;
        sum = fmaf(sum, shrink, lane < B ? e.y * f : 0.0f);
#pragma unroll
        for (int i = 0; i < OV; ++i) acc[i] *= shrink;
#pragma unroll
        for (int x = 0; x < B; ++x) {
            const float fx = __shfl_sync(0xffffffffu, f, x);
            if (x0 + x < count) {
#pragma unroll
                for (int i = 0; i < OV; ++i) acc[i] = fmaf(v[x][i], fx, acc[i]);
            }
        }
    }
#pragma unroll
    for (int q = B / 2; q; q >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, q);
    write_output_row<D>(out, out_type, at, acc, __shfl_sync(0xffffffffu, sum, 0));
}

// One CTA of PAGED_CTAS_PER_SM per SM takes an equal, contiguous share of all
// (sequence, KV head, pass, 128-key) units; its four warps take 32 keys each,
// every warp through a ring of its own that it fills itself by TMA.
// SMALL: pages of 16 keys, two to a tile; else a tile lies in one page.
template <int D, bool SMALL>
__global__ void __launch_bounds__(PAGED_THREADS, PAGED_CTAS_PER_SM)
    attn_decode_i8_kernel(const __grid_constant__ AttnDecodeMaps maps, const AttnDecodeParams p) {
    using L = PagedSmem<D>;
    constexpr uint32_t ST = L::STAGES;
    constexpr int KW = D / 64;   // 16-byte pieces of a key row that one lane holds
    constexpr int VW = D / 32;   // 4-byte words of a value row that one lane holds
    constexpr int NT = D / 8;    // output tiles of 8 dimensions
    constexpr int OP = D + 8;    // pitch of an output row in shared memory
    constexpr int HN = SMALL ? 2 : 1;  // pages of a tile
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_full[PAGED_WARPS][ST];
    __shared__ uint4 s_q[2][D / 16][32];  // query parts as the tile instructions take them
    __shared__ int32_t s_block[PAGED_WARPS][ST][HN];  // a stage's page * n_kv + head, -1: none
    __shared__ float s_m[PAGED_WARPS][PAGED_ROWS], s_l[PAGED_WARPS][PAGED_ROWS];
    __shared__ unsigned long long s_scan[PAGED_WARPS];
    // the CTA's walk through its share, kept here so that it takes no registers: the segment
    // before, this one and the next; next place, the share's end, s_seq's first place
    __shared__ PagedSegment s_sg[3];
    __shared__ unsigned long long s_at, s_end, s_seq_at, s_quota;
    __shared__ uint32_t s_seq, s_extra, s_last, s_abort;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                ~(uintptr_t)1023);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t g = lane >> 2, c = lane & 3u;  // the tile instructions' row and column group
    const uint32_t shift = SMALL ? 4u : p.page_shift;
    const uint32_t passes = (p.group + PAGED_ROWS - 1) / PAGED_ROWS;
    const uint32_t per = (p.group + passes - 1) / passes;  // query heads a pass
    const uint32_t items = p.n_kv * passes;                // items of a sequence
    const uint32_t b = blockIdx.x;
    if (lane == 0)
        for (uint32_t s = 0; s < ST; ++s) mbar_init(&s_full[warp][s], 1);
    if (tid == 0) s_abort = 0;
    fence_mbar_init();
    pdl_launch_dependents();
    pdl_wait();

    auto units_of = [&](int64_t n) -> uint32_t {  // 0 for an empty or refused sequence
        return n <= 0 || n > ((int64_t)p.max_pages << shift)
                   ? 0u
                   : (uint32_t)((n + PAGED_UNIT - 1) / PAGED_UNIT);
    };
    // Places: each item has one for its beginning (its queries and its joining take about
    // a unit's time) and one a unit.  All places, and the sequence where this CTA's begin
    auto places_of = [&](int32_t n) -> uint32_t {
        const uint32_t u = units_of(n);
        return u ? u + 1u : 0u;
    };
    const int32_t my_n = tid < p.n_seqs ? __ldg(p.length + tid) : 0;
    uint64_t total;
    {
        uint64_t sum = places_of(my_n);
        for (uint32_t s = tid + PAGED_THREADS; s < p.n_seqs; s += PAGED_THREADS) sum += places_of(__ldg(p.length + s));
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_scan[warp] = sum;
        __syncthreads();
        total = (s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3]) * items;
    }
    // the first N CTAs have a share: `extra` of them quota + 1 places, the others quota (at
    // least 1)
    const uint32_t N = (uint32_t)min((uint64_t)gridDim.x, total);
    // the segment at place `at` < s_end, in or behind sequence seq, which has n keys and
    // begins at place seq_at
    auto next_segment = [&](PagedSegment &s, uint64_t at, uint32_t seq, uint64_t seq_at, int32_t n) {
        uint32_t places = places_of(n);
        while (at >= seq_at + (uint64_t)places * items) {  // the next sequence with keys
            seq_at += (uint64_t)places * items;
            n = __ldg(p.length + ++seq);
            places = places_of(n);
        }
        const uint32_t item = (uint32_t)div_fast(at - seq_at, places);
        const uint32_t h = passes == 1u ? item : item / passes, pass = item - h * passes;
        const uint64_t item0 = seq_at + (uint64_t)item * places, stop = min((uint64_t)s_end, item0 + places);
        s.seq = seq;
        s.h = h;
        s.head = h * p.group + pass * per;
        s.rows = min(per, p.group - pass * per);
        s.n = (uint32_t)n;
        s.n_units = places - 1u;
        s.u0 = at == item0 ? 0u : (uint32_t)(at - item0) - 1u;
        s.u1 = (uint32_t)(stop - item0) - 1u;
        s.item0 = item0;
        s.valid = s.u0 < s.u1;  // not where the share ends with an item's beginning
        s_seq = seq;
        s_seq_at = seq_at;
        s_at = stop;
    };
    if (b < N) {
        const uint64_t quota = div_fast(total, N);
        const uint32_t extra = (uint32_t)(total - quota * N);
        const uint64_t begin = quota * b + min(b, extra);
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < p.n_seqs; s0 += PAGED_THREADS) {
            const uint32_t s = s0 + tid;
            const int32_t n = s0 == 0 ? my_n : s < p.n_seqs ? __ldg(p.length + s) : 0;
            const uint64_t u = (uint64_t)places_of(n) * items;
            uint64_t incl = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= (uint32_t)o) incl += y;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = incl;
            __syncthreads();
            uint64_t sum = 0;
#pragma unroll
            for (int w = 0; w < PAGED_WARPS; ++w) {
                if (w == (int)warp) incl += before + sum;
                sum += s_scan[w];
            }
            if (u && incl > begin && incl - u <= begin) {  // one thread
                s_end = begin + quota + (b < extra);
                s_quota = quota;
                s_extra = extra;
                next_segment(s_sg[0], begin, s, incl - u, n);
            }
            before += sum;
            if (before > begin) break;  // the same for every thread
        }
        __syncthreads();
    }
    auto *ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(p.workspace) + paged_ml_offset());
    auto *po = reinterpret_cast<float *>(static_cast<uint8_t *>(p.workspace) + paged_o_offset());

    // table entries of this warp's tile of unit u: keys [u * UNIT + warp * TILE, + TILE);
    // -1 where no key is.  Read ahead; checked when the tile is copied.
    struct Pages {
        int32_t id[HN];
    };
    auto pages_of = [&](uint32_t seq, uint32_t n, uint32_t u) {
        const uint32_t t = u * PAGED_UNIT + warp * PAGED_TILE;
        const int32_t *row = p.page_table + (size_t)seq * p.max_pages + (t >> shift);
        Pages r;
#pragma unroll
        for (int a = 0; a < HN; ++a) r.id[a] = t + 16u * a < n ? __ldg(row + a) : -1;
        return r;
    };
    uint8_t *ring = smem + warp * L::WARP;
    uint32_t issued = 0;  // (lane 0) ring entries filled
    // (lane 0) the tile of unit u into ring entry `entry`, each in turn
    auto issue = [&](uint32_t h, uint32_t n, uint32_t u, uint32_t entry, Pages page) {
        issued = entry + 1u;
        const uint32_t st = entry % ST, t = u * PAGED_UNIT + warp * PAGED_TILE;
        uint8_t *dst = ring + st * L::STAGE;
        uint64_t *bar = &s_full[warp][st];
        uint32_t bytes = 0;
#pragma unroll
        for (int a = 0; a < HN; ++a) {
            const bool good = (uint32_t)page.id[a] < p.n_pages;  // negative ids are large ones
            if (!good && t + 16u * a < n) atomicOr(p.status, WL_DEV_ERR_INDEX);
            page.id[a] = good ? page.id[a] * (int32_t)p.n_kv + (int32_t)h : -1;
            s_block[warp][st][a] = page.id[a];
            bytes += good ? L::STAGE / HN : 0u;
        }
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int a = 0; a < HN; ++a) {
            if (page.id[a] >= 0) {
                const uint32_t row = ((uint32_t)page.id[a] << shift) + (t & ((1u << shift) - 1u) & ~31u);
                tma_load_2d_plain(dst + a * (L::HALF / HN), &maps.k, 0, row, bar);
                tma_load_2d_plain(dst + L::HALF + a * (L::HALF / HN), &maps.v, 0, row, bar);
            }
        }
    };

    uint32_t it = 0;   // ring entries consumed
    Pages ahead[2];    // (lane 0) table entries of the next two tiles to copy
    // a segment's loads in one go: table entries, queries (into L1), then the first
    // tiles' copies; one ring entry stays free for the joining of the segment before
    auto begin_segment = [&](const PagedSegment &s) {
        if (g < s.rows)
            prefetch_row_part<D / 4>(p.q, p.type, s.seq * p.q_stride + (size_t)(s.head + g) * D + c * (D / 4));
        if (lane == 0) {
            const uint32_t seq = s.seq, h = s.h, n = s.n, u0 = s.u0, u1 = s.u1;
            Pages first[ST + 1];
#pragma unroll
            for (uint32_t i = 0; i <= ST; ++i)
                if (u0 + i < u1) first[i] = pages_of(seq, n, u0 + i);
#pragma unroll
            for (uint32_t i = 0; i < ST - 1u; ++i)
                if (u0 + i < u1) issue(h, n, u0 + i, it + i, first[i]);
            ahead[0] = first[ST - 1];
            ahead[1] = first[ST];
        }
    };
    if (b < N && s_sg[0].valid) begin_segment(s_sg[0]);
    // rows of sequences without keys
    for (uint32_t s = b; s < p.n_seqs; s += gridDim.x) {
        const int32_t n = __ldg(p.length + s);
        if (units_of(n) == 0u) {
            if (tid == 0 && n != 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
            for (uint32_t i = tid; i < p.n_kv * p.group * D; i += PAGED_THREADS)
                store_typed(p.out, p.out_type, s * p.out_stride + i, 0.0f);
        }
    }
    if (b >= N || !s_sg[0].valid) return;
    // lane's places in a stage: keys' row g, 16-byte pieces of its four dimensions
    // groups; values' rows 2c, 2c + 1 (and 8 more, 16 more), its D / 8 dimensions
    uint32_t koff[KW], voff[2];
    if constexpr (D == 128) {
        koff[0] = g * 128u + (((2u * c) ^ g) << 4);
        koff[1] = g * 128u + (((2u * c + 1u) ^ g) << 4);
        voff[0] = 2u * c * 128u + ((g ^ (2u * c)) << 4);
        voff[1] = (2u * c + 1u) * 128u + ((g ^ (2u * c + 1u)) << 4);
    } else {
        koff[0] = g * 64u + ((c ^ ((g >> 1) & 3u)) << 4);
        voff[0] = 2u * c * 64u + (((g >> 1) ^ c) << 4) + (g & 1u) * 8u;
        voff[1] = voff[0] + 64u;
    }

    bool ok = true, joining = false;
    uint32_t free_at = 0;  // the ring entry that a segment's joining uses, the same in every warp
    for (uint32_t turn = 0, side = 0;; side ^= 1u) {
        const bool more = ok && s_sg[turn].valid;
        float qf = 0.0f;  // scale * log2(e) * 2^-shift
        if (more) {
            // the pass's query rows: row g as f16 parts hi (tile row g) and lo (row
            // g + 8) of q * 2^shift, its largest |q| brought to [2^13, 2^14).  Kept in
            // shared memory: in registers they measured 9.2, 9.7, 66.5 and 74.6 us against
            // 9.0, 9.8, 65.9 and 74.2 (one of 640 keys, 32 to 1024, 64 to 8192, 4 to 100,000)
            const PagedSegment &sg = s_sg[turn];
            if (joining) begin_segment(sg);
            uint4 raw[D / 16];
#pragma unroll
            for (int i = 0; i < D / 16; ++i) raw[i] = make_uint4(0, 0, 0, 0);
            if (g < sg.rows)
                load_row_part<D / 4>(p.q, p.type, sg.seq * p.q_stride + (size_t)(sg.head + g) * D + c * (D / 4), raw);
            float x[D / 4];
            row_part_f32<D / 4>(raw, p.type, x);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(13 - e) for 2^e <= top < 2^(e + 1), in two factors that are floats
            const int e = top > 0.0f && top < INFINITY
                              ? max((int)(__float_as_uint(top) >> 23), 1) - 127 : 0;
            const int s0 = (13 - e) / 2, s1 = 13 - e - s0;
            const float f0 = __uint_as_float((uint32_t)(127 + s0) << 23);
            const float f1 = __uint_as_float((uint32_t)(127 + s1) << 23);
            qf = p.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - s0) << 23) *
                 __uint_as_float((uint32_t)(127 - s1) << 23);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                if (j / (D / 64) != (int)warp) continue;  // a quarter of them by each warp
                uint4 a;
                split_f16(x[4 * j] * f0 * f1, x[4 * j + 1] * f0 * f1, a.x, a.y);
                split_f16(x[4 * j + 2] * f0 * f1, x[4 * j + 3] * f0 * f1, a.z, a.w);
                s_q[side][j][lane] = a;
            }
        }
        __syncthreads();
        const bool stop = s_abort != 0u;  // a wait ran out: nothing more is read or written
        if (joining && !stop) {  // the warps' shares of the segment before, in warp order
            constexpr int OV = D / 32;  // a warp takes a row, a lane D / 32 of its values
            const PagedSegment &sg = s_sg[turn == 0u ? 2u : turn - 1u];
            const bool whole = sg.u0 == 0 && sg.u1 == sg.n_units;
            const size_t to_row = sg.seq * p.out_stride + (size_t)sg.head * D;
            const uint32_t slot = (b * 2u + (sg.u0 != 0 ? 0u : 1u)) * PAGED_ROWS;
            for (uint32_t r = warp; r < sg.rows; r += PAGED_WARPS) {
                const float mx = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
                const float ref = mx == -INFINITY ? 0.0f : mx;
                float sum = 0.0f, acc[OV];
#pragma unroll
                for (int i = 0; i < OV; ++i) acc[i] = 0.0f;
#pragma unroll
                for (int w = 0; w < PAGED_WARPS; ++w) {
                    const float f = ex2_approx(s_m[w][r] - ref);
                    const float *src = reinterpret_cast<const float *>(smem + w * L::WARP + free_at) + r * OP + lane * OV;
                    sum = fmaf(s_l[w][r], f, sum);
#pragma unroll
                    for (int i = 0; i < OV; ++i) acc[i] = fmaf(src[i], f, acc[i]);
                }
                if (whole) {
                    write_output_row<D>(p.out, p.out_type, to_row + (size_t)r * D, acc, sum);
                } else {
#pragma unroll
                    for (int i = 0; i < OV; ++i) po[(slot + r) * D + lane * OV + i] = acc[i];
                    if (lane == 0) ml[slot + r] = make_float2(mx, sum);
                }
            }
            if (!whole) {  // the last CTA to arrive joins the item's parts
                auto cta_of = [&](uint64_t place) -> uint32_t {
                    const uint64_t quota = s_quota, border = (quota + 1u) * s_extra;
                    if (quota >> 31)
                        return (uint32_t)(place < border ? place / (quota + 1u) : s_extra + (place - border) / quota);
                    return (uint32_t)(place < border ? div_fast(place, (uint32_t)quota + 1u)
                                                     : s_extra + div_fast(place - border, (uint32_t)quota));
                };
                const uint32_t first = sg.u0 == 0u ? b : cta_of(sg.item0 + 1u);
                const uint32_t last = sg.u1 == sg.n_units ? b : cta_of(sg.item0 + sg.n_units);
                __syncthreads();
                if (tid == 0) {
                    uint32_t *counter = static_cast<uint32_t *>(p.workspace) + first, arrived;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                 : "=r"(arrived)
                                 : "l"(counter)
                                 : "memory");
                    s_last = arrived == last - first;
                    if (s_last) *counter = 0u;
                }
                __syncthreads();
                if (s_last)
                    for (uint32_t r = warp; r < sg.rows; r += PAGED_WARPS)
                        join_row<D>(p.workspace, first, last - first + 1u, r, p.out, p.out_type, to_row + (size_t)r * D);
            }
        }
        if (stop || !more) break;
        const uint32_t following = turn == 2u ? 0u : turn + 1u;
        if (tid == PAGED_THREADS - 1) {
            s_sg[following].valid = 0u;
            if (s_at < s_end) next_segment(s_sg[following], s_at, s_seq, s_seq_at, __ldg(p.length + s_seq));
        }
        // the joining's reads and writes of the ring come before the copy that follows
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        const PagedSegment &sg = s_sg[turn];
        const uint32_t seq = sg.seq, h = sg.h, n = sg.n, u1 = sg.u1;
        // the entry that the joining of the segment before had used
        if (lane == 0 && sg.u0 + ST - 1u < u1) issue(h, n, sg.u0 + ST - 1u, it + ST - 1u, ahead[0]);
        __syncwarp();
        int32_t block[HN];
        float ks[HN], vs[HN];
        auto scales = [&](uint32_t entry, int32_t (&blk)[HN], float (&k)[HN], float (&v)[HN]) {
#pragma unroll
            for (int a = 0; a < HN; ++a) {
                blk[a] = s_block[warp][entry % ST][a];
                k[a] = blk[a] >= 0 ? __ldg(p.ks + blk[a]) : 0.0f;
                v[a] = blk[a] >= 0 ? __ldg(p.vs + blk[a]) : 0.0f;
            }
        };
        scales(it, block, ks, vs);

        float m = -INFINITY, l = 0.0f, vref = 0.0f;
        float o[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

        for (uint32_t u = sg.u0; u < u1; ++u, ++it) {
            const uint32_t t0 = u * PAGED_UNIT + warp * PAGED_TILE;
            const uint8_t *st = ring + (it % ST) * L::STAGE;
            int32_t block_next[HN];
            float ks_next[HN], vs_next[HN];
            if (u + 1 < u1) scales(it + 1, block_next, ks_next, vs_next);
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[warp][it % ST], (it / ST) & 1u));
            if (!ok) break;
            if (block[0] >= 0 || block[HN - 1] >= 0) {
                float s[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    uint32_t x[4][4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint4 r = lds128(st + koff[w] + t * 8 * D);
                        x[t][0] = r.x ^ 0x80808080u;
                        x[t][1] = r.y ^ 0x80808080u;
                        x[t][2] = r.z ^ 0x80808080u;
                        x[t][3] = r.w ^ 0x80808080u;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 a = lds128(&s_q[side][4 * w + j][lane]);
                        const uint32_t qa[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            mma_f16(s[t], qa, unbias(__byte_perm(x[t][j], EXP1024, 0x4140)),
                                    unbias(__byte_perm(x[t][j], EXP1024, 0x4342)));
                    }
                }
                // z in log2 units, keys 2c, 2c+1 of each 8
                float z[4][2];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float f = qf * ks[SMALL ? t / 2 : 0];
                    z[t][0] = (s[t][0] + s[t][2]) * f;
                    z[t][1] = (s[t][1] + s[t][3]) * f;
                }
                if (t0 + PAGED_TILE > n || (SMALL && (block[0] | block[HN - 1]) < 0)) {  // not all take part
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (t0 + 8u * t + 2u * c + i >= n || block[SMALL ? t / 2 : 0] < 0)
                                z[t][i] = -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; ++t) top = fmaxf(top, fmaxf(z[t][0], z[t][1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float vtop = fmaxf(fabsf(vs[0]), fabsf(vs[HN - 1]));
                if (__any_sync(0xffffffffu, top > m) || vtop > vref) {
                    const float mn = fmaxf(m, top), vn = fmaxf(vref, vtop);
                    const float shrink = mn == -INFINITY ? 0.0f : ex2_approx(m - mn);
                    const float f = vn > 0.0f ? shrink * (vref / vn) : 0.0f;
                    l *= shrink;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        o[i][0] *= f;
                        o[i][1] *= f;
                        o[i][2] *= f;
                        o[i][3] *= f;
                    }
                    m = mn;
                    vref = vn;
                }
                // weights times 2^14, so that the f16 parts of small ones keep their bits,
                // and relative to the largest scale of the values so far
                const float base = 14.0f - (m == -INFINITY ? 0.0f : m);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    uint32_t w[4];
                    const float va = vs[SMALL ? a : 0];
                    const float r = va == vref ? 1.0f : va / vref;  // vref 0 only with va 0: scaled by 0 at the end
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float e0 = ex2_approx(z[2 * a + i][0] + base);
                        const float e1 = ex2_approx(z[2 * a + i][1] + base);
                        l += e0 + e1;
                        split_f16(e0 * r, e1 * r, w[2 * i], w[2 * i + 1]);
                    }
                    uint32_t v[4][VW];  // value rows 2c, 2c + 1, 2c + 8, 2c + 9 of these 16 keys
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint8_t *src = st + L::HALF + voff[k & 1] + (16 * a + 8 * (k >> 1)) * D;
                        if constexpr (D == 128) {
                            const uint4 y = lds128(src);
                            v[k][0] = y.x ^ 0x80808080u;
                            v[k][1] = y.y ^ 0x80808080u;
                            v[k][2] = y.z ^ 0x80808080u;
                            v[k][3] = y.w ^ 0x80808080u;
                        } else {
                            const uint2 y = *reinterpret_cast<const uint2 *>(src);
                            v[k][0] = y.x ^ 0x80808080u;
                            v[k][1] = y.y ^ 0x80808080u;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        const uint32_t a01 = __byte_perm(v[0][i], v[1][i], 0x5140);
                        const uint32_t a23 = __byte_perm(v[0][i], v[1][i], 0x7362);
                        const uint32_t b01 = __byte_perm(v[2][i], v[3][i], 0x5140);
                        const uint32_t b23 = __byte_perm(v[2][i], v[3][i], 0x7362);
                        mma_f16(o[4 * i], w, unbias(__byte_perm(a01, EXP1024, 0x4140)),
                                unbias(__byte_perm(b01, EXP1024, 0x4140)));
                        mma_f16(o[4 * i + 1], w, unbias(__byte_perm(a01, EXP1024, 0x4342)),
                                unbias(__byte_perm(b01, EXP1024, 0x4342)));
                        mma_f16(o[4 * i + 2], w, unbias(__byte_perm(a23, EXP1024, 0x4140)),
                                unbias(__byte_perm(b23, EXP1024, 0x4140)));
                        mma_f16(o[4 * i + 3], w, unbias(__byte_perm(a23, EXP1024, 0x4342)),
                                unbias(__byte_perm(b23, EXP1024, 0x4342)));
                    }
                }
            }
            __syncwarp();  // the entry is free again
            if (lane == 0 && u + ST < u1) {
                issue(h, n, u + ST, it + ST, ahead[1]);
                if (u + ST + 1u < u1) ahead[1] = pages_of(seq, n, u + ST + 1u);
            }
            __syncwarp();
#pragma unroll
            for (int a = 0; a < HN; ++a) {
                block[a] = block_next[a];
                ks[a] = ks_next[a];
                vs[a] = vs_next[a];
            }
        }
        if (!ok) {
            if (lane == 0) {
                atomicOr(p.status - 1, WL_DEV_ERR_TIMEOUT);
                *(volatile uint32_t *)&s_abort = 1u;
            }
        }
        // this warp's share of the segment.  Output tile i, column n stands for dimension
        // n * D / 8 + i; kept at 8 i + n.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float back = vref * 6.103515625e-05f;  // 2^-14
        free_at = ((it + ST - 1u) % ST) * L::STAGE;
        float *so = reinterpret_cast<float *>(ring + free_at);
#pragma unroll
        for (int i = 0; i < NT; ++i)
            *reinterpret_cast<float2 *>(so + g * OP + 8 * i + 2 * c) =
                make_float2((o[i][0] + o[i][2]) * back, (o[i][1] + o[i][3]) * back);
        if (c == 0) {
            s_m[warp][g] = m;
            s_l[warp][g] = l * 6.103515625e-05f;
        }
        joining = true;
        turn = following;
    }
    // after a wait that ran out: the copies still in flight land before the CTA's shared
    // memory goes
    if (lane == 0)
        for (; it < issued; ++it) mbar_drain(&s_full[warp][it % ST], (it / ST) & 1u);
}

}  // namespace wl
