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
constexpr int PAGED_WARPS = PAGED_THREADS / 32;
constexpr int PAGED_TILE = 32;                           // keys of a warp's step
constexpr int PAGED_UNIT = PAGED_TILE * PAGED_WARPS;     // keys of a CTA's step: the unit of work
constexpr int PAGED_CTAS_PER_SM = 2;
constexpr int PAGED_MAX_CTAS = 148 * PAGED_CTAS_PER_SM;
constexpr int PAGED_ROWS = 8;                            // query heads of one pass over the keys

// Caller's workspace: one arrival counter a CTA, then two partial results a
// CTA (max and sum of each row, unnormalised output rows).
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
    static constexpr uint32_t STAGES = D == 128 ? 3 : 6;
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
    uint32_t seq, h, row0, rows;   // sequence, KV head, the pass's query heads within the group
    uint32_t n, u0, u1, n_units;   // keys; units [u0, u1) of the item's n_units
    uint64_t item0;                // the item's first unit
};

__device__ __forceinline__ uint64_t div_fast(uint64_t a, uint32_t b) {
    return a >> 32 ? a / b : (uint64_t)((uint32_t)a / b);
}

// W = D / 4 consecutive elements as f32.
template <int W>
__device__ __forceinline__ void load_row_part(const void *base, uint32_t type, size_t at, float (&x)[W]) {
    if (type == 0u) {
        const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const float4 v = __ldg(src + i);
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
        }
        return;
    }
    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at);
    uint4 raw[W / 8];
#pragma unroll
    for (int i = 0; i < W / 8; ++i) raw[i] = __ldg(src + i);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
        const uint32_t u = i % 4 == 0 ? raw[i / 4].x : i % 4 == 1 ? raw[i / 4].y : i % 4 == 2 ? raw[i / 4].z : raw[i / 4].w;
        if (type == 1u) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(u << 16);
            x[2 * i + 1] = __uint_as_float(u & 0xFFFF0000u);
        }
    }
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
    __shared__ int32_t s_block[PAGED_WARPS][ST][HN];  // a stage's page * n_kv + head, -1: none
    __shared__ float s_m[PAGED_WARPS][PAGED_ROWS], s_l[PAGED_WARPS][PAGED_ROWS];
    __shared__ unsigned long long s_scan[PAGED_WARPS];
    __shared__ unsigned long long s_start;
    __shared__ uint32_t s_seq, s_last, s_abort;
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
    auto units_at = [&](uint32_t s) { return units_of(__ldg(p.length + s)); };
    // all units, and the sequence in which this CTA's share begins
    const uint32_t mine = tid < p.n_seqs ? units_at(tid) : 0u;
    uint64_t total;
    {
        uint64_t sum = mine;
        for (uint32_t s = tid + PAGED_THREADS; s < p.n_seqs; s += PAGED_THREADS) sum += units_at(s);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_scan[warp] = sum;
        __syncthreads();
        total = (s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3]) * items;
    }
    // N CTAs with a share: `extra` of them have quota + 1 units, the others quota (at least 1)
    const uint32_t N = (uint32_t)min((uint64_t)gridDim.x, total);
    const uint64_t quota = N ? div_fast(total, N) : 0u;
    const uint32_t extra = (uint32_t)(total - quota * N);
    const uint64_t begin = quota * b + min(b, extra), end = begin + quota + (b < extra);
    auto cta_of = [&](uint64_t unit) -> uint32_t {
        const uint64_t split = (quota + 1u) * extra;
        if (quota >> 31) return (uint32_t)(unit < split ? unit / (quota + 1u) : extra + (unit - split) / quota);
        return (uint32_t)(unit < split ? div_fast(unit, (uint32_t)quota + 1u)
                                       : extra + div_fast(unit - split, (uint32_t)quota));
    };
    if (b < N) {
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < p.n_seqs; s0 += PAGED_THREADS) {
            const uint32_t s = s0 + tid;
            const uint64_t u = (uint64_t)(s0 == 0 ? mine : s < p.n_seqs ? units_at(s) : 0u) * items;
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
            if (u && incl > begin && incl - u <= begin) {
                s_seq = s;
                s_start = incl - u;
            }
            before += sum;
            if (before > begin) break;  // the same for every thread
        }
        __syncthreads();
    }
    auto *counters = static_cast<uint32_t *>(p.workspace);
    auto *ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(p.workspace) + paged_ml_offset());
    auto *po = reinterpret_cast<float *>(static_cast<uint8_t *>(p.workspace) + paged_o_offset());

    uint32_t seq = s_seq;
    uint64_t seq_unit = s_start;  // the sequence's first unit
    auto segment_at = [&](uint64_t at) {  // at < end, ascending from call to call
        uint32_t n = (uint32_t)__ldg(p.length + seq), nu = units_of((int32_t)n);
        while (at >= seq_unit + (uint64_t)nu * items) {  // the next sequence with keys
            seq_unit += (uint64_t)nu * items;
            ++seq;
            n = (uint32_t)__ldg(p.length + seq);
            nu = units_of((int32_t)n);
        }
        PagedSegment s;
        const uint32_t item = (uint32_t)div_fast(at - seq_unit, nu);
        const uint32_t pass = passes == 1u ? 0u : item % passes;
        s.seq = seq;
        s.h = passes == 1u ? item : item / passes;
        s.row0 = pass * per;
        s.rows = min(per, p.group - s.row0);
        s.n = n;
        s.n_units = nu;
        s.item0 = seq_unit + (uint64_t)item * nu;
        s.u0 = (uint32_t)(at - s.item0);
        s.u1 = (uint32_t)(min(end, s.item0 + nu) - s.item0);
        return s;
    };
    // table entries of this warp's tile of unit u: keys [u * UNIT + warp * TILE, + TILE);
    // -1 where no key is.  Read ahead; checked when the tile is copied.
    struct Pages {
        int32_t id[HN];
    };
    auto pages_of = [&](const PagedSegment &s, uint32_t u) {
        const uint32_t t = u * PAGED_UNIT + warp * PAGED_TILE;
        const int32_t *row = p.page_table + (size_t)s.seq * p.max_pages + (t >> shift);
        Pages r;
#pragma unroll
        for (int a = 0; a < HN; ++a) r.id[a] = t + 16u * a < s.n ? __ldg(row + a) : -1;
        return r;
    };
    uint8_t *ring = smem + warp * L::WARP;
    uint32_t issued = 0;  // (lane 0) ring entries filled
    // (lane 0) the tile of unit u into ring entry `entry`, each in turn
    auto issue = [&](const PagedSegment &s, uint32_t u, uint32_t entry, Pages page) {
        issued = entry + 1u;
        const uint32_t st = entry % ST, t = u * PAGED_UNIT + warp * PAGED_TILE;
        uint8_t *dst = ring + st * L::STAGE;
        uint64_t *bar = &s_full[warp][st];
        uint32_t bytes = 0;
#pragma unroll
        for (int a = 0; a < HN; ++a) {
            const bool good = (uint32_t)page.id[a] < p.n_pages;  // negative ids are large ones
            if (!good && t + 16u * a < s.n) atomicOr(p.status, WL_DEV_ERR_INDEX);
            page.id[a] = good ? page.id[a] * (int32_t)p.n_kv + (int32_t)s.h : -1;
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

    uint64_t at = begin;
    uint32_t it = 0;                     // ring entries consumed
    PagedSegment sg;
    if (b < N) {
        sg = segment_at(at);
        if (lane == 0) {
            Pages first[ST];
#pragma unroll
            for (uint32_t i = 0; i < ST - 1u; ++i)
                if (sg.u0 + i < sg.u1) first[i] = pages_of(sg, sg.u0 + i);
#pragma unroll
            for (uint32_t i = 0; i < ST - 1u; ++i)
                if (sg.u0 + i < sg.u1) issue(sg, sg.u0 + i, it + i, first[i]);
        }
    }
    // rows of sequences without keys
    for (uint32_t s = b; s < p.n_seqs; s += gridDim.x) {
        const int32_t n = __ldg(p.length + s);
        if (units_of(n) == 0u) {
            if (tid == 0 && n != 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
            for (uint32_t i = tid; i < p.n_kv * p.group * D; i += PAGED_THREADS)
                store_typed(p.out, p.out_type, s * p.out_stride + i, 0.0f);
        }
    }
    if (b >= N) return;
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

    bool ok = true;
    for (;;) {
        const uint32_t head = sg.h * p.group + sg.row0;
        // the entry that the joining of the segment before had used, and the pages
        // of the one after it
        Pages ahead;
        if (lane == 0) {
            if (sg.u0 + ST - 1u < sg.u1) issue(sg, sg.u0 + ST - 1u, it + ST - 1u, pages_of(sg, sg.u0 + ST - 1u));
            if (sg.u0 + ST < sg.u1) ahead = pages_of(sg, sg.u0 + ST);
        }
        // the pass's query rows: row g as f16 parts hi (tile row g) and lo (row
        // g + 8) of q * 2^shift, its largest |q| brought to [2^13, 2^14)
        uint32_t qa[D / 16][4];
        float qf;  // scale * log2(e) * 2^-shift
        {
            float x[D / 4];
#pragma unroll
            for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
            if (g < sg.rows)
                load_row_part(p.q, p.type, sg.seq * p.q_stride + (size_t)(head + g) * D + c * (D / 4), x);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(13 - e) for 2^e <= top < 2^(e + 1), in two factors that are floats;
            // e kept so large that its opposite is one too
            const int e = top > 0.0f && top < INFINITY
                              ? max((int)(__float_as_uint(top) >> 23), 1) - 127 : 0;
            const int s0 = (13 - e) / 2, s1 = 13 - e - s0;
            const float f0 = __uint_as_float((uint32_t)(127 + s0) << 23);
            const float f1 = __uint_as_float((uint32_t)(127 + s1) << 23);
            qf = p.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - s0) << 23) *
                 __uint_as_float((uint32_t)(127 - s1) << 23);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                split_f16(x[4 * j] * f0 * f1, x[4 * j + 1] * f0 * f1, qa[j][0], qa[j][1]);
                split_f16(x[4 * j + 2] * f0 * f1, x[4 * j + 3] * f0 * f1, qa[j][2], qa[j][3]);
            }
        }
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

        for (uint32_t u = sg.u0; u < sg.u1; ++u, ++it) {
            const uint32_t t0 = u * PAGED_UNIT + warp * PAGED_TILE;
            const uint8_t *st = ring + (it % ST) * L::STAGE;
            int32_t block_next[HN];
            float ks_next[HN], vs_next[HN];
            if (u + 1 < sg.u1) scales(it + 1, block_next, ks_next, vs_next);
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
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            mma_f16(s[t], qa[4 * w + j], unbias(__byte_perm(x[t][j], EXP1024, 0x4140)),
                                    unbias(__byte_perm(x[t][j], EXP1024, 0x4342)));
                }
                // z in log2 units, keys 2c, 2c+1 of each 8
                float z[4][2];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float f = qf * ks[SMALL ? t / 2 : 0];
                    z[t][0] = (s[t][0] + s[t][2]) * f;
                    z[t][1] = (s[t][1] + s[t][3]) * f;
                }
                if (t0 + PAGED_TILE > sg.n || (SMALL && (block[0] | block[HN - 1]) < 0)) {  // not all take part
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (t0 + 8u * t + 2u * c + i >= sg.n || block[SMALL ? t / 2 : 0] < 0)
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
            if (lane == 0 && u + ST < sg.u1) {
                issue(sg, u + ST, it + ST, ahead);
                if (u + ST + 1u < sg.u1) ahead = pages_of(sg, u + ST + 1u);
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
        // the next segment's first tiles into the entries that the joining does not use
        at = sg.item0 + sg.u1;
        const PagedSegment done = sg;
        if (at < end) {
            sg = segment_at(at);
            if (ok && lane == 0)
                for (uint32_t i = 0; i < ST - 1u && sg.u0 + i < sg.u1; ++i)
                    issue(sg, sg.u0 + i, it + i, pages_of(sg, sg.u0 + i));
        }
        // the warps' shares of the segment, joined in warp order.  Output tile i,
        // column n stands for dimension n * D / 8 + i; kept at 8 i + n.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float back = vref * 6.103515625e-05f;  // 2^-14
        const uint32_t free_at = ((it + ST - 1u) % ST) * L::STAGE;  // the same in every warp
        float *so = reinterpret_cast<float *>(ring + free_at);
#pragma unroll
        for (int i = 0; i < NT; ++i)
            *reinterpret_cast<float2 *>(so + g * OP + 8 * i + 2 * c) =
                make_float2((o[i][0] + o[i][2]) * back, (o[i][1] + o[i][3]) * back);
        if (c == 0) {
            s_m[warp][g] = m;
            s_l[warp][g] = l * 6.103515625e-05f;
        }
        __syncthreads();
        const bool stop = s_abort != 0u;  // a wait ran out: nothing more is read or written
        const bool whole = done.u0 == 0 && done.u1 == done.n_units;
        const size_t slot = (size_t)b * 2u + (done.u0 != 0 ? 0u : 1u);
        // a warp takes a row, a lane D / 32 of its values k: dimensions (k % 8) * D / 8 + k / 8
        constexpr int OV = D / 32;
        auto write_row = [&](uint32_t r, const float (&acc)[OV], float sum) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const size_t to = done.seq * p.out_stride + (size_t)(head + r) * D;
#pragma unroll
            for (int i = 0; i < OV; ++i) {
                const uint32_t k = lane * OV + i;
                store_typed(p.out, p.out_type, to + (k & 7u) * (D / 8) + (k >> 3),
                            sum == 0.0f ? 0.0f : acc[i] * inv);
            }
        };
        if (!stop) {
            for (uint32_t r = warp; r < done.rows; r += PAGED_WARPS) {
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
                    write_row(r, acc, sum);
                } else {
#pragma unroll
                    for (int i = 0; i < OV; ++i) po[(slot * PAGED_ROWS + r) * D + lane * OV + i] = acc[i];
                    if (lane == 0) ml[slot * PAGED_ROWS + r] = make_float2(mx, sum);
                }
            }
            if (!whole) {
                // the CTAs that share the item: the last to arrive joins their parts in order
                const uint32_t first = cta_of(done.item0), last = cta_of(done.item0 + done.n_units - 1u);
                __syncthreads();
                if (tid == 0) {
                    uint32_t before;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                 : "=r"(before)
                                 : "l"(counters + first)
                                 : "memory");
                    s_last = before == last - first;
                    if (s_last) counters[first] = 0u;
                }
                __syncthreads();
                if (s_last) {
                    for (uint32_t r = warp; r < done.rows; r += PAGED_WARPS) {
                        auto part = [&](uint32_t x) { return ((size_t)x * 2u + (x == first)) * PAGED_ROWS + r; };
                        float mx = -INFINITY;
                        for (uint32_t x = first + lane; x <= last; x += 32u) mx = fmaxf(mx, __ldcg(&ml[part(x)]).x);
#pragma unroll
                        for (int q = 16; q; q >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, q));
                        const float ref = mx == -INFINITY ? 0.0f : mx;
                        float sum = 0.0f, acc[OV];
#pragma unroll
                        for (int i = 0; i < OV; ++i) acc[i] = 0.0f;
                        for (uint32_t x0 = first; x0 <= last; x0 += 32u) {
                            float f = 0.0f;
                            if (x0 + lane <= last) {
                                const float2 v = __ldcg(&ml[part(x0 + lane)]);
                                f = ex2_approx(v.x - ref);
                                sum = fmaf(v.y, f, sum);
                            }
                            const uint32_t count = min(32u, last - x0 + 1u);
#pragma unroll 8
                            for (uint32_t k = 0; k < count; ++k) {
                                const float fk = __shfl_sync(0xffffffffu, f, k);
                                const float *src = po + part(x0 + k) * D + lane * OV;
                                if constexpr (OV == 4) {
                                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(src));
                                    acc[0] = fmaf(v.x, fk, acc[0]);
                                    acc[1] = fmaf(v.y, fk, acc[1]);
                                    acc[2] = fmaf(v.z, fk, acc[2]);
                                    acc[3] = fmaf(v.w, fk, acc[3]);
                                } else {
                                    const float2 v = __ldcg(reinterpret_cast<const float2 *>(src));
                                    acc[0] = fmaf(v.x, fk, acc[0]);
                                    acc[1] = fmaf(v.y, fk, acc[1]);
                                }
                            }
                        }
#pragma unroll
                        for (int q = 16; q; q >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, q);
                        write_row(r, acc, sum);
                    }
                }
            }
        }
        if (at >= end || stop) break;
        // the joining's reads and writes of the ring come before the copy that follows
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    // after a wait that ran out: (bounded) the copies still in flight land before
    // the CTA's shared memory goes
    if (lane == 0)
        for (; it < issued; ++it) (void)mbar_wait(&s_full[warp][it % ST], (it / ST) & 1u);
}

}  // namespace wl
