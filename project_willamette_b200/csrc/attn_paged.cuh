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
constexpr int PAGED_CTAS_PER_SM = 3;
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

__device__ __forceinline__ uint4 ldg_stream16(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg_stream8(const void *p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                 : "=r"(v.x), "=r"(v.y)
                 : "l"(p));
    return v;
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

// One CTA of PAGED_CTAS_PER_SM per SM takes an equal, contiguous share of all
// (sequence, KV head, pass, 128-key) units; its four warps take 32 keys each.
template <int D>
__global__ void __launch_bounds__(PAGED_THREADS, PAGED_CTAS_PER_SM)
    attn_decode_i8_kernel(const AttnDecodeParams p) {
    constexpr int KW = D / 64;   // 16-byte loads of a key row by one lane
    constexpr int VW = D / 32;   // 4-byte words of a value row that one lane holds
    constexpr int NT = D / 8;    // output tiles of 8 dimensions
    __shared__ float s_o[PAGED_WARPS][PAGED_ROWS][D + 8];
    __shared__ float s_m[PAGED_WARPS][PAGED_ROWS], s_l[PAGED_WARPS][PAGED_ROWS];
    __shared__ unsigned long long s_scan[PAGED_WARPS];
    __shared__ unsigned long long s_start;
    __shared__ uint32_t s_seq, s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t g = lane >> 2, c = lane & 3u;  // the tile instructions' row and column group
    const uint32_t P = p.page_size, passes = (p.group + PAGED_ROWS - 1) / PAGED_ROWS;
    const uint32_t per = (p.group + passes - 1) / passes;  // query heads a pass
    const uint32_t items = p.n_kv * passes;                // items of a sequence
    const uint64_t b = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();

    auto units_of = [&](uint32_t s) -> uint32_t {  // 0 for an empty or refused sequence
        const int64_t n = __ldg(p.length + s);
        return n <= 0 || n > (int64_t)p.max_pages * P ? 0u
                                                      : (uint32_t)((n + PAGED_UNIT - 1) / PAGED_UNIT);
    };
    // rows of sequences without keys
    for (uint32_t s = (uint32_t)b; s < p.n_seqs; s += gridDim.x) {
        if (units_of(s) == 0u) {
            if (tid == 0 && __ldg(p.length + s) != 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
            for (uint32_t i = tid; i < p.n_kv * p.group * D; i += PAGED_THREADS)
                store_typed(p.out, p.out_type, s * p.out_stride + i, 0.0f);
        }
    }
    // all units, and the sequence in which this CTA's share begins
    uint64_t total = 0;
    {
        uint64_t mine = 0;
        for (uint32_t s = tid; s < p.n_seqs; s += PAGED_THREADS) mine += units_of(s);
#pragma unroll
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) s_scan[warp] = mine;
        __syncthreads();
        for (int w = 0; w < PAGED_WARPS; ++w) total += s_scan[w];
        total *= items;
    }
    const uint64_t N = min((uint64_t)gridDim.x, total);  // CTAs with a share, at least a unit each
    if (b >= N) return;
    const uint64_t begin = b * total / N, end = (b + 1) * total / N;
    {
        uint64_t before = 0;
        for (uint32_t s0 = 0; s0 < p.n_seqs; s0 += PAGED_THREADS) {
            const uint32_t s = s0 + tid;
            const uint64_t u = s < p.n_seqs ? (uint64_t)units_of(s) * items : 0u;
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
    uint32_t seq = s_seq;
    uint64_t seq_unit = s_start;  // the sequence's first unit
    uint64_t at = begin;
    uint32_t n_units = units_of(seq);
    auto *counters = static_cast<uint32_t *>(p.workspace);
    auto *ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(p.workspace) + paged_ml_offset());
    auto *po = reinterpret_cast<float *>(static_cast<uint8_t *>(p.workspace) + paged_o_offset());

    while (at < end) {
        while (at >= seq_unit + (uint64_t)n_units * items) {  // the next sequence with keys
            seq_unit += (uint64_t)n_units * items;
            ++seq;
            n_units = units_of(seq);
        }
        const uint32_t item = (uint32_t)((at - seq_unit) / n_units);
        const uint64_t item0 = seq_unit + (uint64_t)item * n_units, item1 = item0 + n_units;
        const uint32_t u0 = (uint32_t)(at - item0), u1 = (uint32_t)(min(end, item1) - item0);
        const uint32_t h = item / passes, pass = item % passes;
        const uint32_t n = (uint32_t)__ldg(p.length + seq);
        const uint32_t row0 = pass * per, rows = min(per, p.group - row0);
        const uint32_t head = h * p.group + row0;

        // the pass's query rows: row g as f16 parts hi (tile row g) and lo (row
        // g + 8) of q * 2^shift, its largest |q| brought to [2^13, 2^14)
        uint32_t qa[D / 16][4];
        float qf;  // scale * log2(e) * 2^-shift
        {
            float x[D / 4];
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const uint32_t d = (j < 4 ? c * 16u + 4u * j : 64u + c * 16u + 4u * (j - 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[4 * j + i] = g < rows ? load_typed(p.q, p.type, seq * p.q_stride +
                                                                          (size_t)(head + g) * D + d + i)
                                            : 0.0f;
                    top = fmaxf(top, fabsf(x[4 * j + i]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
            // 2^(13 - e) in two factors, each of them a float
            const float f0 = ldexpf(1.0f, (13 - e) / 2), f1 = ldexpf(1.0f, (13 - e) - (13 - e) / 2);
            qf = p.scale * 1.4426950408889634f * ldexpf(1.0f, (e - 13) / 2) *
                 ldexpf(1.0f, (e - 13) - (e - 13) / 2);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                split_f16(x[4 * j] * f0 * f1, x[4 * j + 1] * f0 * f1, qa[j][0], qa[j][1]);
                split_f16(x[4 * j + 2] * f0 * f1, x[4 * j + 3] * f0 * f1, qa[j][2], qa[j][3]);
            }
        }

        float m = -INFINITY, l = 0.0f, vref = 0.0f;
        float o[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

        // keys of this warp's tile of unit u: [u * UNIT + warp * TILE, + TILE), in two
        // halves of 16 that each lie in one page
        uint4 kr[4][KW];
        int32_t pid[2];
        float ks[2], vs[2];
        auto fetch_page = [&](uint32_t u) {
            const uint32_t t0 = u * PAGED_UNIT + warp * PAGED_TILE;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint32_t t = t0 + 16u * a;
                pid[a] = t < n ? __ldg(p.page_table + (size_t)seq * p.max_pages + t / P) : -1;
                if (t < n && (pid[a] < 0 || (uint32_t)pid[a] >= p.n_pages)) {
                    if (lane == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
                    pid[a] = -1;
                }
            }
        };
        auto block_of = [&](int32_t page) { return (size_t)page * p.n_kv + h; };
        auto load_k = [&](uint32_t u) {
            const uint32_t t0 = u * PAGED_UNIT + warp * PAGED_TILE;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                if (pid[a] >= 0) {
                    const size_t block = block_of(pid[a]);
                    ks[a] = __ldg(p.ks + block);
                    vs[a] = __ldg(p.vs + block);
                    const int8_t *k = p.kc + (block * P + ((t0 + 16u * a) & (P - 1u)) + g) * D + c * 16u;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int w = 0; w < KW; ++w)
                            kr[2 * a + i][w] = ldg_stream16(k + 8 * i * D + 64 * w);
                } else {
                    ks[a] = vs[a] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int w = 0; w < KW; ++w) kr[2 * a + i][w] = make_uint4(0, 0, 0, 0);
                }
            }
        };
        fetch_page(u0);
        load_k(u0);
        for (uint32_t u = u0; u < u1; ++u) {
            const uint32_t t0 = u * PAGED_UNIT + warp * PAGED_TILE;
            // this step's values, used after the softmax
            uint32_t vr[2][4][VW];
            const float ks0 = ks[0], ks1 = ks[1], vs0 = vs[0], vs1 = vs[1];
            const bool here[2] = {pid[0] >= 0, pid[1] >= 0};
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int8_t *v = p.vc + (block_of(max(pid[a], 0)) * P + ((t0 + 16u * a) & (P - 1u))) * D +
                                  g * (D / 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t t = 2u * c + (r & 1) + 8u * (r >> 1);
                    if (here[a]) {
                        if constexpr (D == 128) {
                            const uint4 w = ldg_stream16(v + t * D);
                            vr[a][r][0] = w.x;
                            vr[a][r][1] = w.y;
                            vr[a][r][2] = w.z;
                            vr[a][r][3] = w.w;
                        } else {
                            const uint2 w = ldg_stream8(v + t * D);
                            vr[a][r][0] = w.x;
                            vr[a][r][1] = w.y;
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[a][r][w] = 0u;
                    }
                }
            }
            if (u + 1 < u1) fetch_page(u + 1);

            float s[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const uint4 &r = kr[t][j / 4];
                    const uint32_t x =
                        (j % 4 == 0 ? r.x : j % 4 == 1 ? r.y : j % 4 == 2 ? r.z : r.w) ^ 0x80808080u;
                    mma_f16(s[t], qa[j], unbias(__byte_perm(x, EXP1024, 0x4140)),
                            unbias(__byte_perm(x, EXP1024, 0x4342)));
                }
            }
            if (u + 1 < u1) load_k(u + 1);

            // z in log2 units, keys 2c, 2c+1 of each 8; masked at the length and where
            // the page was refused
            float z[4][2];
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float f = qf * (t < 2 ? ks0 : ks1);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t key = t0 + 8u * t + 2u * c + i;
                    z[t][i] = key < n && here[t / 2] ? (s[t][i] + s[t][i + 2]) * f : -INFINITY;
                    top = fmaxf(top, z[t][i]);
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float vtop = fmaxf(fabsf(vs0), fabsf(vs1));
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
            // weights times 2^14, so that the f16 parts of small ones keep their bits
            const float base = 14.0f - (m == -INFINITY ? 0.0f : m);
            const float r0 = vs0 == 0.0f ? 0.0f : vs0 / vref, r1 = vs1 == 0.0f ? 0.0f : vs1 / vref;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                uint32_t w[4];
                const float r = a ? r1 : r0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float e0 = ex2_approx(z[2 * a + i][0] + base);
                    const float e1 = ex2_approx(z[2 * a + i][1] + base);
                    l += e0 + e1;
                    split_f16(e0 * r, e1 * r, w[2 * i], w[2 * i + 1]);
                }
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    uint32_t x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = vr[a][k][i] ^ 0x80808080u;
                    const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), a23 = __byte_perm(x[0], x[1], 0x7362);
                    const uint32_t b01 = __byte_perm(x[2], x[3], 0x5140), b23 = __byte_perm(x[2], x[3], 0x7362);
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
        // the warps' shares of the segment, joined in warp order.  Output tile i,
        // column n stands for dimension n * D / 8 + i; kept at 8 i + n.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float back = vref * 6.103515625e-05f;  // 2^-14
#pragma unroll
        for (int i = 0; i < NT; ++i)
            *reinterpret_cast<float2 *>(&s_o[warp][g][8 * i + 2 * c]) =
                make_float2((o[i][0] + o[i][2]) * back, (o[i][1] + o[i][3]) * back);
        if (c == 0) {
            s_m[warp][g] = m;
            s_l[warp][g] = l * 6.103515625e-05f;
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == n_units;
        const bool tail = u0 != 0;
        const size_t slot = (size_t)b * 2u + (tail ? 0u : 1u);
        for (uint32_t i = tid; i < rows * D; i += PAGED_THREADS) {
            const uint32_t r = i / D, k = i % D;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < PAGED_WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f, acc = 0.0f;
#pragma unroll
            for (int w = 0; w < PAGED_WARPS; ++w) {
                const float f = ex2_approx(s_m[w][r] - ref);
                sum = fmaf(s_l[w][r], f, sum);
                acc = fmaf(s_o[w][r][k], f, acc);
            }
            if (whole) {
                const uint32_t d = (k & 7u) * (D / 8) + (k >> 3);
                store_typed(p.out, p.out_type, seq * p.out_stride + (size_t)(head + r) * D + d,
                            sum == 0.0f ? 0.0f : acc / sum);
            } else {
                po[(slot * PAGED_ROWS + r) * D + k] = acc;
                if (k == 0) ml[slot * PAGED_ROWS + r] = make_float2(mx, sum);
            }
        }
        if (!whole) {
            // the CTAs that share the item: the last to arrive joins their parts in order
            const uint32_t first = (uint32_t)(((item0 + 1) * N - 1) / total);
            const uint32_t last = (uint32_t)((item1 * N - 1) / total);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t before = atomicAdd(counters + first, 1u);
                s_last = before == last - first;
                if (s_last) counters[first] = 0u;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                for (uint32_t i = tid; i < rows * D; i += PAGED_THREADS) {
                    const uint32_t r = i / D, k = i % D;
                    float mx = -INFINITY;
                    for (uint32_t x = first; x <= last; ++x)
                        mx = fmaxf(mx, __ldcg(&ml[((size_t)x * 2u + (x == first)) * PAGED_ROWS + r]).x);
                    const float ref = mx == -INFINITY ? 0.0f : mx;
                    float sum = 0.0f, acc = 0.0f;
#pragma unroll 4
                    for (uint32_t x = first; x <= last; ++x) {
                        const size_t y = ((size_t)x * 2u + (x == first)) * PAGED_ROWS + r;
                        const float2 v = __ldcg(&ml[y]);
                        const float f = ex2_approx(v.x - ref);
                        sum = fmaf(v.y, f, sum);
                        acc = fmaf(__ldcg(&po[y * D + k]), f, acc);
                    }
                    const uint32_t d = (k & 7u) * (D / 8) + (k >> 3);
                    store_typed(p.out, p.out_type, seq * p.out_stride + (size_t)(head + r) * D + d,
                                sum == 0.0f ? 0.0f : acc / sum);
                }
            }
        }
        __syncthreads();  // s_o is free again
        at = item0 + u1;
    }
}

}  // namespace wl
