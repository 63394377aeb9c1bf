// attn_prompt.cuh -- causal attention of packed whole prompts, grouped heads.
//
// Tokens of sequence s are rows [seq_start[s], seq_start[s + 1]) of q, k, v.
// For row i of it and query head h in the group of KV head g:
//   z_j = scale * (q_i . k_j),  j = 0 .. i (rows of the same sequence),
//   out_i = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),  m = max_j z_j.
// Rows outside every sequence are left as they were.
#pragma once

#include <cuda.h>

#include <cstdint>
#include <type_traits>

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

// ------------------------------------------------------------------ tensor cores
// A CTA takes 128 rows of one head and goes through the keys 64 at a time; two CTAs share
// an SM, so that one's softmax runs beside the other's products.  Tensor memory (256
// columns a CTA): the scores of two steps (64 f32 columns each; the weights overwrite
// them as 16-bit pairs) and the output (D f32 columns).
//   warps 0-3  softmax, one thread a row: scores to registers, row maximum, weights
//              2^(z - m + 6) back as 16-bit; the output is rescaled only when the
//              maximum has risen by more than 2^8 over the one in use (weights then stay
//              below 2^14);
//   warp 4     TMA: queries, then ring entries of the keys of step i and the values of
//              step i - 2, which are used together;
//   warp 5     MMA (one thread): weights x values of step j, then queries x keys of step
//              j + 2 into the scores' place that step j leaves, with nothing between
//              them (a commit there cost a tenth of the time).  A softmax warp finds its
//              next scores ready when it hands over its weights.
// The commit of both says that the scores of step j + 2 are there and that the product
// of step j is in the output.
// The masked part of a product is 0 x v, which is NaN where v is not finite: a row whose
// scores or output are not finite is computed again by prompt_row, which does not read
// what the mask leaves out, unless one of its own scores is NaN, which makes all of it NaN.
// That path is slow: where all rows take it (an infinity in an early value row of f16), 2048
// tokens take 10 ms and 2 x 8192 take 99, 200 times as long.
//
// What bounds it: at D = 128 an SM's 128 keys of a tile take 1650 cycles of products (an
// MMA of M = 128 takes 64 to 70 cycles for N = 64 as for N = 128) and 1030 of exponentials
// (16 a cycle and SM), a softmax warp 2400 from scores to weights, and two CTAs overlap
// these to about 1750; long prompts also run into the power limit.  At D = 64 the softmax
// alone bounds it.  Short prompts pay each CTA's beginning and end, 6000 cycles.  Measured
// (median call in a captured chain; in ordinary launches back to back in brackets): 2
// prompts to 8192 tokens, 20 / 5 heads of 128, bf16, 541 to 592 us by the run (638, at 1560 MHz
// under the power limit: 944 TFLOP/s of the causal half, 0.68 of cuBLAS's sustained dense
// rate); 2048 tokens f16 36.0 us (37.8); 32 packed prompts to 1024 tokens, 9 / 3 heads of 64,
// 49.5 us (49.8); 77 tokens 6.0 us (7.4, the host's launches).
// Steps on the way, at 2 x 8192: rows on the CUDA cores 100.8 ms; two tiles a CTA of 10
// warps, 128-key steps 654 us; the masked last step a code path of its own (its 128
// predicates had been kept in registers through every step) 581; one tile a CTA, two CTAs
// an SM 624 (32 packed prompts 77 -> 66); 64-key steps with two score buffers 547 (54);
// sequences in order, not from the last, (49).
// Not kept: weights through shared memory instead of tensor memory (589 against 581),
// a part of the exponentials by polynomial (1 to 20 % slower at each stage: the issue
// slots are what is short), MMAs issued by predicate from a convergent warp (45 against
// 41 us at 2048 tokens).
constexpr int PROMPT_THREADS = 192;
constexpr uint32_t PROMPT_ROWS = 128;
constexpr uint32_t PROMPT_COLUMNS = 256;  // of tensor memory

template <int D>
struct PromptShape {
    static constexpr uint32_t TILE = PROMPT_ROWS * D * 2u;  // the queries; 64 keys and 64 values
    static constexpr uint32_t STAGES = D == 128 ? 2 : 5;
    static constexpr size_t DYN = (1 + STAGES) * TILE + 1024;  // + alignment slack
};

struct AttnPromptMaps {
    CUtensorMap q, k, v;  // [token][head][D] 16-bit, box {64, 1, 128 or 64 (k, v)}, 128-byte swizzle
};

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint32_t x, uint32_t y,
                                            uint32_t z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// D f32, A and B both f16 or both bf16, M = 128; b_mn: B is stored with its N
// dimension contiguous (values), not K (keys).
__device__ __forceinline__ uint32_t umma_idesc_f16(uint32_t bf16, uint32_t b_mn, uint32_t n) {
    return (1u << 4) | (bf16 << 7) | (bf16 << 10) | (b_mn << 16) | ((n >> 3) << 17) | (8u << 24);
}
// Operand stored [k][64 n] with 128-byte rows, 128-byte swizzle: groups of 8 k are
// 1024 bytes apart, blocks of 64 n `block` bytes.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t block) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) |
           ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
#define WL_R8(r, i)                                                                          \
    "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), \
        "=r"(r[i + 6]), "=r"(r[i + 7])
#define WL_IN8(r, i)                                                                      \
    "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), \
        "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this warp's 32 lanes; the caller waits (tmem_wait_ld).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : WL_R8(r, 0), WL_R8(r, 8), WL_R8(r, 16), WL_R8(r, 24)
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::WL_IN8(r, 0),
        WL_IN8(r, 8), WL_IN8(r, 16), WL_IN8(r, 24), "r"(taddr)
        : "memory");
}
#undef WL_R8
#undef WL_IN8
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The largest (smallest) of three, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T, int D>
__global__ void __launch_bounds__(PROMPT_THREADS, 2)
    attn_prompt_kernel(const __grid_constant__ AttnPromptMaps maps, const AttnPromptParams p) {
    using L = PromptShape<D>;
    constexpr uint32_t ST = L::STAGES, TMA_WARP = 4, MMA_WARP = 5;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full, kv_full[ST], kv_empty[ST], s_full[2], p_full[2];
    __shared__ uint32_t s_tmem, s_abort;
    __shared__ SeqExtent s_extent;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                ~(uintptr_t)1023);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    // sequences in the caller's order, the last rows of each (the longest) first, heads side
    // by side: a tail of long tiles at the end of the grid cost 4 of 54 us at 32 prompts
    const uint32_t heads = p.n_kv * p.group, head = blockIdx.x % heads, unit = blockIdx.x / heads;

    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&s_tmem)),
                     "r"(PROMPT_COLUMNS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        // by this warp alone: the next kernel's CTAs may come once this one's tensor memory is
        // allocated.  Before that they could take the columns and wait for this grid's end,
        // which waits for the columns.
        pdl_launch_dependents();
    }
    if (tid == 0) {
        mbar_init(&q_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);  // one arrival a softmax warp
        }
        for (uint32_t s = 0; s < ST; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 1);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == TMA_WARP && lane < 3u) {
        const CUtensorMap *map = lane == 0u ? &maps.q : lane == 1u ? &maps.k : &maps.v;
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    pdl_wait();
    if (warp == TMA_WARP) {
        const SeqExtent e = find_extent(p.seq_start, nullptr, p.n_seqs, PROMPT_ROWS, 1u, unit, lane);
        if (lane == 0) s_extent = e;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // this CTA's rows: [row0, row0 + 128) of the sequence, where there are any
    const int64_t begin = s_extent.begin, stop = s_extent.end, len = stop - begin;
    const bool bad = begin < 0 || stop < begin || stop > (int64_t)p.n_tokens;
    if (bad && tid == 0) atomicOr(p.status, WL_DEV_ERR_INDEX);
    const int64_t tiles = (len + PROMPT_ROWS - 1) / PROMPT_ROWS;
    const int64_t place = (int64_t)unit - (begin / PROMPT_ROWS + (int64_t)s_extent.seq);
    const int64_t row0 = (tiles - 1 - place) * PROMPT_ROWS;
    // steps of 64 keys: to the last that a row of this sequence sees
    const uint32_t n = !bad && place >= 0 && place < tiles ? (uint32_t)(row0 / 64) + (row0 + 64 < len ? 2u : 1u) : 0u;

    auto aborted = [&]() { return *(volatile uint32_t *)&s_abort != 0u; };
    auto wait = [&](uint64_t *bar, uint32_t parity) {  // false: the wait ran out, here or elsewhere
        if (mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = globaltimer_ns(), limit = wait_limit_ns();
        while (!mbar_try_wait(bar, parity)) {
            if (aborted()) return false;
            if (globaltimer_ns() - t0 > limit) {
                atomicOr(p.status - 1, WL_DEV_ERR_TIMEOUT);
                atomicExch(&s_abort, 1u);
                return false;
            }
        }
        return true;
    };
    auto wait_all = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (n == 0u) {
        // no rows
    } else if (warp == TMA_WARP) {
        if (lane == 0) {
            // a box of `rows` x 64 elements of each 64 dimensions
            auto load_tile = [&](uint8_t *dst, const CUtensorMap *map, uint32_t y, uint32_t z, uint32_t rows,
                                 uint64_t *bar) {
#pragma unroll
                for (uint32_t x = 0; x < (uint32_t)D; x += 64) tma_load_3d(dst + x * rows * 2u, map, x, y, z, bar);
            };
            mbar_arrive_expect_tx(&q_full, L::TILE);
            load_tile(smem, &maps.q, head, (uint32_t)(begin + row0), PROMPT_ROWS, &q_full);
            // ring entry i: keys of step i and values of step i - 2, used together
            uint32_t it = 0;
            for (; it < n + 2u; ++it) {
                const uint32_t s = it % ST, h = head / p.group;
                if (it >= ST && !wait(&kv_empty[s], (it / ST - 1u) & 1u)) break;
                uint8_t *dst = smem + (1u + s) * L::TILE;
                mbar_arrive_expect_tx(&kv_full[s], ((it < n) + (it >= 2u)) * (L::TILE / 2u));
                if (it < n) load_tile(dst, &maps.k, h, (uint32_t)begin + it * 64u, 64u, &kv_full[s]);
                if (it >= 2u)
                    load_tile(dst + L::TILE / 2u, &maps.v, h, (uint32_t)begin + (it - 2u) * 64u, 64u, &kv_full[s]);
            }
            // the last copies land before the CTA's shared memory goes
            mbar_drain(&q_full, 0);
            for (uint32_t k = it > ST ? it - ST : 0; k < it; ++k) mbar_drain(&kv_full[k % ST], (k / ST) & 1u);
        }
    } else if (warp == MMA_WARP) {
        if (lane == 0) {
            const uint32_t base = smem_u32(smem);
            const uint32_t bf = pack16<T>(1.0f, 0.0f) == 0x3F80u;
            const uint32_t idesc_s = umma_idesc_f16(bf, 0u, 64u), idesc_o = umma_idesc_f16(bf, 1u, D);
            uint32_t freed = 0;           // ring entries whose reading is committed
            uint32_t told[2] = {0u, 0u};  // commits to s_full
            auto entry = [&](uint32_t it) { return base + (1u + it % ST) * L::TILE; };
            auto loaded = [&](uint32_t it) { return wait(&kv_full[it % ST], (it / ST) & 1u); };
            auto scores = [&](uint32_t s) {  // S = Q K^T of step s, into the place of its parity
                const uint32_t k = entry(s);
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)D / 16; ++i)
                    umma_f16_ss(tmem + (s & 1u) * 64u, umma_desc_sw128(base + (i / 4u) * 16384u + (i % 4u) * 32u),
                                umma_desc_sw128(k + (i / 4u) * 8192u + (i % 4u) * 32u), idesc_s, i != 0u);
            };
            bool ok = wait(&q_full, 0);
            for (uint32_t s = 0; ok && s < min(n, 2u); ++s) {
                if (!(ok = loaded(s))) break;
                tc_fence_after();
                scores(s);
                umma_commit(&s_full[s]);
                told[s] = 1u;
                umma_commit(&kv_empty[freed++ % ST]);
            }
            if (ok && n == 1u) {  // entry 1 holds nothing
                ok = loaded(1);
                if (ok) umma_commit(&kv_empty[freed++ % ST]);
            }
            for (uint32_t j = 0; ok && j < n; ++j) {
                // all that the step needs before its weights, so that nothing comes between
                // the two products
                if (!(ok = loaded(j + 2u) && wait(&p_full[j & 1u], (j >> 1) & 1u))) break;
                tc_fence_after();
                const uint32_t v = entry(j + 2u) + L::TILE / 2u;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)  // O += W V
                    umma_f16_ts(tmem + 128u, tmem + (j & 1u) * 64u + i * 8u, umma_desc_mn_sw128(v + i * 2048u, 8192u),
                                idesc_o, j != 0u || i != 0u);
                if (j + 2u < n) scores(j + 2u);
                umma_commit(&s_full[j & 1u]);  // of step j + 2, and that the product of step j is done
                ++(j & 1u ? told[1] : told[0]);
                umma_commit(&kv_empty[freed++ % ST]);
            }
            // every committed product is done, and has said so, before tensor and shared memory go
            for (uint32_t k = freed > ST ? freed - ST : 0; k < freed; ++k) mbar_drain(&kv_empty[k % ST], (k / ST) & 1u);
            for (uint32_t i = 0; i < 2u; ++i)
                if (told[i]) mbar_drain(&s_full[i], (told[i] - 1u) & 1u);
        }
    } else {
        const uint32_t r = tid;  // row in the tile
        const uint32_t lanes = tmem + ((warp * 32u) << 16), to = lanes + 128u;
        const float sc = p.scale * 1.4426950408889634f;
        float m = 0.0f, l = 0.0f;  // m: the maximum in use, in log2 units
        bool ok = true, fine = true;
        bool none = false;  // a score that the row sees is NaN: so is its sum, and all of its output
        // one step; DIAG: of the last two, where row r sees keys 0 .. `seen` of the 64 (a code
        // path of its own, so that the others carry no masks)
        auto step = [&](uint32_t j, int seen, auto last) {
            constexpr bool DIAG = decltype(last)::value;
            const uint32_t ts = lanes + (j & 1u) * 64u;
            uint32_t s[64];
            tmem_ld32(ts, s);
            tmem_ld32(ts + 32u, s + 32);
            tmem_wait_ld();
            auto score = [&](int i) { return __uint_as_float(s[i]); };
            float hi[4], lo[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) hi[q] = -INFINITY, lo[q] = INFINITY;
            if constexpr (DIAG) {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    if (i <= seen) {
                        hi[i & 3] = max3_nan(hi[i & 3], score(i), score(i));
                        lo[i & 3] = min3_nan(lo[i & 3], score(i), score(i));
                    }
                }
            } else if (sc >= 0.0f) {
#pragma unroll
                for (int i = 0; i < 64; i += 2) hi[(i / 2) & 3] = max3_nan(hi[(i / 2) & 3], score(i), score(i + 1));
            } else {
#pragma unroll
                for (int i = 0; i < 64; i += 2) lo[(i / 2) & 3] = min3_nan(lo[(i / 2) & 3], score(i), score(i + 1));
            }
            float top = sc >= 0.0f ? max3_nan(max3_nan(hi[0], hi[1], hi[2]), hi[3], hi[3])
                                   : min3_nan(min3_nan(lo[0], lo[1], lo[2]), lo[3], lo[3]);
            none = none || top != top;
            top = DIAG && seen < 0 ? -INFINITY : top * sc;
            fine = fine && top < INFINITY;  // NaN or infinite scores: the row is computed again
            if (j == 0) {
                m = top;
            } else if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                // each row by its own maximum: one that has not risen so far keeps what it has
                // (a factor of 1), so that no row's roundings depend on its neighbours
                // the product of step j - 1 is done when the scores of step j + 1 are there
                if (!wait_all(&s_full[(j + 1u) & 1u], ((j + 1u) >> 1) & 1u)) return false;
                tc_fence_after();
                const float mn = top > m + 8.0f ? top : m;
                const float f = mn == -INFINITY ? 1.0f : ex2_approx(m - mn);
                l *= f;
                m = mn;
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    uint32_t o[32];
                    tmem_ld32(to + i, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                    tmem_st32(to + i, o);
                }
            }
            const float base = 6.0f - (m == -INFINITY ? 0.0f : m);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
                const float2 x = f2_fma_rn(make_float2(score(i), score(i + 1)), make_float2(sc, sc),
                                           make_float2(base, base));
                float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                if constexpr (DIAG) {
                    e.x = i <= seen ? e.x : 0.0f;
                    e.y = i + 1 <= seen ? e.y : 0.0f;
                }
                sum[(i / 2) & 1] = f2_add_rn(sum[(i / 2) & 1], e);
                s[i / 2] = pack16<T>(e.x, e.y);
            }
            tmem_st32(ts, s);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[j & 1u]);
            sum[0] = f2_add_rn(sum[0], sum[1]);
            l += sum[0].x + sum[0].y;
            return true;
        };
        const uint32_t plain = (uint32_t)(row0 / 64);  // steps without a mask
        for (uint32_t j = 0; ok && j < n; ++j) {
            if (!(ok = wait_all(&s_full[j & 1u], (j >> 1) & 1u))) break;
            tc_fence_after();
            ok = j < plain ? step(j, 63, std::false_type()) : step(j, (int)r - 64 * (int)(j - plain), std::true_type());
        }
        // the last two products
        if (ok && n > 1u) ok = wait_all(&s_full[n & 1u], (n >> 1) & 1u);
        if (ok && wait_all(&s_full[(n + 1u) & 1u], ((n + 1u) >> 1) & 1u)) {
            tc_fence_after();
            const int64_t row = begin + row0 + r;
            const bool mine = row0 + r < len;
            const float inv = 1.0f / l;
            const size_t at = (size_t)row * p.out_stride + (size_t)head * D;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                uint32_t o[32];
                tmem_ld32(to + i, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = __uint_as_float(o[k + e]) * inv;
                        fine = fine && fabsf(x[e]) < INFINITY;
                    }
                    if (mine) store8(p.out, p.out_type, at + i + k, x);
                }
            }
            uint32_t again = __ballot_sync(0xffffffffu, mine && !fine && !none);
            __syncwarp();  // the lanes of prompt_row store over what the row's own lane stored
            while (again) {
                const uint32_t k = __ffs(again) - 1u;
                again &= again - 1u;
                prompt_row<T, D>(p, begin, row - lane + k, head, lane);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PROMPT_COLUMNS));
    }
}

}  // namespace wl
