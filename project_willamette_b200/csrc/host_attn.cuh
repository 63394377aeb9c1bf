// host_attn.cuh -- host side of the attention operators over caller buffers:
// argument checks and launches of the paged int8 KV append, the decode
// attention over that cache and the packed prompt attention.
//
// Part of the library's single translation unit (see host_core.cuh).
#pragma once

namespace {

// WL_GGML_* of an activation buffer -> the kernels' type index, or -1.
int act_type(uint32_t ggml) {
    return ggml == WL_GGML_F32 ? 0 : ggml == WL_GGML_F16 ? 1 : ggml == WL_GGML_BF16 ? 2 : -1;
}
uint64_t act_size(int type) { return type == 0 ? 4u : 2u; }

// A buffer of rows with `stride` elements between tokens and `width` elements
// used of each: 16-byte aligned rows that do not run into one another.
int check_rows(const char *op, const char *name, const void *p, uint64_t stride, uint64_t width,
               int type) {
    if (!p) return fail(WL_ERR_INVALID_ARGUMENT, "%s: %s is NULL", op, name);
    if (!aligned16(p))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %s is not 16-byte aligned", op, name);
    if (stride < width || stride > (1ull << 31) || stride * act_size(type) % 16u)
        return fail(WL_ERR_INVALID_ARGUMENT,
                    "%s: %s stride %llu must be at least its %llu elements, at most 2^31, and a "
                    "multiple of 16 bytes",
                    op, name, (unsigned long long)stride, (unsigned long long)width);
    return WL_OK;
}

int check_i32(const char *op, const char *name, const int32_t *p) {
    if (!p || (reinterpret_cast<uintptr_t>(p) & 3u))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %s is NULL or not 4-byte aligned", op, name);
    return WL_OK;
}

int check_heads(const char *op, uint32_t n_q, uint32_t n_kv, uint32_t head_dim) {
    if (head_dim != 64 && head_dim != 128)
        return fail(WL_ERR_NOT_IMPLEMENTED, "%s: head_dim %u is neither 64 nor 128", op, head_dim);
    if (!n_kv || !n_q || n_q % n_kv || n_kv > 1024 || n_q > 65535)
        return fail(WL_ERR_INVALID_ARGUMENT,
                    "%s: %u query heads over %u KV heads (a positive multiple, at most 1024 KV and "
                    "65535 query heads)",
                    op, n_q, n_kv);
    return WL_OK;
}

int check_kv_pages(const char *op, const wl_kv_pages_i8 *c) {
    if (!c) return fail(WL_ERR_INVALID_ARGUMENT, "%s: cache is NULL", op);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: page_size %u is not 16, 32, 64 or 128", op,
                    c->page_size);
    if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: k / v pages NULL or not 16-byte aligned", op);
    if (!c->k_scale || !c->v_scale || (reinterpret_cast<uintptr_t>(c->k_scale) & 3u) ||
        (reinterpret_cast<uintptr_t>(c->v_scale) & 3u))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: page scales NULL or not 4-byte aligned", op);
    if (!c->n_pages || (uint64_t)c->n_pages * c->n_kv_heads * c->page_size > 0x7FFFFFFFull)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %u pages of %u heads (at most 2^31 - 1 rows)", op,
                    c->n_pages, c->n_kv_heads);
    return WL_OK;
}

// Tensor map of a cache's codes as rows of head_dim bytes: up to 32 rows of one page
// and head a copy, the swizzle that spans a row.
int encode_pages(EncodeTiledFn enc, CUtensorMap *map, const int8_t *codes, const wl_kv_pages_i8 *c) {
    const uint32_t D = c->head_dim;
    const uint64_t rows = (uint64_t)c->n_pages * c->n_kv_heads * c->page_size;
    return encode_2d(enc, map, codes, D, rows, D, std::min(c->page_size, 32u),
                     D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// Where these operators report a bad index read on the device: the second
// word of the library's status block, so that a bad index is not taken for a
// timed-out wait by the host-buffer calls, which read the first.
int attn_status(const char *op, uint32_t **status) {
    uint32_t *s = status_ptr();
    if (!s) return WL_ERR_NO_DEVICE;
    int dev = -1;
    WL_CUDA(cudaGetDevice(&dev));
    if (dev != ctx().device)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: the current device is %d, the library runs on %d",
                    op, dev, ctx().device);
    *status = s + 1;
    return WL_OK;
}

template <typename T, int ITS, int RT, int HB, bool WHOLE>
int launch_kv_append_as(KvAppendParams &p, cudaStream_t s) {
    if (p.q) {
        // one token a CTA while that leaves room on the SMs, then as many as six CTAs an SM need
        const uint32_t ctas = 6u * (uint32_t)sm_count_for_launch();
        p.q_block = std::min((p.n_tokens + ctas - 1u) / ctas, KV_APPEND_MAX_Q_BLOCK);
        p.q_ctas = (p.n_tokens + p.q_block - 1u) / p.q_block;
    }
    const uint64_t units = (uint64_t)p.n_tokens / p.page_size + 2ull * p.n_seqs;
    const uint64_t ctas = p.q_ctas + units * ((p.n_kv + HB - 1) / HB);
    if (ctas > 0x7FFFFFFFull)
        return fail(WL_ERR_INVALID_ARGUMENT, "rope_kv_append: %u tokens of %u sequences", p.n_tokens, p.n_seqs);
    WL_CUDA(launch(kv_append_kernel<T, ITS, RT, HB, WHOLE>, dim3((uint32_t)ctas), dim3(2 * RT * HB), 0, s, true, p));
    return WL_OK;
}

// Threads by the rows of a page that a call can bring: a step's few tokens a sequence
// fit one warp for K and one for V; whole pages of prompts get four 8-element pieces a
// thread.  CTAs of 256 threads take as many heads as that leaves room for.
template <typename T>
int launch_kv_append(KvAppendParams &p, cudaStream_t s) {
    const uint32_t rows = std::min(p.page_size, (p.n_tokens + p.n_seqs - 1u) / p.n_seqs);
    const uint32_t pieces = rows * p.head_dim / 8u;
    if (p.n_rot % 8u) return launch_kv_append_as<T, 2, 64, 2, false>(p, s);
    if (pieces <= 32) return launch_kv_append_as<T, 1, 32, 4, true>(p, s);
    if (pieces <= 256) return launch_kv_append_as<T, 4, 64, 2, true>(p, s);
    if (pieces <= 512) return launch_kv_append_as<T, 4, 128, 1, true>(p, s);
    return launch_kv_append_as<T, 4, 256, 1, true>(p, s);
}

// Tensor map of [n_tokens][heads][D] 16-bit rows `stride` elements apart: box_rows tokens
// x 64 elements of one head, 128-byte swizzle, zeros behind the last token.
int encode_heads(EncodeTiledFn enc, CUtensorMap *map, const void *base, uint32_t n_tokens,
                 uint32_t heads, uint32_t D, uint64_t stride, uint32_t box_rows) {
    const cuuint64_t dims[3] = {D, heads, n_tokens};
    const cuuint64_t strides[2] = {D * 2ull, stride * 2ull};
    const cuuint32_t box[3] = {64, 1, box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(base), dims, strides, box,
                     estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(WL_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return WL_OK;
}

template <typename T>
int launch_attn_prompt(const AttnPromptParams &p, uint32_t D, cudaStream_t s) {
    EncodeTiledFn enc;
    int rc = get_encode_tiled(&enc);
    if (rc) return rc;
    AttnPromptMaps maps;
    if ((rc = encode_heads(enc, &maps.q, p.q, p.n_tokens, p.n_kv * p.group, D, p.q_stride, PROMPT_ROWS)) ||
        (rc = encode_heads(enc, &maps.k, p.k, p.n_tokens, p.n_kv, D, p.k_stride, 64)) ||
        (rc = encode_heads(enc, &maps.v, p.v, p.n_tokens, p.n_kv, D, p.v_stride, 64)))
        return rc;
    // sequence s owns the units [seq_start[s] / 128 + s, ...), at least as many as it needs
    const uint64_t ctas = ((uint64_t)p.n_tokens / PROMPT_ROWS + p.n_seqs) * p.n_kv * p.group;
    if (ctas > 0x7FFFFFFFull)
        return fail(WL_ERR_INVALID_ARGUMENT, "attn_prompt: %u tokens of %u sequences with %u heads",
                    p.n_tokens, p.n_seqs, p.n_kv * p.group);
    const dim3 grid((uint32_t)ctas), block(PROMPT_THREADS);
    if (D == 64)
        WL_CUDA(launch(attn_prompt_kernel<T, 64>, grid, block, PromptShape<64>::DYN, s, true, maps, p));
    else
        WL_CUDA(launch(attn_prompt_kernel<T, 128>, grid, block, PromptShape<128>::DYN, s, true, maps, p));
    return WL_OK;
}

}  // namespace

extern "C" {

int wl_dev_rope_kv_append_i8(const wl_kv_pages_i8 *cache, const wl_kv_append *a, void *stream) {
    const char *op = "rope_kv_append";
    int rc = check_kv_pages(op, cache);
    if (rc) return rc;
    if (!a) return fail(WL_ERR_INVALID_ARGUMENT, "%s: args is NULL", op);
    const uint32_t D = cache->head_dim, KV = cache->n_kv_heads;
    const uint32_t n_q = a->q ? a->n_q_heads : KV;
    if ((rc = check_heads(op, n_q, KV, D))) return rc;
    const int type = act_type(a->type), out_type = act_type(a->out_type);
    if (type < 0) return fail_type(a->type);
    if (out_type < 0) return fail_type(a->out_type);
    if (a->n_rot % 2 || a->n_rot > D)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: n_rot %u must be even and at most %u", op,
                    a->n_rot, D);
    if (a->rope_pairs > 1)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: rope_pairs %u is neither WL_ROPE_HALF nor "
                    "WL_ROPE_INTERLEAVED", op, a->rope_pairs);
    if (a->n_tokens > 0x7FFFFFFFu || a->n_seqs > 0x3FFFFFFFu)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %u tokens of %u sequences", op, a->n_tokens,
                    a->n_seqs);
    if (a->n_tokens == 0 || a->n_seqs == 0) return WL_OK;
    if ((rc = check_rows(op, "k", a->k, a->k_stride, (uint64_t)KV * D, type)) ||
        (rc = check_rows(op, "v", a->v, a->v_stride, (uint64_t)KV * D, type)) ||
        (a->q && (rc = check_rows(op, "q", a->q, a->q_stride, (uint64_t)n_q * D, type))) ||
        (rc = check_i32(op, "seq_start", a->seq_start)) ||
        (rc = check_i32(op, "position", a->position)) ||
        (rc = check_i32(op, "page_table", a->page_table)))
        return rc;
    if (!a->q != !a->q_out)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: q and q_out go together", op);
    if (!aligned16(a->q_out) || !aligned16(a->k_out) || !aligned16(a->v_out))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: q_out / k_out / v_out not 16-byte aligned", op);
    if (a->n_rot && (!a->rope || !aligned16(a->rope)))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: rope is NULL or not 16-byte aligned", op);
    if (a->max_pages == 0 || a->max_pages > 0x7FFFFFFFu / cache->page_size)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: max_pages %u", op, a->max_pages);
    KvAppendParams p;
    memset(&p, 0, sizeof p);
    if ((rc = attn_status(op, &p.status))) return rc;
    p.kc = cache->k;
    p.vc = cache->v;
    p.ks = cache->k_scale;
    p.vs = cache->v_scale;
    p.n_pages = cache->n_pages;
    p.page_size = cache->page_size;
    p.n_kv = KV;
    p.head_dim = D;
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.seq_start = a->seq_start;
    p.position = a->position;
    p.page_table = a->page_table;
    p.rope = reinterpret_cast<const float2 *>(a->rope);
    p.q_out = a->q_out;
    p.k_out = a->k_out;
    p.v_out = a->v_out;
    p.out_type = (uint32_t)out_type;
    p.n_tokens = a->n_tokens;
    p.n_seqs = a->n_seqs;
    p.group = n_q / KV;
    p.max_pages = a->max_pages;
    p.n_rot = a->n_rot;
    p.rope_len = a->rope_len;
    p.rope_pairs = a->rope_pairs;
    if (type == 0) return launch_kv_append<float>(p, (cudaStream_t)stream);
    if (type == 1) return launch_kv_append<__half>(p, (cudaStream_t)stream);
    return launch_kv_append<__nv_bfloat16>(p, (cudaStream_t)stream);
}

size_t wl_attn_decode_workspace_bytes(uint32_t n_seqs, uint32_t n_q_heads, uint32_t n_kv_heads,
                                      uint32_t head_dim) {
    // one size serves every batch: it follows the GPU's CTAs, not the sequences
    (void)n_seqs;
    (void)n_q_heads;
    (void)n_kv_heads;
    return paged_workspace_bytes(head_dim);
}

int wl_dev_attn_decode_i8(const wl_kv_pages_i8 *cache, const wl_attn_decode *a, void *stream) {
    const char *op = "attn_decode";
    int rc = check_kv_pages(op, cache);
    if (rc) return rc;
    if (!a) return fail(WL_ERR_INVALID_ARGUMENT, "%s: args is NULL", op);
    const uint32_t D = cache->head_dim, KV = cache->n_kv_heads;
    if ((rc = check_heads(op, a->n_q_heads, KV, D))) return rc;
    const int type = act_type(a->type), out_type = act_type(a->out_type);
    if (type < 0) return fail_type(a->type);
    if (out_type < 0) return fail_type(a->out_type);
    if (!std::isfinite(a->scale))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: scale is not finite", op);
    if (a->n_seqs > 65535)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %u sequences (at most 65535)", op, a->n_seqs);
    if (a->n_seqs == 0) return WL_OK;
    const uint64_t width = (uint64_t)a->n_q_heads * D;
    if ((rc = check_rows(op, "q", a->q, a->q_stride, width, type)) ||
        (rc = check_rows(op, "out", a->out, a->out_stride, width, out_type)) ||
        (rc = check_i32(op, "length", a->length)) ||
        (rc = check_i32(op, "page_table", a->page_table)))
        return rc;
    if (a->max_pages == 0 || a->max_pages > 0x7FFFFFFFu / cache->page_size)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: max_pages %u", op, a->max_pages);
    const size_t need = wl_attn_decode_workspace_bytes(a->n_seqs, a->n_q_heads, KV, D);
    if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need)
        return fail(WL_ERR_INVALID_ARGUMENT,
                    "%s: workspace NULL, not 16-byte aligned, or smaller than "
                    "wl_attn_decode_workspace_bytes (%zu)",
                    op, need);
    AttnDecodeParams p;
    memset(&p, 0, sizeof p);
    if ((rc = attn_status(op, &p.status))) return rc;
    EncodeTiledFn enc;
    AttnDecodeMaps maps;
    if ((rc = get_encode_tiled(&enc)) || (rc = encode_pages(enc, &maps.k, cache->k, cache)) ||
        (rc = encode_pages(enc, &maps.v, cache->v, cache)))
        return rc;
    p.ks = cache->k_scale;
    p.vs = cache->v_scale;
    p.n_pages = cache->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(cache->page_size);
    p.n_kv = KV;
    p.q = a->q;
    p.out = a->out;
    p.q_stride = a->q_stride;
    p.out_stride = a->out_stride;
    p.length = a->length;
    p.page_table = a->page_table;
    p.type = (uint32_t)type;
    p.out_type = (uint32_t)out_type;
    p.n_seqs = a->n_seqs;
    p.group = a->n_q_heads / KV;
    p.max_pages = a->max_pages;
    p.scale = a->scale;
    p.workspace = a->workspace;
    // no more CTAs than the longest lengths that the table allows have places of work
    const uint32_t passes = (p.group + PAGED_ROWS - 1) / PAGED_ROWS;
    const uint64_t units = (((uint64_t)a->max_pages << p.page_shift) + PAGED_UNIT - 1) / PAGED_UNIT;
    const uint32_t ctas = (uint32_t)std::min<uint64_t>(
        std::min<uint32_t>((uint32_t)sm_count_for_launch() * PAGED_CTAS_PER_SM, PAGED_MAX_CTAS),
        (units + 1) * KV * passes * a->n_seqs);
    auto kernel = cache->page_size == 16
                      ? (D == 64 ? attn_decode_i8_kernel<64, true> : attn_decode_i8_kernel<128, true>)
                      : (D == 64 ? attn_decode_i8_kernel<64, false> : attn_decode_i8_kernel<128, false>);
    WL_CUDA(launch(kernel, dim3(ctas), dim3(PAGED_THREADS), D == 64 ? PagedSmem<64>::DYN : PagedSmem<128>::DYN,
                   (cudaStream_t)stream, true, maps, p));
    return WL_OK;
}

int wl_dev_attn_prompt(const wl_attn_prompt *a, void *stream) {
    const char *op = "attn_prompt";
    if (!a) return fail(WL_ERR_INVALID_ARGUMENT, "%s: args is NULL", op);
    const uint32_t D = a->head_dim, H = a->n_q_heads, KV = a->n_kv_heads;
    int rc = check_heads(op, H, KV, D);
    if (rc) return rc;
    const int type = act_type(a->type), out_type = act_type(a->out_type);
    if (type < 1) return fail_type(a->type);
    if (out_type < 0 || (out_type && out_type != type)) return fail_type(a->out_type);
    if (!std::isfinite(a->scale))
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: scale is not finite", op);
    if (a->n_tokens > 0x7FFFFFFFu || a->n_seqs > 0x3FFFFFFFu)
        return fail(WL_ERR_INVALID_ARGUMENT, "%s: %u tokens of %u sequences", op, a->n_tokens,
                    a->n_seqs);
    if (a->n_tokens == 0 || a->n_seqs == 0) return WL_OK;
    if ((rc = check_rows(op, "q", a->q, a->q_stride, (uint64_t)H * D, type)) ||
        (rc = check_rows(op, "k", a->k, a->k_stride, (uint64_t)KV * D, type)) ||
        (rc = check_rows(op, "v", a->v, a->v_stride, (uint64_t)KV * D, type)) ||
        (rc = check_rows(op, "out", a->out, a->out_stride, (uint64_t)H * D, out_type)) ||
        (rc = check_i32(op, "seq_start", a->seq_start)))
        return rc;
    AttnPromptParams p;
    memset(&p, 0, sizeof p);
    if ((rc = attn_status(op, &p.status))) return rc;
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.out = a->out;
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.out_stride = a->out_stride;
    p.seq_start = a->seq_start;
    p.out_type = (uint32_t)out_type;
    p.n_tokens = a->n_tokens;
    p.n_seqs = a->n_seqs;
    p.group = H / KV;
    p.n_kv = KV;
    p.scale = a->scale;
    if (type == 1) return launch_attn_prompt<__half>(p, D, (cudaStream_t)stream);
    return launch_attn_prompt<__nv_bfloat16>(p, D, (cudaStream_t)stream);
}

}  // extern "C"
