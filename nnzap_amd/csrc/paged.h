// Ragged batches over a paged KV cache: the argument checks, and the index
// arithmetic that the kernels of paged.hip and paged_attn.hip share.  Plain
// C++ without device code, so that every bound it promises is tested on the
// host (tests/c/paged_host.cc).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "../../include/nnz.h"

#ifdef __HIPCC__
#define NNZ_HD __host__ __device__ __forceinline__
#else
#define NNZ_HD inline
#endif

// What a kernel knows of cache and batch.
struct PagedView {
    const uint32_t *table, *starts, *lens;
    uint32_t num_seqs, width, rows, max_q, max_kv;
    uint32_t num_pages, shift;   // page_size = 1 << shift
    uint32_t hkv;
};

// Sequence s: its rows [row0, row0 + n), the position of the first one (below
// zero if kv_lens counts fewer than n tokens) and its length, all within the
// bounds that the host stated, whatever the device arrays say.
struct PagedSeq {
    uint32_t row0, n, len;
    int32_t first;
};

NNZ_HD uint32_t paged_min(uint32_t a, uint32_t b) { return a < b ? a : b; }

NNZ_HD PagedSeq paged_seq_of(uint32_t start, uint32_t end, uint32_t len, const PagedView &v) {
    PagedSeq s;
    s.row0 = paged_min(start, v.rows);
    end = paged_min(end, v.rows);
    s.n = end > s.row0 ? end - s.row0 : 0;
    s.len = paged_min(len, v.max_kv);
    s.first = (int32_t)s.len - (int32_t)s.n;
    return s;
}

NNZ_HD PagedSeq paged_seq(const PagedView &v, uint32_t s) {
    return paged_seq_of(v.starts[s], v.starts[s + 1], v.lens[s], v);
}

// Page of position j of sequence s; num_pages where there is none.
NNZ_HD uint32_t paged_page(const PagedView &v, uint32_t s, uint32_t j) {
    const uint32_t e = j >> v.shift;
    if (e >= v.width) return v.num_pages;
    const uint32_t p = v.table[(size_t)s * v.width + e];
    return paged_min(p, v.num_pages);
}

// The append's units of work: the aligned groups of 8 positions (which lie in
// one page) that a sequence's rows touch.
NNZ_HD uint32_t paged_first_group(const PagedSeq &s) { return s.first > 0 ? (uint32_t)s.first >> 3 : 0u; }
NNZ_HD uint32_t paged_groups(const PagedSeq &s, const PagedView &v) {
    const int64_t last = (int64_t)s.first + (int64_t)paged_min(s.n, v.max_q) - 1;
    if (s.n == 0 || last < 0) return 0;
    return (uint32_t)(last >> 3) - paged_first_group(s) + 1;
}
// At most this many per sequence with q new tokens.
NNZ_HD uint32_t paged_groups_max(uint32_t q) { return q ? (q + 14u) >> 3 : 0u; }
// The rows of a sequence that stand in group g: i0 .. i1 of it.
NNZ_HD void paged_group_rows(const PagedSeq &s, const PagedView &v, uint32_t g, uint32_t *i0, uint32_t *i1) {
    const int64_t a = (int64_t)g * 8 - s.first, n = paged_min(s.n, v.max_q);
    const int64_t lo = a > 0 ? a : 0, low = s.first < 0 ? -(int64_t)s.first : 0;
    const int64_t b = a + 8;
    *i0 = (uint32_t)(lo > low ? lo : low);
    *i1 = (uint32_t)(b < n ? (b > 0 ? b : 0) : n);
}

// Visible positions [lo, hi) of a row at position p (holes in the page table
// aside).
struct PagedSpan {
    uint32_t lo, hi;
};
NNZ_HD PagedSpan paged_span(int32_t p, uint32_t len, uint32_t prefix, uint32_t window) {
    const int64_t end = (int64_t)p + 1;
    PagedSpan r;
    r.hi = end > 0 ? (uint32_t)end : 0u;
    r.hi = r.hi > prefix ? r.hi : prefix;
    r.hi = paged_min(r.hi, len);
    r.lo = window && end > (int64_t)window ? (uint32_t)(end - window) : 0u;
    return r;
}

// ---- argument checks: the message of the first fault, or null ------------
struct PagedFault {
    int code;
    const char *what;
};

inline PagedFault paged_fault(const nnz_paged_kv *kv, const nnz_paged_batch *b) {
    if (!kv || !b) return {NNZ_EINVAL, "null cache or batch"};
    if (!kv->k_pages || !kv->v_pages) return {NNZ_EINVAL, "null pages"};
    if (!b->page_table || !b->q_starts || !b->kv_lens) return {NNZ_EINVAL, "null page table, q_starts or kv_lens"};
    if (kv->dtype != NNZ_F16 && kv->dtype != NNZ_BF16) return {NNZ_EUNSUPPORTED, "the cache holds f16 or bf16"};
    if (kv->head_dim != 64 && kv->head_dim != 128) return {NNZ_EUNSUPPORTED, "head_dim is 64 or 128"};
    if (kv->page_size < 16 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return {NNZ_EUNSUPPORTED, "page_size is a power of two from 16 to 1024"};
    if (!kv->num_pages || kv->num_pages > 0x7fffffffu) return {NNZ_EINVAL, "num_pages out of range"};
    if (!kv->num_kv_heads || kv->num_kv_heads > 1024) return {NNZ_EINVAL, "num_kv_heads out of range"};
    if (!b->num_seqs || b->num_seqs > 65535) return {NNZ_EINVAL, "num_seqs is 1 to 65535"};
    if (!b->table_width) return {NNZ_EINVAL, "empty page table"};
    if (!b->num_rows || b->num_rows > (1u << 24)) return {NNZ_EINVAL, "num_rows is 1 to 2^24"};
    if (!b->max_q_len || b->max_q_len > b->num_rows) return {NNZ_EINVAL, "max_q_len is 1 to num_rows"};
    if (!b->max_kv_len || b->max_kv_len > (1u << 30)) return {NNZ_EINVAL, "max_kv_len is 1 to 2^30"};
    if ((uint64_t)b->table_width * kv->page_size < b->max_kv_len)
        return {NNZ_EINVAL, "the page table is narrower than max_kv_len"};
    if (((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15) return {NNZ_EINVAL, "pages must be 16-byte aligned"};
    if (((uintptr_t)b->page_table | (uintptr_t)b->q_starts | (uintptr_t)b->kv_lens) & 3)
        return {NNZ_EINVAL, "page table, q_starts and kv_lens must be 4-byte aligned"};
    return {NNZ_OK, nullptr};
}

// A buffer of rows [heads][head_dim] at `stride` elements.
inline PagedFault paged_rows_fault(const void *p, uint32_t stride, uint32_t heads, uint32_t head_dim) {
    if (!p) return {NNZ_EINVAL, "null buffer"};
    if ((uintptr_t)p & 15) return {NNZ_EINVAL, "buffers must be 16-byte aligned"};
    if (stride % 8 || (uint64_t)stride < (uint64_t)heads * head_dim)
        return {NNZ_EINVAL, "a row stride must be a multiple of 8 and hold the row"};
    return {NNZ_OK, nullptr};
}

inline PagedFault paged_append_fault(const nnz_paged_kv *kv, const nnz_paged_batch *b, const void *q, const void *k,
                                     const void *v, const void *q_out, const nnz_paged_append_params *p) {
    if (PagedFault f = paged_fault(kv, b); f.code) return f;
    if (!p) return {NNZ_EINVAL, "null parameters"};
    if (!p->num_query_heads || p->num_query_heads > 1024) return {NNZ_EINVAL, "num_query_heads out of range"};
    if (PagedFault f = paged_rows_fault(q, p->q_stride, p->num_query_heads, kv->head_dim); f.code) return f;
    if (PagedFault f = paged_rows_fault(q_out, p->q_out_stride, p->num_query_heads, kv->head_dim); f.code) return f;
    if (q == q_out && p->q_stride != p->q_out_stride) return {NNZ_EINVAL, "in place with two strides"};
    if (PagedFault f = paged_rows_fault(k, p->k_stride, kv->num_kv_heads, kv->head_dim); f.code) return f;
    if (PagedFault f = paged_rows_fault(v, p->v_stride, kv->num_kv_heads, kv->head_dim); f.code) return f;
    if (p->rotary_dim % 16 || p->rotary_dim > kv->head_dim)
        return {NNZ_EUNSUPPORTED, "rotary_dim is a multiple of 16 up to head_dim"};
    if (p->rope_halves > 1) return {NNZ_EINVAL, "rope_halves is 0 or 1"};
    if (p->rotary_dim && !p->inv_freq && !(p->rope_theta > 0.f && p->rope_theta < 3e38f))
        return {NNZ_EINVAL, "rope_theta must be positive"};
    if (!(p->eps >= 0.f)) return {NNZ_EINVAL, "eps must not be negative"};
    if (((uintptr_t)p->q_scale | (uintptr_t)p->k_scale) & 15) return {NNZ_EINVAL, "norm scales must be 16-byte aligned"};
    if ((uintptr_t)p->inv_freq & 7) return {NNZ_EINVAL, "inv_freq must be 8-byte aligned"};
    return {NNZ_OK, nullptr};
}

inline PagedFault paged_heads_fault(const nnz_paged_kv *kv, uint32_t hq) {
    if (!hq || hq > 1024 || hq % kv->num_kv_heads)
        return {NNZ_EINVAL, "num_query_heads must be a multiple of num_kv_heads, at most 1024"};
    return {NNZ_OK, nullptr};
}

inline PagedFault paged_attn_fault(const nnz_paged_kv *kv, const nnz_paged_batch *b, const void *q, const void *out,
                                   const float *lse, const nnz_paged_attn_params *p) {
    if (PagedFault f = paged_fault(kv, b); f.code) return f;
    if (!p) return {NNZ_EINVAL, "null parameters"};
    if (PagedFault f = paged_heads_fault(kv, p->num_query_heads); f.code) return f;
    if (PagedFault f = paged_rows_fault(q, p->q_stride, p->num_query_heads, kv->head_dim); f.code) return f;
    if (PagedFault f = paged_rows_fault(out, p->out_stride, p->num_query_heads, kv->head_dim); f.code) return f;
    if (q == out) return {NNZ_EINVAL, "the output may not overwrite q"};
    // beyond these what the kernels derive from them leaves float32
    if (p->scale != 0.f && !(p->scale >= 1e-30f && p->scale <= 1e30f))
        return {NNZ_EINVAL, "scale must be from 1e-30 to 1e30, or 0 for 1/sqrt(head_dim)"};
    if (p->softcap != 0.f && !(p->softcap >= 1e-6f && p->softcap <= 1e6f))
        return {NNZ_EINVAL, "softcap must be from 1e-6 to 1e6, or 0 for none"};
    if (((uintptr_t)lse | (uintptr_t)p->slopes | (uintptr_t)p->prefix_lens) & 3)
        return {NNZ_EINVAL, "lse, slopes and prefix_lens must be 4-byte aligned"};
    return {NNZ_OK, nullptr};
}

inline PagedFault logprobs_fault(const void *logits, const uint32_t *tokens, const float *logprobs,
                                 const uint32_t *top_ids, const float *top_logprobs, const nnz_logprobs_dims *d) {
    if (!d || !logits || !tokens || !logprobs) return {NNZ_EINVAL, "null dims, logits, tokens or logprobs"};
    if (d->dtype != NNZ_F32 && d->dtype != NNZ_F16 && d->dtype != NNZ_BF16) return {NNZ_EINVAL, "bad dtype"};
    if (!d->rows || d->rows >= (1u << 24)) return {NNZ_EINVAL, "rows is 1 to 2^24 - 1"};
    if (!d->vocab || d->vocab > (1u << 28)) return {NNZ_EINVAL, "vocab is 1 to 2^28"};
    if (d->row_stride < d->vocab) return {NNZ_EINVAL, "row_stride is less than vocab"};
    if (d->row_stride > (1ull << 32)) return {NNZ_EINVAL, "row_stride out of range"};
    if (d->top_n > 64 || d->top_n > d->vocab) return {NNZ_EINVAL, "top_n is at most 64 and vocab"};
    if (d->top_n && !(top_ids || top_logprobs)) return {NNZ_EINVAL, "top_n without top_ids and top_logprobs"};
    if (!(d->temperature >= 1e-30f && d->temperature <= 1e30f)) return {NNZ_EINVAL, "temperature must be from 1e-30 to 1e30"};
    if ((uintptr_t)logits & (d->dtype == NNZ_F32 ? 3 : 1)) return {NNZ_EINVAL, "logits are not aligned to their type"};
    return {NNZ_OK, nullptr};
}
