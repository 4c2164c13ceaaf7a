// The serving kernels' argument checks and index arithmetic
// (nnzap_amd/csrc/paged.h), exported for tests/test_serving_host.py.
#include "../../nnzap_amd/csrc/paged.h"

// the layouts that nnzap_amd/_lib.py states
static_assert(sizeof(nnz_paged_kv) == 40 && offsetof(nnz_paged_kv, dtype) == 32, "nnz_paged_kv");
static_assert(sizeof(nnz_paged_batch) == 48 && offsetof(nnz_paged_batch, max_kv_len) == 40, "nnz_paged_batch");
static_assert(sizeof(nnz_paged_append_params) == 64 && offsetof(nnz_paged_append_params, eps) == 56, "nnz_paged_append_params");
static_assert(sizeof(nnz_paged_attn_params) == 40 && offsetof(nnz_paged_attn_params, softcap) == 36, "nnz_paged_attn_params");
static_assert(sizeof(nnz_logprobs_dims) == 32 && offsetof(nnz_logprobs_dims, temperature) == 24, "nnz_logprobs_dims");

extern "C" {

static int tell(PagedFault f, const char **what) {
    *what = f.what ? f.what : "";
    return f.code;
}

int h_append(const nnz_paged_kv *kv, const nnz_paged_batch *b, const void *q, const void *k, const void *v,
             const void *q_out, const nnz_paged_append_params *p, const char **what) {
    return tell(paged_append_fault(kv, b, q, k, v, q_out, p), what);
}
int h_attn(const nnz_paged_kv *kv, const nnz_paged_batch *b, const void *q, const void *out, const float *lse,
           const nnz_paged_attn_params *p, const char **what) {
    return tell(paged_attn_fault(kv, b, q, out, lse, p), what);
}
int h_logprobs(const void *x, const uint32_t *tokens, const float *lp, const uint32_t *ids, const float *top,
               const nnz_logprobs_dims *d, const char **what) {
    return tell(logprobs_fault(x, tokens, lp, ids, top, d), what);
}

static PagedView view(const uint32_t *table, const uint32_t *starts, const uint32_t *lens, const uint32_t *n) {
    PagedView v{};
    v.table = table;
    v.starts = starts;
    v.lens = lens;
    v.num_seqs = n[0];
    v.width = n[1];
    v.rows = n[2];
    v.max_q = n[3];
    v.max_kv = n[4];
    v.num_pages = n[5];
    v.shift = n[6];
    return v;
}
// out: row0, n, len, first
void h_seq(const uint32_t *starts, const uint32_t *lens, const uint32_t *n, uint32_t s, int64_t *out) {
    const PagedSeq q = paged_seq(view(nullptr, starts, lens, n), s);
    out[0] = q.row0;
    out[1] = q.n;
    out[2] = q.len;
    out[3] = q.first;
}
uint32_t h_page(const uint32_t *table, const uint32_t *n, uint32_t s, uint32_t j) {
    return paged_page(view(table, nullptr, nullptr, n), s, j);
}
uint32_t h_groups(const uint32_t *starts, const uint32_t *lens, const uint32_t *n, uint32_t s) {
    const PagedView v = view(nullptr, starts, lens, n);
    return paged_groups(paged_seq(v, s), v);
}
uint32_t h_groups_max(uint32_t q) { return paged_groups_max(q); }
void h_group_rows(const uint32_t *starts, const uint32_t *lens, const uint32_t *n, uint32_t s, uint32_t g,
                  uint32_t *out) {
    const PagedView v = view(nullptr, starts, lens, n);
    const PagedSeq q = paged_seq(v, s);
    paged_group_rows(q, v, paged_first_group(q) + g, out, out + 1);
}
void h_span(int32_t p, uint32_t len, uint32_t prefix, uint32_t window, uint32_t *out) {
    const PagedSpan r = paged_span(p, len, prefix, window);
    out[0] = r.lo;
    out[1] = r.hi;
}
}
