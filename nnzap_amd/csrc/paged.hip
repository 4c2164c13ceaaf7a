// Serving batches over a paged KV cache: the append (nnz.h,
// nnz_dispatch_paged_append) -- per-head RMSNorm and rotation of every new
// query and key, and the copy of K and V into their pages.
#include "paged_dev.h"

namespace {

struct AppendArgs {
    PagedView b;
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_pages, *v_pages;
    const float *q_scale, *k_scale;
    const double *inv_freq;
    uint64_t q_stride, k_stride, v_stride, qo_stride;
    uint32_t hq, half, halves;   // half = rotary_dim / 2
    double log2_step;            // log2 of inv_freq[k + 1] / inv_freq[k]
    float eps;
};

// One wave per (row, head of q, k or v); lane l holds dims l, l + 64, ...
template <int D, bool BF>
__global__ __launch_bounds__(64) void append_kernel(AppendArgs a) {
    const uint32_t row = blockIdx.x, head = blockIdx.y, l = threadIdx.x;
    uint32_t s = 0;
    while (s < a.b.num_seqs && a.b.starts[s + 1] <= row) ++s;
    if (s == a.b.num_seqs) return;
    const PagedSeq sq = paged_seq(a.b, s);
    if (row < sq.row0 || row - sq.row0 >= sq.n || row - sq.row0 >= a.b.max_q) return;
    const int32_t p = sq.first + (int32_t)(row - sq.row0);
    if (p < 0) return;
    const uint32_t page = paged_page(a.b, s, (uint32_t)p), slot = (uint32_t)p & ((1u << a.b.shift) - 1);
    if (head >= a.hq && page >= a.b.num_pages) return;
    __shared__ float x[D];
    if (head >= a.hq + a.b.hkv) {
        const uint32_t h = head - a.hq - a.b.hkv;
        const uint16_t *src = a.v + row * a.v_stride + h * D;
        uint16_t *dst = a.v_pages + ((((size_t)page * a.b.hkv + h) * D) << a.b.shift) + slot;
        for (uint32_t d = l; d < D; d += 64) dst[(size_t)d << a.b.shift] = src[d];
        return;
    }
    const bool isq = head < a.hq;
    const uint32_t h = isq ? head : head - a.hq;
    const uint16_t *src = isq ? a.q + row * a.q_stride + h * D : a.k + row * a.k_stride + h * D;
    const float *w = isq ? a.q_scale : a.k_scale;
    float ss = 0.f;
    for (uint32_t d = l; d < D; d += 64) {
        x[d] = paged_load<BF>(src[d]);
        ss += x[d] * x[d];
    }
    if (w) {
        const float r = rsqrtf(wave_sum(ss) / (float)D + a.eps);
        for (uint32_t d = l; d < D; d += 64) x[d] = x[d] * r * w[d];
    }
    __syncthreads();
    for (uint32_t k = l; k < a.half; k += 64) {
        const uint32_t d0 = a.halves ? k : 2 * k, d1 = a.halves ? k + a.half : 2 * k + 1;
        const float2 cs = paged_cos_sin(p, a.inv_freq, a.log2_step, k);
        const float u = x[d0], v = x[d1];
        x[d0] = u * cs.x - v * cs.y;
        x[d1] = u * cs.y + v * cs.x;
    }
    __syncthreads();
    uint16_t *dst = isq ? a.q_out + row * a.qo_stride + h * D
                        : a.k_pages + (((((size_t)page * a.b.hkv + h) << a.b.shift) + slot) * D);
    for (uint32_t d = l; d < D; d += 64) dst[d] = paged_round<BF>(x[d]);
}

template <int D, bool BF>
int launch(nnz_ctx *ctx, const AppendArgs &a) {
    append_kernel<D, BF><<<dim3(a.b.rows, a.hq + 2 * a.b.hkv), 64, 0, ctx->stream>>>(a);
    NNZ_LAUNCHED(ctx);
    return NNZ_OK;
}

}  // namespace

extern "C" int nnz_dispatch_paged_append(nnz_ctx *ctx, const nnz_paged_kv *kv, const nnz_paged_batch *batch,
                                         const void *q, const void *k, const void *v, void *q_out,
                                         const nnz_paged_append_params *p) {
    NNZ_CHECK_CTX(ctx);
    if (const PagedFault f = paged_append_fault(kv, batch, q, k, v, q_out, p); f.code)
        return nnz_fail(ctx, f.code, "paged_append: %s", f.what);
    NnzDeviceScope scope(ctx);
    AppendArgs a{};
    a.b = paged_view(*kv, *batch);
    a.q = (const uint16_t *)q;
    a.k = (const uint16_t *)k;
    a.v = (const uint16_t *)v;
    a.q_out = (uint16_t *)q_out;
    a.k_pages = (uint16_t *)kv->k_pages;
    a.v_pages = (uint16_t *)kv->v_pages;
    a.q_scale = p->q_scale;
    a.k_scale = p->k_scale;
    a.inv_freq = p->inv_freq;
    a.q_stride = p->q_stride;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    a.qo_stride = p->q_out_stride;
    a.hq = p->num_query_heads;
    a.half = p->rotary_dim / 2;
    a.halves = p->rope_halves;
    a.log2_step = a.half && !p->inv_freq ? -log2((double)p->rope_theta) / a.half : 0.0;
    a.eps = p->eps;
    const bool bf = kv->dtype == NNZ_BF16;
    if (kv->head_dim == 128) return bf ? launch<128, true>(ctx, a) : launch<128, false>(ctx, a);
    return bf ? launch<64, true>(ctx, a) : launch<64, false>(ctx, a);
}
