// Attention of a ragged batch over a paged KV cache (nnz.h,
// nnz_dispatch_paged_attention).
#include "paged_dev.h"

namespace {

struct AttnArgs {
    PagedView b;
    const uint16_t *q, *k, *v;
    uint16_t *out;
    float *lse;
    const float *slopes;
    const uint32_t *prefix;
    uint64_t q_stride, o_stride;
    uint32_t hq, G, window;
    float scale, cap;
};

// One wave per (row, query head): 64 keys a step, lane l scores key l, then
// owns dims l, l + 64 of the output.
template <int D, bool BF>
__global__ __launch_bounds__(64) void attn_kernel(AttnArgs a) {
    const uint32_t row = blockIdx.x, h = blockIdx.y, l = threadIdx.x, hk = h / a.G;
    uint32_t s = 0;
    while (s < a.b.num_seqs && a.b.starts[s + 1] <= row) ++s;
    if (s == a.b.num_seqs) return;
    const PagedSeq sq = paged_seq(a.b, s);
    if (row < sq.row0 || row - sq.row0 >= sq.n || row - sq.row0 >= a.b.max_q) return;
    const int32_t p = sq.first + (int32_t)(row - sq.row0);
    const PagedSpan span = paged_span(p, sq.len, a.prefix ? a.prefix[s] : 0u, a.window);
    __shared__ float q[D];
    __shared__ float w[64];
    __shared__ size_t base[64];
    for (uint32_t d = l; d < D; d += 64) q[d] = paged_load<BF>(a.q[row * a.q_stride + h * D + d]);
    __syncthreads();
    float o[D / 64] = {}, m = -INFINITY, sum = 0.f;
    for (uint32_t j0 = span.lo & ~63u; j0 < span.hi; j0 += 64) {
        const uint32_t j = j0 + l, slot = j & ((1u << a.b.shift) - 1);
        const uint32_t page = j >= span.lo && j < span.hi ? paged_page(a.b, s, j) : a.b.num_pages;
        const bool on = page < a.b.num_pages;
        const size_t at = ((size_t)page * a.b.hkv + hk) << a.b.shift;
        float x = -INFINITY;
        if (on) {
            const uint16_t *kr = a.k + (at + slot) * D;
            x = 0.f;
            for (int d = 0; d < D; ++d) x = fmaf(q[d], paged_load<BF>(kr[d]), x);
            x *= a.scale;
            if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
            if (a.slopes) x -= a.slopes[h] * fabsf((float)(p - (int32_t)j));
        }
        const float mn = fmaxf(m, wave_max(x)), ref = mn == -INFINITY ? 0.f : mn;
        const float e = expf(x - ref), alpha = expf(m - ref);
        m = mn;
        sum = sum * alpha + wave_sum(on ? e : 0.f);
        __syncthreads();
        w[l] = on ? e : 0.f;
        base[l] = on ? at * D + slot : ~(size_t)0;
        __syncthreads();
        for (int i = 0; i < D / 64; ++i) {
            o[i] *= alpha;
            for (int t = 0; t < 64; ++t)
                if (base[t] != ~(size_t)0)
                    o[i] = fmaf(w[t], paged_load<BF>(a.v[base[t] + ((size_t)(l + 64 * i) << a.b.shift)]), o[i]);
        }
    }
    const bool none = m == -INFINITY && !(sum != sum);
    for (int i = 0; i < D / 64; ++i)
        a.out[row * a.o_stride + h * D + l + 64 * i] = paged_round<BF>(none ? 0.f : o[i] / sum);
    if (a.lse && l == 0) a.lse[(size_t)row * a.hq + h] = none ? -INFINITY : m + logf(sum);
}

template <int D, bool BF>
int launch(nnz_ctx *ctx, const AttnArgs &a) {
    attn_kernel<D, BF><<<dim3(a.b.rows, a.hq), 64, 0, ctx->stream>>>(a);
    NNZ_LAUNCHED(ctx);
    return NNZ_OK;
}

}  // namespace

extern "C" size_t nnz_paged_attention_workspace_bytes(const nnz_paged_kv *kv, const nnz_paged_batch *batch,
                                                      uint32_t num_query_heads) {
    if (paged_fault(kv, batch).code || paged_heads_fault(kv, num_query_heads).code) return 0;
    return 0;
}

extern "C" int nnz_dispatch_paged_attention(nnz_ctx *ctx, const nnz_paged_kv *kv, const nnz_paged_batch *batch,
                                            const void *q, void *output, float *lse, void *workspace,
                                            size_t workspace_bytes, const nnz_paged_attn_params *p) {
    NNZ_CHECK_CTX(ctx);
    if (const PagedFault f = paged_attn_fault(kv, batch, q, output, lse, p); f.code)
        return nnz_fail(ctx, f.code, "paged_attention: %s", f.what);
    NnzDeviceScope scope(ctx);
    AttnArgs a{};
    a.b = paged_view(*kv, *batch);
    a.q = (const uint16_t *)q;
    a.k = (const uint16_t *)kv->k_pages;
    a.v = (const uint16_t *)kv->v_pages;
    a.out = (uint16_t *)output;
    a.lse = lse;
    a.slopes = p->slopes;
    a.prefix = p->prefix_lens;
    a.q_stride = p->q_stride;
    a.o_stride = p->out_stride;
    a.hq = p->num_query_heads;
    a.G = a.hq / kv->num_kv_heads;
    a.window = p->window;
    a.scale = p->scale > 0.f ? p->scale : 1.f / sqrtf((float)kv->head_dim);
    a.cap = p->softcap;
    const bool bf = kv->dtype == NNZ_BF16;
    if (kv->head_dim == 128) return bf ? launch<128, true>(ctx, a) : launch<128, false>(ctx, a);
    return bf ? launch<64, true>(ctx, a) : launch<64, false>(ctx, a);
}
