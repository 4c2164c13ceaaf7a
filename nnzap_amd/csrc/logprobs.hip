// Log probabilities of given tokens (nnz.h, nnz_dispatch_token_logprobs).
#include "paged_dev.h"

namespace {

struct LpArgs {
    const void *x;
    const uint32_t *tokens;
    float *lp, *lse, *entropy, *top_lp;
    uint32_t *rank, *top_ids;
    uint64_t stride;
    uint32_t vocab, top;
    float inv_t;
};

// (value, lower id first) as one number, larger = earlier; 0 for NaN.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);   // -0 -> 0
    const uint32_t m = u >> 31 ? ~u : u | 0x80000000u;
    return (uint64_t)m << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t m = (uint32_t)(k >> 32);
    return __uint_as_float(m >> 31 ? m & 0x7fffffffu : ~m);
}

// One block per row.
template <int DT>
__global__ __launch_bounds__(256) void logprobs_kernel(LpArgs a) {
    __shared__ float red[3][4];
    __shared__ uint64_t best[4];
    __shared__ uint32_t cnt[4];
    const uint32_t row = blockIdx.x, tid = threadIdx.x, w = tid >> 6;
    const size_t base = row * a.stride;
    const uint32_t tok = a.tokens[row];
    const bool named = tok < a.vocab;
    const float xt = named ? load_as_f32<DT>(a.x, base + tok) : 0.f;
    float m = -INFINITY;
    uint32_t before = 0;
    for (uint32_t i = tid; i < a.vocab; i += 256) {
        const float x = load_as_f32<DT>(a.x, base + i);
        m = fmaxf(m, x);
        before += xt != xt ? (x == x || i < tok) : (x > xt || (x == xt && i < tok));
    }
    m = wave_max(m);
    if ((tid & 63) == 0) red[0][w] = m;
    for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o);
    if ((tid & 63) == 0) cnt[w] = before;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, e = 0.f;
    for (uint32_t i = tid; i < a.vocab; i += 256) {
        const float t = (load_as_f32<DT>(a.x, base + i) - ref) * a.inv_t, p = expf(t);
        s += p;
        e += p * fmaxf(t, -1e30f);
    }
    s = wave_sum(s);
    e = wave_sum(e);
    if ((tid & 63) == 0) red[1][w] = s, red[2][w] = e;
    __syncthreads();
    s = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    e = red[2][0] + red[2][1] + red[2][2] + red[2][3];
    const bool none = s == 0.f;
    const float log_s = logf(s);
    auto lp_of = [&](float x) { return none ? -INFINITY : (x - ref) * a.inv_t - log_s; };
    if (tid == 0) {
        a.lp[row] = s != s ? s : named ? lp_of(xt) : -INFINITY;
        if (a.lse) a.lse[row] = none ? -INFINITY : ref * a.inv_t + log_s;
        if (a.entropy) a.entropy[row] = none ? 0.f : log_s - e / s;
        if (a.rank) a.rank[row] = named ? cnt[0] + cnt[1] + cnt[2] + cnt[3] : a.vocab;
    }
    uint64_t last = ~0ull;
    for (uint32_t n = 0; n < a.top; ++n) {
        uint64_t k = 0;
        for (uint32_t i = tid; i < a.vocab; i += 256) {
            const uint64_t c = order_key(load_as_f32<DT>(a.x, base + i), i);
            if (c < last && c > k) k = c;
        }
        for (int o = 32; o; o >>= 1) {
            const uint64_t c = __shfl_xor((unsigned long long)k, o);
            k = c > k ? c : k;
        }
        __syncthreads();
        if ((tid & 63) == 0) best[w] = k;
        __syncthreads();
        for (int i = 0; i < 4; ++i) k = best[i] > k ? best[i] : k;
        last = k;
        if (tid == 0) {
            const size_t at = (size_t)row * a.top + n;
            if (a.top_ids) a.top_ids[at] = k ? ~(uint32_t)k : 0xFFFFFFFFu;
            if (a.top_lp) a.top_lp[at] = k ? (s != s ? s : lp_of(key_value(k))) : NAN;
        }
    }
}

}  // namespace

extern "C" size_t nnz_token_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top_n) { return 0; }

extern "C" int nnz_dispatch_token_logprobs(nnz_ctx *ctx, const void *logits, const uint32_t *tokens, float *logprobs,
                                           float *lse, float *entropy, uint32_t *rank, uint32_t *top_ids,
                                           float *top_logprobs, void *workspace, size_t workspace_bytes,
                                           const nnz_logprobs_dims *d) {
    NNZ_CHECK_CTX(ctx);
    if (const PagedFault f = logprobs_fault(logits, tokens, logprobs, top_ids, top_logprobs, d); f.code)
        return nnz_fail(ctx, f.code, "token_logprobs: %s", f.what);
    NnzDeviceScope scope(ctx);
    LpArgs a{logits, tokens, logprobs, lse, entropy, top_logprobs, rank, top_ids,
             d->row_stride, d->vocab, d->top_n, 1.f / d->temperature};
    if (d->dtype == NNZ_F32) logprobs_kernel<NNZ_F32><<<d->rows, 256, 0, ctx->stream>>>(a);
    else if (d->dtype == NNZ_F16) logprobs_kernel<NNZ_F16><<<d->rows, 256, 0, ctx->stream>>>(a);
    else logprobs_kernel<NNZ_BF16><<<d->rows, 256, 0, ctx->stream>>>(a);
    NNZ_LAUNCHED(ctx);
    return NNZ_OK;
}
