// Serving batches over a paged KV cache: the append (nnz.h,
// nnz_dispatch_paged_append) -- per-head RMSNorm and rotation of every new
// query and key, and the copy of K and V into their pages.
#include "paged_dev.h"

#include <algorithm>

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

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// Bound by the bytes of q, k and v, read and written once.  A block takes the
// rows of one aligned group of 8 positions of a sequence (they lie in one page)
// and a share of the heads: 8 dims of a row a thread, so that norm and rotation
// stay within 16 (8 at head_dim 64) lanes, with the group's cosines and sines
// computed once into LDS.  V goes to its transposed page two dims a lane, all
// positions of the group in registers: whole groups are two 16-byte stores.
// q and k leave past the caches: 8192 tokens of 32 + 8 heads 60 -> 55 us (201 MB,
// 3.7 TB/s), 4093 tokens of seven prompts 30 -> 25 us; V's 16-byte pieces not,
// they meet in the L2 (past it: 70 us).
template <int D, bool BF>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr uint32_t LPR = D / 8, SETS = 256 / LPR;   // lanes of a row, rows at a time
    __shared__ float2 cs[8][D / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t s = blockIdx.x, g = 0;
    if (a.b.max_q > 1) {
        if (!paged_find(a.b.num_seqs, blockIdx.x, &s, &g,
                        [&](uint32_t i) { return paged_groups(paged_seq(a.b, i), a.b); }))
            return;
    }
    const PagedSeq sq = paged_seq(a.b, s);
    uint32_t i0, i1;
    paged_group_rows(sq, a.b, paged_first_group(sq) + g, &i0, &i1);
    if (i0 >= i1) return;
    const uint32_t nt = i1 - i0, p0 = (uint32_t)(sq.first + (int32_t)i0);
    const uint32_t page = paged_entry(a.b, s, p0, true), slot = p0 & ((1u << a.b.shift) - 1);
    const bool paged = page < a.b.num_pages;
    const size_t row0 = sq.row0 + i0;

    // rows of heads: set i of the block is token i % np of heads i / np, ...
    const uint32_t lg = nt > 4 ? 3 : nt > 2 ? 2 : nt > 1 ? 1 : 0, set = tid / LPR, col = tid % LPR;
    const uint32_t tok = set & ((1u << lg) - 1), step = SETS >> lg, heads = a.hq + (paged ? a.b.hkv : 0);
    const bool on = tok < nt;
    const size_t row = row0 + (on ? tok : 0);
    auto source = [&](uint32_t h) {
        return (h < a.hq ? a.q + row * a.q_stride + h * D : a.k + row * a.k_stride + (h - a.hq) * D) + 8 * col;
    };
    uint32_t h = (set >> lg) + blockIdx.y * step;
    const uint32_t hstep = step * gridDim.y;
    v4u r = {};
    if (on && h < heads) r = *(const v4u *)source(h);

    // V, two dims a lane
    constexpr uint32_t LPV = D / 2, HW = 64 / LPV;
    const uint32_t vd = 2 * (lane % LPV);
    if (paged) {
        for (uint32_t hv = (blockIdx.y * 4 + wave) * HW + lane / LPV; hv < a.b.hkv; hv += 4 * HW * gridDim.y) {
            const uint16_t *src = a.v + row0 * a.v_stride + hv * D + vd;
            uint16_t *dst = a.v_pages + ((((size_t)page * a.b.hkv + hv) * D + vd) << a.b.shift) + slot;
            uint32_t x[8];
#pragma unroll
            for (uint32_t t = 0; t < 8; ++t)
                if (t < nt) x[t] = *(const uint32_t *)(src + t * a.v_stride);
            if (nt == 8) {
                v4u lo, hi;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    lo[i] = (x[2 * i] & 0xFFFFu) | x[2 * i + 1] << 16;
                    hi[i] = x[2 * i] >> 16 | (x[2 * i + 1] & 0xFFFF0000u);
                }
                *(v4u *)dst = lo;
                *(v4u *)(dst + ((size_t)1 << a.b.shift)) = hi;
            } else {
#pragma unroll
                for (uint32_t t = 0; t < 8; ++t)
                    if (t < nt) {
                        dst[t] = (uint16_t)x[t];
                        dst[((size_t)1 << a.b.shift) + t] = (uint16_t)(x[t] >> 16);
                    }
            }
        }
    }

    if ((tid & 63) < a.half)
        for (uint32_t t = tid >> 6; t < nt; t += 4) cs[t][tid & 63] = paged_cos_sin((int32_t)(p0 + t), a.inv_freq, a.log2_step, tid & 63);
    __syncthreads();
    const uint32_t d0 = 8 * col, hl = a.half / 8;   // first dim; lanes of half the rotated dims
    for (; h < heads; h += hstep) {
        v4u next = {};
        if (on && h + hstep < heads) next = *(const v4u *)source(h + hstep);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = paged_load<BF>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
        const float *w = h < a.hq ? a.q_scale : a.k_scale;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
            ss += dpp_move<DPP_XOR1>(ss, 0.f);
            ss += dpp_move<DPP_XOR2>(ss, 0.f);
            ss += dpp_move<DPP_ROW_HALF_MIRROR>(ss, 0.f);
            if constexpr (LPR == 16) ss += dpp_move<DPP_ROW_MIRROR>(ss, 0.f);
            const float f = rsqrtf(ss / (float)D + a.eps);
            const float4 wa = *(const float4 *)(w + d0), wb = *(const float4 *)(w + d0 + 4);
            x[0] *= f * wa.x, x[1] *= f * wa.y, x[2] *= f * wa.z, x[3] *= f * wa.w;
            x[4] *= f * wb.x, x[5] *= f * wb.y, x[6] *= f * wb.z, x[7] *= f * wb.w;
        }
        if (a.halves) {
            const bool first = d0 < a.half, in = d0 < 2 * a.half;   // whole lanes: half is a multiple of 8
            const int from = (int)(first ? lane + hl : lane - hl);
            const uint32_t k0 = first ? d0 : d0 - a.half;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = __shfl(x[e], in ? from : (int)lane);
                if (in) {
                    const float2 c = cs[on ? tok : 0][k0 + e];
                    x[e] = fmaf(x[e], c.x, first ? -y * c.y : y * c.y);
                }
            }
        } else if (d0 < 2 * a.half) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float2 c = cs[on ? tok : 0][(d0 + e) / 2];
                const float u = x[e], v = x[e + 1];
                x[e] = fmaf(u, c.x, -v * c.y);
                x[e + 1] = fmaf(u, c.y, v * c.x);
            }
        }
        v4u y;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            y[i] = (uint32_t)paged_round<BF>(x[2 * i]) | (uint32_t)paged_round<BF>(x[2 * i + 1]) << 16;
        if (on) {
            uint16_t *dst = h < a.hq ? a.q_out + row * a.qo_stride + h * D
                                     : a.k_pages + (((((size_t)page * a.b.hkv + h - a.hq) << a.b.shift) + slot + tok) * D);
            __builtin_nontemporal_store(y, (v4u *)(dst + d0));
        }
        r = next;
    }
}

template <int D, bool BF>
int launch(nnz_ctx *ctx, const AppendArgs &a) {
    // Groups of 8 positions, an upper bound; the heads are shared out until
    // there are about 4096 blocks, down to four rows of heads for a thread (one
    // for single tokens, whose blocks take 16 heads at a time).  1024 blocks:
    // 8192 tokens of 32 + 8 heads 65 us against 60.
    const uint64_t groups = std::min<uint64_t>((uint64_t)a.b.rows / 8 + 2ull * a.b.num_seqs,
                                               (uint64_t)a.b.num_seqs * paged_groups_max(a.b.max_q));
    const uint32_t heads = a.hq + a.b.hkv, most = ceil_div(heads, a.b.max_q > 1 ? 8 : 16);
    const uint32_t shares = std::min(most, (uint32_t)std::max<uint64_t>(1, 4096 / groups));
    append_kernel<D, BF><<<dim3((uint32_t)groups, shares), 256, 0, ctx->stream>>>(a);
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
