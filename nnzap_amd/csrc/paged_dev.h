// Device helpers of the serving kernels.
#pragma once

#include "internal.h"
#include "paged.h"

// Makes the context's device current for the length of a call.
struct NnzDeviceScope {
    int before = -1;
    explicit NnzDeviceScope(const nnz_ctx *ctx) {
        int now = ctx->device;
        if (hipGetDevice(&now) == hipSuccess && now != ctx->device && hipSetDevice(ctx->device) == hipSuccess)
            before = now;
    }
    ~NnzDeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

static inline PagedView paged_view(const nnz_paged_kv &kv, const nnz_paged_batch &b) {
    PagedView v{};
    v.table = b.page_table;
    v.starts = b.q_starts;
    v.lens = b.kv_lens;
    v.num_seqs = b.num_seqs;
    v.width = b.table_width;
    v.rows = b.num_rows;
    v.max_q = b.max_q_len;
    v.max_kv = b.max_kv_len;
    v.num_pages = kv.num_pages;
    v.shift = (uint32_t)__builtin_ctz(kv.page_size);
    v.hkv = kv.num_kv_heads;
    return v;
}

template <bool BF>
__device__ __forceinline__ float paged_load(uint16_t u) {
    return BF ? bf16_to_f32(u) : (float)__builtin_bit_cast(f16_t, u);
}
template <bool BF>
__device__ __forceinline__ uint16_t paged_round(float f) {
    return BF ? f32_to_bf16_rne(f) : __builtin_bit_cast(uint16_t, (f16_t)f);
}

// cos and sin of position p times frequency k, the product and its reduction
// to a part of a turn in 64 bits: at p = 10^6 a float32 product is off by up
// to 0.06 radians.
__device__ __forceinline__ float2 paged_cos_sin(int32_t p, const double *inv_freq, double log2_step, uint32_t k) {
    const double f = inv_freq ? inv_freq[k] : exp2(log2_step * (double)k);
    const double t = (double)p * f * 0.15915494309189533577;   // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    return make_float2(c, s);
}
