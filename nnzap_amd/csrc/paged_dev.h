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

// A table entry through the scalar cache (the table does not change while the
// kernel runs), as it stands there: it names a page only if it is below
// num_pages.  Positions behind the table read its last entry.
__device__ __forceinline__ uint32_t paged_raw(const PagedView &b, uint32_t s, uint32_t key) {
    typedef const uint32_t __attribute__((address_space(4))) *table_t;
    const table_t t = (table_t)(uintptr_t)(b.table + (size_t)s * b.width);
    return t[paged_min(key >> b.shift, b.width - 1)];
}
// num_pages where there is no page or the key is not wanted.
__device__ __forceinline__ uint32_t paged_entry(const PagedView &b, uint32_t s, uint32_t key, bool wanted) {
    return wanted && key >> b.shift < b.width ? paged_min(paged_raw(b, s, key), b.num_pages) : b.num_pages;
}

// Unit u of a batch whose sequence i has count(i) units: which sequence's, and
// which of its units.  By whole waves, 64 sequences at a time.
template <class Count>
__device__ __forceinline__ bool paged_find(uint32_t num_seqs, uint32_t u, uint32_t *s, uint32_t *unit, Count count) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t base = 0; base < num_seqs; base += 64) {
        const uint32_t cnt = base + lane < num_seqs ? count(base + lane) : 0u;
        uint32_t upto = cnt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(upto, o);
            upto += lane >= (uint32_t)o ? t : 0u;
        }
        const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
        if (u - before < all) {
            const uint64_t in = __builtin_amdgcn_ballot_w64(u - before < upto);
            const uint32_t i = __builtin_amdgcn_readfirstlane(__builtin_ctzll(in));
            *s = base + i;
            *unit = u - before - __builtin_amdgcn_readlane(upto - cnt, i);
            return true;
        }
        before += all;
    }
    return false;
}
