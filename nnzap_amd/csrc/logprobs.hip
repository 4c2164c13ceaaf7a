// Log probabilities of given tokens (nnz.h, nnz_dispatch_token_logprobs).
//
// Bound by the logits' bytes, which are read once.  A row is cut into pieces
// (one if there are rows enough to fill the chip), a piece goes to a block of
// four waves, and every wave streams its part with what it needs of it in
// registers:
//   * per lane the running maximum m, s = sum 2^t and w = sum t 2^t with
//     t = (x - m) log2(e) / T; x - m before the scale, so that rows of the
//     type's lowest value stay exact, and w relative to m, so that the entropy
//     log s - w / s is a sum of terms of one sign;
//   * per lane the number of ids that come before the token;
//   * per wave the best top_n so far, one 64-bit key a lane, sorted (value and
//     complemented id: larger is earlier).  A group of 16 values per lane is
//     looked at again only if one of them reaches the last of the list, which
//     after a few groups is rare; what also reaches the top_n-th of the lanes'
//     maxima is gathered in LDS, 64 at a time sorted and merged into the list.
// Keys and counts are integers and the partial sums meet in a fixed order, so a
// call repeats bit for bit.
#include "paged_dev.h"

#include <algorithm>

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr uint32_t WAVES = 4, GROUP = 16;   // values of a lane looked at together
constexpr float LN2 = 0.69314718055994531f, LOG2E = 1.44269504088896341f;

struct LpArgs {
    const void *x;
    const uint32_t *tokens;
    float *lp, *lse, *entropy, *top_lp;
    uint32_t *rank, *top_ids;
    uint64_t stride;
    uint32_t vocab, top, pieces;
    float c, inv_t;        // log2(e) / temperature, 1 / temperature
    float4 *part;          // [row][piece] m, s, w, count (bits)
    uint64_t *part_keys;   // [row][piece][top]
};

// (value, lower id first) as one number, larger = earlier; 0 for NaN.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) {
    const uint32_t u = __float_as_uint(x + 0.f);   // -0 -> 0
    const uint32_t m = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return x != x ? 0 : (uint64_t)m << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t m = (uint32_t)(k >> 32);
    return __uint_as_float(m >> 31 ? m & 0x7fffffffu : ~m);
}

// The value of lane ^ J, with moves of the vector unit only.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    auto dpp = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 0xF, 0xF, false); };
    const uint32_t lane = threadIdx.x & 63;
    if constexpr (J == 1) return dpp(std::integral_constant<int, DPP_XOR1>());
    else if constexpr (J == 2) return dpp(std::integral_constant<int, DPP_XOR2>());
    else if constexpr (J == 4) {
        const uint32_t up = dpp(std::integral_constant<int, 0x104>()), down = dpp(std::integral_constant<int, 0x114>());
        return lane & 4 ? down : up;   // row_shl:4 reads lane + 4, row_shr:4 lane - 4
    } else if constexpr (J == 8) return dpp(std::integral_constant<int, 0x128>());   // row_ror:8
    else if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane & 16 ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return lane & 32 ? r[0] : r[1];
    }
}
template <int J>
__device__ __forceinline__ uint64_t keep(uint64_t k, bool larger) {
    const uint64_t o = (uint64_t)lane_xor<J>((uint32_t)(k >> 32)) << 32 | lane_xor<J>((uint32_t)k);
    return (o > k) == larger ? o : k;
}
// Steps J, J/2, ... 1 of a bitonic merge over runs of K lanes; falling order
// where lane & K is 0 (K = 64: everywhere).
template <int K, int J>
__device__ __forceinline__ uint64_t merge_steps(uint64_t k) {
    const uint32_t lane = threadIdx.x & 63;
    k = keep<J>(k, ((lane & J) == 0) == ((lane & K) == 0));
    if constexpr (J > 1) k = merge_steps<K, J / 2>(k);
    return k;
}
// 64 keys in falling order.
__device__ __forceinline__ uint64_t sort64(uint64_t k) {
    k = merge_steps<2, 1>(k);
    k = merge_steps<4, 2>(k);
    k = merge_steps<8, 4>(k);
    k = merge_steps<16, 8>(k);
    k = merge_steps<32, 16>(k);
    return merge_steps<64, 32>(k);
}
// The 64 largest of two lists, `a` falling and `b` rising over the lanes.
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b) { return merge_steps<64, 32>(a > b ? a : b); }

__device__ __forceinline__ uint64_t lane_key(uint64_t k, uint32_t lane) {
    return (uint64_t)__builtin_amdgcn_readlane((uint32_t)(k >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)k, lane);
}

// A lane's sums, and two of them joined.
struct Sums {
    float m = -INFINITY, s = 0.f, w = 0.f;
    __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void rise(float to, float c) {   // to >= m
        const float d = m == -INFINITY ? 0.f : (m - to) * c, f = __builtin_amdgcn_exp2f(d);
        w = f * fmaf(fmaxf(d, -1e30f), s, w);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void join(Sums o, float c) {
        const float to = fmaxf(m, o.m);
        rise(to, c);
        o.rise(to, c);
        s += o.s;
        w += o.w;
    }
};

// Row-wide results, by one wave: its sums, count and list (lane i holds the
// i-th key).
__device__ __forceinline__ void finish(const LpArgs &a, uint32_t row, const Sums &t, uint32_t before, uint64_t list,
                                       float xt, bool named) {
    const uint32_t lane = threadIdx.x & 63;
    const bool none = t.s == 0.f;   // all -inf
    const float log_s = __builtin_amdgcn_logf(t.s), ref = t.ref();
    auto lp_of = [&](float x) { return none ? -INFINITY : fmaf(x - ref, a.inv_t, -log_s * LN2); };
    if (lane == 0) {
        a.lp[row] = t.s != t.s ? t.s : named ? lp_of(xt) : -INFINITY;
        if (a.lse) a.lse[row] = none ? -INFINITY : fmaf(ref, a.inv_t, log_s * LN2);
        if (a.entropy) a.entropy[row] = none ? 0.f : (log_s - t.w / t.s) * LN2;
        if (a.rank) a.rank[row] = named ? before : a.vocab;
    }
    if (lane < a.top) {
        const size_t at = (size_t)row * a.top + lane;
        if (a.top_ids) a.top_ids[at] = list ? ~(uint32_t)list : 0xFFFFFFFFu;
        if (a.top_lp) a.top_lp[at] = list ? (t.s != t.s ? t.s : lp_of(key_value(list))) : __builtin_nanf("");
    }
}

template <int DT>
__global__ __launch_bounds__(256) void logprobs_kernel(LpArgs a) {
    constexpr uint32_t ESZ = DT == NNZ_F32 ? 4 : 2, VE = 16 / ESZ, U = GROUP / VE;   // values of a vector, vectors of a group
    __shared__ uint64_t pool[WAVES][64 * GROUP + 64];   // under 64 keys wait, a group adds 64 GROUP at most
    __shared__ float4 sums[WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    const unsigned char *const base = (const unsigned char *)a.x + (size_t)row * a.stride * ESZ;
    const uint32_t tok = a.tokens[row];
    const bool named = tok < a.vocab, order = named && a.rank;
    const float xt = named ? load_as_f32<DT>(base, tok) : 0.f;

    // 16-byte vectors from the first aligned one on; what is left over before
    // and after them (under 2 VE values) is piece 0's
    const uint32_t head = paged_min(a.vocab, (uint32_t)(-(intptr_t)base & 15) / ESZ);
    const uint32_t nv = (a.vocab - head) / VE;
    const uint32_t v0 = (uint32_t)((uint64_t)nv * piece / a.pieces), v1 = (uint32_t)((uint64_t)nv * (piece + 1) / a.pieces);
    const v4u *const vec = (const v4u *)(base + (size_t)head * ESZ);

    Sums t;
    uint32_t before = 0, held = 0;     // held: keys waiting in the pool
    uint64_t list = 0, last = 0;       // last: the list's top-th key
    float last_x = -INFINITY;
    auto flush = [&]() __attribute__((always_inline)) {   // the pool's last 64 keys join the list
        const uint32_t n = paged_min(held, 64);
        held -= n;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const uint64_t k = lane < n ? pool[wave][held + lane] : 0;
        // sorted falling, read backwards: rising
        const uint64_t sorted = sort64(k);
        __builtin_amdgcn_wave_barrier();
        pool[wave][held + lane] = sorted;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        list = merge64(list, pool[wave][held + 63 - lane]);
        __builtin_amdgcn_wave_barrier();
        last = lane_key(list, a.top - 1);
        last_x = last ? key_value(last) : -INFINITY;
    };
    // n values of a lane (at most GROUP), ids id(e); those with !on(e) are not there
    auto take = [&](const float *x, auto n_, auto id, auto on, uint32_t first, uint32_t end) __attribute__((always_inline)) {
        constexpr uint32_t n = decltype(n_)::value;
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < n; ++e) mx = fmaxf(mx, x[e]);
        if (__builtin_amdgcn_ballot_w64(mx > t.m)) t.rise(fmaxf(t.m, mx), a.c);
        const float ref = t.ref();
#pragma unroll
        for (uint32_t e = 0; e < n; ++e) {
            const float u = (x[e] - ref) * a.c, p = __builtin_amdgcn_exp2f(u);
            t.s += p;
            t.w = fmaf(p, fmaxf(u, -1e30f), t.w);
        }
        if (order) {
            // [first, end): the ids of the whole wave's group
            if (end <= tok && xt == xt) {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e) before += on(e) && x[e] >= xt;
            } else if (first > tok && xt == xt) {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e) before += on(e) && x[e] > xt;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e)
                    before += on(e) && (xt != xt ? x[e] == x[e] || id(e) < tok : x[e] > xt || (x[e] == xt && id(e) < tok));
            }
        }
        if (a.top && __builtin_amdgcn_ballot_w64(mx >= last_x)) {
            // the top-th largest of the lanes' maxima bounds what can matter
            const float floor_x = key_value(lane_key(sort64(order_key(mx, 0)), a.top - 1));
#pragma unroll
            for (uint32_t e = 0; e < n; ++e) {
                const uint64_t k = on(e) && x[e] >= floor_x ? order_key(x[e], id(e)) : 0;
                const uint64_t in = __builtin_amdgcn_ballot_w64(k > last);
                if (in) {
                    const uint32_t at = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
                    if (k > last) pool[wave][held + at] = k;
                    held += __builtin_popcountll(in);
                }
            }
            while (held >= 64 || (held && !last)) flush();
        }
    };
    auto unpack = [&](const v4u (&r)[U], float *x) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if constexpr (DT == NNZ_F32) {
                    x[4 * u + i] = __uint_as_float(r[u][i]);
                } else {
                    x[8 * u + 2 * i] = paged_load<DT == NNZ_BF16>((uint16_t)r[u][i]);
                    x[8 * u + 2 * i + 1] = paged_load<DT == NNZ_BF16>((uint16_t)(r[u][i] >> 16));
                }
            }
    };
    constexpr uint32_t STEP = 64 * U;   // vectors of a wave's group
    uint32_t v = v0 + wave * STEP;
    v4u r[U];
    auto load = [&](uint32_t at) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) r[u] = __builtin_nontemporal_load(vec + at + 64 * u + lane);
    };
    auto id_of = [&](uint32_t at, uint32_t e) { return head + (at + 64 * (e / VE) + lane) * VE + e % VE; };
    if (v + STEP <= v1) load(v);
    for (; v + STEP <= v1; v += WAVES * STEP) {   // whole groups, the next one's loads in flight
        float x[GROUP];
        unpack(r, x);
        if (v + WAVES * STEP + STEP <= v1) load(v + WAVES * STEP);
        take(x, std::integral_constant<uint32_t, GROUP>(), [&](uint32_t e) { return id_of(v, e); }, [](uint32_t) { return true; },
             head + v * VE, head + (v + STEP) * VE);
    }
    if (v < v1) {   // the last, partial one
        float x[GROUP];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) r[u] = v + 64 * u + lane < v1 ? vec[v + 64 * u + lane] : (v4u){0, 0, 0, 0};
        unpack(r, x);
#pragma unroll
        for (uint32_t e = 0; e < GROUP; ++e) x[e] = v + 64 * (e / VE) + lane < v1 ? x[e] : -INFINITY;
        take(x, std::integral_constant<uint32_t, GROUP>(), [&](uint32_t e) { return id_of(v, e); },
             [&](uint32_t e) { return v + 64 * (e / VE) + lane < v1; }, 0u, a.vocab);
    }
    if (piece == 0 && wave == WAVES - 1) {
        const uint32_t tail = head + nv * VE, left = head + (a.vocab - tail);
        if (left) {
            const uint32_t id = lane < head ? lane : tail + (lane - head);
            const bool on = lane < left;
            const float x = on ? load_as_f32<DT>(base, id) : -INFINITY;
            take(&x, std::integral_constant<uint32_t, 1>(), [&](uint32_t) { return id; }, [&](uint32_t) { return on; }, 0u, a.vocab);
        }
    }
    if (a.top && held) flush();

    // the wave's lanes, then the block's waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        Sums other;
        other.m = __shfl_xor(t.m, o);
        other.s = __shfl_xor(t.s, o);
        other.w = __shfl_xor(t.w, o);
        t.join(other, a.c);
        before += __shfl_xor(before, o);
    }
    if (lane == 0) sums[wave] = make_float4(t.m, t.s, t.w, __uint_as_float(before));
    pool[wave][lane] = list;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (uint32_t i = 1; i < WAVES; ++i) {
        const float4 f = sums[i];
        Sums other;
        other.m = f.x;
        other.s = f.y;
        other.w = f.z;
        t.join(other, a.c);
        before += __float_as_uint(f.w);
        if (a.top) list = merge64(list, pool[i][63 - lane]);
    }
    if (a.pieces == 1) {
        finish(a, row, t, before, list, xt, named);
        return;
    }
    if (lane == 0) a.part[blockIdx.x] = make_float4(t.m, t.s, t.w, __uint_as_float(before));
    if (lane < a.top) a.part_keys[(size_t)blockIdx.x * a.top + lane] = list;
}

// The pieces of a row joined: 16 waves take them in turn, then pair by pair.
template <int DT>
__global__ __launch_bounds__(1024) void logprobs_join_kernel(LpArgs a) {
    __shared__ uint64_t lists[16][64];
    __shared__ float4 sums[16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
    const uint32_t tok = a.tokens[row];
    const bool named = tok < a.vocab;
    const float xt = named ? load_as_f32<DT>(a.x, (size_t)row * a.stride + tok) : 0.f;
    Sums t;
    uint32_t before = 0;
    uint64_t list = 0;
    auto add = [&](float4 f) {
        Sums o;
        o.m = f.x;
        o.s = f.y;
        o.w = f.z;
        t.join(o, a.c);
        before += __float_as_uint(f.w);
    };
    for (uint32_t p = wave; p < a.pieces; p += 16) {
        const size_t at = (size_t)row * a.pieces + p;
        add(a.part[at]);
        if (a.top) list = merge64(list, 63 - lane < a.top ? a.part_keys[at * a.top + 63 - lane] : 0);
    }
    for (uint32_t half = 8; half; half /= 2) {
        if (wave >= half && wave < 2 * half) {
            lists[wave][lane] = list;
            if (lane == 0) sums[wave] = make_float4(t.m, t.s, t.w, __uint_as_float(before));
        }
        __syncthreads();
        if (wave < half) {
            add(sums[wave + half]);
            list = merge64(list, lists[wave + half][63 - lane]);
        }
    }
    if (wave == 0) finish(a, row, t, before, list, xt, named);
}

// Blocks for about four per CU, each with a group of values per lane at least.
uint32_t pieces_of(uint32_t rows, uint32_t vocab) {
    const uint32_t want = std::max(1u, 1024u / rows), most = std::max(1u, vocab / (WAVES * 64 * GROUP));
    return std::min(want, most);
}

template <int DT>
void start(hipStream_t stream, const LpArgs &a, uint32_t rows) {
    logprobs_kernel<DT><<<rows * a.pieces, 256, 0, stream>>>(a);
    if (a.pieces > 1) logprobs_join_kernel<DT><<<rows, 1024, 0, stream>>>(a);
}

}  // namespace

extern "C" size_t nnz_token_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top_n) {
    if (!rows || !vocab) return 0;
    const uint32_t pieces = pieces_of(rows, vocab);
    return pieces > 1 ? (size_t)rows * pieces * (16 + 8 * (size_t)top_n) : 0;
}

extern "C" int nnz_dispatch_token_logprobs(nnz_ctx *ctx, const void *logits, const uint32_t *tokens, float *logprobs,
                                           float *lse, float *entropy, uint32_t *rank, uint32_t *top_ids,
                                           float *top_logprobs, void *workspace, size_t workspace_bytes,
                                           const nnz_logprobs_dims *d) {
    NNZ_CHECK_CTX(ctx);
    if (const PagedFault f = logprobs_fault(logits, tokens, logprobs, top_ids, top_logprobs, d); f.code)
        return nnz_fail(ctx, f.code, "token_logprobs: %s", f.what);
    const size_t need = nnz_token_logprobs_workspace_bytes(d->rows, d->vocab, d->top_n);
    NNZ_REQUIRE(ctx, need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), NNZ_EINVAL,
                "token_logprobs: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", need, workspace_bytes);
    NnzDeviceScope scope(ctx);
    LpArgs a{};
    a.x = logits;
    a.tokens = tokens;
    a.lp = logprobs;
    a.lse = lse;
    a.entropy = entropy;
    a.top_lp = top_logprobs;
    a.rank = rank;
    a.top_ids = top_ids;
    a.stride = d->row_stride;
    a.vocab = d->vocab;
    a.top = d->top_n;
    a.pieces = pieces_of(d->rows, d->vocab);
    a.c = LOG2E / d->temperature;
    a.inv_t = 1.f / d->temperature;
    a.part = (float4 *)workspace;
    a.part_keys = (uint64_t *)((char *)workspace + (size_t)d->rows * a.pieces * 16);
    if (d->dtype == NNZ_F32) start<NNZ_F32>(ctx->stream, a, d->rows);
    else if (d->dtype == NNZ_F16) start<NNZ_F16>(ctx->stream, a, d->rows);
    else start<NNZ_BF16>(ctx->stream, a, d->rows);
    NNZ_LAUNCHED(ctx);
    return NNZ_OK;
}
