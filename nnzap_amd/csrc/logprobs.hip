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
//   * the number of ids that come before the token, counted from the compares'
//     lane masks;
//   * candidates for the best top_n, which wait in LDS with their ids.  A group of
//     16 values per lane is looked at again only if one of them reaches the bound,
//     a value that top_n values of the block's part are known to reach: the
//     top_n-th largest of a wave's lane maxima (16 ballots find its upper half).
//     When more than 48 + top_n wait, the same over them raises the bound and
//     leaves about top_n.  Where values are equal it leaves too many: they are
//     sorted into a list of keys (value and complemented id: larger is earlier),
//     whose last bounds what follows.  Ids rise along a wave's part, so that a
//     full list lets no equal value in: rows of equal values cost one list.
// At the end the largest of the waves' bounds leaves a few dozen of the block's
// candidates, which one sort puts in order; the pieces' lists likewise.
// Measured: 2048 x 151936 f32 193 us (6.4 TB/s), one row of 151669 14 us, of it 4
// the join; the candidates cost calls of few rows most (one row without: 11 us).
// Keys and counts are integers and the partial sums meet in a fixed order, so a
// call repeats bit for bit.
#include "paged_dev.h"

#include <algorithm>

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr uint32_t WAVES = 4, GROUP = 16;   // values of a lane looked at together
constexpr uint32_t WAITING = 112;           // most candidates of a wave that wait (48 + top)
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
    __device__ __forceinline__ void join_lanes(float c) {   // the same in every lane
        rise(wave_max(m), c);
        s = wave_sum(s);
        w = wave_sum(w);
    }
};

// The upper half of order_key, and back.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t m) {   // what lies below -inf counts as it
    return m <= 0x007FFFFFu ? -INFINITY : __uint_as_float(m >> 31 ? m & 0x7fffffffu : ~m);
}
// The n-th largest of the lanes' values, its lower 16 bits cleared: n of them
// reach it.
__device__ __forceinline__ uint32_t reached_by(uint32_t k, uint32_t n) {
    uint32_t f = 0;
#pragma unroll
    for (int b = 31; b >= 16; --b) {
        const uint32_t up = f | 1u << b;
        f = __builtin_popcountll(__builtin_amdgcn_ballot_w64(k >= up)) >= (int)n ? up : f;
    }
    return f;
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The 64 largest of n keys, falling, by one wave.  More than 64 are first cut to
// those that reach what `top` of the lanes' largest do, by way of `room` in LDS (up
// to 640 of them); where many are equal, 64 at a time are sorted and merged.
template <class Key>
__device__ __forceinline__ uint64_t sort_some(uint32_t n, uint32_t top, Key key_at, uint64_t *room) {
    const uint32_t lane = threadIdx.x & 63;
    bool moved = false;
    if (n > 64 && n <= 640) {
        uint32_t k = 0;
        for (uint32_t j = lane; j < n; j += 64) {
            const uint32_t m = (uint32_t)(key_at(j) >> 32);
            k = m > k ? m : k;
        }
        const uint32_t f = reached_by(k, top);
        uint32_t kept = 0;
        for (uint32_t j = 0; j < n; j += 64) {
            const uint64_t v = j + lane < n ? key_at(j + lane) : 0;
            const uint64_t in = __builtin_amdgcn_ballot_w64(v != 0 && (uint32_t)(v >> 32) >= f);
            if (in >> lane & 1) room[kept + lanes_below(in)] = v;
            kept += __builtin_popcountll(in);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        n = kept;
        moved = true;
    }
    uint64_t list = 0;
    for (uint32_t j = 0; j < n; j += 64) {
        uint64_t k = sort64(j + lane < n ? (moved ? room[j + lane] : key_at(j + lane)) : 0);
        if (j) {   // two falling lists: the second one backwards
            const uint32_t lo = __shfl((uint32_t)k, 63 - lane), hi = __shfl((uint32_t)(k >> 32), 63 - lane);
            k = merge64(list, (uint64_t)hi << 32 | lo);
        }
        list = k;
    }
    return list;
}

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
    __shared__ uint2 pool[WAVES][WAITING + 64 * GROUP + 64];   // value and id; later keys
    __shared__ float4 sums[WAVES];
    __shared__ float bounds[WAVES];   // the waves' bounds, as they rise
    __shared__ uint32_t counts[WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    const unsigned char *const base = (const unsigned char *)a.x + (size_t)row * a.stride * ESZ;
    // 16-byte vectors from the first aligned one on; what is left over before
    // and after them (under 2 VE values) is piece 0's
    const uint32_t head = paged_min(a.vocab, (uint32_t)(-(intptr_t)base & 15) / ESZ);
    const uint32_t nv = (a.vocab - head) / VE;
    const uint32_t v0 = (uint32_t)((uint64_t)nv * piece / a.pieces), v1 = (uint32_t)((uint64_t)nv * (piece + 1) / a.pieces);
    const v4u *const vec = (const v4u *)(base + (size_t)head * ESZ);

    constexpr uint32_t STEP = 64 * U;   // vectors of a wave's group
    uint32_t v = v0 + wave * STEP;
    v4u r[U];
    auto load = [&](uint32_t at) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) r[u] = __builtin_nontemporal_load(vec + at + 64 * u + lane);
    };
    if (v + STEP <= v1) load(v);   // before the token's value, which takes two rounds to memory

    const uint32_t tok = a.tokens[row];
    const bool named = tok < a.vocab, order = named && a.rank;
    const float xt = named ? load_as_f32<DT>(base, tok) : 0.f;

    if (threadIdx.x < WAVES) bounds[threadIdx.x] = -INFINITY;
    __syncthreads();
    const uint32_t waiting = 48 + a.top;
    Sums t;
    uint32_t before = 0, held = 0;   // held: candidates waiting in the pool
    uint64_t list = 0;
    float bound = -INFINITY;         // what a candidate reaches, or, with `above`, passes
    bool above = false;
    auto tell = [&]() __attribute__((always_inline)) {
        if (lane == 0) __hip_atomic_store(&bounds[wave], bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    auto settle = [&]() __attribute__((always_inline)) {   // LDS written by this wave is there for it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    // Raises the bound to what top of the lanes' largest candidates reach, and
    // leaves the candidates that do.
    auto narrow = [&]() __attribute__((always_inline)) {
        settle();
        uint32_t k = 0;
        for (uint32_t at = 0; at < held; at += 64) {
            const uint32_t m = order_of(__uint_as_float(pool[wave][at + lane].x));
            k = at + lane < held && m > k ? m : k;
        }
        const float to = value_of(reached_by(k, a.top));
        if (to > bound) {
            bound = to;
            above = false;
            tell();
        }
        uint32_t kept = 0;
        for (uint32_t at = 0; at < held; at += 64) {
            const uint2 f = pool[wave][at + lane];
            const uint64_t in = __builtin_amdgcn_ballot_w64(at + lane < held && __uint_as_float(f.x) >= bound);
            settle();
            if (in >> lane & 1) pool[wave][kept + lanes_below(in)] = f;
            settle();
            kept += __builtin_popcountll(in);
        }
        held = kept;
    };
    // Where values are equal that leaves too many: sorted into a list of keys,
    // whose last id bounds them too.
    auto drain = [&]() __attribute__((always_inline)) {
        narrow();
        if (held <= waiting) return;
        for (uint32_t at = 0; at < held; at += 64) {
            const uint2 f = pool[wave][at + lane];
            const uint64_t k = sort64(at + lane < held ? order_key(__uint_as_float(f.x), f.y) : 0);
            settle();
            pool[wave][at + lane] = make_uint2((uint32_t)k, (uint32_t)(k >> 32));
            settle();
            const uint2 r = pool[wave][at + 63 - lane];
            list = merge64(list, (uint64_t)r.y << 32 | r.x);
            settle();
        }
        held = 0;
        const uint64_t last = lane_key(list, a.top - 1);
        if (last && key_value(last) >= bound) {
            bound = key_value(last);
            above = true;
            tell();
        }
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
            auto add = [&](bool yes) __attribute__((always_inline)) { before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(yes)); };
            // [first, end): the ids of the whole wave's group
            if (end <= tok && xt == xt) {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e) add(on(e) && x[e] >= xt);
            } else if (first > tok && xt == xt) {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e) add(on(e) && x[e] > xt);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < n; ++e)
                    add(on(e) && (xt != xt ? x[e] == x[e] || id(e) < tok : x[e] > xt || (x[e] == xt && id(e) < tok)));
            }
        }
        if (!a.top) return;
        // any wave's bound is one of the block's
        float others = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < WAVES; ++i)
            others = fmaxf(others, __hip_atomic_load(&bounds[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
        if (others > bound) {
            bound = others;
            above = false;
        }
        const uint64_t reach = __builtin_amdgcn_ballot_w64(above ? mx > bound : mx >= bound);
        if (reach) {
            if (__builtin_popcountll(reach) >= (int)a.top) {   // else it cannot rise
                const float to = value_of(reached_by(order_of(mx), a.top));
                if (to > bound) {
                    bound = to;
                    above = false;
                    tell();
                }
            }
#pragma unroll
            for (uint32_t q = 0; q < n; q += 4) {
                float m4 = x[q];
#pragma unroll
                for (uint32_t e = q + 1; e < q + 4 && e < n; ++e) m4 = fmaxf(m4, x[e]);
                if (!__builtin_amdgcn_ballot_w64(m4 >= bound)) continue;
#pragma unroll
                for (uint32_t e = q; e < q + 4 && e < n; ++e) {
                    const bool mine = on(e) && (above ? x[e] > bound : x[e] >= bound);
                    const uint64_t in = __builtin_amdgcn_ballot_w64(mine);
                    if (in) {
                        if (mine) pool[wave][held + lanes_below(in)] = make_uint2(__float_as_uint(x[e]), id(e));
                        held += __builtin_popcountll(in);
                    }
                }
            }
            if (held > waiting) drain();
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
    auto id_of = [&](uint32_t at, uint32_t e) { return head + (at + 64 * (e / VE) + lane) * VE + e % VE; };
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
            above = false;   // its ids may be lower than the list's
            const uint32_t id = lane < head ? lane : tail + (lane - head);
            const bool on = lane < left;
            const float x = on ? load_as_f32<DT>(base, id) : -INFINITY;
            take(&x, std::integral_constant<uint32_t, 1>(), [&](uint32_t) { return id; }, [&](uint32_t) { return on; }, 0u, a.vocab);
        }
    }

    // the wave's lanes, then the block's waves
    if (held > a.top) narrow();
    t.join_lanes(a.c);
    if (lane == 0) {
        sums[wave] = make_float4(t.m, t.s, t.w, __uint_as_float(before));
        bounds[wave] = bound;
    }
    __syncthreads();
    if (a.top) {
        // what reaches every wave's bound moves to the front of the wave's pool, as keys
        const float reach = fmaxf(fmaxf(bounds[0], bounds[1]), fmaxf(bounds[2], bounds[3]));
        uint32_t kept = 0;
        auto put = [&](uint64_t k) __attribute__((always_inline)) {
            const uint64_t in = __builtin_amdgcn_ballot_w64(k != 0);
            settle();
            if (k) pool[wave][kept + lanes_below(in)] = make_uint2((uint32_t)k, (uint32_t)(k >> 32));
            settle();
            kept += __builtin_popcountll(in);
        };
        for (uint32_t at = 0; at < held; at += 64) {
            const uint2 f = pool[wave][at + lane];
            const float x = __uint_as_float(f.x);
            put(at + lane < held && x >= reach ? order_key(x, f.y) : 0);
        }
        if (__builtin_amdgcn_ballot_w64(list != 0)) put(lane < a.top ? list : 0);
        if (lane == 0) counts[wave] = kept;
        __syncthreads();
    }
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
    }
    if (a.top) {
        const uint32_t n0 = counts[0], n1 = n0 + counts[1], n2 = n1 + counts[2];
        uint32_t n = n2 + counts[3];
        auto key_at = [&](uint32_t i) {
            const uint2 f = i < n0 ? pool[0][i] : i < n1 ? pool[1][i - n0] : i < n2 ? pool[2][i - n1] : pool[3][i < n ? i - n2 : 0];
            return i < n ? (uint64_t)f.y << 32 | f.x : 0;
        };
        list = sort_some(n, a.top, key_at, (uint64_t *)&pool[0][2 * WAITING]);
    }
    if (a.pieces == 1) {
        finish(a, row, t, before, list, xt, named);
        return;
    }
    if (lane == 0) a.part[blockIdx.x] = make_float4(t.m, t.s, t.w, __uint_as_float(before));
    if (lane < a.top) a.part_keys[(size_t)blockIdx.x * a.top + lane] = list;
}

// The pieces of a row joined: sums by wave 0, a piece a lane; keys that reach
// every piece's last one, and what `top` of the pieces' first few reach, are
// gathered in LDS, a few dozen, and sorted.  (Where pieces are equal in value the
// last keys differ by id, so that the bound, the largest of them, leaves fewer
// than 64 of each.)  One row of 151669, top 64: by last keys alone 47 us, now 26.
template <int DT>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LpArgs a) {
    extern __shared__ uint64_t kept[];   // [pieces * top]
    __shared__ uint64_t reach[WAVES], room[640];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const float4 *const part = a.part + (size_t)row * a.pieces;
    const uint64_t *const keys = a.part_keys + (size_t)row * a.pieces * a.top;
    const uint32_t nk = a.pieces * a.top, tok = a.tokens[row];
    // every load at once: the first part of a lane, the pieces' last keys (at most
    // 96, a thread each), the first four keys of a thread
    const float4 first = lane < a.pieces ? part[lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    const uint64_t last = a.top && tid < a.pieces ? keys[(size_t)tid * a.top + a.top - 1] : 0;
    // what r lanes' j-th keys reach, r j keys do (a lane is one piece or two; about
    // two thirds of them are asked for)
    const uint32_t lanes = paged_min(a.pieces, 64u), j = (3 * a.top + 2 * lanes - 1) / (2 * lanes);
    uint32_t jth = 0;
    if (a.top)
        for (uint32_t p = lane; p < a.pieces; p += 64) {
            const uint32_t m = (uint32_t)(keys[(size_t)p * a.top + j - 1] >> 32);
            jth = m > jth ? m : jth;
        }
    uint64_t mine[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) mine[i] = tid + 256 * i < nk ? keys[tid + 256 * i] : 0;
    const bool named = tok < a.vocab;
    const float xt = named ? load_as_f32<DT>(a.x, (size_t)row * a.stride + tok) : 0.f;
    if (a.top) {
        uint64_t k = last;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t v = __shfl_xor((unsigned long long)k, o);
            k = v > k ? v : k;
        }
        if (lane == 0) reach[wave] = k;
        if (tid == 0) count = 0;
        const uint32_t m = reached_by(jth, (a.top + j - 1) / j);   // the same in every wave
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < WAVES; ++i) k = reach[i] > k ? reach[i] : k;
        k = (uint64_t)m << 32 > k ? (uint64_t)m << 32 : k;
        auto put = [&](uint64_t v) {
            if (v && v >= k) kept[atomicAdd(&count, 1u)] = v;   // any order: they are sorted next
        };
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) put(mine[i]);
        for (uint32_t i = tid + 1024; i < nk; i += 256) put(keys[i]);
        __syncthreads();
    }
    if (wave) return;
    Sums t;
    uint32_t before = 0;
    for (uint32_t p = lane; p < a.pieces; p += 64) {
        const float4 f = p == lane ? first : part[p];
        Sums o;
        o.m = f.x;
        o.s = f.y;
        o.w = f.z;
        t.join(o, a.c);
        before += __float_as_uint(f.w);
    }
    t.join_lanes(a.c);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) before += __shfl_xor(before, o);
    const uint64_t list = a.top ? sort_some(count, a.top, [&](uint32_t i) { return kept[i]; }, room) : 0;
    finish(a, row, t, before, list, xt, named);
}

// Blocks for about four per CU, each with a group of values per lane at least.
// (512, 1024 and 2048 blocks: 333 x 50257 bf16 34.8, 25.0 and 31.0 us.)
// At most 96: the join's keys (64 each) stay within 48 KB of LDS.
uint32_t pieces_of(uint32_t rows, uint32_t vocab) {
    const uint32_t want = std::max(1u, 1024u / rows), most = std::max(1u, vocab / (WAVES * 64 * GROUP));
    return std::min({want, most, 96u});
}

template <int DT>
void start(hipStream_t stream, const LpArgs &a, uint32_t rows) {
    logprobs_kernel<DT><<<rows * a.pieces, 256, 0, stream>>>(a);
    if (a.pieces > 1) logprobs_join_kernel<DT><<<rows, 256, (size_t)a.pieces * a.top * 8, stream>>>(a);
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
