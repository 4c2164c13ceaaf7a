// Attention of a ragged batch over a paged KV cache (nnz.h,
// nnz_dispatch_paged_attention), on the matrix cores.
//
// The rows of a sequence and KV head are the pairs (token, query head of the
// group), row r = token * G + head, so that one pass over K and V serves all G
// heads, and a single token of G heads is a matrix product too.  Both kernels
// compute scores transposed, S^T[key][row] = K . Q^T, with K as the A operand
// in a key order that leaves the accumulators holding, per lane, the eight
// consecutive keys that the second product O^T[dim][row] += V^T . P^T wants of
// it as its B operand: the weights never move between lanes.  V's pages are
// transposed, so V^T's A operand is 16 contiguous bytes of a page.
//
//   few_part    at most 16 rows (single tokens, drafts): bound by the bytes of
//               K and V, which go straight from memory into the operand
//               registers, each byte once; keys are split over waves and blocks;
//   chunk_part  more rows (chunks of prompts): bound by the matrix cores and the
//               softmax's vector work beside them; 128 rows a block, K and V
//               tiles of 64 keys in LDS; keys are split over two groups of waves,
//               and over blocks where there are few rows.
// join_kernel joins what blocks computed of one row.
//
// Measured (kernels' time): one token over 131072 (32 + 8 heads of 128, bf16, 537
// MB) 95 + 8 us, 5.6 TB/s; 64 chats of up to 8191 (1.17 GB) 238 + 5, 4.9 TB/s; 2048
// tokens over 8192 (16 + 8 heads of 128, 155 GFLOP) 165-172 us, 0.9 PFLOP/s: there 256
// KB of LDS reads a turn take 3000 of a CU's 4400 cycles, vector instructions 2600,
// the matrix cores 2048; 64 rows a wave would halve the reads, but leave one wave
// a SIMD.
//
// The softmax is the online one in base 2: sums are kept relative to a
// reference M per row, which follows the row's maximum only when that runs
// ahead by more than 2^8 (weights up to 2^8 cost no precision: f16 and bf16
// weights are relative to themselves and the sums are f32), so that most steps
// rescale nothing.
#include "paged_dev.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

constexpr uint32_t FEW = 16;      // most rows of few_part
constexpr uint32_t TILE_ROWS = 128;
constexpr uint32_t KT = 64;       // keys per tile of chunk_part
constexpr float LN2 = 0.69314718055994531f, LOG2E = 1.44269504088896341f;

struct AttnArgs {
    PagedView b;
    const uint16_t *q, *k, *v;
    uint16_t *out;
    float *lse;
    const float *slopes;
    const uint32_t *prefix;
    uint64_t q_stride, o_stride;
    uint32_t hq, G, window;
    float scale;          // of the scores, times log2 e
    float unbias;         // 1 / scale before that: a bias in units of products
    float cap_in, cap;    // softcap: cap * tanh(x) with 2 log2(e) x = cap_in * (q . k); cap times log2 e
    // Sequences of at most `few` rows (0: none) are few_part's: keys in chunks of
    // few_steps steps, at most few_splits of them, a block each, few_blocks in all.
    uint32_t few, few_splits, few_steps, few_blocks;
    // The others' are chunk_part's: `units` row tiles in the whole batch, an upper
    // bound, keys in chunks of chunk_tiles tiles, at most chunk_splits of them.
    uint32_t units, chunk_splits, chunk_tiles;
    uint32_t few_rows;              // most rows of a sequence in few_part
    float *few_o, *few_ml, *chunk_o, *chunk_ml;
};

template <bool BF>
__device__ __forceinline__ float4v mfma16(v4u a, v4u b, float4v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ float16v mfma32(v4u a, v4u b, float16v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Two values rounded to nearest into one word.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const float2v f = {a, b};
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf2v));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, half2v));
}

// A step that some rows see only in part must not let a hidden key's weight of
// 0 meet NaN or infinities in V.  Such steps multiply by V without those;
// where one was met (odd), the rows that do see it get it afterwards, in a pass
// of its own over the wave's keys (odd_value).
template <bool BF>
__device__ __forceinline__ v4u finite_part(v4u v, uint32_t &odd) {
    constexpr uint32_t EXP = BF ? 0x7F807F80u : 0x7C007C00u, STEP = BF ? 0x00800080u : 0x04000400u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = ((v[i] & EXP) + STEP) & 0x80008000u;   // of each half: all exponent bits set
        odd |= t;
        v[i] &= ~((t - (t >> 15)) | t);
    }
    return v;
}
template <bool BF>
__device__ __forceinline__ float odd_value(uint16_t v, bool seen) {
    const float f = paged_load<BF>(v);
    return seen && !(fabsf(f) < INFINITY) ? f : 0.f;
}

// How a product becomes a score.  Without a softcap scores stay in units of
// products, a bias too, and are scaled in the exponent; capped ones are in log2 units.
enum { PLAIN, BIASED, CAPPED, CAPPED_BIASED };
constexpr bool biased(int sc) { return sc & 1; }
constexpr bool capped(int sc) { return sc & 2; }
template <int SC>
__device__ __forceinline__ float score_of(const AttnArgs &a, float s, float slope, int32_t distance) {
    if constexpr (capped(SC))   // tanh(x) = 1 - 2 / (e^2x + 1)
        s = a.cap * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a.cap_in * s) + 1.f), 1.f);
    if constexpr (biased(SC)) s = fmaf(-slope, fabsf((float)distance), s);
    return s;
}

// ---------------------------------------------------------------- few rows
// A step is 32 keys of a wave: K as two A operands of 16 keys (row m of operand
// i is key 8 (m >> 2) + 4 i + (m & 3), so lane group g's accumulators hold keys
// 8 g .. 8 g + 7), V^T as D/16 A operands.  With AHEAD the next step's loads are
// issued before the current one is computed.  Block = W waves that take the steps
// of a chunk in turn.
template <int D, bool BF>
struct FewStep {
    v4u k[2][D / 32], v[D / 16];
    uint32_t bad;   // groups of 16 keys without a page
};

template <int D, int W>
struct FewShared {
    float4v o[W][D / 16][64];
    float m[W][16], l[W][16];
};

template <int D, bool BF, int SC, int W, bool AHEAD>
__device__ __forceinline__ void few_part(const AttnArgs &a, uint32_t block, FewShared<D, W> &sh) {
    constexpr int NKS = D / 32, NDT = D / 16;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    const uint32_t hkv = a.b.hkv, kvh = block % hkv, z = block / hkv % a.few_splits, s = block / hkv / a.few_splits;
    const PagedSeq sq = paged_seq(a.b, s);
    const uint32_t n = paged_min(sq.n, a.b.max_q), R = n * a.G;
    if (R == 0 || R > FEW) return;
    const uint32_t prefix = a.prefix ? a.prefix[s] : 0u;
    const PagedSpan sp0 = paged_span(sq.first, sq.len, prefix, a.window);
    const PagedSpan sp1 = paged_span(sq.first + (int32_t)n - 1, sq.len, prefix, a.window);
    const uint32_t lo = sp0.lo & ~31u, hi = sp1.hi, steps = hi > lo ? (hi - lo + 31) / 32 : 0;
    const uint32_t nz = steps > a.few_steps ? (steps + a.few_steps - 1) / a.few_steps : 1;
    if (z >= nz) return;
    const uint32_t st1 = paged_min(steps, (z + 1) * a.few_steps);

    const uint32_t r = paged_min((uint32_t)c, R - 1), tok = r / a.G, head = kvh * a.G + r % a.G;
    const int32_t pos = sq.first + (int32_t)tok;
    const PagedSpan sp = paged_span(pos, sq.len, prefix, a.window);
    const float slope = biased(SC) ? a.slopes[head] * (capped(SC) ? LOG2E : a.unbias) : 0.f;
    v4u qf[NKS];
    {
        const uint16_t *qp = a.q + (sq.row0 + tok) * a.q_stride + head * D;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[ks] = *(const v4u *)(qp + 32 * ks + 8 * g);
    }

    // elements of a page; this head's part of page 0
    const uint32_t pmask = (1u << a.b.shift) - 1, page_len = (hkv * D) << a.b.shift;
    const uint16_t *const kh = a.k + (((size_t)kvh * D) << a.b.shift), *const vh = a.v + (((size_t)kvh * D) << a.b.shift);
    auto load = [&](FewStep<D, BF> &f, uint32_t st) __attribute__((always_inline)) {
        const uint32_t k0 = lo + 32 * st;
        uint32_t pa = paged_raw(a.b, s, k0), pb = paged_raw(a.b, s, k0 + 16);
        f.bad = (pa < a.b.num_pages ? 0u : 1u) | (k0 + 16 < hi && pb < a.b.num_pages ? 0u : 2u);
        pa = f.bad & 1 ? 0u : pa;   // any page: the keys are masked
        pb = f.bad & 2 ? 0u : pb;
        const uint64_t ha = (uint64_t)pa * page_len, hb = (uint64_t)pb * page_len;
        const uint32_t oa = k0 & pmask, ob = (k0 + 16) & pmask;
        const uint16_t *ka = kh + ha + oa * D, *kb = kh + hb + ob * D;
        const uint16_t *kp = (c < 8 ? ka : kb) + (8 * (c >> 2 & 1) + (c & 3)) * D + 8 * g;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) f.k[i][ks] = *(const v4u *)(kp + 4 * i * D + 32 * ks);
        const uint16_t *va = vh + ha + oa, *vb = vh + hb + ob;
        const uint16_t *vp = (g < 2 ? va : vb) + ((size_t)c << a.b.shift) + 8 * (g & 1);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) f.v[dt] = *(const v4u *)(vp + ((size_t)(16 * dt) << a.b.shift));
    };

    float4v o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = (float4v){0.f, 0.f, 0.f, 0.f};
    const float cs = capped(SC) ? 1.f : a.scale, ahead = 8.f / cs;
    float m = -INFINITY, nm = 0.f, l = 0.f;   // reference score, minus it in log2 units, sum of this lane's weights
    uint32_t odd = 0;
    auto in_part = [&](uint32_t k0, uint32_t bad) { return k0 < sp1.lo || k0 + 32 > sp0.hi || bad; };   // wave-uniform
    auto compute = [&](const FewStep<D, BF> &f, uint32_t st) __attribute__((always_inline)) {
        const uint32_t k0 = lo + 32 * st;
        float sc[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float4v t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) t = mfma16<BF>(f.k[i][ks], qf[ks], t);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[4 * i + e] = t[e];
        }
        const uint32_t key = k0 + 8 * g;
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e] = score_of<SC>(a, sc[e], slope, pos - (int32_t)(key + e));
        const bool masked = in_part(k0, f.bad);
        if (masked) {
            const bool on = !(f.bad >> (g >> 1) & 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) sc[e] = on && key + e >= sp.lo && key + e < sp.hi ? sc[e] : -INFINITY;
        }
        float mx = sc[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
        if (__builtin_amdgcn_ballot_w64(mx > m + ahead)) {   // wave-uniform
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const bool move = mx > m + ahead;
            const float nm2 = move ? -mx * cs : nm;
            const float alpha = move && m != -INFINITY ? __builtin_amdgcn_exp2f(nm2 - nm) : 1.f;
            m = move ? mx : m;
            nm = nm2;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], cs, nm));
            l += sc[e];
        }
        v4u p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pack2<BF>(sc[2 * i], sc[2 * i + 1]);
        if (masked) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] = mfma16<BF>(finite_part<BF>(f.v[dt], odd), p, o[dt]);
        } else {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] = mfma16<BF>(f.v[dt], p, o[dt]);
        }
    };

    uint32_t st = z * a.few_steps + (uint32_t)w;
    if constexpr (!AHEAD) {
        for (; st < st1; st += W) {   // wave-uniform
            FewStep<D, BF> f;
            load(f, st);
            compute(f, st);
        }
    } else if (st < st1) {   // wave-uniform, all of it
        FewStep<D, BF> f0, f1;
        load(f0, st);
        for (;;) {
            if (st + W < st1) load(f1, st + W);
            compute(f0, st);
            st += W;
            if (st >= st1) break;
            if (st + W < st1) load(f0, st + W);
            compute(f1, st);
            st += W;
            if (st >= st1) break;
        }
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, 0)) {   // wave-uniform
        for (st = z * a.few_steps + (uint32_t)w; st < st1; st += W) {
            const uint32_t k0 = lo + 32 * st;
            const bool hole = paged_entry(a.b, s, k0, true) == a.b.num_pages ||
                              paged_entry(a.b, s, k0 + 16, k0 + 16 < hi) == a.b.num_pages;
            if (!in_part(k0, hole)) continue;   // whole steps had V as it is
            for (uint32_t key = k0; key < k0 + 32; ++key) {
                const uint32_t page = paged_entry(a.b, s, key, key < hi);
                if (page == a.b.num_pages) continue;
                const uint16_t *vp = vh + (uint64_t)page * page_len + (key & pmask);
                const bool seen = key >= sp.lo && key < sp.hi;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[dt][e] += odd_value<BF>(vp[(16 * dt + 4 * g + e) << a.b.shift], seen);
                    __builtin_amdgcn_sched_barrier(0);   // all loads at once would take registers
                }
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' parts, relative to the largest reference
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) sh.o[w][dt][lane] = o[dt];
    if (g == 0) {
        sh.m[w][c] = m == -INFINITY ? -INFINITY : -nm;
        sh.l[w][c] = l;
    }
    __syncthreads();
    float M = sh.m[0][c], wt[W];
#pragma unroll
    for (int i = 1; i < W; ++i) M = fmaxf(M, sh.m[i][c]);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        wt[i] = sh.m[i][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sh.m[i][c] - M);
        l += wt[i] * sh.l[i][c];   // NaN stays NaN, times 0 too
    }
    const bool mine = (uint32_t)c < R;
    if (nz == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t *op = a.out + (sq.row0 + tok) * a.o_stride + head * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            if (dt % W != w) continue;
            float4v t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; ++i) t += sh.o[i][dt][lane] * wt[i];
            if (mine)
                *(uint2 *)(op + 16 * dt) = make_uint2(pack2<BF>(t[0] * inv, t[1] * inv), pack2<BF>(t[2] * inv, t[3] * inv));
        }
        if (a.lse && mine && g == 0 && w == 0)
            a.lse[(size_t)(sq.row0 + tok) * a.hq + head] = l == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * LN2;
        return;
    }
    const size_t part = (((size_t)s * hkv + kvh) * a.few_splits + z) * a.few_rows + (uint32_t)c;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
        if (dt % W != w) continue;
        float4v t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; ++i) t += sh.o[i][dt][lane] * wt[i];
        if (mine) *(float4v *)(a.few_o + part * D + 16 * dt + 4 * g) = t;
    }
    if (mine && g == 0 && w == 0) {
        a.few_ml[2 * part] = M;
        a.few_ml[2 * part + 1] = l;
    }
}

// ------------------------------------------------------------ chunks of rows
// 16 bytes per lane from memory straight into LDS: lane i's to lds + 16 i.
__device__ __forceinline__ void load_to_lds(const void *sbase, uint32_t voff, uint32_t lds) {
    // five wait states between a VALU write of an SGPR and its use as address
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds) : "memory");
}

// What unit u of the batch's row tiles is: tile `tile` of sequence `s`.
__device__ __forceinline__ bool find_tile(const AttnArgs &a, uint32_t u, uint32_t *s, uint32_t *tile) {
    return paged_find(a.b.num_seqs, u, s, tile, [&](uint32_t i) {
        const uint32_t rows = paged_min(paged_seq(a.b, i).n, a.b.max_q) * a.G;
        return rows <= a.few ? 0u : (rows + TILE_ROWS - 1) / TILE_ROWS;
    });
}

// Tile `tile` of sequence s: its rows and its keys, in tiles of KT.
struct RowTile {
    PagedSeq sq;
    uint32_t R, r0, prefix, lo, hi, t0, t1, nz;
};
__device__ __forceinline__ RowTile row_tile(const AttnArgs &a, uint32_t s, uint32_t tile) {
    RowTile t;
    t.sq = paged_seq(a.b, s);
    t.R = paged_min(t.sq.n, a.b.max_q) * a.G;
    t.r0 = tile * TILE_ROWS;
    t.prefix = a.prefix ? a.prefix[s] : 0u;
    const uint32_t last = paged_min(t.r0 + TILE_ROWS, t.R) - 1;
    t.lo = paged_span(t.sq.first + (int32_t)(t.r0 / a.G), t.sq.len, t.prefix, a.window).lo;
    t.hi = paged_span(t.sq.first + (int32_t)(last / a.G), t.sq.len, t.prefix, a.window).hi;
    t.t0 = t.lo / KT;
    t.t1 = t.hi > t.lo ? (t.hi + KT - 1) / KT : t.t0;
    t.nz = a.chunk_splits > 1 && t.t1 - t.t0 > a.chunk_tiles ? (t.t1 - t.t0 + a.chunk_tiles - 1) / a.chunk_tiles : 1;
    return t;
}

// A block owns 128 rows of one KV head, a wave 32 of them
// (v_mfma_f32_32x32x16); accumulator register 4 j + e of lane half hh is row
// 8 j + 4 hh + e of a 32-key A operand, whose row m is key m with bits 2 and 3
// swapped: registers 8 i .. 8 i + 7 are keys 16 i + 8 hh ...  K rows lie in
// LDS with their 16-byte pieces rotated (piece p of row r at slot p ^ r), V as
// its pages have it, [16-key group][dim][16 keys], where a wave's operand is
// one contiguous run.
//
// The block's eight waves are two groups of four that hold the same rows and
// take the key tiles in turn, half a tile apart: a SIMD has a wave of each, and
// while one multiplies K and Q the other runs its softmax and the product with
// V, so that matrix and vector instructions of the two overlap.  A barrier ends
// every half.  At the end the second group's sums join the first's.
template <int D>
struct ChunkShared {
    union {
        struct {
            uint16_t k[2][2][KT * D], v[2][2][KT * D];   // [group][buffer]
        };
        float join[4][D / 2 + 2][64];   // [wave][register][lane]
    };
    uint32_t odd[2][4];   // [group][wave]
};

template <int D, bool BF, int SC>
__device__ __forceinline__ void chunk_part(const AttnArgs &a, uint32_t block, ChunkShared<D> &sh) {
    constexpr int NKS = D / 16, NDT = D / 32, PIECES = D / 8;   // pieces of 16 bytes in a K row
    constexpr int TILE = KT * D, LOADS = TILE / 8 / 256;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5, c = lane & 31;
    const uint32_t group = __builtin_amdgcn_readfirstlane(tid >> 8);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6 & 3);
    // KV head fastest: with 8 of them each XCD keeps one head's K and V in its L2;
    // the last tiles, which see the most keys, first
    const uint32_t hkv = a.b.hkv, kvh = block % hkv, z = block / hkv % a.chunk_splits;
    const uint32_t u = a.units - 1 - block / hkv / a.chunk_splits;
    uint32_t s, tile;
    if (!find_tile(a, u, &s, &tile)) return;
    const RowTile rt = row_tile(a, s, tile);
    if (z >= rt.nz) return;
    const uint32_t t0 = a.chunk_splits > 1 ? rt.t0 + z * a.chunk_tiles : rt.t0;
    const uint32_t t1 = a.chunk_splits > 1 ? paged_min(rt.t1, t0 + a.chunk_tiles) : rt.t1;

    const uint32_t w0 = rt.r0 + 32u * (uint32_t)wave;
    const bool any = w0 < rt.R;   // wave-uniform
    const uint32_t wl = paged_min(w0 + 31, rt.R - 1), r = paged_min(w0 + (uint32_t)c, rt.R - 1);
    auto span_of = [&](uint32_t row) {
        return paged_span(rt.sq.first + (int32_t)(row / a.G), rt.sq.len, rt.prefix, a.window);
    };
    const PagedSpan first = span_of(paged_min(w0, rt.R - 1)), last = span_of(wl), sp = span_of(r);
    const uint32_t tok = r / a.G, head = kvh * a.G + r % a.G;
    const int32_t pos = rt.sq.first + (int32_t)tok;
    const float slope = biased(SC) ? a.slopes[head] * (capped(SC) ? LOG2E : a.unbias) : 0.f;

    // Wave w stages group w of a tile's four groups of 16 keys, K and V alike:
    // one page.  Piece i of a lane: 16 bytes of K row 64 i / PIECES + lane / PIECES,
    // of V^T row 32 i + lane / 2.
    constexpr uint32_t RPW = 64 / PIECES;   // K rows of the wave's piece
    uint32_t koff[LOADS];
    const uint32_t voff = (((uint32_t)lane / 2) << a.b.shift) * 2u + ((uint32_t)lane & 1) * 16u;
#pragma unroll
    for (uint32_t i = 0; i < LOADS; ++i) {
        const uint32_t row = i * RPW + (uint32_t)lane / PIECES;
        koff[i] = (row * D + 8 * (((uint32_t)lane % PIECES) ^ (row & (PIECES - 1)))) * 2u;
    }
    // elements of a page; this head's part of page 0
    const uint32_t pmask = (1u << a.b.shift) - 1, page_len = (hkv * D) << a.b.shift;
    const uint16_t *const kh = a.k + (((size_t)kvh * D) << a.b.shift), *const vh = a.v + (((size_t)kvh * D) << a.b.shift);
    struct Pages {
        uint32_t p[4];   // table entries of the tile's groups of 16 keys, as they stand there
    };
    auto pages_of = [&](uint32_t t) __attribute__((always_inline)) {
        Pages p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p.p[i] = paged_raw(a.b, s, t * KT + 16 * i);
        return p;
    };
    auto has_page = [&](const Pages &p, uint32_t t, int i) { return t * KT + 16 * i < rt.hi && p.p[i] < a.b.num_pages; };
    const uint32_t lds_k = __builtin_amdgcn_readfirstlane(
        (uint32_t)(size_t)(__attribute__((address_space(3))) uint16_t *)(sh.k[group][0] + 16 * D * wave));
    const uint32_t lds_v = __builtin_amdgcn_readfirstlane(
        (uint32_t)(size_t)(__attribute__((address_space(3))) uint16_t *)(sh.v[group][0] + 16 * D * wave));
    auto stage = [&](uint32_t t, uint32_t entry, uint32_t half) __attribute__((always_inline)) {
        const uint32_t key = t * KT + 16 * (uint32_t)wave, buf = half * (TILE * 2);
        // any page where there is none: the keys are masked
        const uint32_t page = key < rt.hi && entry < a.b.num_pages ? entry : 0u, slot = key & pmask;
        const uint64_t at = (uint64_t)page * page_len;
        const uint16_t *const kp = kh + at + slot * D, *const vp = vh + at + slot;
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) {
            load_to_lds(kp, koff[i], lds_k + buf + 1024 * i);
            load_to_lds(vp + ((32 * i) << a.b.shift), voff, lds_v + buf + 1024 * i);
        }
    };
    auto bad_of = [&](const Pages &p, uint32_t t) __attribute__((always_inline)) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= (has_page(p, t, i) ? 0u : 1u) << i;
        return bad;
    };

    // table entries: this wave's of the group's next tile, all of this one and the next
    const uint32_t ta = t0 + group;
    Pages cur{}, next{};
    uint32_t ahead_entry = 0;
    if (ta < t1) {
        cur = pages_of(ta);
        stage(ta, paged_raw(a.b, s, ta * KT + 16 * (uint32_t)wave), 0);
        next = pages_of(ta + 2);
        ahead_entry = paged_raw(a.b, s, (ta + 2) * KT + 16 * (uint32_t)wave);
    }
    v4u qf[NKS];
    {
        const uint16_t *qp = a.q + (rt.sq.row0 + tok) * a.q_stride + head * D;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[ks] = *(const v4u *)(qp + 16 * ks + 8 * hh);
    }
    float16v o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    const float cs = capped(SC) ? 1.f : a.scale, ahead = 8.f / cs;
    float m = -INFINITY, nm = 0.f, l = 0.f;
    bool odd = false;   // wave-uniform
    // tiles that some rows of the wave, of the block, see only in part
    auto in_part = [&](uint32_t k0, uint32_t gone) { return k0 < last.lo || k0 + KT > first.hi || gone; };
    const uint32_t lo_most = span_of(paged_min(rt.r0 + TILE_ROWS, rt.R) - 1).lo, hi_least = span_of(rt.r0).hi;
    auto block_part = [&](uint32_t k0, uint32_t gone) { return k0 < lo_most || k0 + KT > hi_least || gone; };
    const int krm = (c & 19) | ((c & 4) << 1) | ((c & 8) >> 1);   // key of A row c

    auto barrier = [&]() __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const uint32_t turns = (t1 - t0 + 1) / 2;   // of both groups; the second's last tile may not be there
    if (group) barrier();
    for (uint32_t i = 0; i < turns; ++i) {
        const uint32_t t = ta + 2 * i, k0 = t * KT;
        // the group's loads of this tile have arrived, and its waves are done
        // with the other buffer
        __builtin_amdgcn_s_waitcnt(7 << 4);   // vmcnt 0, lgkmcnt 0
        const uint32_t bad = bad_of(cur, t);
        if (t < t1 && block_part(k0, bad)) {   // the 16 keys that this wave has staged
            uint16_t *const mine = sh.v[group][i & 1] + 16 * D * wave + 8 * lane;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                v4u *const at = (v4u *)(mine + 512 * j);
                uint32_t met = 0;
                const v4u v = finite_part<BF>(*at, met);
                if (met) *at = v;
                odd |= __builtin_amdgcn_ballot_w64(met != 0) != 0;
            }
            __builtin_amdgcn_s_waitcnt(7 << 4);
        }
        barrier();
        if (t + 2 < t1) {   // group-uniform
            stage(t + 2, ahead_entry, (i + 1) & 1);
            cur = next;
            next = pages_of(t + 4);
            ahead_entry = paged_raw(a.b, s, (t + 4) * KT + 16 * (uint32_t)wave);
        }
        if (t >= t1 || !any || k0 >= last.hi || k0 + KT <= first.lo) {   // wave-uniform
            barrier();
            continue;
        }
        // computed anew in every turn where registers are short: the asm hides that they need not be
        uint32_t krow = krm * D + 8 * (hh ^ (krm & (PIECES - 1)));
        if constexpr (D == 64) asm volatile("" : "+v"(krow));
        const uint16_t *const Kt = sh.k[group][i & 1], *const Vt = sh.v[group][i & 1];
        // scores of both halves of the tile; the operands of a half are all read
        // before its products, the second half's during the first one's
        float16v sc[2];
        v4u kf[2][NKS];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) kf[kt][ks] = *(const v4u *)(Kt + 32 * kt * D + (krow ^ 16 * ks));
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[kt][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) sc[kt] = mfma32<BF>(kf[kt][ks], qf[ks], sc[kt]);
        }
        // V^T of the first 16 keys, read while the softmax runs
        v4u vf[NDT];
        auto read_v = [&](int st) __attribute__((always_inline)) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) vf[dt] = *(const v4u *)(Vt + st * (16 * D) + (32 * dt + c) * 16 + 8 * hh);
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        barrier();
        // at head_dim 128 the sums go first: measured without and with it, 2048 rows
        // over 8192 184.9 and 179.1 us, 1500 over 3000 76.2 and 72.6; at 64, 102 and
        // 103 (capped), 51.3 and 54.0 (five prompts, biased)
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
        uint32_t key = k0 + 8 * hh;   // register e of half kt: key + 32 kt + 16 (e >> 3) + (e & 7)
        int32_t rel = pos - (int32_t)key;
        if constexpr (D == 64) asm volatile("" : "+v"(key), "+v"(rel));
        auto few_at_once = [](int e) __attribute__((always_inline)) {   // chains in flight take registers
            if (D == 64 && e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (capped(SC)) {
            const float cap2 = -2.f * a.cap;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                sc[e >> 4][e & 15] = fmaf(cap2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a.cap_in * sc[e >> 4][e & 15]) + 1.f), a.cap);
                few_at_once(e);
            }
        }
        if constexpr (biased(SC)) {
            const float d = (float)rel;   // distances are exact up to 2^24, and as good as the scores beyond
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                sc[e >> 4][e & 15] = fmaf(-slope, fabsf(d - (float)(16 * (e >> 3) + (e & 7))), sc[e >> 4][e & 15]);
                few_at_once(e);
            }
        }
        const bool masked = in_part(k0, bad);
        if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const uint32_t j = key + 16 * (e >> 3) + (e & 7);
                const bool on = j >= sp.lo && j < sp.hi && !(bad >> (e >> 3) & 1);
                sc[e >> 4][e & 15] = on ? sc[e >> 4][e & 15] : -INFINITY;
                few_at_once(e);
            }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
        if (__builtin_amdgcn_ballot_w64(mx > m + ahead)) {   // wave-uniform
            const float2 both = swap32(mx, mx);
            mx = fmaxf(both.x, both.y);
            const bool move = mx > m + ahead;
            const float nm2 = move ? -mx * cs : nm;
            const float alpha = move && m != -INFINITY ? __builtin_amdgcn_exp2f(nm2 - nm) : 1.f;
            m = move ? mx : m;
            nm = nm2;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        }
        // Weights of two keys, and a word of the B operand of the 16 keys they are in
        auto weigh = [&](int i) __attribute__((always_inline)) {
            const float x = __builtin_amdgcn_exp2f(fmaf(sc[i >> 3][2 * (i & 7)], cs, nm));
            const float y = __builtin_amdgcn_exp2f(fmaf(sc[i >> 3][2 * (i & 7) + 1], cs, nm));
            l += x;
            l += y;
            return pack2<BF>(x, y);
        };
        // a wave issues in order: between the products of 16 keys come the weights
        // of the next 16, or the vector unit would wait for the matrix cores, which
        // the other group shares
        v4u p, ahead_p = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = weigh(i);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            v4u v[NDT];
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) v[dt] = vf[dt];
            if (st < 3) read_v(st + 1);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                o[dt] = mfma32<BF>(v[dt], p, o[dt]);
                if (st < 3)
#pragma unroll
                    for (int i = dt * 4 / NDT; i < (dt + 1) * 4 / NDT; ++i) ahead_p[i] = weigh(4 * (st + 1) + i);
                __builtin_amdgcn_sched_barrier(0);   // keep this order
            }
            p = ahead_p;
        }
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
    }
    if (!group) barrier();
    const float2 lp = swap32(l, l);
    l = lp.x + lp.y;
    float M = m == -INFINITY ? -INFINITY : -nm;
    if (lane == 0) sh.odd[group][wave] = odd;
    __syncthreads();
    if (__builtin_expect(sh.odd[group][0] | sh.odd[group][1] | sh.odd[group][2] | sh.odd[group][3], 0)) {   // group-uniform
        for (uint32_t t = ta; t < t1; t += 2) {
            const uint32_t k0 = t * KT;
            if (!block_part(k0, bad_of(pages_of(t), t))) continue;   // whole tiles had V as it is
            for (uint32_t key = k0; key < k0 + KT; ++key) {
                const uint32_t page = paged_entry(a.b, s, key, key < rt.hi);
                if (page == a.b.num_pages) continue;
                const uint16_t *vp = vh + (uint64_t)page * page_len + (key & pmask);
                const bool seen = key >= sp.lo && key < sp.hi;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        o[dt][e] += odd_value<BF>(vp[(32 * dt + 8 * (e >> 2) + 4 * hh + (e & 3)) << a.b.shift], seen);
                        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    }
    // where the lane's results go, computed here: kept over the loop that costs registers
    uint32_t none = 0, G = a.G;
    asm volatile("" : "+s"(none), "+s"(G));
    const uint32_t ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none)), lh = ln >> 5, row = w0 + (ln & 31);
    float (&join)[D / 2 + 2][64] = sh.join[wave];
    if (group) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) join[16 * dt + e][ln] = o[dt][e];
        join[D / 2][ln] = M;
        join[D / 2 + 1][ln] = l;
    }
    __syncthreads();
    if (group || !any || row >= rt.R) return;
    {
        const float M2 = join[D / 2][ln], to = fmaxf(M, M2);
        const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - to);
        const float f2 = M2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M2 - to);
        l = l * f + join[D / 2 + 1][ln] * f2;
        M = to;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * f + join[16 * dt + e][ln] * f2;
    }
    if (rt.nz > 1) {
        const size_t part = (((size_t)u * hkv + kvh) * a.chunk_splits + z) * TILE_ROWS + (row - rt.r0);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(float4v *)(a.chunk_o + part * D + 32 * dt + 8 * j + 4 * lh) =
                    (float4v){o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
        if (lh == 0) {
            a.chunk_ml[2 * part] = M;
            a.chunk_ml[2 * part + 1] = l;
        }
        return;
    }
    const uint32_t of = row / G, hd = kvh * G + row % G;   // token, head
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *const op = a.out + (rt.sq.row0 + of) * a.o_stride + hd * D;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(uint2 *)(op + 32 * dt + 8 * j + 4 * lh) =
                make_uint2(pack2<BF>(o[dt][4 * j] * inv, o[dt][4 * j + 1] * inv),
                           pack2<BF>(o[dt][4 * j + 2] * inv, o[dt][4 * j + 3] * inv));
    if (a.lse && lh == 0)
        a.lse[(size_t)(rt.sq.row0 + of) * a.hq + hd] = l == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * LN2;
}

// One launch for a batch, chunk_part's blocks first: they take longest, and
// few_part's then fill the CUs beside them.  Measured with few_part's first and
// last: 18 single tokens and 6 chunks in a window of 512 (head_dim 64, capped)
// 31.9 and 24.5 us, at head_dim 128 41.3 and 38.8, 24 sequences without a window
// 90.3 and 93.1.
// At head_dim 64 chunk_part keeps to 128 registers, so that a CU holds two of its
// blocks; few_part beside it then has no room to load a step ahead, and need not,
// with four waves a SIMD (24 sequences, 1 and 2 blocks a CU: 40.8 and 33.8 us).
enum { FEW_4, FEW_8, CHUNK, BOTH };   // few_part by 4 or 8 waves, chunk_part, both
constexpr int threads_of(int kind) { return kind == FEW_4 ? 256 : 512; }
constexpr int waves_of(int head_dim, int kind) { return head_dim == 64 && (kind == CHUNK || kind == BOTH) ? 4 : 2; }
template <int D, bool BF, int SC, int KIND>
__global__ __launch_bounds__(threads_of(KIND)) __attribute__((amdgpu_waves_per_eu(waves_of(D, KIND)))) void attn_kernel(AttnArgs a) {
    constexpr int W = threads_of(KIND) / 64;
    constexpr bool AHEAD = waves_of(D, KIND) == 2;
    __shared__ __align__(16) union {
        char none;
        typename std::conditional<KIND != CHUNK, FewShared<D, W>, char>::type few;
        typename std::conditional<KIND == CHUNK || KIND == BOTH, ChunkShared<D>, char>::type chunk;
    } sh;
    const uint32_t chunk_blocks = gridDim.x - a.few_blocks;
    if constexpr (KIND == CHUNK) chunk_part<D, BF, SC>(a, blockIdx.x, sh.chunk);
    else if constexpr (KIND != BOTH) few_part<D, BF, SC, W, AHEAD>(a, blockIdx.x, sh.few);
    else if (blockIdx.x < chunk_blocks) chunk_part<D, BF, SC>(a, blockIdx.x, sh.chunk);
    else few_part<D, BF, SC, W, AHEAD>(a, blockIdx.x - chunk_blocks, sh.few);
}

// ------------------------------------------------------------- parts joined
// A row takes D/4 threads (four dims each) times 1, 2, 4 or 8 sets that share
// its parts out; a block holds as many rows as fit.  few_part's rows first, by
// (sequence, KV head, row), then chunk_part's, by (row tile, KV head, row).
// Bound by its loads' latency: with one set everywhere one token over 131072 keys
// takes 130 us for 104, over 16000 23.5 for 19.3; with eight 12 sequences of chunks
// and single tokens 260 for 236.
constexpr uint32_t MOST_SPLITS = 256;
struct JoinArgs {
    uint64_t few_rows;            // rows of few_part's, rounded up to whole blocks
    uint32_t few_sets, chunk_sets;
};

// The parts first + z step, z = set, set + sets, ..., then the sets' sums.
template <int D, bool BF>
__device__ __forceinline__ void join_parts(const float *po, const float *ml, size_t first, size_t step, uint32_t nz,
                                           uint32_t sets, bool mine, uint16_t *out, float *lse) {
    constexpr uint32_t LANES = D / 4;
    __shared__ float4v part[256];
    __shared__ float2 stat[256 / LANES];
    const uint32_t tid = threadIdx.x, d = tid % LANES, team = tid / LANES, set = team % sets;
    float M = -INFINITY, l = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float m2, float l2, float4v o2) {
        const float to = fmaxf(M, m2);
        const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - to);
        const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - to);
        M = to;
        l = l * f + l2 * f2;
        o = o * f + o2 * f2;
    };
    constexpr uint32_t AHEAD = 4;   // parts whose loads are in flight together
    if (mine) {
        for (uint32_t z0 = set; z0 < nz; z0 += AHEAD * sets) {
            float2 f[AHEAD];
            float4v v[AHEAD];
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i) {
                const size_t p = first + paged_min(z0 + i * sets, nz - 1) * step;
                f[i] = *(const float2 *)(ml + 2 * p);
                v[i] = *(const float4v *)(po + p * D + 4 * d);
            }
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                if (z0 + i * sets < nz) add(f[i].x, f[i].y, v[i]);
        }
    }
    if (sets > 1) {   // block-uniform
        part[tid] = o;
        if (d == 0) stat[team] = make_float2(M, l);
        __syncthreads();
        if (set) return;
        for (uint32_t i = 1; i < sets; ++i) {
            const float2 f = stat[team + i];
            add(f.x, f.y, part[tid + i * LANES]);
        }
    }
    if (!mine) return;
    o *= l == 0.f ? 0.f : 1.f / l;
    *(uint2 *)(out + 4 * d) = make_uint2(pack2<BF>(o[0], o[1]), pack2<BF>(o[2], o[3]));
    if (lse && d == 0) *lse = l == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(l)) * LN2;
}

template <int D, bool BF>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a, JoinArgs j) {
    constexpr uint32_t TEAMS = 256 / (D / 4);
    const uint32_t hkv = a.b.hkv, team = threadIdx.x / (D / 4);
    const uint32_t few_blocks = (uint32_t)(j.few_rows / (TEAMS / j.few_sets));
    bool mine = false;
    size_t first = 0, step = 0, row = 0;
    uint32_t nz = 0, head = 0, sets;
    const float *po, *ml;
    if (blockIdx.x < few_blocks) {
        sets = j.few_sets;
        po = a.few_o;
        ml = a.few_ml;
        const uint32_t i = blockIdx.x * (TEAMS / sets) + team / sets;
        const uint32_t r = i % a.few_rows, unit = i / a.few_rows, kvh = unit % hkv, s = unit / hkv;
        if (s < a.b.num_seqs) {
            const PagedSeq sq = paged_seq(a.b, s);
            const uint32_t n = paged_min(sq.n, a.b.max_q), R = n * a.G;
            const uint32_t prefix = a.prefix ? a.prefix[s] : 0u;
            const uint32_t lo = paged_span(sq.first, sq.len, prefix, a.window).lo & ~31u;
            const uint32_t hi = paged_span(sq.first + (int32_t)n - 1, sq.len, prefix, a.window).hi;
            const uint32_t steps = hi > lo ? (hi - lo + 31) / 32 : 0;
            mine = r < R && R <= FEW && steps > a.few_steps;
            nz = (steps + a.few_steps - 1) / a.few_steps;
            first = (size_t)unit * a.few_splits * a.few_rows + r;
            step = a.few_rows;
            row = sq.row0 + r / a.G;
            head = kvh * a.G + r % a.G;
        }
    } else {
        sets = j.chunk_sets;
        po = a.chunk_o;
        ml = a.chunk_ml;
        const uint32_t per = TEAMS / sets, block = blockIdx.x - few_blocks;   // rows of a block: in one tile
        const uint32_t unit = block / (TILE_ROWS / per), r = block % (TILE_ROWS / per) * per + team / sets;
        const uint32_t kvh = unit % hkv;
        uint32_t s, tile;
        if (!find_tile(a, unit / hkv, &s, &tile)) return;   // block-uniform
        const RowTile rt = row_tile(a, s, tile);
        if (rt.nz == 1) return;
        mine = rt.r0 + r < rt.R;
        nz = rt.nz;
        first = (size_t)unit * a.chunk_splits * TILE_ROWS + r;
        step = TILE_ROWS;
        row = rt.sq.row0 + (rt.r0 + r) / a.G;
        head = kvh * a.G + (rt.r0 + r) % a.G;
    }
    join_parts<D, BF>(po, ml, first, step, nz, sets, mine, a.out + row * a.o_stride + head * D,
                      a.lse ? a.lse + row * a.hq + head : nullptr);
}

// ------------------------------------------------------------------- launch
// Which parts run and how keys are split, from the host's bounds alone.
// few_part: about 1024 blocks (one token over 131072: 512, 1024 and 2048 blocks
// 101, 104 and 111 us; 64 chats 251, 243 and 239), of 16 steps at least (8, 16 and
// 32: 513 keys 13.7, 10.0 and 10.6 us, four tokens over 2000 14.7, 16.0 and 26,
// 32 over 500-1500 at head_dim 64 19.6, 17.1 and 15.6); 256 beside chunks (more
// change nothing).
// chunk_part: as many blocks as the CUs hold, 256 at head_dim 128 and 512 at 64
// (512 tokens over 25000, 256 and 512 blocks: 132 and 146 us, 85 and 76); 512 for
// several sequences, whose lengths differ and whose row tiles are bounded from
// above only (12 of up to 30300 keys, head_dim 128, 311 and 235 us, three prompts
// 75 and 64; two prompts of one length lose, 54 and 61); four tiles of keys at
// least (2 and 4: 300 tokens alone 17.5 and 13.4 us; 8 and 4: 64 over 2000 21.7 and
// 19.0).
struct Plan {
    uint32_t few_rows = 0, few_splits = 0, few_steps = 0;          // 0 splits: not launched
    uint32_t units = 0, chunk_splits = 0, chunk_tiles = 0;
    size_t few_parts = 0, chunk_parts = 0;                         // rows of partial results
};

// window: where no row's keys are more than that, else 0.  A few rows (16 tokens)
// then see window + 15 keys, of them up to 31 more for whole steps of 32; a row
// tile (128 tokens) window + 127, up to 63 more for whole tiles.
Plan plan_of(const nnz_paged_kv &kv, const nnz_paged_batch &b, uint32_t hq, uint32_t window = 0) {
    Plan p;
    auto keys = [&](uint32_t more) {
        return window ? (uint32_t)std::min<uint64_t>(b.max_kv_len, (uint64_t)window + more) : b.max_kv_len;
    };
    const uint32_t G = hq / kv.num_kv_heads, hkv = kv.num_kv_heads;
    const uint64_t most = (uint64_t)b.max_q_len * G;   // rows of a sequence
    const bool chunks = most > FEW;
    // One sequence whose bound passes 16 rows goes to chunk_part, whatever its
    // length turns out to be; a batch of several may hold both kinds.
    if (G <= FEW && (!chunks || b.num_seqs > 1)) {
        const uint32_t steps = (keys(48) + 31) / 32, blocks = b.num_seqs * hkv;   // below 2^26
        const uint32_t want = std::max(1u, (chunks ? 256u : 1024u) / blocks), most_splits = std::max(1u, steps / 16);
        const uint32_t splits = std::min({want, most_splits, MOST_SPLITS});
        p.few_rows = (uint32_t)std::min<uint64_t>(most, FEW);
        p.few_steps = (steps + splits - 1) / splits;
        p.few_splits = (steps + p.few_steps - 1) / p.few_steps;
        if (p.few_splits > 1) p.few_parts = (size_t)blocks * p.few_splits * p.few_rows;
    }
    if (chunks) {
        const uint64_t by_rows = (uint64_t)b.num_rows * G / TILE_ROWS + b.num_seqs;
        const uint64_t by_seqs = (uint64_t)b.num_seqs * ((most + TILE_ROWS - 1) / TILE_ROWS);
        p.units = (uint32_t)std::min(by_rows, by_seqs);
        const uint32_t tiles = (keys(192) + KT - 1) / KT;
        const uint32_t blocks = kv.head_dim == 64 || b.num_seqs > 1 ? 512 : 256;
        const uint32_t want = (uint32_t)std::max<uint64_t>(1, blocks / ((uint64_t)p.units * hkv)), most_splits = std::max(1u, tiles / 4);
        const uint32_t splits = std::min({want, most_splits, MOST_SPLITS});
        p.chunk_tiles = (tiles + splits - 1) / splits;
        p.chunk_splits = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
        if (p.chunk_splits > 1) p.chunk_parts = (size_t)p.units * hkv * p.chunk_splits * TILE_ROWS;
    }
    return p;
}

uint64_t blocks_of(const Plan &p, const nnz_paged_batch &b, uint32_t hkv) {
    return (uint64_t)b.num_seqs * hkv * p.few_splits + (uint64_t)p.units * hkv * p.chunk_splits;
}
size_t bytes_of(const Plan &p, uint32_t head_dim) { return (p.few_parts + p.chunk_parts) * (head_dim + 2) * 4; }

template <int D, bool BF, int SC>
void start(hipStream_t stream, const Plan &p, AttnArgs a, float *ws) {
    const uint32_t hkv = a.b.hkv;
    a.few = p.few_splits ? FEW : 0;
    a.few_rows = p.few_rows;
    a.few_splits = p.few_splits;
    a.few_steps = p.few_steps;
    a.few_blocks = a.b.num_seqs * hkv * p.few_splits;
    a.units = p.units;
    a.chunk_splits = p.chunk_splits;
    a.chunk_tiles = p.chunk_tiles;
    a.few_o = ws;
    a.few_ml = a.few_o + p.few_parts * D;
    a.chunk_o = a.few_ml + p.few_parts * 2;
    a.chunk_ml = a.chunk_o + p.chunk_parts * D;
    const uint32_t chunk_blocks = p.units * hkv * p.chunk_splits;
    // 8 waves a block where blocks are fewer than CUs (4 and 8: one token over 4000
    // 16.3 and 15.3 us), 4 beyond, two blocks a CU (8 and 4: 131072 107 and 104, 64
    // chats 245 and 242)
    if (!chunk_blocks && a.few_blocks > 256) attn_kernel<D, BF, SC, FEW_4><<<a.few_blocks, 256, 0, stream>>>(a);
    else if (!chunk_blocks) attn_kernel<D, BF, SC, FEW_8><<<a.few_blocks, 512, 0, stream>>>(a);
    else if (!a.few_blocks) attn_kernel<D, BF, SC, CHUNK><<<chunk_blocks, 512, 0, stream>>>(a);
    else attn_kernel<D, BF, SC, BOTH><<<a.few_blocks + chunk_blocks, 512, 0, stream>>>(a);
    if (!p.few_parts && !p.chunk_parts) return;
    auto sets_of = [](uint32_t splits) { return splits > 32 ? 8u : splits > 8 ? 4u : splits > 4 ? 2u : 1u; };
    constexpr uint32_t TEAMS = 256 / (D / 4);
    JoinArgs j{0, sets_of(p.few_splits), sets_of(p.chunk_splits)};
    const uint32_t per = TEAMS / j.few_sets;   // few_part's rows of a block
    if (p.few_parts) j.few_rows = ((uint64_t)a.b.num_seqs * hkv * p.few_rows + per - 1) / per * per;
    const uint32_t chunk_join = p.chunk_parts ? p.units * hkv * TILE_ROWS / (TEAMS / j.chunk_sets) : 0;
    join_kernel<D, BF><<<(uint32_t)(j.few_rows / per) + chunk_join, 256, 0, stream>>>(a, j);
}

template <int D, bool BF>
void start_scores(hipStream_t stream, const Plan &p, const AttnArgs &a, float *ws) {
    if (a.cap > 0.f && a.slopes) start<D, BF, CAPPED_BIASED>(stream, p, a, ws);
    else if (a.cap > 0.f) start<D, BF, CAPPED>(stream, p, a, ws);
    else if (a.slopes) start<D, BF, BIASED>(stream, p, a, ws);
    else start<D, BF, PLAIN>(stream, p, a, ws);
}

}  // namespace

extern "C" size_t nnz_paged_attention_workspace_bytes(const nnz_paged_kv *kv, const nnz_paged_batch *batch,
                                                      uint32_t num_query_heads) {
    if (paged_fault(kv, batch).code || paged_heads_fault(kv, num_query_heads).code) return 0;
    return bytes_of(plan_of(*kv, *batch, num_query_heads), kv->head_dim);
}

extern "C" int nnz_dispatch_paged_attention(nnz_ctx *ctx, const nnz_paged_kv *kv, const nnz_paged_batch *batch,
                                            const void *q, void *output, float *lse, void *workspace,
                                            size_t workspace_bytes, const nnz_paged_attn_params *p) {
    NNZ_CHECK_CTX(ctx);
    if (const PagedFault f = paged_attn_fault(kv, batch, q, output, lse, p); f.code)
        return nnz_fail(ctx, f.code, "paged_attention: %s", f.what);
    Plan plan = plan_of(*kv, *batch, p->num_query_heads);
    const size_t need = bytes_of(plan, kv->head_dim);
    if (p->window && !p->prefix_lens) {   // fewer keys to split, in the workspace that the bounds ask for
        const Plan narrow = plan_of(*kv, *batch, p->num_query_heads, p->window);
        if (bytes_of(narrow, kv->head_dim) <= need) plan = narrow;
    }
    NNZ_REQUIRE(ctx, blocks_of(plan, *batch, kv->num_kv_heads) < (1u << 23), NNZ_EUNSUPPORTED,
                "paged_attention: more than 2^23 blocks; split the batch");
    NNZ_REQUIRE(ctx, need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), NNZ_EINVAL,
                "paged_attention: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", need, workspace_bytes);
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
    const float scale = p->scale > 0.f ? p->scale : 1.f / sqrtf((float)kv->head_dim);
    a.scale = scale * LOG2E;
    a.unbias = 1.f / scale;
    a.cap = p->softcap * LOG2E;
    a.cap_in = p->softcap > 0.f ? 2.f * LOG2E * scale / p->softcap : 0.f;
    const bool bf = kv->dtype == NNZ_BF16;
    float *ws = (float *)workspace;
    if (kv->head_dim == 128) bf ? start_scores<128, true>(ctx->stream, plan, a, ws) : start_scores<128, false>(ctx->stream, plan, a, ws);
    else bf ? start_scores<64, true>(ctx->stream, plan, a, ws) : start_scores<64, false>(ctx->stream, plan, a, ws);
    NNZ_LAUNCHED(ctx);
    return NNZ_OK;
}
