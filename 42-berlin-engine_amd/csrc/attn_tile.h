// attn_tile.h -- tiles of query rows over pages: what the attention of a batch behind
// a prefix (prefix.hip) and of trees of drafts (tree.hip) share.
#pragma once

#include <algorithm>
#include <type_traits>

#include "be42_common.h"
#include "paged_dev.h"

namespace be42 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

struct PrefixArgs {
    const void *q;
    void *out;
    const int *slots, *lens;
    float *part_o, *part_ml;  // [parts][rows][head_dim], [parts][rows][2]; rows = n_queries * n_heads
    size_t q_stride;
    int n_queries, n_heads, prefix_slot, prefix_len, max_len;
    float scale;
    // the cut: parts of the prefix and of the own tokens, tokens of each, tiles of
    // rows that a KV head has over the prefix and over one query (of 16), and rows
    // of a prefix tile
    int parts_p, parts_o, chunk_p, chunk_o, tiles_p, tiles_o, rows_p;
    bool whole;               // one launch: k_prefix_whole
};

// The first `want` tokens of a slot, cut at what it holds (0 for a slot outside
// the pool).  How full the last page is takes two more dependent loads, which
// only those who look at it wait for.
__device__ __forceinline__ int slot_tokens(const be42_kv_pool &P, int slot, int want)
{
    if (slot < 0 || slot >= P.n_layers || want <= 0)
        return 0;
    const int pages = min(P.n_logical[slot], P.max_logical);
    if (want <= (pages - 1) * kPage || pages <= 0)
        return max(min(want, pages * kPage), 0);
    const int last = P.page_table[(size_t)slot * P.max_logical + pages - 1];
    if (last < 0 || last >= P.capacity)
        return 0;
    return min(want, (pages - 1) * kPage + min(P.ntok[last], kPage));
}

// Physical page of a slot's logical page.  Asked for before it is known how many
// pages the slot has: what lies past them is some page of the pool, whose tokens
// are masked.
__device__ __forceinline__ int table_page(const be42_kv_pool &P, int slot, int logical)
{
    const size_t at = (size_t)min(max(slot, 0), P.n_layers - 1) * P.max_logical + min(logical, P.max_logical - 1);
    return min(max(P.page_table[at], 0), P.capacity - 1);
}

// Eight fp32 as N bf16 parts: each part the rest rounded to bf16, so that three
// hold all 24 bits and one is a plain rounding.
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&p)[N])
{
    uint32_t w[N][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        v2f r = {x[2 * j], x[2 * j + 1]};
#pragma unroll
        for (int n = 0; n < N; n++) {
            w[n][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
            if (n + 1 < N) {
                r[0] -= __uint_as_float(w[n][j] << 16);
                r[1] -= __uint_as_float(w[n][j] & 0xFFFF0000u);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; n++)
        p[n] = __builtin_bit_cast(bf16x8, make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]));
}

// bytes 0 .. 7 of two words as bf16 (exact)
__device__ __forceinline__ bf16x8 codes8(uint32_t a, uint32_t b)
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t u = j < 2 ? a : b;
        const v2f r = {(float)(int8_t)(u >> (16 * (j & 1))), (float)(int8_t)(u >> (16 * (j & 1) + 8))};
        w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
    }
    return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

__device__ __forceinline__ v4f mfma16(bf16x8 a, bf16x8 b, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ v16f mfma32(bf16x8 a, bf16x8 b, v16f c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// eight elements of a query row from element `at` on, in NP parts, negated for a
// negative scale
template <int NP>
__device__ __forceinline__ void load_q(const PrefixArgs &a, size_t at, bf16x8 (&Q)[NP])
{
    const bool flip = a.scale < 0.0f;
    if constexpr (NP == 1) {
        uint32_t w[4];
        __builtin_memcpy(w, (const uint16_t *)a.q + at, 16);
#pragma unroll
        for (int j = 0; j < 4; j++)
            w[j] ^= flip ? 0x80008000u : 0u;
        Q[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    } else {
        float x[8];
        __builtin_memcpy(x, (const float *)a.q + at, 32);
#pragma unroll
        for (int j = 0; j < 8; j++)
            x[j] = flip ? -x[j] : x[j];
        split8<NP>(x, Q);
    }
}

// The scores' factor c, log2(e) |scale| (load_q has the sign), and not 0: times the
// -infinity of a token past the part that would be NaN.
__device__ __forceinline__ float log2_scale(const PrefixArgs &a)
{
    return fmaxf(fabsf(a.scale) * 1.44269504088896340736f, 1.17549435e-38f);
}

// The largest of three, NaN if one is.  (fmaxf adds a canonicalizing move for
// each operand; in inline assembly the wait states after a matrix product would
// be missing.)
__device__ __forceinline__ float max3(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// x and the other half's x (lane ^ 32), in either order; with quarters of a wave
// (lane ^ 16) likewise
__device__ __forceinline__ void halves(float x, float &a, float &b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void quarters(float x, float &a, float &b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}

// A read of LDS that direct-to-LDS loads fill, after the barrier that waited for
// them.  The argument's promise not to alias keeps the compiler from waiting for
// every such load in flight before each read (32 queries over 8192 tokens took 32 us
// with the wait and 21 without, when the ring was brought in).
template <class T>
__device__ __forceinline__ T ring_read(const void *__restrict__ p)
{
    return *(const T *)p;
}

// What a row's sums count from, m, is a score as the products give it, and may lie
// this much (a factor of 256) below the largest so far: the sums are rescaled past
// that only.  With the exact
// maximum some of a wave's 32 rows has a new one in most steps, and the rescaling
// was a third of the vector work.
constexpr float kSlack = 8.0f;
// the least m of a row that has seen a token (-infinity: none)
constexpr float kLowest = -3.402823466e38f;

constexpr int kPartWaves = 4;
constexpr int kStep = 32;         // tokens of a wave's step: two pages

template <int HD, int N = kPartWaves>
struct PartShared {
    float o[N][16][HD + 4];
    float m[N][16], l[N][16];
};

// Rows of a part in 16x16 tiles.  Both products are formed transposed, S^T =
// K Q^T (operand rows are tokens, columns are query rows) and O^T = V^T P^T, so
// that a lane keeps one query row from the scores to the output: column c =
// lane % 16, and with g = lane / 16 the lane's eight scores of a step of 32
// tokens are tokens 8 g .. 8 g + 7 -- row 4 g + i of score tile t is given to
// token 8 g + 4 t + i -- which is the operand the second product takes from
// it.  Weights go from one product to the other in registers.
//
// `share` waves take the steps in turn, from step `first` on this one; its sums
// go to rows to .. to + rows - row0 - 1 of place `at` in LDS.  `seen` says which
// tokens each row sees: every one, or those of a path (SeesPath).
struct SeesAll {
    static constexpr bool kSome = false;
};
// In LDS, for each row of the tile, a bit for each token from lo on; lo is a page's
// first token, those of the tree are from .. to - 1 from there.
struct SeesPath {
    static constexpr bool kSome = true;
    static constexpr int kWords = 9;       // 256 tokens from somewhere in the first page on
    const uint32_t *bits;                  // [16][kWords]
    int from, to;
    __device__ __forceinline__ uint32_t row(int c, int step) const { return bits[c * kWords + step]; }
    __device__ __forceinline__ uint32_t tree(int step) const
    {
        const int a = min(max(from - 32 * step, 0), 32), b = min(max(to - 32 * step, 0), 32);
        return (uint32_t)((1ull << b) - (1ull << min(a, b)));
    }
};

// of a word's two bf16, the bits of those that are finite
__device__ __forceinline__ uint32_t tame_bf16(uint32_t w)
{
    return ((w & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
}

template <bool KV8, int HD, int NP, int PP, class Shared, class Seen = SeesAll>
__device__ __forceinline__ void part16(const be42_kv_pool &P, const PrefixArgs &a, Shared &S, int slot, int lo, int hi, int kvh,
                                       int b0, int row0, int rows, int first, int share, int at, int to, Seen seen = Seen())
{
    constexpr int NK = HD / 32, NE = HD / 16;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int G = a.n_heads / P.n_kv;
    const int ns = (hi - lo + kStep - 1) / kStep;
    const int mine = ns > first ? (ns - first + share - 1) / share : 0;      // steps first, first + share, ..

    // the lane's query row, eight elements a k block: bf16 pages take element
    // 32 kb + 8 g + j there, INT8 pages (16 codes a load) 64 (kb / 2) + 16 g + 8 (kb % 2) + j
    bf16x8 Q[NK][NP];
    {
        const int ri = min(row0 + c, rows - 1);
        const size_t row = (size_t)(b0 + ri / G) * a.q_stride + (size_t)(kvh * G + ri % G) * HD;
#pragma unroll
        for (int kb = 0; kb < NK; kb++)
            load_q<NP>(a, row + (KV8 ? 64 * (kb / 2) + 16 * g + 8 * (kb % 2) : 32 * kb + 8 * g), Q[kb]);
    }
    const float sc = log2_scale(a);

    v4f O[NE];
#pragma unroll
    for (int e = 0; e < NE; e++)
        O[e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    uint4 K[2][KV8 ? NK / 2 : NK];
    uint4 V[KV8 ? 1 : NE];
    uint32_t V8[KV8 ? 8 : 1][HD / 64];
    float4 ks[2], vs[2];
    // physical pages of the wave's next 32 steps: lane 2 i + e holds page e of step i
    int pages = 0;
    auto load_pages = [&](int i0) {
        pages = table_page(P, slot, lo / kPage + 2 * (first + share * (i0 + lane / 2)) + (lane & 1));
    };
    auto head_of = [&](int i, int e) {
        return (size_t)__builtin_amdgcn_readlane(pages, 2 * (i & 31) + e) * P.n_kv + kvh;
    };
    const int kg = c >> 2, ktok = 8 * (kg & 1) + (c & 3);      // token (of its page) that operand row c of tile 0 is
    auto load_k = [&](int i) {
        const size_t h0 = head_of(i, 0), h1 = head_of(i, 1), hk = kg >> 1 ? h1 : h0, hv = g >> 1 ? h1 : h0;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const size_t row = (hk * kPage + ktok + 4 * t) * HD;
#pragma unroll
            for (int x = 0; x < (KV8 ? NK / 2 : NK); x++)
                K[t][x] = KV8 ? *(const uint4 *)((const int8_t *)P.k + row + 64 * x + 16 * g)
                              : *(const uint4 *)((const uint16_t *)P.k + row + 32 * x + 8 * g);
        }
        if constexpr (KV8)
#pragma unroll
            for (int t = 0; t < 2; t++)
                ks[t] = *(const float4 *)(P.k_scale + hv * kPage + 8 * (g & 1) + 4 * t);
    };
    auto load_v = [&](int i) {
        const size_t h0 = head_of(i, 0), h1 = head_of(i, 1), hv = g >> 1 ? h1 : h0;
        if constexpr (KV8) {
            // eight tokens of NE dims: tile e's row r is dim NE r + e
#pragma unroll
            for (int j = 0; j < 8; j++)
                __builtin_memcpy(V8[j], (const int8_t *)P.v + (hv * kPage + 8 * (g & 1) + j) * HD + NE * c, HD / 16);
#pragma unroll
            for (int t = 0; t < 2; t++)
                vs[t] = *(const float4 *)(P.v_scale + hv * kPage + 8 * (g & 1) + 4 * t);
        } else {
#pragma unroll
            for (int e = 0; e < NE; e++)
                V[e] = *(const uint4 *)((const uint16_t *)P.v + (hv * HD + 16 * e + c) * kPage + 8 * (g & 1));
        }
    };

    if (mine) {
        load_pages(0);
        load_k(0);
        load_v(0);
    }
    for (int i = 0; i < mine; i++) {
        const int left = hi - lo - (first + share * i) * kStep;      // tokens from this step on
        v4f s[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int kb = 0; kb < NK; kb++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const bf16x8 k = KV8 ? (kb & 1 ? codes8(K[t][kb / 2].z, K[t][kb / 2].w) : codes8(K[t][kb / 2].x, K[t][kb / 2].y))
                                     : __builtin_bit_cast(bf16x8, K[t][KV8 ? 0 : kb]);
#pragma unroll
                for (int n = NP - 1; n >= 0; n--)
                    s[t] = mfma16(k, Q[kb][n], s[t]);
            }
        float p[8], vsc[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = s[j >> 2][j & 3];
            if constexpr (KV8) {
                p[j] *= ((const float *)&ks[j >> 2])[j & 3];
                vsc[j] = ((const float *)&vs[j >> 2])[j & 3];
            }
        }
        const bool more = i + 1 < mine;
        if (more) {
            if (((i + 1) & 31) == 0)
                load_pages(i + 1);
            load_k(i + 1);
        }
        uint32_t mine_of = 0, tree_of = 0;           // the lane's eight tokens: seen by its row, of the tree
        if constexpr (Seen::kSome) {
            mine_of = seen.row(c, first + share * i) >> (8 * g);
            tree_of = seen.tree(first + share * i) >> (8 * g);
        }
        if (Seen::kSome || left < kStep)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool out = Seen::kSome ? !(mine_of >> j & 1) : 8 * g + j >= left;
                p[j] = out ? -INFINITY : p[j];
                if (KV8)
                    vsc[j] = out ? 0.0f : vsc[j];
            }
        float top = max3(max3(p[0], p[1], p[2]), max3(p[3], p[4], p[5]), max3(p[6], p[7], p[7])), other;
        quarters(top, top, other);
        top = max3(top, other, other);
        halves(top, top, other);
        top = fmaxf(max3(top, other, other), kLowest);
        if constexpr (Seen::kSome)
            top = seen.row(c, first + share * i) ? top : -INFINITY;     // a row that sees nothing here
        if (__any((top - m) * sc > kSlack)) {
            const float now = fmaxf(m, top), f = Seen::kSome && m == now ? 1.0f : __builtin_amdgcn_exp2f((m - now) * sc);
            l *= f;
#pragma unroll
            for (int e = 0; e < NE; e++)
                O[e] *= f;
            m = now;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = Seen::kSome && !(mine_of >> j & 1) ? 0.0f : __builtin_amdgcn_exp2f((p[j] - m) * sc);
            l += p[j];
            if (KV8)
                p[j] *= vsc[j];
        }
        bf16x8 W[PP];
        split8<PP>(p, W);
        // V of tokens past the part is whatever the page held: a weight of zero
        // times a NaN pattern would be NaN
        if (!KV8 && (Seen::kSome || left < kStep)) {
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                keep[j] = Seen::kSome ? (tree_of >> (2 * j) & 1 ? 0xFFFFu : 0u) | (tree_of >> (2 * j + 1) & 1 ? 0xFFFF0000u : 0u)
                                      : (8 * g + 2 * j < left ? 0xFFFFu : 0u) | (8 * g + 2 * j + 1 < left ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int e = 0; e < (KV8 ? 0 : NE); e++) {
                V[e].x &= keep[0];
                V[e].y &= keep[1];
                V[e].z &= keep[2];
                V[e].w &= keep[3];
            }
        }
        // an infinity or NaN among the tree's values reaches only the rows that see
        // its token: the tokens one by one, each for those rows; times the weight's
        // first part (a later one may be 0 or below)
        bool wild = false;
        if constexpr (Seen::kSome && !KV8) {
#pragma unroll
            for (int e = 0; e < NE; e++)
                wild |= (tame_bf16(V[e].x) & tame_bf16(V[e].y) & tame_bf16(V[e].z) & tame_bf16(V[e].w)) != ~0u;
            wild = __any(wild);
            if (wild) {
                const uint32_t row = seen.row(c, first + share * i);
#pragma unroll 1
                for (int t = 0; t < kStep; t++) {
                    const bool sees = row >> t & 1;
                    const uint32_t half = t >> 3 == g ? (t & 1 ? 0xFFFF0000u : 0xFFFFu) : 0u;
                    const int word = t >> 1 & 3;
#pragma unroll
                    for (int e = 0; e < NE; e++) {
                        const uint4 one = make_uint4(word == 0 ? V[e].x & half : 0u, word == 1 ? V[e].y & half : 0u,
                                                     word == 2 ? V[e].z & half : 0u, word == 3 ? V[e].w & half : 0u);
                        v4f o = O[e];
                        const uint4 fine = make_uint4(one.x & tame_bf16(one.x), one.y & tame_bf16(one.y),
                                                      one.z & tame_bf16(one.z), one.w & tame_bf16(one.w));
#pragma unroll
                        for (int n = PP - 1; n > 0; n--)
                            o = mfma16(__builtin_bit_cast(bf16x8, fine), W[n], o);
                        o = mfma16(__builtin_bit_cast(bf16x8, one), W[0], o);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            O[e][j] = sees ? o[j] : O[e][j];
                    }
                }
            }
        }
        if (!wild)
#pragma unroll
        for (int e = 0; e < NE; e++) {
            bf16x8 v;
            if constexpr (KV8) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int word = e >> 2, at = 8 * (e & 3);
                    const v2f r = {(float)(int8_t)(V8[2 * j][word] >> at), (float)(int8_t)(V8[2 * j + 1][word] >> at)};
                    w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
                }
                v = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
            } else {
                v = __builtin_bit_cast(bf16x8, V[KV8 ? 0 : e]);
            }
#pragma unroll
            for (int n = PP - 1; n >= 0; n--)
                O[e] = mfma16(v, W[n], O[e]);
        }
        if (more)
            load_v(i + 1);
    }

    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    if (row0 + c >= rows)
        return;
    if (g == 0) {
        S.m[at][to + c] = m;
        S.l[at][to + c] = l;
    }
#pragma unroll
    for (int e = 0; e < NE; e++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            S.o[at][to + c][KV8 ? NE * (4 * g + i) + e : 16 * e + 4 * g + i] = O[e][i];
}

// Weight of a partial result that counts from m against one from the largest m of
// all; one without tokens weighs nothing.
__device__ __forceinline__ float part_weight(float m, float top, float sc)
{
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * sc);
}

// 1 / the sum of a row's weights, 0 for a row that saw no token
__device__ __forceinline__ float row_inverse(float top, float sum)
{
    return top == -INFINITY ? 0.0f : 1.0f / sum;
}

template <bool QB>
__device__ __forceinline__ void store_out4(void *out, size_t at, float4 v)
{
    if constexpr (QB) {
        const v2f a = {v.x, v.y}, b = {v.z, v.w};
        const uint2 w = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf16x2)),
                                   __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf16x2)));
        __builtin_memcpy((uint16_t *)out + at, &w, 8);
    } else {
        __builtin_memcpy((float *)out + at, &v, 16);
    }
}

// ---- many rows ------------------------------------------------------------------
// Rows of the prefix in 32x32 tiles: of a workgroup's four waves, R share the
// tokens and take 32 rows each, and T = 4 / R share the rows and take each the
// next two pages, whose sums are joined in LDS at the end.  Pages come through a
// ring in LDS that direct-to-LDS loads fill ahead, a stage of T steps at a time.
// The products are transposed as in part16: a lane keeps query row c = lane %
// 32, and with h = lane / 32 its sixteen scores are tokens 8 h .. 8 h + 7 of the
// first page, then of the second (operand row i is token 8 (i / 4 % 2) +
// 4 (i / 8 % 2) + i % 4 of page i / 16).
template <bool KV8, int HD, int R>
struct WideShared {
    static constexpr int T = kPartWaves / R, kPageBytes = kPage * HD * (KV8 ? 1 : 2);
    struct Step {
        alignas(16) char k[2][kPageBytes], v[2][kPageBytes];
        float scale[KV8 ? 2 : 1][2][kPage];     // of K and V, of each page
    };
    static constexpr int NS = T * 4 * kPageBytes > 16 * 1024 ? 2 : 4;       // a ring of 64 KB at most, where two workgroups a CU fit
    struct Sums {
        float o[T][32 * R][HD + 4];
        float m[T][32 * R], l[T][32 * R];
    };
    union {
        Step ring[NS][T];
        Sums sums;
    };
};

template <bool KV8, int HD, int NP, int PP, int R>
__device__ __forceinline__ void part32(const be42_kv_pool &P, const PrefixArgs &a, WideShared<KV8, HD, R> &S, int slot,
                                       int lo, int want, int kvh, int b0, int row0, int rows)
{
    using Shared = WideShared<KV8, HD, R>;
    constexpr int NK = HD / 16, NE = HD / 32, kRowBytes = HD * (KV8 ? 1 : 2), kRowWords = kRowBytes / 16;
    constexpr int T = Shared::T, NS = Shared::NS, kStage = T * kStep;
    constexpr int kPageLoads = Shared::kPageBytes / 1024;             // of a wave, 1 KB each
    constexpr int kStepLoads = 4 * kPageLoads, kWaveLoads = T * kStepLoads / kPartWaves;
    // a wave's loads of a stage; scales: a load a step, by one wave of each T
    constexpr int kLoads = kWaveLoads + (KV8 ? 1 : 0);
    static_assert(kWaveLoads >= 1 && T <= kPartWaves, "each wave loads");
    constexpr int D = NS - 1;                  // stages that are loaded ahead
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
    const int rg = wave % R, tg = wave / R;
    const int G = a.n_heads / P.n_kv;
    // physical pages of the next stages: lane 2 T i + p holds page p of stage i
    constexpr int kHeld = kWave / (2 * T);
    int pages = table_page(P, slot, lo / kPage + lane);

    // the lane's query row: bf16 pages take element 16 kb + 8 h + j in k block
    // kb, INT8 pages (16 codes a read) 32 (kb / 2) + 16 h + 8 (kb % 2) + j
    bf16x8 Q[NK][NP];
    const int rc = min(row0 + 32 * rg + c, rows - 1);
    const size_t qat = (size_t)(b0 + rc / G) * a.q_stride + (size_t)(kvh * G + rc % G) * HD;
#pragma unroll
    for (int kb = 0; kb < NK; kb++)
        load_q<NP>(a, qat + (KV8 ? 32 * (kb / 2) + 16 * h + 8 * (kb % 2) : 16 * kb + 8 * h), Q[kb]);
    const float sc = log2_scale(a);

    // K rows of kRowWords 16-byte words: word x of row t lies at x ^ swz(t), so
    // that the rows of an operand spread over the banks
    auto swz = [](int t) { return t / (16 / kRowWords) % kRowWords; };
    auto load = [&](int i) {
        if (i && i % kHeld == 0)
            pages = table_page(P, slot, (lo + i * kStage) / kPage + lane);
#pragma unroll
        for (int x = 0; x < kWaveLoads; x++) {
            const int y = x * kPartWaves + wave, step = y / kStepLoads, z = y % kStepLoads;      // K pages, then V pages
            const bool of_k = z < 2 * kPageLoads;
            const int page = z / kPageLoads % 2, at = z % kPageLoads * 64 + lane, t = at / kRowWords;
            const size_t head = (size_t)__builtin_amdgcn_readlane(pages, 2 * (i % kHeld * T + step) + page) * P.n_kv + kvh;
            const char *base = (const char *)(of_k ? P.k : P.v) + head * Shared::kPageBytes;
            const int from = of_k ? t * kRowWords + (at % kRowWords ^ swz(t)) : at;
            typename Shared::Step &st = S.ring[i % NS][step];
            __builtin_amdgcn_global_load_lds((const void *)(base + 16 * from),
                                             (lds_void *)((of_k ? st.k[page] : st.v[page]) + z % kPageLoads * 1024), 16, 0, 0);
        }
        if constexpr (KV8) {
            // (every wave loads the scales of a step, so that all wait for the same number of loads)
            const int step = wave % T, at = 2 * (i % kHeld * T + step);
            const size_t h0 = (size_t)__builtin_amdgcn_readlane(pages, at) * P.n_kv + kvh;
            const size_t h1 = (size_t)__builtin_amdgcn_readlane(pages, at + 1) * P.n_kv + kvh;
            const float *from = (lane < 32 ? P.k_scale : P.v_scale) + (lane & 16 ? h1 : h0) * kPage + lane % 16;
            __builtin_amdgcn_global_load_lds((const void *)from, (lds_void *)&S.ring[i % NS][step].scale[0][0][0], 4, 0, 0);
        }
        // (the counts that are waited for assume that stages are loaded in order)
        asm volatile("" ::: "memory");
    };
    // the first stages are asked for before it is known how many there are
    for (int i = 0; i < D; i++)
        load(i);
    const int hi = max(lo, slot_tokens(P, slot, want)), ns = (hi - lo + kStage - 1) / kStage;

    v16f O[NE];
#pragma unroll
    for (int e = 0; e < NE; e++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            O[e][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int kpage = c >> 4, ktok = 8 * (c >> 2 & 1) + 4 * (c >> 3 & 1) + (c & 3), kswz = swz(ktok);

    // stage i is in LDS, and every wave is done with the stage whose place the
    // next load takes
    auto begin = [&](int i) {
        if (i + D - 1 < ns)
            stage_barrier<(D - 1) * kLoads>();
        else
            stage_barrier<0>();
        if (i + D < ns)
            load(i + D);
    };
    auto scores = [&](int i, v16f &s) {
        const typename Shared::Step &st = S.ring[i % NS][tg];
#pragma unroll
        for (int j = 0; j < 16; j++)
            s[j] = 0.0f;
        // all of K's operands are asked for before the first product, V's (the
        // first page's where registers are short) before the softmax: read as
        // they are needed they cost a wait of 130 cycles every two products
        constexpr int NR = KV8 ? NK / 2 : NK;
        const char *krow = st.k[kpage] + ktok * kRowBytes;
        uint4 kw[NR];
#pragma unroll
        for (int x = 0; x < NR; x++)
            kw[x] = ring_read<uint4>(krow + 16 * ((2 * x + h) ^ kswz));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kb = 0; kb < NK; kb++) {
            bf16x8 k;
            if constexpr (KV8)
                k = kb % 2 ? codes8(kw[kb / 2].z, kw[kb / 2].w) : codes8(kw[kb / 2].x, kw[kb / 2].y);
            else
                k = __builtin_bit_cast(bf16x8, kw[KV8 ? 0 : kb]);
#pragma unroll
            for (int n = NP - 1; n >= 0; n--)
                s = mfma32(k, Q[kb][n], s);
        }
    };
    auto values = [&](int i, const v16f &s, auto cut) {
        constexpr bool CUT = decltype(cut)::value;     // the part ends within the stage
        const typename Shared::Step &st = S.ring[i % NS][tg];
        const int left = CUT ? hi - lo - i * kStage - tg * kStep : kStep;
        uint4 vw[2][KV8 ? 1 : NE];
        uint32_t v8[2][KV8 ? 8 : 1];
        auto read_v = [&](int pg) {
            if constexpr (KV8) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    v8[pg][j] = NE == 4 ? ring_read<uint32_t>(st.v[pg] + (8 * h + j) * HD + NE * c)
                                        : ring_read<uint16_t>(st.v[pg] + (8 * h + j) * HD + NE * c);
            } else {
#pragma unroll
                for (int e = 0; e < NE; e++)
                    vw[pg][e] = ring_read<uint4>(st.v[pg] + (32 * e + c) * 32 + 16 * h);
            }
        };
        read_v(0);
        if (NP == 1)
            read_v(1);
        __builtin_amdgcn_sched_barrier(0);
        float p[16];
#pragma unroll
        for (int j = 0; j < 16; j++)
            p[j] = s[j];
        if constexpr (KV8)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 x = ring_read<float4>(&st.scale[0][j / 8][8 * h + j % 8]);
                p[j] *= x.x;
                p[j + 1] *= x.y;
                p[j + 2] *= x.z;
                p[j + 3] *= x.w;
            }
        if constexpr (CUT)
#pragma unroll
            for (int j = 0; j < 16; j++)
                p[j] = 16 * (j / 8) + 8 * h + j % 8 >= left ? -INFINITY : p[j];
        float top = max3(p[0], p[1], p[2]), other;
#pragma unroll
        for (int j = 3; j < 15; j += 2)
            top = max3(top, p[j], p[j + 1]);
        top = max3(top, p[15], p[15]);
        halves(top, top, other);
        top = fmaxf(max3(top, other, other), kLowest);
        if (__any((top - m) * sc > kSlack)) {
            const float now = fmaxf(m, top), f = __builtin_amdgcn_exp2f((m - now) * sc);
            l *= f;
#pragma unroll
            for (int e = 0; e < NE; e++)
                O[e] *= f;
            m = now;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
            p[j] = __builtin_amdgcn_exp2f((p[j] - m) * sc);
            l += p[j];
        }
        if constexpr (KV8)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 x = ring_read<float4>(&st.scale[KV8 ? 1 : 0][j / 8][8 * h + j % 8]);
                const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int q = 0; q < 4; q++)
                    p[j + q] *= CUT && 16 * (j / 8) + 8 * h + j % 8 + q >= left ? 0.0f : v[q];
            }
#pragma unroll
        for (int pg = 0; pg < 2; pg++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = p[8 * pg + j];
            bf16x8 W[PP];
            split8<PP>(x, W);
            if (pg == 0 && NP > 1)
                read_v(1);
#pragma unroll
            for (int e = 0; e < NE; e++) {
                uint4 w;
                if constexpr (KV8) {
                    uint32_t x[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const v2f r = {(float)(int8_t)(v8[pg][2 * j] >> (8 * e)), (float)(int8_t)(v8[pg][2 * j + 1] >> (8 * e))};
                        x[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
                    }
                    w = make_uint4(x[0], x[1], x[2], x[3]);
                } else {
                    w = vw[pg][KV8 ? 0 : e];
                    // V of tokens past the part is whatever the page held: a weight
                    // of zero times a NaN pattern would be NaN
                    if constexpr (CUT) {
                        const int ok = left - 16 * pg - 8 * h;        // of the lane's eight tokens
                        w.x &= (ok > 0 ? 0xFFFFu : 0u) | (ok > 1 ? 0xFFFF0000u : 0u);
                        w.y &= (ok > 2 ? 0xFFFFu : 0u) | (ok > 3 ? 0xFFFF0000u : 0u);
                        w.z &= (ok > 4 ? 0xFFFFu : 0u) | (ok > 5 ? 0xFFFF0000u : 0u);
                        w.w &= (ok > 6 ? 0xFFFFu : 0u) | (ok > 7 ? 0xFFFF0000u : 0u);
                    }
                }
                const bf16x8 v = __builtin_bit_cast(bf16x8, w);
#pragma unroll
                for (int n = PP - 1; n >= 0; n--)
                    O[e] = mfma32(v, W[n], O[e]);
            }
        }
    };
    const int whole = (hi - lo) / kStage;
    const bool any = row0 + 32 * rg < rows;                           // else the wave only loads
    const bool mine = any && hi - lo - whole * kStage > tg * kStep;   // of the stage that the part's end cuts
    v16f s;
    for (int i = 0; i < whole; i++) {
        begin(i);
        if (!any)
            continue;
        scores(i, s);
        values(i, s, std::false_type());
    }
    if (whole < ns) {
        begin(whole);
        if (mine) {
            scores(whole, s);
            values(whole, s, std::true_type());
        }
    }

    // the sums of the T waves of each row; dims of operand row x = 8 (i / 4) +
    // 4 h + i % 4 of tile e: 32 e + x, INT8 pages NE x + e
    l += __shfl_xor(l, 32, kWave);
    stage_barrier<0>();                    // every wave is done with the ring, and its loads are
    const int r = 32 * rg + c;
    if (h == 0) {
        S.sums.m[tg][r] = m;
        S.sums.l[tg][r] = l;
    }
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
        for (int e = 0; e < NE; e++) {
            const int x = 8 * (i / 4) + 4 * h + i % 4;
            S.sums.o[tg][r][KV8 ? NE * x + e : 32 * e + x] = O[e][i];
        }
    __syncthreads();
}

// Writes the rows of a part, row0 .. rows - 1 of the tile's, whose waves (or groups
// of them) left their sums in LDS: m, l [NW][ROWS], o [NW][ROWS][HD + 4].  HD / 4
// threads a row; a thread reads kAt rows at once (one at a time a tile of 64 rows
// took 2.6 us, LDS's latency four times over for each).
template <int HD, bool QB, int NW, int ROWS, class S>
__device__ __forceinline__ void write_part(const PrefixArgs &a, const S &sums, int row0, int rows, int b0, int kvh, int G,
                                           int part)
{
    constexpr int L = HD / 4, kApart = 64 * kPartWaves / L, kAt = ROWS / kApart < 4 ? ROWS / kApart : 4;
    const size_t all = (size_t)a.n_queries * a.n_heads;
    const bool last = a.parts_p + a.parts_o == 1;
    const float sc = log2_scale(a);
    const int d = 4 * (threadIdx.x % L), more_q = kApart / G, more_h = kApart % G;
    int c = threadIdx.x / L, qi = (row0 + c) / G, hi = (row0 + c) % G;       // query and head of the group of row c
#pragma unroll 1
    while (row0 + c < rows && c < ROWS) {
        float m[kAt][NW], l[kAt][NW];
        float4 o[kAt][NW];
#pragma unroll
        for (int i = 0; i < kAt; i++)
#pragma unroll
            for (int x = 0; x < NW; x++) {
                m[i][x] = sums.m[x][c + i * kApart];
                l[i][x] = sums.l[x][c + i * kApart];
                o[i][x] = *(const float4 *)&sums.o[x][c + i * kApart][d];
            }
#pragma unroll
        for (int i = 0; i < kAt; i++) {
            float top = m[i][0], sum = 0.0f;
#pragma unroll
            for (int x = 1; x < NW; x++)
                top = fmaxf(top, m[i][x]);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < NW; x++) {
                const float w = part_weight(m[i][x], top, sc);
                sum += w * l[i][x];
                v.x = __fmaf_rn(w, o[i][x].x, v.x);
                v.y = __fmaf_rn(w, o[i][x].y, v.y);
                v.z = __fmaf_rn(w, o[i][x].z, v.z);
                v.w = __fmaf_rn(w, o[i][x].w, v.w);
            }
            if (row0 + c < rows) {
                const size_t row = (size_t)(b0 + qi) * a.n_heads + kvh * G + hi;
                if (last) {
                    const float inv = row_inverse(top, sum);
                    store_out4<QB>(a.out, row * HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    if (d == 0)
                        *(float2 *)(a.part_ml + 2 * (part * all + row)) = make_float2(top, sum);
                    // (k_prefix_join reads no values of a part without tokens)
                    if (top != -INFINITY)
                        *(float4 *)(a.part_o + (part * all + row) * HD + d) = v;
                }
            }
            c += kApart;
            qi += more_q;
            hi += more_h;
            if (hi >= G) {
                hi -= G;
                qi++;
            }
        }
    }
}

// One wave per row: its parts by weight.  Lanes of head_dim / 4 words take the
// parts in turn, kAhead loads each in flight: one at a time, 32 parts of 1024
// rows took 11.6 us.
template <int HD, bool QB>
__device__ __forceinline__ void join_row(const PrefixArgs &a, int parts, size_t row)
{
    constexpr int L = HD / 4, PER = kWave / L, kAhead = 8;
    const size_t all = (size_t)a.n_queries * a.n_heads;
    const int lane = threadIdx.x & 63, sub = lane / L;
    const float2 *ml = (const float2 *)a.part_ml;
    float top = -INFINITY;
    for (int p = lane; p < parts; p += kWave)
        top = fmaxf(top, ml[p * all + row].x);
    top = wave_max(top);
    const float sc = log2_scale(a);
    float l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p0 = sub; p0 < parts; p0 += kAhead * PER) {
        float4 o[kAhead];
        float2 x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const size_t at = (size_t)min(p0 + i * PER, parts - 1) * all + row;
            x[i] = ml[at];
            o[i] = *(const float4 *)(a.part_o + at * HD + 4 * (lane % L));
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            // (a part without tokens left no values)
            const bool in = p0 + i * PER < parts && x[i].x != -INFINITY;
            const float w = in ? __builtin_amdgcn_exp2f((x[i].x - top) * sc) : 0.0f;
            l = in ? __fmaf_rn(w, x[i].y, l) : l;
            v.x = in ? __fmaf_rn(w, o[i].x, v.x) : v.x;
            v.y = in ? __fmaf_rn(w, o[i].y, v.y) : v.y;
            v.z = in ? __fmaf_rn(w, o[i].z, v.z) : v.z;
            v.w = in ? __fmaf_rn(w, o[i].w, v.w) : v.w;
        }
    }
#pragma unroll
    for (int o = L; o < kWave; o <<= 1) {
        l += __shfl_xor(l, o, kWave);
        v.x += __shfl_xor(v.x, o, kWave);
        v.y += __shfl_xor(v.y, o, kWave);
        v.z += __shfl_xor(v.z, o, kWave);
        v.w += __shfl_xor(v.w, o, kWave);
    }
    const float inv = row_inverse(top, l);
    if (sub == 0)
        store_out4<QB>(a.out, row * HD + 4 * lane, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
}

// Tokens of a slot that a call may name: their sums stay within 32 bits.  Rows
// (queries x heads) that it may have: the join's launch, a wave each, has less than
// 2^32 threads.  (The workspace's size is given up to twice as many: the plan's
// numbers of tiles fit an int.)
constexpr int kMaxTokens = 1 << 30;
constexpr size_t kMaxRows = 4 * (size_t)kMaxBlocks;

// The cut of the tokens: as many parts as give `want` workgroups, of at least
// `unit` tokens.
inline void cut(int tokens, long tiles, int unit, long want, int *parts, int *chunk)
{
    *parts = *chunk = 0;
    if (!tokens)
        return;
    const long units = ((long)tokens + unit - 1) / unit;
    const long n = std::min(units, (want + tiles - 1) / tiles);
    *chunk = (int)((units + n - 1) / n * unit);
    *parts = (int)(((long)tokens + *chunk - 1) / *chunk);
}

}  // namespace be42
