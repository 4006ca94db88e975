// prefix.hip -- attention of a batch that shares a prefix: queries over the
// tokens of one shared slot of the page pool and of their own slots.
//
//   out[b][h] = sum_t softmax_t(scale * q[b][h] . k_t) v_t
// over the first prefix_len tokens of slot prefix_slot and the first lens[b]
// tokens of slot slots[b].
//
// Where there are few tokens, a workgroup sees a few queries' all
// (k_prefix_whole).  Else they are cut into parts, some of the prefix and some of
// each query's own tokens; one workgroup forms, for a tile of rows (query, head) of one KV head
// and one part, with s = q.k and c = log2(e) * scale, m = max s, l = sum
// 2^((s - m) c) and o = sum 2^((s - m) c) v, and k_prefix_join adds the parts of a
// row with weights 2^((m - max m) c).  (Differences are taken before they are
// scaled: s c - m c with a rounded m c is off by that rounding, past a score of
// 2^30 by more than an exponent holds.  It costs an instruction a score, 1 - 3%
// where those bound the tile.)  Rows of the prefix are those of all queries, so
// its pages are read once for a tile of up to 128 rows.
//
// What bounds it, of a pass (kernel times; a large copy runs at 5.2 to 5.5 TB/s, a
// large bf16 product at 1.2 PFLOP/s here): 512 bf16 rows over 32768 tokens 121 us,
// 0.85 PFLOP/s with the weights' second part; matrix units are busy for 41% of a
// SIMD's cycles, vector units for 45%, both at once for 15% (forming the next
// step's scores beside this one's weights changed nothing); 128 sequences of up to
// 1024 own tokens behind the same prefix 156 us, 2.6 TB/s, each byte read once; own
// tokens alone 64 us, 4.3 TB/s; 128 fp32 rows over 8190 tokens 30 us, of which 4.5
// until the first pages are there, 14 products (three bf16 parts each of q and the
// weights, 0.45 PFLOP/s of them; one wave a SIMD), 3 results and 4.4 the join; the
// smallest call 7.9 us in one launch, a chain of loads (page table, pages) and steps.
#include <algorithm>
#include <cmath>
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
// go to rows to .. to + rows - row0 - 1 of place `at` in LDS.
template <bool KV8, int HD, int NP, int PP, class Shared>
__device__ __forceinline__ void part16(const be42_kv_pool &P, const PrefixArgs &a, Shared &S, int slot, int lo, int hi, int kvh,
                                       int b0, int row0, int rows, int first, int share, int at, int to)
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
        if (left < kStep)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool out = 8 * g + j >= left;
                p[j] = out ? -INFINITY : p[j];
                if (KV8)
                    vsc[j] = out ? 0.0f : vsc[j];
            }
        float top = max3(max3(p[0], p[1], p[2]), max3(p[3], p[4], p[5]), max3(p[6], p[7], p[7])), other;
        quarters(top, top, other);
        top = max3(top, other, other);
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
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f((p[j] - m) * sc);
            l += p[j];
            if (KV8)
                p[j] *= vsc[j];
        }
        bf16x8 W[PP];
        split8<PP>(p, W);
        // V of tokens past the part is whatever the page held: a weight of zero
        // times a NaN pattern would be NaN
        if (!KV8 && left < kStep) {
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                keep[j] = (8 * g + 2 * j < left ? 0xFFFFu : 0u) | (8 * g + 2 * j + 1 < left ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int e = 0; e < (KV8 ? 0 : NE); e++) {
                V[e].x &= keep[0];
                V[e].y &= keep[1];
                V[e].z &= keep[2];
                V[e].w &= keep[3];
            }
        }
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
                                       int lo, int want, int kvh, int row0, int rows)
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
    const size_t qat = (size_t)(rc / G) * a.q_stride + (size_t)(kvh * G + rc % G) * HD;
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
    const bool mine = hi - lo - whole * kStage > tg * kStep;          // of the stage that the part's end cuts
    v16f s;
    for (int i = 0; i < whole; i++) {
        begin(i);
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

// One workgroup a tile of rows and part: of the prefix by part32 (R > 0) or
// part16, of own tokens by part16.  fp32 queries and their weights enter the
// products with all 24 bits, in three parts.  For bf16 queries, whose output is
// rounded to bf16 (2^-8 of it at most), the weights are rounded to 16 bits, in two
// parts, whatever the batch: over 32768 tokens the output is off by 0.0017 of
// itself, its rounding alone.  (One part, bf16, made that 0.0023, and 0.0026 from
// the same query's in a batch of few; 128 queries over 32768 tokens and up to 1024
// of their own 133 us instead of 158.)
template <bool KV8, int HD, bool QB, int R>
__global__ __launch_bounds__(64 * kPartWaves, 2) void k_prefix_part(const be42_kv_pool P, const PrefixArgs a)
{
    __shared__ union {
        PartShared<HD> few;
        std::conditional_t<R != 0, WideShared<KV8, HD, R ? R : 4>, char> many;
    } S;
    constexpr int NP = QB ? 1 : 3, kRows = R ? 32 * R : 16;
    const int G = a.n_heads / P.n_kv;
    const unsigned of_prefix = (unsigned)P.n_kv * a.tiles_p * a.parts_p;
    unsigned id = blockIdx.x;
    int slot, n, chunk, part, b0, row0, rows;
    const bool own = id >= of_prefix;
    if (own)
        id -= of_prefix;
    const int kvh = (int)(id % (unsigned)P.n_kv);
    id /= (unsigned)P.n_kv;
    if (own) {
        row0 = 16 * (int)(id % (unsigned)a.tiles_o);
        id /= (unsigned)a.tiles_o;
        b0 = (int)(id % (unsigned)a.n_queries);
        part = (int)(id / (unsigned)a.n_queries);
        rows = G;
        slot = a.slots ? a.slots[b0] : b0;
        n = a.lens ? min(a.lens[b0], a.max_len) : a.max_len;
        chunk = a.chunk_o;
    } else {
        row0 = kRows * (int)(id % (unsigned)a.tiles_p);
        part = (int)(id / (unsigned)a.tiles_p);
        b0 = 0;
        rows = a.n_queries * G;
        slot = a.prefix_slot;
        n = a.prefix_len;
        chunk = a.chunk_p;
    }
    const int lo = part * chunk;
    n = min(n, lo + chunk);
    part += own ? a.parts_p : 0;
    if constexpr (R != 0)
        if (!own) {
            part32<KV8, HD, NP, QB ? 2 : 3, R>(P, a, S.many, slot, lo, n, kvh, row0, rows);
            write_part<HD, QB, kPartWaves / R, kRows>(a, S.many.sums, row0, rows, b0, kvh, G, part);
            return;
        }
    const int wave = threadIdx.x >> 6;
    part16<KV8, HD, NP, QB ? 2 : 3>(P, a, S.few, slot, lo, max(lo, slot_tokens(P, slot, n)), kvh, b0, row0, rows, wave, kPartWaves,
                                    wave, 0);
    __syncthreads();
    write_part<HD, QB, kPartWaves, 16>(a, S.few, row0, rows, b0, kvh, G, part);
}

// A call with few tokens in one launch: a workgroup takes as many queries as 16
// rows hold, the prefix with all its waves, then each wave the own tokens of every
// fourth query.  (Those keep sums of their own: in the tile of all rows a weight
// of zero times a NaN in one query's pages would reach the others.)
template <bool KV8, int HD, bool QB>
__global__ __launch_bounds__(64 * kPartWaves, 2) void k_prefix_whole(const be42_kv_pool P, const PrefixArgs a)
{
    __shared__ PartShared<HD, kPartWaves + 1> S;
    constexpr int NP = QB ? 1 : 3, PP = QB ? 2 : 3;
    const int G = a.n_heads / P.n_kv, fit = 16 / G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = (int)(blockIdx.x % (unsigned)P.n_kv), b0 = (int)(blockIdx.x / (unsigned)P.n_kv) * fit;
    const int rows = min(fit, a.n_queries - b0) * G;
    part16<KV8, HD, NP, PP>(P, a, S, a.prefix_slot, 0, slot_tokens(P, a.prefix_slot, a.prefix_len), kvh, b0, 0, rows, wave,
                            kPartWaves, wave, 0);
    for (int j = wave; j * G < rows; j += kPartWaves) {
        const int b = b0 + j, slot = a.slots ? a.slots[b] : b, n = a.lens ? min(a.lens[b], a.max_len) : a.max_len;
        part16<KV8, HD, NP, PP>(P, a, S, slot, 0, slot_tokens(P, slot, n), kvh, b, 0, G, 0, 1, kPartWaves, j * G);
    }
    __syncthreads();
    write_part<HD, QB, kPartWaves + 1, 16>(a, S, 0, rows, b0, kvh, G, 0);
}

// One wave per row: its parts by weight.  Lanes of head_dim / 4 words take the
// parts in turn, kAhead loads each in flight: one at a time, 32 parts of 1024
// rows took 11.6 us.
template <int HD, bool QB>
__global__ __launch_bounds__(256) void k_prefix_join(const PrefixArgs a, int parts)
{
    constexpr int L = HD / 4, PER = kWave / L, kAhead = 8;
    const size_t all = (size_t)a.n_queries * a.n_heads, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, sub = lane / L;
    if (row >= all)
        return;
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
static void cut(int tokens, long tiles, int unit, long want, int *parts, int *chunk)
{
    *parts = *chunk = 0;
    if (!tokens)
        return;
    const long units = ((long)tokens + unit - 1) / unit;
    const long n = std::min(units, (want + tiles - 1) / tiles);
    *chunk = (int)((units + n - 1) / n * unit);
    *parts = (int)(((long)tokens + *chunk - 1) / *chunk);
}

// Rows of a prefix tile: up to 32 rows of a KV head go in tiles of 16 (fp32, 32
// rows over 2000 tokens 12.1 us, 14.1 in one of 64; over 32000 39.8 and 40.5; over
// 8192 20.9 and 19.4; four rows 9.6 and 12.1, 34.0 and 38.9, 18.5 and 18.4), up to
// 256 in tiles of 64 (128 rows over 8192: 27.9 us, 31.0 in one of 128), more in
// tiles of 128 (32768 tokens, 512 bf16 rows and own tokens: 157 us, 178 in tiles of
// 64).  The prefix gets a workgroup a CU, so that own tokens, which wait for memory,
// run beside it (two: 162 us; 128 fp32 rows over 8190 tokens and up to 256 own
// tokens 30.0, two 35.7); where there are few of those and the parts stay long, it
// gets two (512 rows alone 121 us, 142 with one; 128 fp32 rows over 32000 tokens 64
// and 68, over 16000 41.5 and 40.5; heads of 64, half the work a token, 64 rows over
// 32768 tokens 31.4 and 27.9).
static void plan_prefix(PrefixArgs &a, int n_kv, int head_dim)
{
    const int G = a.n_heads / n_kv, unit = kPartWaves * kStep;
    const long rows = (long)a.n_queries * G;
    // Short prefixes and own tokens go in one launch where a wave's steps of 32
    // tokens are few, up to 32 rows of a KV head five, up to 256 eight, more twelve.
    // fp32, 32 heads on 8 KV heads, 40 own tokens, in us: one query over 300 tokens
    // 9.6, in parts 9.4, over 600 12.3 and 9.5 (besides a second launch's 3 us of the
    // caller's time); 64 queries over 300 13.0 and 17.4, over 600 (seven steps) 16.1
    // and 18.4, over 1200 (twelve) 22.4 and 20.5; 512 over 300 35 and 60, over 1200 69
    // and 77, over 1600 (fifteen) 84 and 82.
    const long turns = G <= 16 ? std::min((long)a.n_queries, 16L / G) : 0, each = (turns + kPartWaves - 1) / kPartWaves;
    const long steps = (a.prefix_len + unit - 1L) / unit + each * ((a.max_len + kStep - 1L) / kStep);
    a.whole = G <= 16 && steps <= (rows > 256 ? 12 : rows > 32 ? 8 : 5);
    if (a.whole) {
        a.parts_p = 1;
        return;
    }
    a.rows_p = rows > 256 ? 128 : rows > 32 ? 64 : 16;
    a.tiles_p = (int)((rows + a.rows_p - 1) / a.rows_p);
    a.tiles_o = (G + 15) / 16;
    const long tiles = (long)a.tiles_p * n_kv, read = (long)a.prefix_len * a.tiles_p;
    const bool two = a.rows_p == 16 || ((double)a.prefix_len * tiles * head_dim >= 1L << 25 && 2L * a.n_queries * a.max_len < read);
    cut(a.prefix_len, tiles, unit, two ? 512 : 256, &a.parts_p, &a.chunk_p);
    cut(a.max_len, (long)a.tiles_o * n_kv * a.n_queries, unit, 512, &a.parts_o, &a.chunk_o);
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_prefix_attention_workspace_bytes(int n_queries, int n_heads, int n_kv, int head_dim,
                                                        int prefix_len, int max_len)
{
    if (n_queries <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || (head_dim != 64 && head_dim != 128) ||
        prefix_len < 0 || prefix_len > kMaxTokens || max_len < 0 || max_len > kMaxTokens ||
        (size_t)n_queries * n_heads > 2 * kMaxRows)
        return 0;
    PrefixArgs a = {};
    a.n_queries = n_queries;
    a.n_heads = n_heads;
    a.prefix_len = prefix_len;
    a.max_len = max_len;
    plan_prefix(a, n_kv, head_dim);
    const int parts = a.parts_p + a.parts_o;
    return 16 + (parts > 1 ? (size_t)parts * n_queries * n_heads * (head_dim + 2) * sizeof(float) : 0);
}

extern "C" int be42_prefix_attention(const be42_kv_pool *pool, const void *q, int q_bf16, int q_stride, int n_queries,
                                     int n_heads, int prefix_slot, int prefix_len, const int *slots, const int *lens,
                                     int max_len, float scale, void *out, void *workspace, size_t workspace_bytes,
                                     void *stream)
{
    BE42_CHECK(pool && (n_queries == 0 || (q && out)), "be42_prefix_attention: null pointer");
    const be42_kv_pool &P = *pool;
    BE42_CHECK(n_heads > 0 && n_heads % P.n_kv == 0, "be42_prefix_attention: %d heads over %d kv heads", n_heads,
               P.n_kv);
    BE42_CHECK(P.head_dim == 64 || P.head_dim == 128, "be42_prefix_attention: head_dim %d (64 or 128)", P.head_dim);
    BE42_CHECK(n_queries >= 0 && q_stride >= (long)n_heads * P.head_dim, "be42_prefix_attention: %d queries at stride %d",
               n_queries, q_stride);
    BE42_CHECK(prefix_slot >= 0 && prefix_slot < P.n_layers, "be42_prefix_attention: prefix slot %d of %d", prefix_slot,
               P.n_layers);
    const long held = (long)P.max_logical * kPage;
    BE42_CHECK(prefix_len >= 0 && prefix_len <= std::min(held, (long)kMaxTokens) && max_len >= 0 && max_len <= kMaxTokens,
               "be42_prefix_attention: prefix %d, max_len %d (a slot holds %ld tokens)", prefix_len, max_len, held);
    BE42_CHECK(std::fabs(scale) <= 1e30f, "be42_prefix_attention: scale %g", (double)scale);
    BE42_CHECK(!(((uintptr_t)q | (uintptr_t)out) & (q_bf16 ? 1 : 3)), "be42_prefix_attention: unaligned pointer");
    // without slots query b reads slot b
    BE42_CHECK(slots || max_len == 0 || n_queries <= P.n_layers, "be42_prefix_attention: %d queries over %d slots",
               n_queries, P.n_layers);
    if (n_queries == 0)
        return BE42_OK;
    const size_t rows = (size_t)n_queries * n_heads;
    BE42_CHECK(rows <= kMaxRows, "be42_prefix_attention: %d queries of %d heads", n_queries, n_heads);
    PrefixArgs a = {q, out, slots, lens, nullptr, nullptr, (size_t)q_stride, n_queries, n_heads, prefix_slot, prefix_len,
                    max_len, scale};
    plan_prefix(a, P.n_kv, P.head_dim);
    const int parts = a.parts_p + a.parts_o;
    const long blocks = (long)P.n_kv * ((long)a.tiles_p * a.parts_p + (long)a.tiles_o * n_queries * a.parts_o);
    BE42_CHECK(blocks <= kMaxBlocks, "be42_prefix_attention: %d queries of %d heads", n_queries, n_heads);
    const size_t need = be42_prefix_attention_workspace_bytes(n_queries, n_heads, P.n_kv, P.head_dim, prefix_len,
                                                              max_len);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_prefix_attention: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    hipStream_t s = as_stream(stream);
    // (whether or not these sizes use it)
    BE42_CHECK(workspace || !captured(s), "be42_prefix_attention: a captured call needs a workspace of the caller's");
    if (parts > 1) {
        if (!workspace)
            workspace = be42::workspace(need, s);
        if (!workspace)
            return BE42_ENOMEM;
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + (size_t)parts * rows * P.head_dim;
    }
    const int fit = a.whole ? 16 * P.n_kv / n_heads : 1;
    auto go = [&](auto kv8, auto hd, auto qb) {
        constexpr bool KV8 = decltype(kv8)::value, QB = decltype(qb)::value;
        constexpr int HD = decltype(hd)::value;
        const dim3 g((unsigned)blocks), t(64 * kPartWaves);
        if (a.whole) {
            hipLaunchKernelGGL((k_prefix_whole<KV8, HD, QB>), dim3((unsigned)((n_queries + fit - 1) / fit * P.n_kv)), t, 0, s, P, a);
            return;
        }
        if (parts && a.rows_p == 128)
            hipLaunchKernelGGL((k_prefix_part<KV8, HD, QB, 4>), g, t, 0, s, P, a);
        else if (parts && a.rows_p == 64)
            hipLaunchKernelGGL((k_prefix_part<KV8, HD, QB, 2>), g, t, 0, s, P, a);
        else if (parts)
            hipLaunchKernelGGL((k_prefix_part<KV8, HD, QB, 0>), g, t, 0, s, P, a);
        if (parts != 1)
            hipLaunchKernelGGL((k_prefix_join<HD, QB>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, parts);
    };
    auto of_type = [&](auto kv8, auto hd) { q_bf16 ? go(kv8, hd, std::true_type()) : go(kv8, hd, std::false_type()); };
    auto of_dim = [&](auto kv8) {
        P.head_dim == 64 ? of_type(kv8, std::integral_constant<int, 64>()) : of_type(kv8, std::integral_constant<int, 128>());
    };
    P.kind == BE42_KV_INT8 ? of_dim(std::true_type()) : of_dim(std::false_type());
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
