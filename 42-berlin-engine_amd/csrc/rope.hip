// rope.hip -- tokens into the pages of several slots at once: norms of queries and
// keys, rotation and append in one pass (be42_rope_append), and drafted tokens that
// were right behind their sequences (be42_kv_accept).
//
// A workgroup takes the tokens of a call that go into one page, for one KV head: the
// query heads of its group, its K and its V row.  Pages are planned on the host and
// go with the launch by value, so nothing is copied to the device beforehand; the
// workgroup of KV head 0 seals the page where its last position is written.
#include <algorithm>
#include <new>
#include <type_traits>

#include "be42_common.h"
#include "paged_dev.h"
#include "paged_step.h"

namespace be42 {

// What a launch takes: pieces of runs, whose physical pages follow one another (new ones
// mostly do: no list, and prompts of any length in one launch) or are listed.
constexpr int kPieces = 64, kPiecePages = 480;
constexpr int kMaxGridYZ = 65535;
struct Piece {
    int slot, pos0, n, tok0, page0;    // page0: its first page's workgroup
    int entry0, step;                  // page j is entry0 + step * j, with step 0 pages[entry0 + j]
};
struct RopeArgs {
    int n, n_pages, n_listed;
    Piece piece[kPieces];
    int pages[kPiecePages];
};

struct RopeIn {
    const void *q, *k, *v;
    void *q_out;
    const uint16_t *q_norm, *k_norm;
    const float *cos_t, *sin_t;
    const int *positions;
    size_t q_stride, k_stride, v_stride, q_out_stride;
    int n_heads, rope_len, rope_dim, interleaved;
    float eps;
};
// (arguments of a kernel are at most 4 KB, with the padding between them)
constexpr size_t kMostArgs = 4096 - 16;
static_assert(sizeof(be42_kv_pool) + sizeof(RopeArgs) + sizeof(RopeIn) <= kMostArgs, "arguments of a launch");

// The entry of page j of a piece: its physical page, and kNewPage.
__device__ __forceinline__ int page_entry(const RopeArgs &a, const Piece &p, int j)
{
    return p.step ? p.entry0 + p.step * j : a.pages[p.entry0 + j];
}

// The piece that page `at` of a launch belongs to: lanes compare, one each.
template <class A>
__device__ __forceinline__ int piece_of(const A &a, int at)
{
    if (a.n == 1)
        return 0;
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(lane < a.n && a.piece[min(lane, kPieces - 1)].page0 <= at)) - 1;
}

// The page table's and the page's words, by the workgroup of KV head 0.  A launch may hold
// several pieces of one run, whose ends are not the run's, and their workgroups are here
// at once: the slot's counts grow by atomic maxima, which leave the run's in any order.
__device__ __forceinline__ void publish(const be42_kv_pool &P, int slot, int pos0, int n, int blk, int phys, bool fresh)
{
    const int end = pos0 + n;
    if (fresh) {
        P.page_table[(size_t)slot * P.max_logical + blk] = phys;
        // (a replay may come after appends behind the captured ones, whose pages stay)
        if (end <= (blk + 1) * kPage)
            atomicMax(&P.n_logical[slot], blk + 1);
    }
    // the page ends with what was written last, as be42_kv_append leaves it: a call at
    // earlier positions, and a replay like it, takes the page's later tokens off
    P.ntok[phys] = min(end - blk * kPage, kPage);
    // the last page that the piece fills
    if (end >= (blk + 1) * kPage && end < (blk + 2) * kPage)
        atomicMax(&P.n_indexed[slot], blk + 1);
}

// seal_page of a page whose rows the workgroup has just written, the same sums in the
// same order; the projection was brought to LDS while the rows were on their way (by
// load_projection: the chain of the hash's products waits for a load of it every few
// terms otherwise, and a seal takes 5 us; accepted drafts of 28 layers 6.6
// us with it, 4.6 without).
template <int HD = 256>
struct SealShared {
    float hp[HD * 16], c[HD];
};
template <class S_>
__device__ __forceinline__ void load_projection(const be42_kv_pool &P, S_ &S)
{
    for (int i = threadIdx.x; i < P.head_dim * 4; i += 256)
        *(float4 *)&S.hp[4 * i] = *(const float4 *)(P.hpT + 4 * i);
}
template <bool BF16, class S_>
__device__ __forceinline__ void seal_written(const be42_kv_pool &P, S_ &S, int slot, int blk, int phys)
{
    const int d = threadIdx.x, hd = P.head_dim;
    __syncthreads();                       // the page's rows are in memory
    const size_t head0 = (size_t)phys * P.n_kv * kPage;
    if (d < hd) {
        float x[kPage], acc = 0.0f;
#pragma unroll
        for (int t = 0; t < kPage; t++)
            x[t] = BF16 ? bf16_to_f32(((const uint16_t *)P.k)[(head0 + t) * hd + d])
                        : (float)((const int8_t *)P.k)[(head0 + t) * hd + d] * P.k_scale[head0 + t];
#pragma unroll
        for (int t = 0; t < kPage; t++)
            acc = acc + x[t];
        acc = acc * (1.0f / (float)kPage);
        S.c[d] = acc;
        P.centroid[(size_t)phys * hd + d] = acc;
    }
    __syncthreads();
    if (d >= kWave)
        return;
    // (head_dim is a multiple of 8)
    float s = 0.0f;
    if (d < 16)
        for (int i = 0; i < hd; i += 8) {
            float c[8], h[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                c[j] = S.c[i + j];
                h[j] = S.hp[(i + j) * 16 + d];
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                s = __fmaf_rn(c[j], h[j], s);
        }
    const unsigned long long m = __ballot(d < 16 && s > 0.0f);
    if (d == 0)
        P.page_hash[(size_t)slot * P.max_logical + blk] = (uint16_t)(m & 0xFFFFu);
}

template <bool BF16>
__device__ __forceinline__ float act_at(const void *p, size_t i)
{
    return BF16 ? bf16_to_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

// op over the lanes of a group of L (8, 16 or 32), in every one, by lane moves.
template <int L, class T, class F>
__device__ __forceinline__ T group_all(T v, F &&op)
{
    v = op(v, dpp_mov<0xB1>(v, v));            // neighbours, pairs, halves of 8, of 16
    v = op(v, dpp_mov<0x4E>(v, v));
    v = op(v, dpp_mov<0x141>(v, v));
    if constexpr (L >= 16)
        v = op(v, dpp_mov<0x140>(v, v));
    if constexpr (L >= 32)
        v = op(v, __shfl_xor(v, 16, kWave));
    return v;
}

// Four elements from `at` on (any alignment).
template <bool BF16>
__device__ __forceinline__ void load4(const void *p, size_t at, float *v)
{
    if constexpr (BF16) {
        uint32_t u[2];
        __builtin_memcpy(u, (const uint16_t *)p + at, 8);
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[j] = __uint_as_float(j & 1 ? u[j / 2] & 0xFFFF0000u : u[j / 2] << 16);
    } else {
        __builtin_memcpy(v, (const float *)p + at, 16);
    }
}
__device__ __forceinline__ uint2 bf16_4(const float *v)
{
    return make_uint2(f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16, f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16);
}

// Heads of 64, 128 or 256, a rotation of a multiple of 8 elements.  A group of HD / 8
// lanes takes a row: lane u the pairs 4 u .. 4 u + 3 of the rotation in two words of
// four, or eight elements of what is not rotated.  A workgroup takes two heads' rows of
// the tokens of a page, K and V or two query heads (blockIdx.z), all its loads in
// flight together and one pair of table words for both heads; rows of V go through LDS
// where the whole page is written, so that they leave as its lines.  Bound by HBM: 11801 bf16
// tokens with norms, 32 query heads on 8 KV heads of 128, 79 us, 3.7 TB/s (243 us in the
// form below; with all 740 pages listed, in two launches, 85); 218 INT8 tokens 6.9 us (25).
template <bool KV8, bool BF16, int HD>
__global__ __launch_bounds__(256) void k_rope_append_words(const be42_kv_pool P, const RopeArgs a, const RopeIn x)
{
    constexpr int L = HD / 8, PER = 256 / L, TOKENS = PER < kPage ? PER : kPage, VS = kPage + 8;
    __shared__ __align__(16) SealShared<HD> seal;
    __shared__ __align__(16) uint16_t vt[KV8 ? 1 : HD][VS];
    const int h = blockIdx.y, z = blockIdx.z, grp = threadIdx.x / L, l = threadIdx.x % L;
    const Piece &p = a.piece[piece_of(a, blockIdx.x)];
    const int blk = p.pos0 / kPage + ((int)blockIdx.x - p.page0);
    const int entry = page_entry(a, p, (int)blockIdx.x - p.page0), phys = entry & ~kNewPage;
    const int lo = max(p.pos0, blk * kPage), T = min(p.pos0 + p.n, (blk + 1) * kPage) - lo;
    const int tok0 = p.tok0 + lo - p.pos0, off0 = lo - blk * kPage;
    const int G = x.n_heads / P.n_kv, half = x.rope_dim / 2;
    const bool kv = z == 0, two = kv || 2 * z <= G;
    const int head = h * G + 2 * (z - 1);
    const bool seals = kv && h == 0 && off0 + T == kPage;
    if (seals)
        load_projection(P, seal);
    if (kv && h == 0 && threadIdx.x == 0)
        publish(P, p.slot, p.pos0, p.n, blk, phys, entry & kNewPage);
    // the lane's two words
    const bool turns = 8 * l < x.rope_dim;
    const int c0 = turns && !x.interleaved ? 4 * l : 8 * l, c1 = turns && !x.interleaved ? half + 4 * l : 8 * l + 4;
    const uint16_t *w = kv ? x.k_norm : x.q_norm;
    for (int i = grp; i < T && grp < TOKENS; i += TOKENS) {
        const int tok = tok0 + i;
        float y[2][8], cs[4], sn[4], wt[8];
        const size_t at0 = kv ? tok * x.k_stride + (size_t)h * HD : tok * x.q_stride + (size_t)head * HD;
        const size_t at1 = kv ? tok * x.v_stride + (size_t)h * HD : at0 + HD;
        const void *from0 = kv ? x.k : x.q, *from1 = kv ? x.v : x.q;
        load4<BF16>(from0, at0 + c0, y[0]);
        load4<BF16>(from0, at0 + c1, y[0] + 4);
        if (two) {
            load4<BF16>(from1, at1 + c0, y[1]);
            load4<BF16>(from1, at1 + c1, y[1] + 4);
        }
        const int pos = x.positions ? x.positions[tok] : lo + i;
        const bool turn = turns && pos >= 0 && pos < x.rope_len;
        if (turn) {
            load4<false>(x.cos_t, (size_t)pos * half + 4 * l, cs);
            load4<false>(x.sin_t, (size_t)pos * half + 4 * l, sn);
        }
        if (w) {
            load4<true>(w, c0, wt);
            load4<true>(w, c1, wt + 4);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (j && (!two || kv))
                break;
            if (w) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    ss = fma((double)y[j][e], (double)y[j][e], ss);
                ss = group_all<L>(ss, [](double a, double b) { return a + b; });
                const double s = 1.0 / sqrt(ss / HD + (double)x.eps);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    y[j][e] = (float)((double)y[j][e] * s * (double)wt[e]);
            }
            if (turn)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float &u = x.interleaved ? y[j][2 * e] : y[j][e], &v = x.interleaved ? y[j][2 * e + 1] : y[j][4 + e];
                    const float u0 = u, v0 = v;
                    u = __fmaf_rn(u0, cs[e], -(v0 * sn[e]));
                    v = __fmaf_rn(u0, sn[e], v0 * cs[e]);
                }
        }
        if (!kv) {
            const size_t to = tok * x.q_out_stride + (size_t)head * HD;
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (j == 0 || two)
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const size_t at = to + j * HD + (e ? c1 : c0);
                        if constexpr (BF16) {
                            const uint2 b = bf16_4(y[j] + e);
                            __builtin_memcpy((uint16_t *)x.q_out + at, &b, 8);
                        } else {
                            __builtin_memcpy((float *)x.q_out + at, y[j] + e, 16);
                        }
                    }
            continue;
        }
        const int off = off0 + i;
        const size_t row = ((size_t)phys * P.n_kv + h) * kPage + off;
        if constexpr (KV8) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    m = fmaxf(m, fabsf(y[j][e]));
                m = group_all<L>(m, [](float a, float b) { return fmaxf(a, b); });
                const float sc = m > 0.0f ? m / 127.0f : 1.0f, inv = m > 0.0f ? 127.0f / m : 1.0f;
                int8_t *to = (int8_t *)(j ? P.v : P.k) + row * HD;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    uint32_t code = 0;
#pragma unroll
                    for (int d = 0; d < 4; d++)
                        code |= (uint32_t)(uint8_t)max(min((int)roundf(y[j][e + d] * inv), 127), -127) << (8 * d);
                    *(uint32_t *)(to + (e ? c1 : c0)) = code;
                }
                if (l == 0)
                    (j ? P.v_scale : P.k_scale)[row] = sc;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *(uint2 *)((uint16_t *)P.k + row * HD + (e ? c1 : c0)) = bf16_4(y[0] + e);
            uint16_t *to = (uint16_t *)P.v + (row / kPage) * HD * kPage + off;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = (e < 4 ? c0 : c1 - 4) + e;
                if (T == kPage)
                    vt[d][i] = f32_to_bf16(y[1][e]);
                else
                    to[(size_t)d * kPage] = f32_to_bf16(y[1][e]);
            }
        }
    }
    if (!kv)
        return;
    if constexpr (!KV8)
        if (T == kPage) {
            __syncthreads();
            uint16_t *to = (uint16_t *)P.v + ((size_t)phys * P.n_kv + h) * HD * kPage;
            for (int i = threadIdx.x; i < 2 * HD; i += 256)
                *(uint4 *)(to + 8 * i) = *(const uint4 *)&vt[i / 2][8 * (i % 2)];
        }
    if (seals)
        seal_written<!KV8>(P, seal, p.slot, blk, phys);
}

// Any other head, or rotation: one wave a row, a lane a pair of elements (two pairs where head_dim is past 128):
// the pairs of the rotation, then neighbours behind them.
template <bool KV8, bool BF16, int NP>
__global__ __launch_bounds__(256) void k_rope_append(const be42_kv_pool P, const RopeArgs a, const RopeIn x)
{
    __shared__ __align__(16) SealShared<> seal;
    const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Piece &u = a.piece[piece_of(a, blockIdx.x)];
    const int blk = u.pos0 / kPage + ((int)blockIdx.x - u.page0);
    const int entry = page_entry(a, u, (int)blockIdx.x - u.page0), phys = entry & ~kNewPage;
    const int lo = max(u.pos0, blk * kPage), T = min(u.pos0 + u.n, (blk + 1) * kPage) - lo;
    const int tok0 = u.tok0 + lo - u.pos0, off0 = lo - blk * kPage;
    const int hd = P.head_dim, G = x.n_heads / P.n_kv, half = x.rope_dim / 2;
    const bool seals = h == 0 && off0 + T == kPage;
    if (seals)
        load_projection(P, seal);
    if (h == 0 && threadIdx.x == 0)
        publish(P, u.slot, u.pos0, u.n, blk, phys, entry & kNewPage);
    for (int r = wave; r < T * (G + 2); r += 4) {
        const int kind = r / T, i = r % T, tok = tok0 + i;     // query heads, then K, then V
        const bool is_v = kind == G + 1, is_k = kind == G;
        const size_t at = is_v ? tok * x.v_stride + (size_t)h * hd
                        : is_k ? tok * x.k_stride + (size_t)h * hd
                               : tok * x.q_stride + (size_t)(h * G + kind) * hd;
        const void *from = is_v ? x.v : is_k ? x.k : x.q;
        const uint16_t *w = is_v ? nullptr : is_k ? x.k_norm : x.q_norm;
        int e0[NP], e1[NP];
        float y0[NP], y1[NP];
        bool in[NP];
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int p = lane + 64 * j;
            in[j] = p < hd / 2;
            const bool apart = p < half && !x.interleaved;
            e0[j] = apart ? p : 2 * p;
            e1[j] = apart ? p + half : 2 * p + 1;
            y0[j] = in[j] ? act_at<BF16>(from, at + e0[j]) : 0.0f;
            y1[j] = in[j] ? act_at<BF16>(from, at + e1[j]) : 0.0f;
        }
        if (w) {
            double ss = 0.0;
#pragma unroll
            for (int j = 0; j < NP; j++)
                ss = fma((double)y1[j], (double)y1[j], fma((double)y0[j], (double)y0[j], ss));
            const double s = 1.0 / sqrt(wave_sum_d(ss) / hd + (double)x.eps);
#pragma unroll
            for (int j = 0; j < NP; j++)
                if (in[j]) {
                    y0[j] = (float)((double)y0[j] * s * (double)bf16_to_f32(w[e0[j]]));
                    y1[j] = (float)((double)y1[j] * s * (double)bf16_to_f32(w[e1[j]]));
                }
        }
        const int pos = x.positions ? x.positions[tok] : lo + i;
        if (!is_v && pos >= 0 && pos < x.rope_len)
#pragma unroll
            for (int j = 0; j < NP; j++) {
                const int p = lane + 64 * j;
                if (p < half) {
                    const float cs = x.cos_t[(size_t)pos * half + p], sn = x.sin_t[(size_t)pos * half + p];
                    const float z0 = __fmaf_rn(y0[j], cs, -(y1[j] * sn)), z1 = __fmaf_rn(y0[j], sn, y1[j] * cs);
                    y0[j] = z0;
                    y1[j] = z1;
                }
            }
        if (!is_v && !is_k) {
            const size_t to = tok * x.q_out_stride + (size_t)(h * G + kind) * hd;
#pragma unroll
            for (int j = 0; j < NP; j++)
                if (in[j]) {
                    if (BF16) {
                        ((uint16_t *)x.q_out)[to + e0[j]] = f32_to_bf16(y0[j]);
                        ((uint16_t *)x.q_out)[to + e1[j]] = f32_to_bf16(y1[j]);
                    } else {
                        ((float *)x.q_out)[to + e0[j]] = y0[j];
                        ((float *)x.q_out)[to + e1[j]] = y1[j];
                    }
                }
            continue;
        }
        const size_t head = (size_t)phys * P.n_kv + h;
        const int off = off0 + i;
        if constexpr (KV8) {
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < NP; j++)
                m = fmaxf(m, fmaxf(fabsf(y0[j]), fabsf(y1[j])));
            m = wave_top(m);
            const float sc = m > 0.0f ? m / 127.0f : 1.0f, inv = m > 0.0f ? 127.0f / m : 1.0f;
            int8_t *to = (int8_t *)(is_k ? P.k : P.v) + (head * kPage + off) * hd;
#pragma unroll
            for (int j = 0; j < NP; j++)
                if (in[j]) {
                    const int c0 = (int)roundf(y0[j] * inv), c1 = (int)roundf(y1[j] * inv);
                    to[e0[j]] = (int8_t)max(min(c0, 127), -127);
                    to[e1[j]] = (int8_t)max(min(c1, 127), -127);
                }
            if (lane == 0)
                (is_k ? P.k_scale : P.v_scale)[head * kPage + off] = sc;
        } else {
            // (V pages are [dim][16 tokens])
            uint16_t *to = is_k ? (uint16_t *)P.k + (head * kPage + off) * hd : (uint16_t *)P.v + head * kPage * hd + off;
            const int step = is_k ? 1 : kPage;
#pragma unroll
            for (int j = 0; j < NP; j++)
                if (in[j]) {
                    to[e0[j] * step] = f32_to_bf16(y0[j]);
                    to[e1[j] * step] = f32_to_bf16(y1[j]);
                }
        }
    }
    if (seals)
        seal_written<!KV8>(P, seal, u.slot, blk, phys);
}

// Pieces of a launch of be42_kv_accept, the same for each of its layers, and the tokens
// to take.  Pages that are old in every layer are looked up in the page tables; the
// others are listed, layer after layer (a page for every one of 28 layers x 25 pages
// would take two launches).
constexpr int kTakes = 64, kTaken = 248, kTakePages = 352;
struct TakeArgs {
    int n, n_pages, n_listed, layer0, from_step, to_step;
    struct {
        int from, slot, pos0;
        short n, tok0, page0, list0;   // list0: its first listed page's place in a layer's
        uint32_t listed;               // which of its pages (at most 17)
    } piece[kTakes];
    int index[kTaken];
    int pages[kTakePages];
};
static_assert(sizeof(be42_kv_pool) + sizeof(TakeArgs) <= kMostArgs, "arguments of a launch");
static_assert(kTaken <= 16 * kPage, "at most 17 pages of a piece");

template <bool KV8>
__global__ __launch_bounds__(256) void k_kv_accept(const be42_kv_pool P, const TakeArgs a)
{
    __shared__ __align__(16) SealShared<> seal;
    const int h = blockIdx.y, layer = blockIdx.z, hd = P.head_dim;
    const auto &u = a.piece[piece_of(a, blockIdx.x)];
    const int from = u.from + (a.layer0 + layer) * a.from_step, slot = u.slot + (a.layer0 + layer) * a.to_step;
    const int blk = u.pos0 / kPage + ((int)blockIdx.x - u.page0);
    const int j = (int)blockIdx.x - u.page0;
    const int entry = u.listed >> j & 1 ? a.pages[layer * a.n_listed + u.list0 + __popc(u.listed & ((1u << j) - 1))]
                                        : P.page_table[(size_t)slot * P.max_logical + blk];
    const int phys = entry & ~kNewPage;
    // a replay after the slot was reset: it has no such page
    if (entry < 0 || phys >= P.capacity)
        return;
    const int lo = max(u.pos0, blk * kPage), T = min(u.pos0 + u.n, (blk + 1) * kPage) - lo;
    const int off0 = lo - blk * kPage;
    const bool seals = h == 0 && off0 + T == kPage;
    if (seals)
        load_projection(P, seal);
    if (h == 0 && threadIdx.x == 0)
        publish(P, slot, u.pos0, u.n, blk, phys, entry & kNewPage);
    // eight elements of a token's row a thread, all tokens beside each other: one chain of
    // loads (page table, row), whatever the page takes
    const size_t head = (size_t)phys * P.n_kv + h;
    const int nw = hd / 8;
    for (int i = threadIdx.x; i < T * nw; i += 256) {
        const int t = i / nw, d = 8 * (i % nw), src = a.index[u.tok0 + lo - u.pos0 + t], off = off0 + t, so = src % kPage;
        const int page = min(max(P.page_table[(size_t)from * P.max_logical + src / kPage], 0), P.capacity - 1);
        const size_t sh = (size_t)page * P.n_kv + h, sr = (sh * kPage + so) * hd + d, dr = (head * kPage + off) * hd + d;
        if constexpr (KV8) {
            const uint2 k = *(const uint2 *)((const int8_t *)P.k + sr), v = *(const uint2 *)((const int8_t *)P.v + sr);
            if (d == 0) {
                P.k_scale[head * kPage + off] = P.k_scale[sh * kPage + so];
                P.v_scale[head * kPage + off] = P.v_scale[sh * kPage + so];
            }
            *(uint2 *)((int8_t *)P.k + dr) = k;
            *(uint2 *)((int8_t *)P.v + dr) = v;
        } else {
            const uint4 k = *(const uint4 *)((const uint16_t *)P.k + sr);
            uint16_t v[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = ((const uint16_t *)P.v)[(sh * hd + d + e) * kPage + so];
            *(uint4 *)((uint16_t *)P.k + dr) = k;
#pragma unroll
            for (int e = 0; e < 8; e++)
                ((uint16_t *)P.v)[(head * hd + d + e) * kPage + off] = v[e];
        }
    }
    if (seals)
        seal_written<!KV8>(P, seal, slot, blk, phys);
}

static int rope_append(be42_kv_pool *pool, const be42_kv_run *runs, int n_runs, const RopeIn &x, bool bf16, hipStream_t s)
{
    be42_kv_pool &P = *pool;
    std::vector<int> pages;
    const int rc = plan_runs(pool, "be42_rope_append", runs, n_runs, nullptr, pages);
    if (rc)
        return rc;
    RopeArgs a;
    a.n = a.n_pages = a.n_listed = 0;
    auto launch = [&]() {
        const int z = 1 + (x.n_heads / P.n_kv + 1) / 2;
        auto words = [&](auto kv8, auto act, auto hd) {
            hipLaunchKernelGGL((k_rope_append_words<decltype(kv8)::value, decltype(act)::value, decltype(hd)::value>),
                               dim3(a.n_pages, P.n_kv, z), dim3(256), 0, s, P, a, x);
        };
        auto pairs = [&](auto kv8, auto act, auto np) {
            hipLaunchKernelGGL((k_rope_append<decltype(kv8)::value, decltype(act)::value, decltype(np)::value>),
                               dim3(a.n_pages, P.n_kv), dim3(256), 0, s, P, a, x);
        };
        auto of_dim = [&](auto kv8, auto act) {
            if (x.rope_dim % 8 == 0 && P.head_dim == 64)
                words(kv8, act, std::integral_constant<int, 64>());
            else if (x.rope_dim % 8 == 0 && P.head_dim == 128)
                words(kv8, act, std::integral_constant<int, 128>());
            else if (x.rope_dim % 8 == 0 && P.head_dim == 256)
                words(kv8, act, std::integral_constant<int, 256>());
            else if (P.head_dim > 128)
                pairs(kv8, act, std::integral_constant<int, 2>());
            else
                pairs(kv8, act, std::integral_constant<int, 1>());
        };
        auto of_kind = [&](auto act) { P.kind == BE42_KV_INT8 ? of_dim(std::true_type(), act) : of_dim(std::false_type(), act); };
        bf16 ? of_kind(std::true_type()) : of_kind(std::false_type());
        a.n = a.n_pages = a.n_listed = 0;
    };
    // of `want` pages from `at` on, how many follow one another (and how)
    auto in_order = [&](size_t at, int want, int &step) {
        step = want > 1 ? pages[at + 1] - pages[at] : 0;
        int n = 1;
        if (step == 1 || step == -1)
            while (n < want && pages[at + n] - pages[at + n - 1] == step)
                n++;
        return n;
    };
    constexpr int kInOrder = 16;               // fewer are listed
    size_t at = 0;
    int tok = 0;
    for (int r = 0; r < n_runs; r++) {
        int pos = runs[r].pos0, left = runs[r].count;
        while (left) {
            const int want = (pos + left - 1) / kPage - pos / kPage + 1;
            int step, take = std::min(in_order(at, want, step), kMaxBlocks - a.n_pages);
            const bool listed = take < kInOrder;
            if (listed) {
                // up to where some follow one another, as many as the launch has room for
                const int room = std::min({want, kPiecePages - a.n_listed, kMaxBlocks - a.n_pages});
                for (step = 0; take < room;) {
                    int by;
                    const int n = in_order(at + take, want - take, by);
                    if (n >= kInOrder)
                        break;
                    take += n;
                }
                take = std::min(take, room);
            }
            if (a.n == kPieces || take <= 0) {
                launch();
                continue;
            }
            const int n = std::min(left, (pos / kPage + take) * kPage - pos);
            a.piece[a.n++] = {runs[r].slot, pos, n, tok, a.n_pages, listed ? a.n_listed : pages[at], step};
            if (listed) {
                std::copy_n(pages.begin() + at, take, a.pages + a.n_listed);
                a.n_listed += take;
            }
            a.n_pages += take;
            at += take;
            pos += n;
            tok += n;
            left -= n;
        }
    }
    if (a.n)
        launch();
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

static int kv_accept(be42_kv_pool *pool, const be42_kv_take *runs, int n_runs, const int *index, size_t n_index, int n_layers,
                     int from_step, int to_step, hipStream_t s)
{
    be42_kv_pool &P = *pool;
    std::vector<be42_kv_run> all;
    std::vector<int> from, pages, last(n_runs, -1);          // last: the largest token that a run names
    all.reserve((size_t)n_runs * n_layers);
    from.reserve((size_t)n_runs * n_layers);
    size_t at = 0;
    for (int r = 0; r < n_runs; r++) {
        BE42_CHECK(runs[r].count >= 0 && (size_t)runs[r].count <= n_index - at, "be42_kv_accept: %zu tokens, the runs have more", n_index);
        for (int i = 0; i < runs[r].count; i++, at++) {
            BE42_CHECK(index[at] >= 0, "be42_kv_accept: token %d", index[at]);
            last[r] = std::max(last[r], index[at]);
        }
    }
    BE42_CHECK(at == n_index, "be42_kv_accept: %zu tokens, the runs have %zu", n_index, at);
    for (int l = 0; l < n_layers; l++)
        for (int r = 0; r < n_runs; r++) {
            const long a = runs[r].from + (long)l * from_step, b = runs[r].to + (long)l * to_step;
            BE42_CHECK(a >= 0 && a < P.n_layers && b >= 0 && b < P.n_layers, "be42_kv_accept: slot %ld or %ld out of range", a, b);
            BE42_CHECK(last[r] < 0 || last[r] / kPage < slot_pages(pool, (int)a), "be42_kv_accept: token %d of slot %ld, which has %d pages",
                       last[r], a, slot_pages(pool, (int)a));
            from.push_back((int)a);
            all.push_back({(int)b, runs[r].pos0, runs[r].count});
        }
    const int rc = plan_runs(pool, "be42_kv_accept", all.data(), (int)all.size(), from.data(), pages);
    if (rc)
        return rc;
    const size_t per_layer = pages.size() / n_layers;        // positions are every layer's
    TakeArgs a;
    a.from_step = from_step;
    a.to_step = to_step;
    a.n = a.n_pages = 0;
    size_t first = 0;                                        // of the pages of a layer
    int toks = 0;
    auto launch = [&]() {
        // the pages that are new somewhere
        a.n_listed = 0;
        for (int i = 0; i < a.n; i++) {
            auto &u = a.piece[i];
            const int np = (i + 1 < a.n ? a.piece[i + 1].page0 : a.n_pages) - u.page0;
            u.list0 = (short)a.n_listed;
            u.listed = 0;
            for (int j = 0; j < np; j++)
                for (int l = 0; l < n_layers; l++)
                    if (pages[l * per_layer + first + u.page0 + j] & kNewPage) {
                        u.listed |= 1u << j;
                        a.n_listed++;
                        break;
                    }
        }
        const int most = std::min(a.n_listed ? kTakePages / a.n_listed : n_layers, kMaxGridYZ);
        for (int l = 0; l < n_layers; l += most) {
            const int n = std::min(most, n_layers - l);
            a.layer0 = l;
            int at = 0;
            for (int k = 0; a.n_listed && k < n; k++)
                for (int i = 0; i < a.n; i++)
                    for (int j = 0; a.piece[i].listed >> j; j++)
                        if (a.piece[i].listed >> j & 1)
                            a.pages[at++] = pages[(l + k) * per_layer + first + a.piece[i].page0 + j];
            const dim3 g(a.n_pages, P.n_kv, n);
            if (P.kind == BE42_KV_INT8)
                hipLaunchKernelGGL(k_kv_accept<true>, g, dim3(256), 0, s, P, a);
            else
                hipLaunchKernelGGL(k_kv_accept<false>, g, dim3(256), 0, s, P, a);
        }
        first += a.n_pages;
        a.n = a.n_pages = toks = 0;
    };
    at = 0;
    for (int r = 0; r < n_runs; r++) {
        int pos = runs[r].pos0, left = runs[r].count;
        while (left) {
            // as many tokens as the launch has room for; a piece ends with a page or
            // with its run
            int n = std::min(left, kTaken - toks);
            if (n < left)
                n = std::max((pos + n) / kPage * kPage - pos, 0);
            const int np = (pos + n - 1) / kPage - pos / kPage + 1;
            if (a.n == kTakes || n <= 0 || a.n_pages + np > kTakePages) {
                launch();
                continue;
            }
            a.piece[a.n++] = {runs[r].from, runs[r].to, pos, (short)n, (short)toks, (short)a.n_pages, 0, 0};
            std::copy_n(index + at, n, a.index + toks);
            a.n_pages += np;
            toks += n;
            at += n;
            pos += n;
            left -= n;
        }
    }
    if (a.n)
        launch();
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

}  // namespace be42

using namespace be42;

extern "C" int be42_rope_append(be42_kv_pool *pool, const be42_kv_run *runs, int n_runs, int n_tokens, const void *q,
                                int q_stride, int n_heads, const void *k, int k_stride, const void *v, int v_stride, int act_bf16,
                                const uint16_t *q_norm, const uint16_t *k_norm, float eps, const be42_rope *rope,
                                const int *positions, void *q_out, int q_out_stride, void *stream)
{
    BE42_CHECK(pool && (n_runs == 0 || runs), "be42_rope_append: null pointer");
    const be42_kv_pool &P = *pool;
    BE42_CHECK(n_runs >= 0 && n_tokens >= 0, "be42_rope_append: %d runs, %d tokens", n_runs, n_tokens);
    long tokens = 0;
    for (int r = 0; r < n_runs; r++)
        tokens += std::max(runs[r].count, 0);
    BE42_CHECK(tokens == n_tokens, "be42_rope_append: %d tokens, the runs have %ld", n_tokens, tokens);
    BE42_CHECK(tokens == 0 || (k && v), "be42_rope_append: null pointer");
    BE42_CHECK(n_heads >= 0 && n_heads % P.n_kv == 0 && (!tokens || (n_heads == 0) == (q == nullptr)),
               "be42_rope_append: %d query heads over %d kv heads", n_heads, P.n_kv);
    BE42_CHECK(!q || q_out, "be42_rope_append: null q_out");
    BE42_CHECK(P.n_kv <= kMaxGridYZ && n_heads / P.n_kv <= kMaxGridYZ, "be42_rope_append: %d query heads, %d kv heads", n_heads, P.n_kv);
    const long row = (long)P.n_kv * P.head_dim, qrow = (long)n_heads * P.head_dim;
    BE42_CHECK(k_stride >= row && v_stride >= row && (!q || (q_stride >= qrow && q_out_stride >= qrow)),
               "be42_rope_append: strides %d, %d, %d, %d of rows of %ld and %ld", q_stride, k_stride, v_stride,
               q_out_stride, qrow, row);
    BE42_CHECK(!q || q != q_out || q_stride == q_out_stride, "be42_rope_append: q in place at strides %d and %d",
               q_stride, q_out_stride);
    BE42_CHECK((!q_norm && !k_norm) || (eps >= 0.0f && eps < INFINITY), "be42_rope_append: eps %g", (double)eps);
    BE42_CHECK(!rope || (rope->len >= 0 && rope->dim >= 0 && rope->dim % 2 == 0 && rope->dim <= P.head_dim),
               "be42_rope_append: a rope of %d positions, %d elements (head_dim %d)", rope->len, rope->dim, P.head_dim);
    BE42_CHECK(!rope || !rope->len || !rope->dim || (rope->cos && rope->sin), "be42_rope_append: null table");
    BE42_CHECK(!(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & (act_bf16 ? 1 : 3)) &&
                   !(((uintptr_t)q_norm | (uintptr_t)k_norm) & 1) && !((uintptr_t)positions & 3) &&
                   (!rope || !(((uintptr_t)rope->cos | (uintptr_t)rope->sin) & 3)),
               "be42_rope_append: unaligned pointer");
    const RopeIn x = {q, k, v, q_out, q_norm, k_norm, rope ? rope->cos : nullptr, rope ? rope->sin : nullptr, positions,
                      (size_t)q_stride, (size_t)k_stride, (size_t)v_stride, (size_t)q_out_stride, n_heads,
                      rope ? rope->len : 0, rope ? rope->dim : 0, rope ? rope->interleaved : 0, eps};
    try {
        return rope_append(pool, runs, n_runs, x, act_bf16, as_stream(stream));
    } catch (const std::bad_alloc &) {
        set_error("be42_rope_append: out of host memory");
        return BE42_ENOMEM;
    }
}

extern "C" int be42_kv_accept(be42_kv_pool *pool, const be42_kv_take *runs, int n_runs, const int *index, int n_index,
                              int n_layers, int from_step, int to_step, void *stream)
{
    BE42_CHECK(pool && (n_runs == 0 || runs) && (n_index == 0 || index), "be42_kv_accept: null pointer");
    BE42_CHECK(n_runs >= 0 && n_index >= 0 && n_layers >= 0 && (long)n_runs * n_layers <= pool->n_layers,
               "be42_kv_accept: %d runs of %d layers over %d slots", n_runs, n_layers, pool->n_layers);
    BE42_CHECK(n_runs || !n_index, "be42_kv_accept: %d tokens without a run", n_index);
    BE42_CHECK(pool->n_kv <= kMaxGridYZ, "be42_kv_accept: %d kv heads", pool->n_kv);
    if (!n_runs || !n_layers)
        return BE42_OK;
    try {
        return kv_accept(pool, runs, n_runs, index, (size_t)n_index, n_layers, from_step, to_step, as_stream(stream));
    } catch (const std::bad_alloc &) {
        set_error("be42_kv_accept: out of host memory");
        return BE42_ENOMEM;
    }
}
