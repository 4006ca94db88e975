// score.hip -- log probabilities of given tokens, entropy and the top
// alternatives of logits rows.
//
// With z = (x - m) / T, m the row's maximum, s = sum e^z and t = sum z e^z:
//   log p(i) = z_i - log s,   H = log s - t / s.
// A row is cut into slices that one workgroup holds in registers, so that it
// is read once: each slice leaves its m, s, t and its top_k largest entries,
// and a second launch (none where a row is one slice) joins a row's slices.
#include <algorithm>
#include <cmath>

#include "be42_common.h"

namespace be42 {

constexpr int kTopMax = 64;
constexpr int kScoreT = 256, kScoreW = kScoreT / kWave;
constexpr int kScoreE = 32;                 // entries a thread holds
constexpr int kGroup = 8;                   // entries that are looked through together
constexpr int kSlice = kScoreT * kScoreE;
constexpr int kScoreCand = 512;             // candidates of a slice that are ranked together
constexpr int kJoinCand = 1024;             // of a row's slices

// One number per (value, id) that is larger for a larger value, then for a
// lower id: the value's bits as an order-preserving integer, then ~id.  -0 is
// taken for +0 and a NaN for -infinity.  No key is 0.
__device__ __forceinline__ uint32_t order_bits(float x)
{
    const uint32_t u = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_key(float x, int id)
{
    return (unsigned long long)order_bits(x) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(unsigned long long k)
{
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

struct ScoreArgs {
    const void *logits;
    size_t row_stride;
    float *lp, *entropy, *top_lp;
    int *top_ids;
    const int *tokens;
    int n_tokens, top_k, n, slices;
    float temp, c;                          // c = log2(e) / T: exponents are kept in base 2
    float4 *stats;                          // [rows][slices]: m, s, t (of base-2 exponents)
    unsigned long long *keys;               // [rows][slices][top_k], descending
};

template <bool BF16>
__device__ __forceinline__ float logit(const void *row, int i)
{
    return BF16 ? bf16_to_f32(((const uint16_t *)row)[i]) : ((const float *)row)[i];
}

template <bool BF16>
__device__ __forceinline__ const void *row_of(const ScoreArgs &a, int row)
{
    return (const char *)a.logits + (size_t)row * a.row_stride * (BF16 ? 2 : 4);
}

// What a row's sums say: log s is NaN for a row without a distribution (s is
// NaN where an entry was NaN or +infinity).
struct RowSums {
    double m, ls, H;
};
__device__ __forceinline__ RowSums row_sums(float m, double s, double t)
{
    const double ls = m == -INFINITY ? (double)NAN : log(s);
    return {m, ls, ls - t / s * 0.69314718055994530942};
}
__device__ __forceinline__ float log_prob(const ScoreArgs &a, const RowSums &r, float x)
{
    return r.ls != r.ls ? NAN : (float)(((double)x - r.m) / (double)a.temp - r.ls);
}

// the wave's largest value, in every lane (lane moves)
__device__ __forceinline__ float wave_top(float v)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_prefix_max(v)), 63));
}
template <int CTRL, int ROWMASK = 0xF>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v)
{
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWMASK, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_top_u(uint32_t v)
{
    v = dpp_max_u<0x111>(v);          // row_shr:1, 2, 4, 8
    v = dpp_max_u<0x112>(v);
    v = dpp_max_u<0x114>(v);
    v = dpp_max_u<0x118>(v);
    v = dpp_max_u<0x142, 0xA>(v);     // row_bcast:15 into rows 1, 3
    v = dpp_max_u<0x143, 0xC>(v);     // row_bcast:31 into rows 2, 3
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// One set of entries' m, s and t as they count under the maximum `top` of several.
__device__ __forceinline__ void rebase(const ScoreArgs &a, const float4 &p, float top, double &s, double &t)
{
    const float d = p.x == -INFINITY ? 0.0f : (p.x - top) * a.c, w = __builtin_amdgcn_exp2f(d);
    s = (double)w * p.y;
    t = (double)w * ((double)p.z + (double)fmaxf(d, -200.0f) * p.y);
}

// the given tokens and the entropy of a row
template <bool BF16>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int row, const RowSums &r, int tid, int threads)
{
    if (tid == 0 && a.entropy)
        a.entropy[row] = (float)r.H;
    for (int j = tid; j < a.n_tokens; j += threads) {
        const int id = a.tokens[(size_t)row * a.n_tokens + j];
        a.lp[(size_t)row * a.n_tokens + j] =
            log_prob(a, r, id >= 0 && id < a.n ? logit<BF16>(row_of<BF16>(a, row), id) : -INFINITY);
    }
}

__device__ __forceinline__ void write_top(const ScoreArgs &a, int row, const RowSums &r, int rank,
                                          unsigned long long key)
{
    a.top_ids[(size_t)row * a.top_k + rank] = key_id(key);
    a.top_lp[(size_t)row * a.top_k + rank] = log_prob(a, r, key_value(key));
}

__device__ __forceinline__ unsigned long long larger(unsigned long long p, unsigned long long q) { return p > q ? p : q; }

// Calls out(rank, key) for the k largest of n distinct keys in LDS: a key's
// rank is the number of larger ones.
template <class F>
__device__ __forceinline__ void rank_keys(const unsigned long long *cand, int n, int k, F &&out)
{
    for (int i = threadIdx.x; i < n; i += kScoreT) {
        const unsigned long long mine = cand[i];
        int rank = 0;
        for (int j = 0; j < n; j++)
            rank += cand[j] > mine;
        if (rank < k)
            out(rank, mine);
    }
}

// The same where there are too many keys to rank together: one after the
// other, best(last) being the thread's largest key below `last` (0: none).
template <class B, class F>
__device__ __forceinline__ void pull_keys(unsigned long long *sh, int k, B &&best, F &&out)
{
    unsigned long long last = ~0ull;
    for (int r = 0; r < k; r++) {
        unsigned long long b = best(last);
        for (int o = 32; o > 0; o >>= 1)
            b = larger(b, __shfl_xor(b, o, kWave));
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            sh[threadIdx.x >> 6] = b;
        __syncthreads();
        last = larger(larger(sh[0], sh[1]), larger(sh[2], sh[3]));
        if (threadIdx.x == 0)
            out(r, last);
        if (last == 0)
            last = 1;                       // nothing is left: the other ranks are 0 too
    }
}

// One slice of a row: block (row, slice).  The candidates of the slice's top_k
// are the entries not below a bound that at least top_k threads' maxima reach:
// the bound is bisected over the 256 maxima until few more than top_k do.
template <bool BF16>
__global__ __launch_bounds__(kScoreT) void k_score_slice(const ScoreArgs a)
{
    constexpr int VE = BF16 ? 8 : 4, U = kScoreE / VE;     // entries of a 16-byte word, words a thread
    __shared__ float4 part[kScoreW];
    __shared__ uint32_t tops[kScoreT];
    __shared__ unsigned long long cand[kScoreCand];
    __shared__ int n_cand;
    const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top_k;
    const void *xr = row_of<BF16>(a, row);
    // words lie on 16 bytes of memory: word w of the row holds entries VE w - off ..
    const int off = (int)((uintptr_t)xr / (BF16 ? 2 : 4) % VE);
    float x[kScoreE];
    const int first = slice * kSlice - off;
    auto id_of = [&](int i) { return first + (i / VE * kScoreT + tid) * VE + i % VE; };
    // every thread loads whole words, all in flight together (one that is not
    // wholly of the row reads the row's first whole word instead); entries of
    // the words that the row's ends cut are then loaded singly
    const bool inside = first >= 0 && first <= a.n - kSlice;
    const int whole = off ? VE - off : 0;
    auto is_whole = [&](int e0) { return inside || (e0 >= 0 && e0 <= a.n - VE); };
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int e0 = id_of(u * VE);
        w[u] = make_uint4(0, 0, 0, 0);
        if (inside || whole <= a.n - VE)
            w[u] = *(const uint4 *)((const char *)xr + (ptrdiff_t)(is_whole(e0) ? e0 : whole) * (BF16 ? 2 : 4));
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int e0 = id_of(u * VE);
        const uint32_t v[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (BF16) {
                x[u * VE + 2 * j] = __uint_as_float(v[j] << 16);
                x[u * VE + 2 * j + 1] = __uint_as_float(v[j] & 0xFFFF0000u);
            } else {
                x[u * VE + j] = __uint_as_float(v[j]);
            }
        }
        if (!inside && !is_whole(e0)) {
#pragma unroll
            for (int j = 0; j < VE; j++)
                x[u * VE + j] = -INFINITY;
            if (e0 > -VE && e0 < a.n) {
                float y[VE];
#pragma unroll
                for (int j = 0; j < VE; j++)
                    y[j] = logit<BF16>(xr, min(max(e0 + j, 0), a.n - 1));
#pragma unroll
                for (int j = 0; j < VE; j++)
                    x[u * VE + j] = e0 + j >= 0 && e0 + j < a.n ? y[j] : -INFINITY;
            }
        }
    }
    float mg[kScoreE / kGroup], mt = -INFINITY;     // maxima of groups of entries, and of all
#pragma unroll
    for (int g = 0; g < kScoreE / kGroup; g++) {
        mg[g] = x[g * kGroup];
#pragma unroll
        for (int i = 1; i < kGroup; i++)
            mg[g] = fmaxf(mg[g], x[g * kGroup + i]);
        mt = fmaxf(mt, mg[g]);
    }
    const float m = wave_top(mt), mf = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < kScoreE; i++) {
        // an entry of -infinity adds 0 to t, not 0 * -infinity
        const float z = (x[i] - mf) * a.c, e = __builtin_amdgcn_exp2f(z);
        s += e;
        t = __fmaf_rn(e, fmaxf(z, -200.0f), t);
    }
    s = wave_sum_dpp(s);
    t = wave_sum_dpp(t);
    if (lane == 0)
        part[wave] = make_float4(m, s, t, 0.0f);
    tops[tid] = order_bits(mt);
    if (tid == 0)
        n_cand = 0;
    __syncthreads();

    const float top = fmaxf(fmaxf(part[0].x, part[1].x), fmaxf(part[2].x, part[3].x));
    double bs = 0.0, bt = 0.0;
    const bool single = a.slices == 1;
    if (tid == 0 || single)
        for (int w = 0; w < kScoreW; w++) {
            double sw, tw;
            rebase(a, part[w], top, sw, tw);
            bs += sw;
            bt += tw;
        }
    RowSums r = {};
    if (single) {
        r = row_sums(top, bs, bt);
        write_row<BF16>(a, row, r, tid, kScoreT);
    } else if (tid == 0) {
        a.stats[blockIdx.x] = make_float4(top, (float)bs, (float)bt, 0.0f);
    }
    if (!k)
        return;

    // every wave bisects by itself: at least k maxima are >= lo, fewer than k >= hi
    uint32_t q[kScoreW], lo = ~0u, hi = 0;
#pragma unroll
    for (int w = 0; w < kScoreW; w++) {
        q[w] = tops[w * kWave + lane];
        lo = min(lo, q[w]);
        hi = max(hi, q[w]);
    }
    lo = ~wave_top_u(~lo);
    hi = wave_top_u(hi) + 1;
    int reach = kScoreT;
    while (hi - lo > 1 && reach > k + k / 4) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int w = 0; w < kScoreW; w++)
            c += __popcll(__ballot(q[w] >= mid));
        if (c >= k) {
            lo = mid;
            reach = c;
        } else {
            hi = mid;
        }
    }
    const float bound = key_value((unsigned long long)lo << 32);
#pragma unroll
    for (int g = 0; g < kScoreE / kGroup; g++)
        // (a group of nothing but NaN has the maximum NaN)
        if (!(mg[g] < bound))
#pragma unroll
            for (int i = g * kGroup; i < (g + 1) * kGroup; i++) {
                const int id = id_of(i);
                if (!(x[i] < bound) && (inside || (id >= 0 && id < a.n))) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kScoreCand)
                        cand[at] = order_key(x[i], id);
                }
            }
    __syncthreads();
    const int found = n_cand;
    auto out = [&](int rank, unsigned long long key) {
        if (single)
            write_top(a, row, r, rank, key);
        else
            a.keys[(size_t)blockIdx.x * k + rank] = key;
    };
    if (found <= kScoreCand) {
        rank_keys(cand, found, k, out);
        for (int i = found + tid; i < k; i += kScoreT)
            out(i, 0);                      // a row's last slice may hold fewer entries (a single one holds k)
        return;
    }
    // ties, or large entries of few threads
    pull_keys(cand, k,
              [&](unsigned long long last) {
                  unsigned long long best = 0;
#pragma unroll
                  for (int i = 0; i < kScoreE; i++) {
                      const int id = id_of(i);
                      const unsigned long long key = order_key(x[i], id);
                      best = id >= 0 && id < a.n && key < last ? larger(best, key) : best;
                  }
                  return best;
              },
              out);
}

// The slices of a row, one block a row.
template <bool BF16>
__global__ __launch_bounds__(kScoreT) void k_score_join(const ScoreArgs a)
{
    __shared__ double sums[2][kScoreW];
    __shared__ float maxs[kScoreW];
    __shared__ unsigned long long bounds[kScoreW], cand[kJoinCand];
    __shared__ int n_cand;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top_k;
    const float4 *st = a.stats + (size_t)row * a.slices;
    const unsigned long long *keys = a.keys + (size_t)row * a.slices * k;
    float m = -INFINITY;
    unsigned long long bound = 0;           // the best slice's last key: k keys of the row reach it
    for (int i = tid; i < a.slices; i += kScoreT) {
        m = fmaxf(m, st[i].x);
        if (k)
            bound = larger(bound, keys[(size_t)i * k + k - 1]);
    }
    m = wave_top(m);
    for (int o = 32; o > 0; o >>= 1)
        bound = larger(bound, __shfl_xor(bound, o, kWave));
    if (lane == 0) {
        maxs[wave] = m;
        bounds[wave] = bound;
    }
    if (tid == 0)
        n_cand = 0;
    __syncthreads();
    m = fmaxf(fmaxf(maxs[0], maxs[1]), fmaxf(maxs[2], maxs[3]));
    bound = larger(larger(bounds[0], bounds[1]), larger(bounds[2], bounds[3]));
    double s = 0.0, t = 0.0;
    for (int i = tid; i < a.slices; i += kScoreT) {
        double si, ti;
        rebase(a, st[i], m, si, ti);
        s += si;
        t += ti;
    }
    for (int o = 32; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, kWave);
        t += __shfl_xor(t, o, kWave);
    }
    if (lane == 0) {
        sums[0][wave] = s;
        sums[1][wave] = t;
    }
    const int all = a.slices * k;
    for (int i = tid; i < all; i += kScoreT) {
        const unsigned long long key = keys[i];
        if (key && key >= bound) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kJoinCand)
                cand[at] = key;
        }
    }
    __syncthreads();
    const RowSums r = row_sums(m, (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]),
                               (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]));
    write_row<BF16>(a, row, r, tid, kScoreT);
    if (!k)
        return;
    const int found = n_cand;
    auto out = [&](int rank, unsigned long long key) { write_top(a, row, r, rank, key); };
    if (found <= kJoinCand)
        rank_keys(cand, found, k, out);
    else
        pull_keys(cand, k,
                  [&](unsigned long long last) {
                      unsigned long long best = 0;
                      for (int i = tid; i < all; i += kScoreT)
                          best = keys[i] < last ? larger(best, keys[i]) : best;
                      return best;
                  },
                  out);
}

// Slices of a row of n entries, whose first word may begin before it.
static long score_slices(int n) { return ((long)n + 7 + kSlice - 1) / kSlice; }

}  // namespace be42

using namespace be42;

extern "C" size_t be42_logprobs_workspace_bytes(int n, int rows, int top_k)
{
    if (n <= 0 || rows <= 0 || top_k < 0 || top_k > kTopMax || top_k > n)
        return 0;
    const size_t per = (size_t)rows * score_slices(n);
    return per * (sizeof(float4) + top_k * sizeof(unsigned long long));
}

extern "C" int be42_logprobs(float *logprobs, float *entropy, int *top_ids, float *top_logprobs, const void *logits,
                             int logits_bf16, int row_stride, int n, int rows, float temp, const int *tokens,
                             int n_tokens, int top_k, void *workspace, size_t workspace_bytes, void *stream)
{
    BE42_CHECK(n > 0 && n <= 1 << 30 && rows >= 0 && row_stride >= n, "be42_logprobs: %d rows of %d at stride %d", rows, n, row_stride);
    BE42_CHECK(temp > 0.0f && std::isfinite(temp) && std::isfinite(1.0f / temp), "be42_logprobs: temperature %g",
               (double)temp);
    if (rows == 0)
        return BE42_OK;
    BE42_CHECK(logits, "be42_logprobs: null pointer");
    BE42_CHECK(n_tokens >= 0 && (n_tokens == 0 || (tokens && logprobs)), "be42_logprobs: %d tokens a row, %s", n_tokens,
               tokens ? "no logprobs" : "no ids");
    BE42_CHECK(top_k >= 0 && top_k <= kTopMax && top_k <= n, "be42_logprobs: top %d of %d (at most %d)", top_k, n,
               kTopMax);
    BE42_CHECK(top_k == 0 || (top_ids && top_logprobs), "be42_logprobs: top %d without arrays", top_k);
    BE42_CHECK(n_tokens || top_k || entropy, "be42_logprobs: nothing asked for");
    BE42_CHECK(!((uintptr_t)logits & (logits_bf16 ? 1 : 3)), "be42_logprobs: unaligned logits");
    const size_t need = be42_logprobs_workspace_bytes(n, rows, top_k);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_logprobs: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    const long slices = score_slices(n), blocks = slices * rows;
    BE42_CHECK(blocks <= 0x7FFFFFFF, "be42_logprobs: %d rows of %d", rows, n);
    ScoreArgs a = {logits, (size_t)row_stride, logprobs, entropy, top_logprobs, top_ids, tokens, n_tokens, top_k, n,
                   (int)slices, temp, (float)(1.44269504088896340736 / (double)temp)};
    hipStream_t s = as_stream(stream);
    if (slices > 1) {
        if (!workspace)
            workspace = be42::workspace(need, s);
        if (!workspace)
            return BE42_ENOMEM;
        a.stats = (float4 *)workspace;
        a.keys = (unsigned long long *)(a.stats + blocks);
    }
    const dim3 g((unsigned)blocks), t(kScoreT);
    if (logits_bf16)
        hipLaunchKernelGGL(k_score_slice<true>, g, t, 0, s, a);
    else
        hipLaunchKernelGGL(k_score_slice<false>, g, t, 0, s, a);
    if (slices > 1) {
        if (logits_bf16)
            hipLaunchKernelGGL(k_score_join<true>, dim3(rows), t, 0, s, a);
        else
            hipLaunchKernelGGL(k_score_join<false>, dim3(rows), t, 0, s, a);
    }
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
