// score.hip -- log probabilities of given tokens, entropy and the top
// alternatives of logits rows.
//
// With exponents to base 2, c = log2(e) / T, z = (x - m) c for the largest entry
// m, s = sum 2^z and t = sum 2^z z:
//   log p(i) = ln 2 (z_i - log2 s),   H = ln 2 (log2 s - t / s).
// A workgroup reads a run of a row once.  Its waves take chunks of 64 x 8 words
// of 16 bytes in turn and keep s and t of each lane and the largest entries so
// far; they share a bound that top_k entries are known to reach, so that few
// entries past the first chunks are looked at again.  A second launch (none
// where a row is one run) joins the runs of a row.  Sums of lanes, waves and
// runs are joined in 64 bits.
//
// Instruction bound for bf16 (an entry costs a shift or mask, half a maximum, a
// difference, a product, the exponential -- four times as long as another
// instruction --, an add and an fma): 2000 x 128256 with five alternatives 109 us,
// 4.7 TB/s.  Memory bound for fp32: 1000 x 128256 98 us without alternatives, 5.2
// TB/s.  One row of 128256 takes 11.2 us, two launches of which the loads are 2.4.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "be42_common.h"

namespace be42 {

constexpr int kTopMax = 64;
constexpr int kScoreW = 4;                  // waves of a workgroup, each on its own
constexpr int kScoreWide = 8;               // of one that has a row to itself
constexpr int kScoreU = 8;                  // words of 16 bytes a lane holds
constexpr int kChunkBytes = kWave * kScoreU * 16;
constexpr int kTopCap = 576;                // a wave's candidates: top_k, and the entries of 64 words
constexpr int kJoinKeys = 8;                // keys of the runs that a lane of the joining wave holds

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
__device__ __forceinline__ unsigned long long larger(unsigned long long p, unsigned long long q) { return p > q ? p : q; }

// s and t of a set of entries and m c, which they count from (-infinity: no
// entry but -infinity)
struct Sums {
    double ref;
    float s, t;
};

struct ScoreArgs {
    const void *logits;
    size_t row_stride;
    float *lp, *entropy, *top_lp;
    int *top_ids;
    const int *tokens;
    int n_tokens, top_k, n;
    float c;
    int chunks, per, runs;                  // chunks of a row, of a run, runs of a row
    Sums *sums;                             // [rows][runs]
    unsigned long long *keys;               // [rows][runs][top_k], descending, 0 past the last entry
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

// What a row's sums say: NaN for a row without a distribution (s is NaN or
// infinite where an entry was NaN or +infinity).
struct RowSums {
    double ref, ls, H;                      // log p(x) = ln 2 (x c - ref - ls)
};
__device__ __forceinline__ RowSums row_sums(double ref, double s, double t)
{
    const double ls = ref > -INFINITY && s < INFINITY ? log2(s) : (double)NAN;
    return {ref, ls, (ls - t / s) * 0.69314718055994530942};
}
// (the reference first: ls would be lost beside one past 2^53 of it)
__device__ __forceinline__ float log_prob(const ScoreArgs &a, const RowSums &r, float x)
{
    return r.ls != r.ls ? NAN : (float)((((double)x * (double)a.c - r.ref) - r.ls) * 0.69314718055994530942);
}

// s and t under the reference `top` >= p.ref
__device__ __forceinline__ void rebase(const Sums &p, double top, double &s, double &t)
{
    const double d = p.ref == -INFINITY ? 0.0 : p.ref - top;
    const double w = (double)__builtin_amdgcn_exp2f((float)d);
    s = w * p.s;
    t = w * ((double)p.t + fmax(d, -1000.0) * p.s);
}

// joins the lanes' sums; every lane gets the reference and the sums
__device__ __forceinline__ void join_lanes(const Sums &mine, double &ref, double &s, double &t)
{
    ref = wave_max_d(mine.ref);
    rebase(mine, ref, s, t);
    s = wave_sum_d(s);
    t = wave_sum_d(t);
}

// the logit of given token j of a row (one outside the row: -infinity)
template <bool BF16>
__device__ __forceinline__ float given_logit(const ScoreArgs &a, int row, int j)
{
    const int id = a.tokens[(size_t)row * a.n_tokens + j];
    return id >= 0 && id < a.n ? logit<BF16>(row_of<BF16>(a, row), id) : -INFINITY;
}

// the given tokens (x0: the logit of token `lane`) and the entropy of a row, by one wave
template <bool BF16>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int row, const RowSums &r, int lane, float x0)
{
    if (lane == 0 && a.entropy)
        a.entropy[row] = (float)r.H;
    if (lane < a.n_tokens)
        a.lp[(size_t)row * a.n_tokens + lane] = log_prob(a, r, x0);
    for (int j = kWave + lane; j < a.n_tokens; j += kWave)
        a.lp[(size_t)row * a.n_tokens + j] = log_prob(a, r, given_logit<BF16>(a, row, j));
}

__device__ __forceinline__ void write_top(const ScoreArgs &a, int row, const RowSums &r, int rank,
                                          unsigned long long key)
{
    a.top_ids[(size_t)row * a.top_k + rank] = key_id(key);
    a.top_lp[(size_t)row * a.top_k + rank] = log_prob(a, r, key_value(key));
}

// LDS written by other lanes of the wave before this point may be read after it
__device__ __forceinline__ void wave_lds()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// Calls out(rank, key) for the k largest of the n <= N * 64 distinct keys that a
// wave keeps in LDS (with room for 8 more): a key's rank is the number of larger
// ones.  All keys are read before the first call.
template <int N, class F>
__device__ __forceinline__ void rank_keys(unsigned long long *cand, int n, int k, int lane, F &&out)
{
    if (lane < 8)
        cand[n + lane] = 0;
    wave_lds();
    unsigned long long mine[N];
    int rank[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        mine[i] = lane + i * kWave < n ? cand[lane + i * kWave] : 0;
        rank[i] = mine[i] ? 0 : k;
    }
    for (int j = 0; j < n; j += 8)
#pragma unroll
        for (int x = 0; x < 8; x++) {
            const unsigned long long other = cand[j + x];
#pragma unroll
            for (int i = 0; i < N; i++)
                rank[i] += other > mine[i];
        }
    wave_lds();
#pragma unroll
    for (int i = 0; i < N; i++)
        if (rank[i] < k)
            out(rank[i], mine[i]);
    wave_lds();
}

// A wave's run of a row.  Places past the row's ends are set to -infinity, which
// adds nothing to the sums under any reference and temperature (any number does
// beside a lane whose own entries lie below it), and are left out of the maxima.
template <bool BF16>
struct Run {
    static constexpr int VE = BF16 ? 8 : 4;    // entries of a word
    static constexpr int kEntries = kWave * kScoreU * VE;
    const void *xr;
    int n, off, lane;
    // words lie on 16 bytes of memory: word w of the row holds entries VE w - off ..
    __device__ __forceinline__ Run(const ScoreArgs &a, int row, int ln) : xr(row_of<BF16>(a, row)), n(a.n), lane(ln)
    {
        off = (int)((uintptr_t)xr / (BF16 ? 2 : 4) % VE);
    }
    __device__ __forceinline__ int id(int chunk, int u, int j) const
    {
        return chunk * kEntries - off + (u * kWave + lane) * VE + j;
    }
    __device__ __forceinline__ bool inside(int chunk) const
    {
        return chunk * kEntries - off >= 0 && chunk * kEntries - off <= n - kEntries;
    }
    // All words in flight together.  One that is not wholly of the row reads the
    // row's first whole word instead; entries of words that the row's ends cut
    // are then loaded singly.
    __device__ __forceinline__ void load(int chunk, uint4 (&w)[kScoreU]) const
    {
        const char *base = (const char *)xr;
        if (inside(chunk)) {
#pragma unroll
            for (int u = 0; u < kScoreU; u++)
                w[u] = *(const uint4 *)(base + (ptrdiff_t)id(chunk, u, 0) * (BF16 ? 2 : 4));
            return;
        }
        const int whole = off ? VE - off : 0;
        auto is_whole = [&](int e0) { return e0 >= 0 && e0 <= n - VE; };
#pragma unroll
        for (int u = 0; u < kScoreU; u++) {
            const int e0 = id(chunk, u, 0);
            w[u] = make_uint4(0, 0, 0, 0);
            if (whole <= n - VE)
                w[u] = *(const uint4 *)(base + (ptrdiff_t)(is_whole(e0) ? e0 : whole) * (BF16 ? 2 : 4));
        }
        constexpr uint32_t none = BF16 ? 0xFF80FF80u : 0xFF800000u;
#pragma unroll
        for (int u = 0; u < kScoreU; u++) {
            const int e0 = id(chunk, u, 0);
            if (is_whole(e0))
                continue;
            w[u] = make_uint4(none, none, none, none);
            if (e0 > -VE && e0 < n) {
                uint32_t y[VE], z[4];
#pragma unroll
                for (int j = 0; j < VE; j++)
                    y[j] = __float_as_uint(logit<BF16>(xr, min(max(e0 + j, 0), n - 1)));
#pragma unroll
                for (int j = 0; j < VE; j++)
                    y[j] = e0 + j >= 0 && e0 + j < n ? y[j] : BF16 ? none & 0xFFFF0000u : none;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    z[j] = BF16 ? y[2 * j % VE] >> 16 | y[(2 * j + 1) % VE] : y[j];
                w[u] = make_uint4(z[0], z[1], z[2], z[3]);
            }
        }
    }
    // entry j of a word; of a bf16 pair's upper entry, `raw` leaves the lower one's bits behind it
    static __device__ __forceinline__ float entry(const uint4 &v, int j, bool raw = false)
    {
        const int at = BF16 ? j / 2 : j;
        const uint32_t part = at == 0 ? v.x : at == 1 ? v.y : at == 2 ? v.z : v.w;
        return __uint_as_float(!BF16 || (raw && (j & 1)) ? part : j & 1 ? part & 0xFFFF0000u : part << 16);
    }
    // Maxima of a lane's words, and of all of them; a NaN counts as -infinity.
    // The bits behind a bf16 pair's upper entry do not change which entry is the
    // largest, but make an infinity a NaN.  So a maximum that keeps NaN is taken
    // first, and once more with care where it finds one.
    __device__ __forceinline__ float tops(int chunk, const uint4 (&w)[kScoreU], float (&mg)[kScoreU]) const
    {
        float top = -INFINITY;
        bool fine = inside(chunk);
        if (fine) {
#pragma unroll
            for (int u = 0; u < kScoreU; u++) {
                mg[u] = entry(w[u], 0, true);
#pragma unroll
                for (int j = 1; j < VE; j++)
                    mg[u] = __builtin_elementwise_maximum(mg[u], entry(w[u], j, true));
                top = __builtin_elementwise_maximum(top, mg[u]);
            }
            fine = !__any(top != top);
        }
        if (fine) {
#pragma unroll
            for (int u = 0; u < (BF16 ? kScoreU : 0); u++)
                mg[u] = __uint_as_float(__float_as_uint(mg[u]) & 0xFFFF0000u);
            return BF16 ? __uint_as_float(__float_as_uint(top) & 0xFFFF0000u) : top;
        }
        top = -INFINITY;
#pragma unroll
        for (int u = 0; u < kScoreU; u++) {
            mg[u] = -INFINITY;
#pragma unroll
            for (int j = 0; j < VE; j++) {
                const float x = entry(w[u], j);
                mg[u] = x > mg[u] && (unsigned)id(chunk, u, j) < (unsigned)n ? x : mg[u];
            }
            top = fmaxf(top, mg[u]);
        }
        return top;
    }
};

// Makes the compiler take a chunk's words apart again at their next use: kept
// apart, 64 bf16 entries a lane take 165 registers.
__device__ __forceinline__ void keep_packed(uint4 (&w)[kScoreU])
{
#pragma unroll
    for (int u = 0; u < kScoreU; u++)
        asm volatile("" : "+v"(w[u].x), "+v"(w[u].y), "+v"(w[u].z), "+v"(w[u].w));
}

// The largest entries of a wave's chunks, so far, in the wave's part of LDS: keys
// of entries, words that have yet to be looked through, and a bound that top_k
// entries of the run are known to reach, shared by the workgroup's waves as the
// order bits of a value.  (They read and raise it without waiting for each
// other: which entries are looked at depends on that, which are found does not.)
// Only words are noted where they are seen, and read again in batches of 64:
// looking into a word's entries there and then kept 64 bf16 entries apart in
// 207 registers (2000 rows of 128256 with 5 alternatives 300 us).
struct TopKeys {
    unsigned long long *cand, least;        // candidates have keys > least
    int *words;                             // indexes of 16-byte words of the row
    uint32_t *shared;
    int n, n_words;
    __device__ __forceinline__ float bound() const
    {
        // (the lowest order bits of a number are those of -infinity)
        return (uint32_t)(least >> 32) < 0x007FFFFFu ? -INFINITY : key_value(least);
    }
};

// the wave's largest number, in every lane
__device__ __forceinline__ uint32_t wave_top(uint32_t v)
{
    auto step = [&](auto ctrl, auto rows) {
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());       // row_shr:1, 2, 4, 8
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());       // row_bcast:15, 31
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The largest value, or one with few more above, that at least k <= 64 of the
// lanes' N order bits reach (0: fewer than k are there).  Looked for between the
// lanes' largest and the least of them, where k lanes have one: from 0 on the
// search took 1.7 us of the joining launch.
template <int N>
__device__ __forceinline__ uint32_t reached(const uint32_t (&q)[N], int k)
{
    uint32_t mine = q[0];
#pragma unroll
    for (int i = 1; i < N; i++)
        mine = max(mine, q[i]);
    const uint32_t top = wave_top(mine), least = ~wave_top(~(mine ? mine : top));
    uint32_t lo = __popcll(__ballot(mine != 0)) >= k ? least : 0, hi = top + 1;
    int reach = N * kWave;                  // at least k are >= lo, fewer than k >= hi
    while (hi - lo > 1 && reach > k + k / 4) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
            c += __popcll(__ballot(q[i] >= mid));
        if (c >= k) {
            lo = mid;
            reach = c;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ __forceinline__ void raise(TopKeys &T, unsigned long long least, int lane)
{
    if (least <= T.least)
        return;
    T.least = least;
    if (lane == 0)
        atomicMax(T.shared, (uint32_t)(least >> 32));
}

// leaves the k largest
__device__ __forceinline__ void compress(TopKeys &T, int k, int lane)
{
    auto keep = [&](int rank, unsigned long long key) { T.cand[rank] = key; };
    if (T.n <= kWave)
        rank_keys<1>(T.cand, T.n, k, lane, keep);
    else if (T.n <= 4 * kWave)
        rank_keys<4>(T.cand, T.n, k, lane, keep);
    else
        rank_keys<kTopCap / kWave>(T.cand, T.n, k, lane, keep);
    T.n = min(T.n, k);
    if (T.n == k)
        raise(T, T.cand[k - 1], lane);
}

// notes the words of a chunk that hold entries at the bound or above
__device__ __forceinline__ void note(TopKeys &T, int chunk, const float (&mg)[kScoreU], float top, int k, int lane)
{
    T.least = larger(T.least, (unsigned long long)*(volatile uint32_t *)T.shared << 32);
    float bound = T.bound();
    const int reach = __popcll(__ballot(!(top < bound)));
    if (!reach)
        return;
    if (reach > k + k / 4) {                // the first chunk, rising entries
        const uint32_t q[1] = {order_bits(top)};
        raise(T, (unsigned long long)reached<1>(q, k) << 32, lane);
        bound = T.bound();
    }
#pragma unroll
    for (int u = 0; u < kScoreU; u++) {
        const bool in = !(mg[u] < bound);
        const unsigned long long who = __ballot(in);
        if (in)
            T.words[T.n_words + __popcll(who & ((1ull << lane) - 1))] = (chunk * kScoreU + u) * kWave + lane;
        T.n_words += __popcll(who);
    }
}

// looks through the noted words
template <bool BF16>
__device__ __forceinline__ void look(TopKeys &T, const Run<BF16> &run, int k, int lane)
{
    constexpr int VE = Run<BF16>::VE;
    wave_lds();
    for (int i0 = 0; i0 < T.n_words; i0 += kWave) {
        const int first = i0 + lane < T.n_words ? T.words[i0 + lane] * VE - run.off : run.n;
        float x[VE];
#pragma unroll
        for (int j = 0; j < VE; j++)
            x[j] = logit<BF16>(run.xr, min(max(first + j, 0), run.n - 1));
#pragma unroll
        for (int j = 0; j < VE; j++) {
            const unsigned long long key = (unsigned)(first + j) < (unsigned)run.n ? order_key(x[j], first + j) : 0;
            const unsigned long long who = __ballot(key > T.least);
            if (key > T.least)
                T.cand[T.n + __popcll(who & ((1ull << lane) - 1))] = key;
            T.n += __popcll(who);
        }
        if (T.n > k)
            compress(T, k, lane);
    }
    T.n_words = 0;
}

// Calls out(rank, key) for the k largest of the keys that the lanes hold (0: none),
// all distinct: those that reach a value which few more than k do are ranked.
// Returns how many there were.
template <int N, class F>
__device__ __forceinline__ int select_keys(const unsigned long long (&key)[N], unsigned long long *cand, int k, int lane, F &&out)
{
    uint32_t q[N];
#pragma unroll
    for (int x = 0; x < N; x++)
        q[x] = (uint32_t)(key[x] >> 32);
    const uint32_t lo = reached<N>(q, k);
    int found = 0;
#pragma unroll
    for (int x = 0; x < N; x++) {
        const bool in = key[x] && q[x] >= lo;
        const unsigned long long who = __ballot(in);
        if (in)
            cand[found + __popcll(who & ((1ull << lane) - 1))] = key[x];
        found += __popcll(who);
    }
    if (found <= kWave)
        rank_keys<1>(cand, found, k, lane, out);
    else
        rank_keys<N>(cand, found, k, lane, out);
    return found;
}

// block: (row, run)
template <bool BF16, int W>
__global__ __launch_bounds__(kWave *W) void k_score_run(const ScoreArgs a)
{
    __shared__ unsigned long long lds[W][kTopCap + 8];
    __shared__ int words[W][(kScoreU + 1) * kWave];
    __shared__ unsigned long long merged[W * kTopMax + 8];
    __shared__ Sums sums[W];
    __shared__ uint32_t shared;
    constexpr bool AHEAD = W > 4;            // few rows: a wave loads the next chunk beside this one
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k = a.top_k;
    const int row = (int)(blockIdx.x / (unsigned)a.runs), part = (int)(blockIdx.x % (unsigned)a.runs);
    const int c0 = part * a.per, c1 = min(c0 + a.per, a.chunks);
    const Run<BF16> run(a, row, lane);
    const bool single = a.runs == 1;
    const float x0 = single && wave == 0 && lane < a.n_tokens ? given_logit<BF16>(a, row, lane) : 0.0f;
    if (threadIdx.x == 0)
        shared = 0;
    __syncthreads();
    TopKeys T = {lds[wave], 0, words[wave], &shared, 0, 0};
    uint4 w[kScoreU], next[kScoreU];
    float mg[kScoreU];
    // each lane by itself: its largest entry and its sums, z = (x - m) c
    float m = -INFINITY, ref = 0.0f, s = 0.0f, t = 0.0f;
    if (AHEAD && c0 + wave < c1)
        run.load(c0 + wave, next);
    for (int c = c0 + wave; c < c1; c += W) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int u = 0; u < kScoreU; u++)
                w[u] = next[u];
            if (c + W < c1)
                run.load(c + W, next);
        } else {
            run.load(c, w);
        }
        const float top = run.tops(c, w, mg);
        keep_packed(w);
        if (__any(top > m)) {
            const float r2 = top > m ? top : ref, d = m == -INFINITY ? 0.0f : (ref - r2) * a.c;
            const float f = __builtin_amdgcn_exp2f(d);
            t = f * __fmaf_rn(fmaxf(d, -200.0f), s, t);
            s *= f;
            ref = r2;
            m = fmaxf(m, top);
        }
        // -infinity (0 * -infinity in t) takes a second, careful pass, with exponents
        // held where they underflow; a chunk that the row's ends cut, whose filling
        // is that, goes straight there
        bool careful = !run.inside(c);
        if (!careful) {
            const float s0 = s, t0 = t;
#pragma unroll
            for (int u = 0; u < kScoreU; u++)
#pragma unroll
                for (int j = 0; j < Run<BF16>::VE; j++) {
                    const float z = (Run<BF16>::entry(w[u], j) - ref) * a.c, e = __builtin_amdgcn_exp2f(z);
                    s += e;
                    t = __fmaf_rn(e, z, t);
                }
            keep_packed(w);
            careful = __any(!(fabsf(t) < INFINITY));
            if (careful) {
                s = s0;
                t = t0;
            }
        }
        if (careful) {
#pragma unroll
            for (int u = 0; u < kScoreU; u++)
#pragma unroll
                for (int j = 0; j < Run<BF16>::VE; j++) {
                    const float z = (Run<BF16>::entry(w[u], j) - ref) * a.c, e = __builtin_amdgcn_exp2f(z);
                    s += e;
                    t = __fmaf_rn(e, fmaxf(z, -200.0f), t);
                }
            keep_packed(w);
        }
        if (k) {
            note(T, c, mg, top, k, lane);
            if (T.n_words >= kWave || c + W >= c1)
                look<BF16>(T, run, k, lane);
        }
    }
    const Sums mine = {(double)m * (double)a.c, s, t};
    double rs, ss, tt;
    join_lanes(mine, rs, ss, tt);
    if (lane == 0)
        sums[wave] = {rs, (float)ss, (float)tt};
    if (lane < k)
        merged[wave * k + lane] = lane < T.n ? T.cand[lane] : 0;
    __syncthreads();
    if (wave)
        return;
    join_lanes(lane < W ? sums[lane] : Sums{-INFINITY, 0.0f, 0.0f}, rs, ss, tt);
    RowSums r = {};
    if (single) {
        r = row_sums(rs, ss, tt);
        write_row<BF16>(a, row, r, lane, x0);
    } else if (lane == 0) {
        a.sums[blockIdx.x] = {rs, (float)ss, (float)tt};
    }
    if (!k)
        return;
    if (!single && lane < k)
        a.keys[(size_t)blockIdx.x * k + lane] = 0;      // a row's last run may hold fewer than k entries
    auto out = [&](int rank, unsigned long long key) {
        if (single)
            write_top(a, row, r, rank, key);
        else
            a.keys[(size_t)blockIdx.x * k + rank] = key;
    };
    unsigned long long key[W];
#pragma unroll
    for (int x = 0; x < W; x++)
        key[x] = x * kWave + lane < W * k ? merged[x * kWave + lane] : 0;
    wave_lds();
    select_keys<W>(key, merged, k, lane, out);
}

// The runs of a row, one wave a row.
template <bool BF16>
__global__ __launch_bounds__(kWave) void k_score_join(const ScoreArgs a)
{
    __shared__ unsigned long long cand[kJoinKeys * kWave + 8];
    const int row = blockIdx.x, lane = threadIdx.x, k = a.top_k, all = a.runs * k;
    const Sums *st = a.sums + (size_t)row * a.runs;
    const unsigned long long *keys = a.keys + (size_t)row * all;
    // a chain of dependent loads would be most of a short call: what the first
    // 64 runs, 512 keys and 64 tokens need is asked for at once
    Sums mine = {-INFINITY, 0.0f, 0.0f};
    if (lane < a.runs)
        mine = st[lane];
    unsigned long long key[kJoinKeys];
#pragma unroll
    for (int x = 0; x < kJoinKeys; x++)
        key[x] = x * kWave + lane < all ? keys[x * kWave + lane] : 0;
    const float x0 = lane < a.n_tokens ? given_logit<BF16>(a, row, lane) : 0.0f;

    for (int i = lane + kWave; i < a.runs; i += kWave) {
        const Sums b = st[i];
        const double top = fmax(mine.ref, b.ref);
        double s, t, s2, t2;
        rebase(mine, top, s, t);
        rebase(b, top, s2, t2);
        mine = {top, (float)(s + s2), (float)(t + t2)};
    }
    double ref, s, t;
    join_lanes(mine, ref, s, t);
    const RowSums r = row_sums(ref, s, t);
    write_row<BF16>(a, row, r, lane, x0);
    if (!k)
        return;
    // the keys that reach a value which few more than k do; keys past those that
    // the lanes hold replace them in turn
    for (int i0 = kJoinKeys * kWave;; i0 += (kJoinKeys - 1) * kWave) {
        const bool last = i0 >= all;
        auto out = [&](int rank, unsigned long long kk) {
            if (last)
                write_top(a, row, r, rank, kk);
            else
                cand[rank] = kk;
        };
        const int found = select_keys<kJoinKeys>(key, cand, k, lane, out);
        if (last)
            return;
        key[0] = lane < min(found, k) ? cand[lane] : 0;
#pragma unroll
        for (int x = 1; x < kJoinKeys; x++) {
            const int i = i0 + (x - 1) * kWave + lane;
            key[x] = i < all ? keys[i] : 0;
        }
        wave_lds();
    }
}

// How a row of n entries is cut: chunks (the first word may begin `before`
// entries before the row), chunks of a run, runs, and the waves of a workgroup.
// Up to 256 rows, a workgroup of eight waves takes a whole row where that has up
// to 80 K entries, or where the rows come near to filling the chip (fp32, top 5, in
// us: 1 x 32000 8.6, cut 9.6; 1 x 64000 11.4, cut 9.6 and a second launch's 4 us of
// the caller's time; 1 x 128256 17, cut 10.4; 64 x 128256 19.4, cut 16.6; 120 x
// 128256 19.4, cut 23.5; 200 x 32000 12.7, cut 16.0; in a captured graph, where a
// launch costs no caller's time, 1 x 32000 9.6, cut 10.5, 64 x 32000 10.4 and 12.0, 64
// x 64000 13.7 and 14.0, but 1 x 64000 12.2 and 10.1); rows of up to four
// chunks do with four waves (200 x 8000 8.3, eight 8.7).  Other rows are cut
// until there are four workgroups a CU; a run has at least a chunk for each wave,
// and four where the rows alone fill the chip, since joining runs costs a launch
// of 4 us (333 x 32003 without alternatives 14.3 uncut).
static void cut_row(int n, int before, int rows, bool bf16, long *chunks, long *per, long *runs, int *waves)
{
    const long entries = kChunkBytes / (bf16 ? 2 : 4);
    *chunks = ((long)n + before + entries - 1) / entries;
    const bool whole = rows <= 256 && *chunks > kScoreW && (*chunks * entries <= 80 * 1024 || rows > 96);
    *waves = whole ? kScoreWide : kScoreW;
    const long least = rows >= 256 ? 4 * kScoreW : kScoreW;
    *runs = whole ? 1 : std::min((*chunks + least - 1) / least, (1024 + (long)rows - 1) / rows);
    *per = (*chunks + *runs - 1) / *runs;
    *runs = (*chunks + *per - 1) / *per;
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_logprobs_workspace_bytes(int n, int rows, int top_k)
{
    if (n <= 0 || rows <= 0 || top_k < 0 || top_k > kTopMax || top_k > n)
        return 0;
    size_t most = 0;                        // of either type
    for (int i = 0; i < 4; i++) {           // and alignment
        long chunks, per, runs;
        int waves;
        cut_row(n, i & 1 ? 7 : 0, rows, i >> 1, &chunks, &per, &runs, &waves);
        if (runs > 1)
            most = std::max(most, (size_t)rows * runs);
    }
    return 16 + most * (sizeof(Sums) + top_k * sizeof(unsigned long long));
}

extern "C" int be42_logprobs(float *logprobs, float *entropy, int *top_ids, float *top_logprobs, const void *logits,
                             int logits_bf16, int row_stride, int n, int rows, float temp, const int *tokens,
                             int n_tokens, int top_k, void *workspace, size_t workspace_bytes, void *stream)
{
    BE42_CHECK(n > 0 && n <= 1 << 30 && rows >= 0 && row_stride >= n, "be42_logprobs: %d rows of %d at stride %d", rows,
               n, row_stride);
    const float c = (float)(1.44269504088896340736 / (double)temp);
    BE42_CHECK(temp > 0.0f && std::isfinite(temp) && std::isfinite(c) && c >= 1e-30f, "be42_logprobs: temperature %g",
               (double)temp);
    if (rows == 0)
        return BE42_OK;
    BE42_CHECK(logits, "be42_logprobs: null pointer");
    BE42_CHECK(n_tokens >= 0 && n_tokens <= 1 << 30 && (n_tokens == 0 || (tokens && logprobs)),
               "be42_logprobs: %d tokens a row, %s", n_tokens, tokens ? "no logprobs" : "no ids");
    BE42_CHECK(top_k >= 0 && top_k <= kTopMax && top_k <= n, "be42_logprobs: top %d of %d (at most %d)", top_k, n,
               kTopMax);
    BE42_CHECK(top_k == 0 || (top_ids && top_logprobs), "be42_logprobs: top %d without arrays", top_k);
    BE42_CHECK(n_tokens || top_k || entropy, "be42_logprobs: nothing asked for");
    BE42_CHECK(!((uintptr_t)logits & (logits_bf16 ? 1 : 3)), "be42_logprobs: unaligned logits");
    const size_t need = be42_logprobs_workspace_bytes(n, rows, top_k);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_logprobs: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    long chunks, per, runs;
    int waves;
    const bool aligned = !((uintptr_t)logits & 15) && row_stride % (logits_bf16 ? 8 : 4) == 0;
    cut_row(n, aligned ? 0 : 7, rows, logits_bf16 != 0, &chunks, &per, &runs, &waves);
    const long blocks = runs * rows;
    BE42_CHECK(blocks <= kMaxBlocks, "be42_logprobs: %d rows of %d (at most %d)", rows, n, kMaxBlocks);
    ScoreArgs a = {logits, (size_t)row_stride, logprobs, entropy, top_logprobs, top_ids, tokens, n_tokens, top_k, n, c,
                   (int)chunks, (int)per, (int)runs};
    hipStream_t s = as_stream(stream);
    // (whether or not these sizes use it)
    BE42_CHECK(workspace || !captured(s), "be42_logprobs: a captured call needs a workspace of the caller's");
    if (runs > 1) {
        if (!workspace)
            workspace = be42::workspace(need, s);
        if (!workspace)
            return BE42_ENOMEM;
        a.sums = (Sums *)workspace;
        a.keys = (unsigned long long *)(a.sums + blocks);
    }
    const dim3 g((unsigned)blocks), t(kWave * waves);
    auto run = [&](auto bf16) {
        constexpr bool BF16 = decltype(bf16)::value;
        if (waves == kScoreWide)
            hipLaunchKernelGGL((k_score_run<BF16, kScoreWide>), g, t, 0, s, a);
        else
            hipLaunchKernelGGL((k_score_run<BF16, kScoreW>), g, t, 0, s, a);
    };
    logits_bf16 ? run(std::true_type()) : run(std::false_type());
    if (runs > 1) {
        const dim3 w(kWave);
        if (logits_bf16)
            hipLaunchKernelGGL(k_score_join<true>, dim3(rows), w, 0, s, a);
        else
            hipLaunchKernelGGL(k_score_join<false>, dim3(rows), w, 0, s, a);
    }
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
