// score.hip -- log probabilities of given tokens, entropy and the top
// alternatives of logits rows.
//
// With z = (x - m) / T, m the row's maximum, s = sum e^z and t = sum z e^z:
//   log p(i) = z_i - log s,   H = log s - t / s.
// Both follow from one pass over the row; sums are joined in 64 bits.
#include <cmath>

#include "be42_common.h"

namespace be42 {

constexpr int kTopMax = 64;

// One number per (value, id) that is larger for a larger value, then for a
// lower id: the value's bits as an order-preserving integer, then ~id.  -0 is
// taken for +0 and a NaN for -infinity.
__device__ __forceinline__ unsigned long long order_key(float x, int id)
{
    const uint32_t u = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(unsigned long long k)
{
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

template <bool BF16>
__device__ __forceinline__ float logit(const void *row, int i)
{
    return BF16 ? bf16_to_f32(((const uint16_t *)row)[i]) : ((const float *)row)[i];
}

struct ScoreArgs {
    float *lp, *entropy, *top_lp;
    int *top_ids;
    const int *tokens;
    int n_tokens, top_k, n;
    float inv_temp;
};

constexpr int kScoreT = 256;

// one block per row
template <bool BF16>
__global__ __launch_bounds__(kScoreT) void k_logprobs(const ScoreArgs a, const void *logits, size_t row_stride)
{
    __shared__ double sd[kScoreT];
    __shared__ unsigned long long sk[kScoreT];
    const int b = blockIdx.x, tid = threadIdx.x;
    const void *x = (const char *)logits + (size_t)b * row_stride * (BF16 ? 2 : 4);
    auto all = [&](auto *sh, auto v, auto &&op) {
        __syncthreads();
        sh[tid] = v;
        __syncthreads();
        for (int o = kScoreT / 2; o > 0; o >>= 1) {
            if (tid < o)
                sh[tid] = op(sh[tid], sh[tid + o]);
            __syncthreads();
        }
        return sh[0];
    };
    auto larger = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    auto add = [](double p, double q) { return p + q; };
    bool bad = false;
    unsigned long long best = 0;
    for (int i = tid; i < a.n; i += kScoreT) {
        const float v = logit<BF16>(x, i);
        bad |= !(v < INFINITY);
        best = larger(best, order_key(v, i));
    }
    best = all(sk, best, larger);
    const float m = key_value(best);
    bad = __syncthreads_or(bad) || m == -INFINITY;
    double s = 0.0, t = 0.0;
    for (int i = tid; i < a.n; i += kScoreT) {
        const float z = (logit<BF16>(x, i) - m) * a.inv_temp;
        const double e = exp((double)z);
        s += e;
        t += e > 0.0 ? e * z : 0.0;
    }
    s = all(sd, s, add);
    t = all(sd, t, add);
    const double ls = bad ? (double)NAN : log(s);
    if (tid == 0 && a.entropy)
        a.entropy[b] = (float)(ls - t / s);
    for (int j = tid; j < a.n_tokens; j += kScoreT) {
        const int id = a.tokens[(size_t)b * a.n_tokens + j];
        const float v = id >= 0 && id < a.n ? logit<BF16>(x, id) : -INFINITY;
        a.lp[(size_t)b * a.n_tokens + j] = bad ? NAN : (float)((double)(v - m) * a.inv_temp - ls);
    }
    for (int k = 0; k < a.top_k; k++) {
        if (tid == 0) {
            a.top_ids[(size_t)b * a.top_k + k] = key_id(best);
            a.top_lp[(size_t)b * a.top_k + k] = bad ? NAN : (float)((double)(key_value(best) - m) * a.inv_temp - ls);
        }
        unsigned long long next = 0;
        for (int i = tid; i < a.n; i += kScoreT) {
            const unsigned long long key = order_key(logit<BF16>(x, i), i);
            next = key < best ? larger(next, key) : next;
        }
        best = all(sk, next, larger);
    }
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_logprobs_workspace_bytes(int n, int rows, int top_k)
{
    if (n <= 0 || rows <= 0 || top_k < 0 || top_k > kTopMax || top_k > n)
        return 0;
    return 16;
}

extern "C" int be42_logprobs(float *logprobs, float *entropy, int *top_ids, float *top_logprobs, const void *logits,
                             int logits_bf16, int row_stride, int n, int rows, float temp, const int *tokens,
                             int n_tokens, int top_k, void *workspace, size_t workspace_bytes, void *stream)
{
    BE42_CHECK(n > 0 && rows >= 0 && row_stride >= n, "be42_logprobs: %d rows of %d at stride %d", rows, n, row_stride);
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
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) &&
                              workspace_bytes >= be42_logprobs_workspace_bytes(n, rows, top_k)),
               "be42_logprobs: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes,
               be42_logprobs_workspace_bytes(n, rows, top_k));
    const ScoreArgs a = {logprobs, entropy, top_logprobs, top_ids, tokens, n_tokens, top_k, n, 1.0f / temp};
    hipStream_t s = as_stream(stream);
    if (logits_bf16)
        hipLaunchKernelGGL(k_logprobs<true>, dim3(rows), dim3(kScoreT), 0, s, a, logits, (size_t)row_stride);
    else
        hipLaunchKernelGGL(k_logprobs<false>, dim3(rows), dim3(kScoreT), 0, s, a, logits, (size_t)row_stride);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
