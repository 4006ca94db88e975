// prefix.hip -- attention of a batch that shares a prefix: queries over the
// tokens of one shared slot of the page pool and of their own slots.
//
//   out[b][h] = sum_t softmax_t(scale * q[b][h] . k_t) v_t
// over the first prefix_len tokens of slot prefix_slot and the first lens[b]
// tokens of slot slots[b].
#include <algorithm>
#include <cmath>

#include "be42_common.h"
#include "paged_dev.h"

namespace be42 {

struct PrefixArgs {
    const void *q;
    void *out;
    const int *slots, *lens;
    float *part;              // workspace
    size_t q_stride;
    int n_queries, n_heads, prefix_slot, prefix_len, max_len;
    float scale;
};

// tokens a slot holds (0 for a slot outside the pool)
__device__ __forceinline__ int slot_tokens(const be42_kv_pool &P, int slot)
{
    if (slot < 0 || slot >= P.n_layers)
        return 0;
    const int pages = min(P.n_logical[slot], P.max_logical);
    if (pages <= 0)
        return 0;
    const int last = P.page_table[(size_t)slot * P.max_logical + pages - 1];
    if (last < 0 || last >= P.capacity)
        return 0;
    return (pages - 1) * kPage + min(P.ntok[last], kPage);
}

template <bool BF16>
__device__ __forceinline__ float kv_elem(const be42_kv_pool &P, bool v, size_t page_head, int t, int d)
{
    const void *p = v ? P.v : P.k;
    if (BF16)
        return bf16_to_f32(((const uint16_t *)p)[v ? (page_head * P.head_dim + d) * kPage + t
                                                   : (page_head * kPage + t) * P.head_dim + d]);
    return (float)((const int8_t *)p)[(page_head * kPage + t) * P.head_dim + d] *
           (v ? P.v_scale : P.k_scale)[page_head * kPage + t];
}

// one wave per (query, head), one token at a time
template <bool BF16, bool QB>
__global__ __launch_bounds__(64) void k_prefix_attn(const be42_kv_pool P, const PrefixArgs a)
{
    const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int hd = P.head_dim, per = hd / kWave, kvh = h / (a.n_heads / P.n_kv);
    float q[2], o[2] = {0.0f, 0.0f};
    for (int i = 0; i < per; i++) {
        const size_t at = (size_t)b * a.q_stride + (size_t)h * hd + lane + i * kWave;
        q[i] = QB ? bf16_to_f32(((const uint16_t *)a.q)[at]) : ((const float *)a.q)[at];
    }
    float m = -INFINITY, l = 0.0f;
    for (int part = 0; part < 2; part++) {
        const int slot = part ? (a.slots ? a.slots[b] : b) : a.prefix_slot;
        int n = slot_tokens(P, slot);
        n = min(n, part ? (a.lens ? min(a.lens[b], a.max_len) : a.max_len) : a.prefix_len);
        for (int t = 0; t < n; t++) {
            const int phys = P.page_table[(size_t)slot * P.max_logical + t / kPage];
            if (phys < 0 || phys >= P.capacity)
                continue;
            const size_t ph = (size_t)phys * P.n_kv + kvh;
            float s = 0.0f;
            for (int i = 0; i < per; i++)
                s = __fmaf_rn(q[i], kv_elem<BF16>(P, false, ph, t % kPage, lane + i * kWave), s);
            s = wave_sum(s) * a.scale;
            const float mn = fmaxf(m, s), c = expf(m - mn), p = expf(s - mn);
            l = l * c + p;
            for (int i = 0; i < per; i++)
                o[i] = __fmaf_rn(p, kv_elem<BF16>(P, true, ph, t % kPage, lane + i * kWave), o[i] * c);
            m = mn;
        }
    }
    for (int i = 0; i < per; i++) {
        const size_t at = ((size_t)b * a.n_heads + h) * hd + lane + i * kWave;
        const float v = l == 0.0f ? 0.0f : o[i] / l;
        if (QB)
            ((uint16_t *)a.out)[at] = f32_to_bf16(v);
        else
            ((float *)a.out)[at] = v;
    }
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_prefix_attention_workspace_bytes(int n_queries, int n_heads, int n_kv, int head_dim,
                                                        int prefix_len, int max_len)
{
    if (n_queries <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || (head_dim != 64 && head_dim != 128) ||
        prefix_len < 0 || max_len < 0)
        return 0;
    return 16;
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
    BE42_CHECK(n_queries >= 0 && q_stride >= n_heads * P.head_dim, "be42_prefix_attention: %d queries at stride %d",
               n_queries, q_stride);
    BE42_CHECK(prefix_slot >= 0 && prefix_slot < P.n_layers, "be42_prefix_attention: prefix slot %d of %d", prefix_slot,
               P.n_layers);
    const long held = (long)P.max_logical * kPage;
    BE42_CHECK(prefix_len >= 0 && prefix_len <= held && max_len >= 0,
               "be42_prefix_attention: prefix %d, max_len %d (a slot holds %ld tokens)", prefix_len, max_len, held);
    BE42_CHECK(std::isfinite(scale), "be42_prefix_attention: scale %g", (double)scale);
    BE42_CHECK(!(((uintptr_t)q | (uintptr_t)out) & (q_bf16 ? 1 : 3)), "be42_prefix_attention: unaligned pointer");
    // without slots query b reads slot b
    BE42_CHECK(slots || max_len == 0 || n_queries <= P.n_layers, "be42_prefix_attention: %d queries over %d slots",
               n_queries, P.n_layers);
    if (n_queries == 0)
        return BE42_OK;
    const size_t need = be42_prefix_attention_workspace_bytes(n_queries, n_heads, P.n_kv, P.head_dim, prefix_len,
                                                              max_len);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_prefix_attention: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    PrefixArgs a = {q, out, slots, lens, nullptr, (size_t)q_stride, n_queries, n_heads, prefix_slot, prefix_len,
                    max_len, scale};
    const dim3 g(n_queries, n_heads), b(64);
    hipStream_t s = as_stream(stream);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, b, 0, s, P, a); };
    if (P.kind == BE42_KV_BF16) {
        if (q_bf16) go(k_prefix_attn<true, true>);
        else go(k_prefix_attn<true, false>);
    } else {
        if (q_bf16) go(k_prefix_attn<false, true>);
        else go(k_prefix_attn<false, false>);
    }
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
