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

#include "attn_tile.h"
#include "be42_common.h"
#include "paged_dev.h"

namespace be42 {


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
            part32<KV8, HD, NP, QB ? 2 : 3, R>(P, a, S.many, slot, lo, n, kvh, b0, row0, rows);
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

template <int HD, bool QB>
__global__ __launch_bounds__(256) void k_prefix_join(const PrefixArgs a, int parts)
{
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row < (size_t)a.n_queries * a.n_heads)
        join_row<HD, QB>(a, parts, row);
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
