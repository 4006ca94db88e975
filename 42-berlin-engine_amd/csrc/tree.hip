// tree.hip -- attention of trees of drafted tokens: every draft over its sequence's
// context and over its own path in the tree.
//
//   out[i][h] = sum_t softmax_t(scale * q[i][h] . k_t) v_t
// over the first lens[b] tokens of slot slots[b], and over draft i and what lies above
// it in its tree, which are tokens of the slot that holds all the drafts.
//
// Rows (draft, head) of one tree and KV head go in tiles over the context, which is
// cut into parts as the prefix's tokens are (attn_tile.h); the drafts are one part
// more, whose tiles of 16 rows have a bit for each row and draft.  The parts of a row
// are joined by weight.  Where there are few tokens, one launch does all.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_tile.h"
#include "be42_common.h"
#include "paged_dev.h"

namespace be42 {

constexpr int kMaxTree = 256;

struct TreeArgs : PrefixArgs {     // n_queries: tokens; parts_p, chunk_p, tiles_p, rows_p: of the contexts
    const int *starts, *parents;
    int n_trees, max_tree, draft_slot;
};

// Tokens first .. first + n - 1 of tree b.
__device__ __forceinline__ int tree_tokens(const TreeArgs &a, int b, int &first)
{
    first = min(max(a.starts[b], 0), a.n_queries);
    return min(min(max(a.starts[b + 1], first), a.n_queries) - first, a.max_tree);
}

struct TreePaths {
    static constexpr int kWords = kMaxTree / 32;
    int up[kMaxTree];
    uint32_t above[kMaxTree][kWords + 1];         // (rows on distinct banks)
};
template <int HD, int N>
struct TreeShared {
    union {
        PartShared<HD, N> sums;
        TreePaths paths;                          // done with before there are sums
    };
    uint32_t bits[16][SeesPath::kWords];
};
static_assert(SeesPath::kWords == TreePaths::kWords + 1 && kMaxTree == 64 * kPartWaves, "a tree from anywhere in a page on; a draft a thread");

// The paths of a tile's rows, from row `row0` of the tree on; bit 0 is token `lo` of
// the drafts' slot.  A parent that is no earlier draft ends the path, as -1 does.  A
// thread has a draft and what is known of its path, and doubles it each time: the path
// of the draft where its own ends so far.  (With a thread a row that walks up draft by
// draft, calls of four chains of 256 took 40 us, with this 16.)
template <class S>
__device__ __forceinline__ SeesPath tree_mask(const TreeArgs &a, S &shared, int first, int n, int lo, int hi, int row0, int rows, int G)
{
    constexpr int W = TreePaths::kWords;
    TreePaths &M = shared.paths;
    const int i = threadIdx.x, last = min(row0 + 15, rows - 1) / G;
    uint32_t path[W];
#pragma unroll
    for (int w = 0; w < W; w++)
        path[w] = i >> 5 == w ? 1u << (i & 31) : 0u;
    int up = -1;
    if (i <= last) {
        up = a.parents ? a.parents[first + i] : i - 1;
        up = up < i ? max(up, -1) : -1;
    }
    while (true) {
        M.up[i] = up;
#pragma unroll
        for (int w = 0; w < W; w++)
            M.above[i][w] = path[w];
        if (!__syncthreads_or(up >= 0))
            break;
        int next = -1;
        if (up >= 0) {
            next = M.up[up];
#pragma unroll
            for (int w = 0; w < W; w++)
                path[w] |= M.above[up][w];
        }
        up = next;
        __syncthreads();
    }
    // from the tree's first draft to the page's first token, and no further than the slot
    for (int x = threadIdx.x; x < 16 * SeesPath::kWords; x += blockDim.x) {
        const int r = x / SeesPath::kWords, w = x % SeesPath::kWords, at = min(row0 + r, rows - 1) / G, shift = first - lo;
        auto held = [&](int v) {
            const int left = hi - first - 32 * v;
            return v < 0 || v >= W || left <= 0 ? 0u : M.above[at][v] & (left < 32 ? (1u << left) - 1 : ~0u);
        };
        shared.bits[r][w] = held(w) << shift | (uint32_t)((uint64_t)held(w - 1) << shift >> 32);
    }
    __syncthreads();
    return {&shared.bits[0][0], first - lo, hi - lo};
}

template <bool KV8, int HD, bool QB, int R>
__global__ __launch_bounds__(64 * kPartWaves, 2) void k_tree_part(const be42_kv_pool P, const TreeArgs a)
{
    __shared__ union {
        TreeShared<HD, kPartWaves> few;
        std::conditional_t<R != 0, WideShared<KV8, HD, R ? R : 4>, char> many;
    } S;
    constexpr int NP = QB ? 1 : 3, PP = QB ? 2 : 3, kRows = R ? 32 * R : 16;
    const int G = a.n_heads / P.n_kv, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (the drafts last: they are short, and end beside the last contexts)
    const unsigned of_contexts = (unsigned)P.n_kv * a.tiles_p * a.n_trees * a.parts_p;
    unsigned id = blockIdx.x;
    const bool drafts = id >= of_contexts;
    if (drafts)
        id -= of_contexts;
    const int kvh = (int)(id % (unsigned)P.n_kv);
    id /= (unsigned)P.n_kv;
    const unsigned tiles = drafts ? a.tiles_o : a.tiles_p;
    const int row0 = (drafts ? 16 : kRows) * (int)(id % tiles);
    id /= tiles;
    const int b = (int)(id % (unsigned)a.n_trees), part = (int)(id / (unsigned)a.n_trees);
    int first;
    const int n = tree_tokens(a, b, first), rows = n * G;
    if (row0 >= rows)
        return;
    if (drafts) {
        const int lo = first / kPage * kPage, hi = max(first, slot_tokens(P, a.draft_slot, first + n));
        const SeesPath seen = tree_mask(a, S.few, first, n, lo, hi, row0, rows, G);
        part16<KV8, HD, NP, PP>(P, a, S.few.sums, a.draft_slot, lo, hi, kvh, first, row0, rows, wave, kPartWaves, wave, 0, seen);
        __syncthreads();
        write_part<HD, QB, kPartWaves, 16>(a, S.few.sums, row0, rows, first, kvh, G, a.parts_p);
        return;
    }
    const int slot = a.slots ? a.slots[b] : b, lo = part * a.chunk_p;
    const int want = min(a.lens ? min(a.lens[b], a.max_len) : a.max_len, lo + a.chunk_p);
    if constexpr (R != 0) {
        part32<KV8, HD, NP, PP, R>(P, a, S.many, slot, lo, want, kvh, first, row0, rows);
        write_part<HD, QB, kPartWaves / R, kRows>(a, S.many.sums, row0, rows, first, kvh, G, part);
    } else {
        part16<KV8, HD, NP, PP>(P, a, S.few.sums, slot, lo, max(lo, slot_tokens(P, slot, want)), kvh, first, row0, rows, wave, kPartWaves,
                                wave, 0);
        __syncthreads();
        write_part<HD, QB, kPartWaves, 16>(a, S.few.sums, row0, rows, first, kvh, G, part);
    }
}

// Few tokens: a workgroup takes a tile's context and drafts.
template <bool KV8, int HD, bool QB>
__global__ __launch_bounds__(64 * kPartWaves, 2) void k_tree_whole(const be42_kv_pool P, const TreeArgs a)
{
    __shared__ TreeShared<HD, 2 * kPartWaves> S;
    constexpr int NP = QB ? 1 : 3, PP = QB ? 2 : 3;
    const int G = a.n_heads / P.n_kv, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)P.n_kv);
    id /= (unsigned)P.n_kv;
    const int row0 = 16 * (int)(id % (unsigned)a.tiles_o), b = (int)(id / (unsigned)a.tiles_o);
    int first;
    const int n = tree_tokens(a, b, first), rows = n * G;
    if (row0 >= rows)
        return;
    const int lo = first / kPage * kPage, hi = max(first, slot_tokens(P, a.draft_slot, first + n));
    const SeesPath seen = tree_mask(a, S, first, n, lo, hi, row0, rows, G);
    const int slot = a.slots ? a.slots[b] : b;
    const int want = a.lens ? min(a.lens[b], a.max_len) : a.max_len;
    part16<KV8, HD, NP, PP>(P, a, S.sums, slot, 0, slot_tokens(P, slot, want), kvh, first, row0, rows, wave, kPartWaves, wave, 0);
    part16<KV8, HD, NP, PP>(P, a, S.sums, a.draft_slot, lo, hi, kvh, first, row0, rows, wave, kPartWaves, kPartWaves + wave, 0, seen);
    __syncthreads();
    write_part<HD, QB, 2 * kPartWaves, 16>(a, S.sums, row0, rows, first, kvh, G, 0);
}

// The parts of the rows that trees have (the others' are left as they are), a workgroup a
// few rows of a tree's.  MANY parts: a wave a row (join_row).  Few: HD / 4 lanes a row,
// all its loads in flight together.  (With four rows for the same lanes, one after the
// other, 6168 rows took 9 us.)
constexpr int kFewParts = 8;
template <int HD>
constexpr int kJoinRows = 256 / (HD / 4);
template <int HD, bool QB, bool MANY>
__global__ __launch_bounds__(256) void k_tree_join(const TreeArgs a, int parts, int chunks)
{
    constexpr int L = HD / 4, ROWS = MANY ? 4 : kJoinRows<HD>;
    const int b = (int)(blockIdx.x / (unsigned)chunks), c0 = (int)(blockIdx.x % (unsigned)chunks) * ROWS;
    int first;
    const int rows = tree_tokens(a, b, first) * a.n_heads, d = 4 * (threadIdx.x % L);
    const size_t all = (size_t)a.n_queries * a.n_heads, row0 = (size_t)first * a.n_heads;
    if constexpr (MANY) {
        const int r = c0 + (threadIdx.x >> 6);
        if (r < rows)
            join_row<HD, QB>(a, parts, row0 + r);
    } else {
        const int r = c0 + threadIdx.x / L;
        if (r >= rows)
            return;
        const float2 *ml = (const float2 *)a.part_ml;
        const float sc = log2_scale(a);
        const size_t row = row0 + r;
        float2 x[kFewParts];
        float4 o[kFewParts];
#pragma unroll
        for (int j = 0; j < kFewParts; j++)
            if (j < parts) {
                const size_t at = j * all + row;
                x[j] = ml[at];
                o[j] = *(const float4 *)(a.part_o + at * HD + d);
            }
        float top = -INFINITY, l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < kFewParts; j++)
            if (j < parts)
                top = fmaxf(top, x[j].x);
#pragma unroll
        for (int j = 0; j < kFewParts; j++)
            // (a part without tokens left no values)
            if (j < parts && x[j].x != -INFINITY) {
                const float w = __builtin_amdgcn_exp2f((x[j].x - top) * sc);
                l = __fmaf_rn(w, x[j].y, l);
                v.x = __fmaf_rn(w, o[j].x, v.x);
                v.y = __fmaf_rn(w, o[j].y, v.y);
                v.z = __fmaf_rn(w, o[j].z, v.z);
                v.w = __fmaf_rn(w, o[j].w, v.w);
            }
        const float inv = row_inverse(top, l);
        store_out4<QB>(a.out, row * HD + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
}

// Rows of a context's tile: 16 where all of a tree fit (64 trees of 4 INT8 drafts, four
// heads a KV head, over up to 2048 tokens 38 us, 57 in tiles of 64), up to 192 in tiles
// of 64 (32 bf16 rows over 8 x 8192 tokens fp32 42 us, 16: 49, 128: 56; 183 INT8 rows 60,
// 128: 67), more in tiles of 128 (256 rows over 32768 tokens 459, 64: 483).  Two
// workgroups a CU (four of tiles of 16), of no less than 512 tokens (128), since each
// takes 5 us before and after its tokens (one tree of 128 rows over 8192 tokens 23 us, in
// parts of 256 28), and of no more than 4096: lengths differ, and the longest is the last
// (32768 tokens in parts of 16384 650 us).
static void plan_tree(TreeArgs &a, int n_kv)
{
    const int G = a.n_heads / n_kv, unit = kPartWaves * kStep;
    const long rows = (long)a.max_tree * G;
    const long steps = (a.max_len + unit - 1L) / unit + (a.max_tree + kPage + unit - 1) / unit;
    a.tiles_o = (int)((rows + 15) / 16);
    a.whole = steps <= 5;
    if (a.whole) {
        a.parts_p = 1;
        return;
    }
    a.rows_p = rows > 192 ? 128 : rows > 16 ? 64 : 16;
    a.tiles_p = (int)((rows + a.rows_p - 1) / a.rows_p);
    a.parts_o = 1;
    const long tiles = (long)a.tiles_p * n_kv * a.n_trees;
    cut(a.max_len, tiles, a.rows_p == 16 ? unit : 4 * unit, std::max(a.rows_p == 16 ? 1024L : 512L, tiles * ((a.max_len + 4095L) / 4096)), &a.parts_p, &a.chunk_p);
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_tree_attention_workspace_bytes(int n_tokens, int n_trees, int n_heads, int n_kv, int head_dim,
                                                      int max_tree, int max_len)
{
    if (n_tokens <= 0 || n_trees <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || (head_dim != 64 && head_dim != 128) ||
        max_tree <= 0 || max_tree > kMaxTree || max_len < 0 || max_len > kMaxTokens || (size_t)n_tokens * n_heads > kMaxRows)
        return 0;
    TreeArgs a = {};
    a.n_heads = n_heads;
    a.max_len = max_len;
    a.n_trees = n_trees;
    a.max_tree = max_tree;
    plan_tree(a, n_kv);
    const int parts = a.parts_p + a.parts_o;
    return 16 + (parts > 1 ? (size_t)parts * n_tokens * n_heads * (head_dim + 2) * sizeof(float) : 0);
}

extern "C" int be42_tree_attention(const be42_kv_pool *pool, const void *q, int q_bf16, int q_stride, int n_tokens,
                                   int n_heads, const int *starts, int n_trees, int max_tree, const int *parents,
                                   int draft_slot, const int *slots, const int *lens, int max_len, float scale, void *out,
                                   void *workspace, size_t workspace_bytes, void *stream)
{
    BE42_CHECK(pool && (n_tokens == 0 || n_trees == 0 || (q && out && starts)), "be42_tree_attention: null pointer");
    const be42_kv_pool &P = *pool;
    BE42_CHECK(n_heads > 0 && n_heads % P.n_kv == 0, "be42_tree_attention: %d heads over %d kv heads", n_heads, P.n_kv);
    BE42_CHECK(P.head_dim == 64 || P.head_dim == 128, "be42_tree_attention: head_dim %d (64 or 128)", P.head_dim);
    BE42_CHECK(n_tokens >= 0 && q_stride >= (long)n_heads * P.head_dim, "be42_tree_attention: %d drafts at stride %d",
               n_tokens, q_stride);
    BE42_CHECK(n_trees >= 0 && max_tree > 0 && max_tree <= kMaxTree, "be42_tree_attention: %d trees of up to %d drafts (at most %d)",
               n_trees, max_tree, kMaxTree);
    BE42_CHECK(draft_slot >= 0 && draft_slot < P.n_layers, "be42_tree_attention: draft slot %d of %d", draft_slot, P.n_layers);
    BE42_CHECK(max_len >= 0 && max_len <= kMaxTokens, "be42_tree_attention: max_len %d", max_len);
    BE42_CHECK(std::fabs(scale) <= 1e30f, "be42_tree_attention: scale %g", (double)scale);
    BE42_CHECK(!(((uintptr_t)q | (uintptr_t)out) & (q_bf16 ? 1 : 3)) &&
                   !(((uintptr_t)starts | (uintptr_t)parents | (uintptr_t)slots | (uintptr_t)lens) & 3),
               "be42_tree_attention: unaligned pointer");
    // without slots tree b reads slot b
    BE42_CHECK(slots || max_len == 0 || n_trees <= P.n_layers, "be42_tree_attention: %d trees over %d slots", n_trees,
               P.n_layers);
    if (n_tokens == 0 || n_trees == 0)
        return BE42_OK;
    const size_t rows = (size_t)n_tokens * n_heads;
    BE42_CHECK(rows <= kMaxRows, "be42_tree_attention: %d drafts of %d heads", n_tokens, n_heads);
    TreeArgs a = {};
    a.q = q;
    a.out = out;
    a.slots = slots;
    a.lens = lens;
    a.q_stride = (size_t)q_stride;
    a.n_queries = n_tokens;
    a.n_heads = n_heads;
    a.max_len = max_len;
    a.scale = scale;
    a.starts = starts;
    a.parents = parents;
    a.n_trees = n_trees;
    a.max_tree = max_tree;
    a.draft_slot = draft_slot;
    plan_tree(a, P.n_kv);
    const int parts = a.parts_p + a.parts_o;
    const double blocks = (double)P.n_kv * n_trees * (a.whole ? a.tiles_o : (double)a.tiles_p * a.parts_p + a.tiles_o);
    BE42_CHECK(blocks <= kMaxBlocks, "be42_tree_attention: %d trees of up to %d drafts of %d heads", n_trees, max_tree, n_heads);
    const int join_rows = parts > kFewParts ? 4 : P.head_dim == 64 ? kJoinRows<64> : kJoinRows<128>;
    const long chunks = ((long)max_tree * n_heads + join_rows - 1) / join_rows;
    BE42_CHECK(chunks * n_trees <= kMaxBlocks, "be42_tree_attention: %d trees of up to %d drafts of %d heads", n_trees, max_tree, n_heads);
    const size_t need = be42_tree_attention_workspace_bytes(n_tokens, n_trees, n_heads, P.n_kv, P.head_dim, max_tree, max_len);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_tree_attention: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    hipStream_t s = as_stream(stream);
    // (whether or not these sizes use it)
    BE42_CHECK(workspace || !captured(s), "be42_tree_attention: a captured call needs a workspace of the caller's");
    if (parts > 1) {
        if (!workspace)
            workspace = be42::workspace(need, s);
        if (!workspace)
            return BE42_ENOMEM;
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + (size_t)parts * rows * P.head_dim;
    }
    auto go = [&](auto kv8, auto hd, auto qb) {
        constexpr bool KV8 = decltype(kv8)::value, QB = decltype(qb)::value;
        constexpr int HD = decltype(hd)::value;
        const dim3 g((unsigned)blocks), t(64 * kPartWaves);
        if (a.whole) {
            hipLaunchKernelGGL((k_tree_whole<KV8, HD, QB>), g, t, 0, s, P, a);
            return;
        }
        if (a.rows_p == 128)
            hipLaunchKernelGGL((k_tree_part<KV8, HD, QB, 4>), g, t, 0, s, P, a);
        else if (a.rows_p == 64)
            hipLaunchKernelGGL((k_tree_part<KV8, HD, QB, 2>), g, t, 0, s, P, a);
        else
            hipLaunchKernelGGL((k_tree_part<KV8, HD, QB, 0>), g, t, 0, s, P, a);
        if (parts > 1) {
            if (parts > kFewParts)
                hipLaunchKernelGGL((k_tree_join<HD, QB, true>), dim3((unsigned)(n_trees * chunks)), dim3(256), 0, s, a, parts, (int)chunks);
            else
                hipLaunchKernelGGL((k_tree_join<HD, QB, false>), dim3((unsigned)(n_trees * chunks)), dim3(256), 0, s, a, parts, (int)chunks);
        }
    };
    auto of_type = [&](auto kv8, auto hd) { q_bf16 ? go(kv8, hd, std::true_type()) : go(kv8, hd, std::false_type()); };
    auto of_dim = [&](auto kv8) {
        P.head_dim == 64 ? of_type(kv8, std::integral_constant<int, 64>()) : of_type(kv8, std::integral_constant<int, 128>());
    };
    P.kind == BE42_KV_INT8 ? of_dim(std::true_type()) : of_dim(std::false_type());
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
