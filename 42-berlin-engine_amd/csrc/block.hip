// block.hip -- E4M3 products with a scale for each block of 128: activations with one
// for 128 elements of a row, weights with one for 128 x 128.
//
//   y[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] w[n][k]
//
// The sum of a block is formed by the matrix cores from the codes and then enters y's
// sum with its scale, in fp32.
#include <algorithm>
#include <type_traits>

#include "be42_common.h"
#include "fp8_codec.h"

namespace be42 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 128;

int upload_fp8_thresholds(int device);       // quant.hip

int upload_block_thresholds(const float *thr)
{
    BE42_HIP(hipMemcpyToSymbol(HIP_SYMBOL(c_fp8_thr), thr, sizeof c_fp8_thr));
    return BE42_OK;
}

// eight E4M3 codes as bf16 (exact)
__device__ __forceinline__ bf16x8 codes_bf16(uint2 c)
{
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, 1.0f, true);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, 1.0f, false), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// Chunk slot of 16-byte chunk c in LDS row R: rows are 128 bytes, and the rows of an
// operand read at one chunk fall on distinct banks.
__device__ __forceinline__ int chunk_slot(int R, int c) { return c ^ ((R & 7) ^ ((R >> 3) & 1)); }

// Sixteen rows' fragment of a block: lane (r, g) has the 32 codes from 32 g on of row r.
union Codes {
    v8i w;
    uint2 d[4];
};

// One 16x16 tile's sum over a block.  The 8-bit instruction takes all 128 at once, at
// twice the bf16 rate (4096 x 14336 x 4096 to bf16 272 us); it aligns the products of
// eight elements to the largest's power of two and cuts each towards zero below 2^-13
// of it, then adds the eights in fp32 (seen with codes of single bits, the same for any
// eight).  A bf16 output keeps 8 bits: for normal values 1.5% of the outputs become a
// neighbouring one and the relative error against 64 bits is 1.65763e-3, with exact sums
// 1.65756e-3; large terms that cancel leave more of it.  fp32 outputs take four bf16
// instructions of the lane's codes eight at a time (either operand's the same way, so
// that equal k meet), in which products are exact and sums fp32.
struct Wide {
    bf16x8 v[4];
};
__device__ __forceinline__ void widen(const Codes &c, Wide &x)
{
#pragma unroll
    for (int s = 0; s < 4; s++)
        x.v[s] = codes_bf16(c.d[s]);
}
__device__ __forceinline__ v4f block_sum(const Codes &a, const Codes &b)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.w, b.w, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 127, 0, 127);
}
__device__ __forceinline__ v4f block_sum(const Wide &a, const Wide &b)
{
    v4f t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; s++)
        t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[s], b.v[s], t, 0, 0, 0);
    return t;
}

template <bool YB>
__device__ __forceinline__ void store_y(void *Y, size_t at, int left, bool words, v4f v)
{
    if (words) {
        if (YB) {
            const uint2 w = make_uint2(f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16, f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16);
            *(uint2 *)((uint16_t *)Y + at) = w;
        } else {
            *(v4f *)((float *)Y + at) = v;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left) {
            if (YB)
                ((uint16_t *)Y)[at + e] = f32_to_bf16(v[e]);
            else
                ((float *)Y)[at + e] = v[e];
        }
}

// The ring of blocks in LDS: codes of BT tokens, then of BF features, 128 bytes a row,
// and the tokens' scales.  A wave loads DPW times eight rows, and 64 scales, through
// buffer descriptors: an offset of the lane and one of the wave, where 64-bit addresses
// would take 16 registers and an instruction a load.  CUT: K is no multiple of 128; a
// row's chunks behind its end are given an offset past the descriptor's, which reads
// zeros.
#ifdef __HIP_DEVICE_COMPILE__
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)bytes, 0x00027000);
}
template <int SIZE>
__device__ __forceinline__ void buffer_to_lds(buffer_t b, void *to, uint32_t lane_off, uint32_t wave_off)
{
    if constexpr (SIZE == 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void *)to, 16, lane_off, wave_off, 0, 0);
    else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (lds_void *)to, 4, lane_off, wave_off, 0, 0);
}
#else                                          // (the host's pass does not know the type)
typedef void *buffer_t;
__device__ buffer_t buffer_of(const void *p, uint32_t bytes);
template <int SIZE>
__device__ void buffer_to_lds(buffer_t b, void *to, uint32_t lane_off, uint32_t wave_off);
#endif
constexpr int kMaxK = 1 << 22;                 // 256 rows of it are 2^30 bytes
constexpr uint32_t kPastEnd = 0x80000000u, kMostBytes = 0x7FFFFFFFu;
template <int BT, int BF, int NW, int NS, bool CUT>
struct Loader {
    static constexpr int ROWS = BT + BF, DPW = ROWS / 8 / NW, kLoads = DPW + 1, SCH = BT < 64 ? 1 : BT / 64;
    static constexpr int SBYTES = ROWS * 128 + SCH * 256;
    static_assert(ROWS % (8 * NW) == 0 && BT % 8 == 0 && SCH <= NW && (BT < 64 || BT % 64 == 0), "loads divide over the waves");
    buffer_t xr, wr, sr;
    uint32_t src[DPW], soff;
    int K, wave, lane;
    static __device__ __forceinline__ buffer_t rsrc(const void *p, size_t bytes)
    {
        return buffer_of(p, (uint32_t)(bytes < kMostBytes ? bytes : kMostBytes));
    }
    __device__ __forceinline__ void init(const uint8_t *X, const uint8_t *W, const float *sx, int M, int N, int K_, int m0, int n0,
                                         int wave_, int lane_)
    {
        K = K_;
        wave = wave_;
        lane = lane_;
        const int kb = (K + kBlock - 1) / kBlock;
        xr = rsrc(X + (size_t)m0 * K, (size_t)(M - m0) * K);
        wr = rsrc(W + (size_t)n0 * K, (size_t)(N - n0) * K);
        sr = rsrc(sx + (size_t)m0 * kb, (size_t)(M - m0) * kb * sizeof(float));
        // rows past M or N read the last one and are not stored
#pragma unroll
        for (int j = 0; j < DPW; j++) {
            const int row = (wave * DPW + j) * 8 + (lane >> 3);
            src[j] = (uint32_t)(row < BT ? min(row, M - 1 - m0) : min(row - BT, N - 1 - n0)) * (uint32_t)K + chunk_slot(row, lane & 7) * 16;
        }
        soff = (uint32_t)min(wave % SCH * 64 + (BT < 64 ? min(lane, BT - 1) : lane), M - 1 - m0) * (uint32_t)kb * 4;
    }
    __device__ __forceinline__ void issue(uint8_t *lds, int b, int place) const
    {
        uint8_t *base = lds + place % NS * SBYTES;
#pragma unroll
        for (int j = 0; j < DPW; j++) {
            const int row0 = (wave * DPW + j) * 8;
            const bool past = CUT && b * kBlock + chunk_slot(row0 + (lane >> 3), lane & 7) * 16 >= K;
            buffer_to_lds<16>(row0 < BT ? xr : wr, base + row0 * 128, past ? kPastEnd : src[j], b * kBlock);
        }
        buffer_to_lds<4>(sr, base + ROWS * 128 + wave % SCH * 256, soff, b * 4);
        // (the counts that are waited for assume that blocks are loaded in order)
        asm volatile("" ::: "memory");
    }
};

// Workgroups of one XCD walk neighbouring tiles, runs of 8 tiles of tokens.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int &tm, int &tn)
{
    const int nb = gridDim.x, per = nb / 8, rem = nb % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
    const int tile = (x < rem ? x * (per + 1) : rem * (per + 1) + (x - rem) * per) + i;
    const int span = 8 * tiles_n, first = tile / span * 8, gsz = min(tiles_m - first, 8), t = tile % span;
    tm = first + t % gsz;
    tn = t / gsz;
}

// A workgroup of WF x WT waves owns WF * TF * 16 features x WT * TT * 16 tokens, a wave
// TF x TT tiles of 16 x 16, rows of the products features and columns tokens, so that
// a lane has one token of a tile and with it one scale.  Blocks of 128 codes of all
// rows, and the tokens' scales of the block, come into a ring of NS in LDS by
// direct-to-LDS loads.  Before the last tokens of a block the next one is waited for
// and its place's successor asked for: by then every wave holds what is left of the
// block in registers.
template <bool F8, bool YB, int WF, int WT, int TF, int TT, int NS, bool CUT, bool PART>
__global__ __launch_bounds__(WF *WT * 64, WF *WT == 4 ? 2 : 1) void k_block_dma(void *__restrict__ Y, const uint8_t *__restrict__ X,
                                                           const float *__restrict__ sx, const uint8_t *__restrict__ W,
                                                           const float *__restrict__ sw, int M, int N, int K, int tiles_m,
                                                           int tiles_n, int tile0)
{
    constexpr int NW = WF * WT, BF = WF * TF * 16, BT = WT * TT * 16, ROWS = BF + BT;
    constexpr int kLoads = Loader<BT, BF, NW, NS, CUT>::kLoads, SBYTES = Loader<BT, BF, NW, NS, CUT>::SBYTES;
    static_assert(128 % (TF * 16) == 0, "a wave's features lie in one block");
    extern __shared__ __align__(1024) uint8_t lds_dyn[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    int tm, tn;
    tile_of(tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BT, n0 = (tile0 + tn) * BF;             // tile0: the first of the features' tiles
    const int wf = wave / WT, wt = wave % WT, blocks = (K + kBlock - 1) / kBlock;
    // this workgroup's blocks: all, or with parts an equal share
    const int first = (int)((long)blocks * blockIdx.y / gridDim.y), kb = (int)((long)blocks * (blockIdx.y + 1) / gridDim.y) - first;

    Loader<BT, BF, NW, NS, CUT> in;
    in.init(X, W, sx, M, N, K, m0, n0, wave, lane);
    auto issue = [&](int b) { in.issue(lds_dyn, first + b, b); };
    v4f acc[TF][TT];
#pragma unroll
    for (int i = 0; i < TF; i++)
#pragma unroll
        for (int j = 0; j < TT; j++)
            acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const float *swp = sw + (size_t)min((n0 + wf * TF * 16) / kBlock, (N - 1) / kBlock) * blocks + first;
    // a wave's operands of a block, and its tokens' scales
    struct Block {
        Codes a[TF], b[TT];
        float s[TT];
    };
    const int xrow = wt * TT * 16, wrow = BT + wf * TF * 16;
    // (addresses of a step are four sums; the compiler would keep one for each
    // operand and place of the ring)
    const uint32_t xlo = (xrow + r) * 128 + chunk_slot(r, 2 * g) * 16, wlo = xlo + (wrow - xrow) * 128, slo = ROWS * 128 + (xrow + r) * 4;
    struct At {
        const uint8_t *x0, *x1, *w0, *w1, *s;
    };
    auto place = [&](int b) {
        uint32_t off = (uint32_t)(b % NS) * SBYTES;
        asm volatile("" : "+s"(off));
        const uint8_t *L = lds_dyn + off;
        return At{L + xlo, L + (xlo ^ 16), L + wlo, L + (wlo ^ 16), L + slo};
    };
    auto read = [&](const At &at, Block &f, int i) {
        const int up = (i < TT ? i : i - TT) * 2048;
        const v4i lo = *(const v4i *)((i < TT ? at.x0 : at.w0) + up), hi = *(const v4i *)((i < TT ? at.x1 : at.w1) + up);
        (i < TT ? f.b[i < TT ? i : 0] : f.a[i < TT ? 0 : i - TT]).w = v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (i < TT)
            f.s[i < TT ? i : 0] = *(const float *)(at.s + i * 64);
    };
    // The products of a block.  Beside each tile's the next block's operands are read,
    // and an earlier tile's sums scaled: some before, since a sum is there only after
    // the next instructions.  8-bit operands go to registers of their own (now, next);
    // ones that are widened leave theirs free (now is next), and are read in program
    // order: the compiler would read them all at once, for which it has no registers.
    auto products = [&](int b, Block &f, Block &next, float swv) {
        constexpr int LAG = F8 ? 3 : 1, Q = TF * TT;
        float sc[TT];
        v4f t[LAG + 1];
        const At at = place(b + 1);
        [[maybe_unused]] Wide A[TF], B;
        if constexpr (!F8) {
#pragma unroll
            for (int i = 0; i < TF; i++) {
                widen(f.a[i], A[i]);
                asm volatile("" : "+v"(A[i].v[0]), "+v"(A[i].v[1]), "+v"(A[i].v[2]), "+v"(A[i].v[3])::"memory");
            }
#pragma unroll
            for (int i = 0; i < TF; i++)
                read(at, next, TT + i);
        }
#pragma unroll
        for (int q = 0; q < Q + LAG; q++) {
            if (q < Q) {
                const int i = q % TF, j = q / TF;
                if (i == 0) {
                    sc[j] = f.s[j] * swv;
                    if constexpr (!F8) {
                        widen(f.b[j], B);
                        asm volatile("" : "+v"(B.v[0]), "+v"(B.v[1]), "+v"(B.v[2]), "+v"(B.v[3]), "+v"(sc[j])::"memory");
                        read(at, next, j);
                    }
                }
                if constexpr (F8) {
                    t[q % (LAG + 1)] = block_sum(f.a[i], f.b[j]);
                    // operands, spread over the tiles
#pragma unroll
                    for (int x = q * (TF + TT) / Q; x < (q + 1) * (TF + TT) / Q; x++)
                        read(at, next, x);
                } else {
                    t[q % (LAG + 1)] = block_sum(A[i], B);
                }
            }
            if (q >= LAG) {
                const int p = q - LAG, i = p % TF, j = p / TF;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    acc[i][j][e] = __fmaf_rn(t[p % (LAG + 1)][e], sc[j], acc[i][j][e]);
            }
            if constexpr (F8)
                __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int b = 0; b < NS; b++)
        if (b < kb)
            issue(b);
    if (kb >= NS)
        stage_barrier<(NS - 1) * kLoads>();
    else
        stage_barrier<0>();
    Block F[F8 ? 2 : 1];
    float swv = swp[0];
    {
        const At at = place(0);
#pragma unroll
        for (int i = 0; i < TF + TT; i++)
            read(at, F[0], i);
    }
    // block b is in registers; the next one is read while its products are formed
    // (past the last: some block's codes, not used)
    auto step = [&](int b, Block &now, Block &next) {
        if (b + NS - 1 < kb)
            stage_barrier<(NS - 2) * kLoads>();
        else
            stage_barrier<0>();
        if (b + NS < kb)
            issue(b + NS);
        const float sc = swv;
        swv = swp[min(b + 1, kb - 1)];
        __builtin_amdgcn_sched_barrier(0);
        products(b, now, next, sc);
    };
    if constexpr (F8) {
        for (int b = 0; b < kb; b += 2) {
            step(b, F[0], F[1]);
            if (b + 1 < kb)
                step(b + 1, F[1], F[0]);
        }
    } else {
#pragma unroll 1
        for (int b = 0; b < kb; b++)
            step(b, F[0], F[0]);
    }
    const bool words = N % 4 == 0 && n0 + BF <= N;           // whole tiles, rows on 16 (8) bytes
#pragma unroll
    for (int j = 0; j < TT; j++) {
        const int tok = m0 + xrow + 16 * j + r;
        if (tok >= M)
            continue;
#pragma unroll
        for (int i = 0; i < TF; i++) {
            const int n = n0 + wf * TF * 16 + 16 * i + 4 * g;
            store_y<YB && !PART>(Y, ((size_t)(PART ? blockIdx.y : 0) * M + tok) * N + n, N - n, words, acc[i][j]);
        }
    }
}

// The parts of a product, in their order.
template <bool YB>
__global__ __launch_bounds__(256) void k_block_join(void *__restrict__ Y, const float *__restrict__ part, size_t all, int parts)
{
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= all)
        return;
    if (all % 4 == 0) {
        v4f v = *(const v4f *)(part + at);
        for (int p = 1; p < parts; p++)
            v += *(const v4f *)(part + p * all + at);
        store_y<YB>(Y, at, 4, true, v);
    } else {
        for (size_t i = at; i < all && i < at + 4; i++) {
            v4f v = {part[i], 0.0f, 0.0f, 0.0f};
            for (int p = 1; p < parts; p++)
                v[0] += part[p * all + i];
            store_y<YB>(Y, i, 1, false, v);
        }
    }
}

// 256 x 256 for bf16 outputs: eight waves of 128 features x 64 tokens, in 8-bit
// products.  What bounds it is LDS: 64 KB in and 192 KB out a block for 2048 cycles of
// a SIMD's products, half of what tiles of 128 x 128 take a product.  The tokens'
// operands of a block stay in registers, the features' pass through two places; the
// next block is waited for before the last 16 features, beside which its first
// operands are read into what they leave.
template <bool YB, bool CUT>
__global__ __launch_bounds__(512, 1) void k_block_big(void *__restrict__ Y, const uint8_t *__restrict__ X, const float *__restrict__ sx,
                                                      const uint8_t *__restrict__ W, const float *__restrict__ sw, int M, int N, int K,
                                                      int tiles_m, int tiles_n)
{
    constexpr int BT = 256, BF = 256, NW = 8, NS = 2, TF = 8, TT = 4, LAG = 3;
    using In = Loader<BT, BF, NW, NS, CUT>;
    extern __shared__ __align__(1024) uint8_t lds_dyn[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    int tm, tn;
    tile_of(tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BT, n0 = tn * BF, wf = wave >> 2, wt = wave & 3, kb = (K + kBlock - 1) / kBlock;
    In in;
    in.init(X, W, sx, M, N, K, m0, n0, wave, lane);
    const float *swp = sw + (size_t)min(n0 / kBlock + wf, (N - 1) / kBlock) * kb;
    const int xrow = wt * TT * 16, wrow = BT + wf * TF * 16;
    const uint32_t xlo = (xrow + r) * 128 + chunk_slot(r, 2 * g) * 16, wlo = xlo + (wrow - xrow) * 128, slo = In::ROWS * 128 + (xrow + r) * 4;
    v4f acc[TF][TT], t[LAG + 1];
#pragma unroll
    for (int i = 0; i < TF; i++)
#pragma unroll
        for (int j = 0; j < TT; j++)
            acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i <= LAG; i++)
        t[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    auto operand = [&](const uint8_t *lo, const uint8_t *hi, int up) {
        const v4i a = *(const v4i *)(lo + up), b = *(const v4i *)(hi + up);
        return Codes{v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
    };
    Codes A[2], B[TT];
    float s[TT], sc[TT], before[TT];
#pragma unroll
    for (int j = 0; j < TT; j++)
        before[j] = sc[j] = 0.0f;
    in.issue(lds_dyn, 0, 0);
    if (kb > 1) {
        in.issue(lds_dyn, 1, 1);
        stage_barrier<In::kLoads>();
    } else {
        stage_barrier<0>();
    }
    A[0] = operand(lds_dyn + wlo, lds_dyn + (wlo ^ 16), 0);
#pragma unroll
    for (int j = 0; j < TT; j++) {
        B[j] = operand(lds_dyn + xlo, lds_dyn + (xlo ^ 16), 2048 * j);
        s[j] = *(const float *)(lds_dyn + slo + 64 * j);
    }
    float swv = swp[0];
#pragma unroll 1
    for (int b = 0; b < kb; b++) {
        uint32_t off = (uint32_t)(b % NS) * In::SBYTES, noff = (uint32_t)((b + 1) % NS) * In::SBYTES;
        asm volatile("" : "+s"(off), "+s"(noff));
        const uint8_t *w0 = lds_dyn + off + wlo, *w1 = lds_dyn + off + (wlo ^ 16);
#pragma unroll
        for (int j = 0; j < TT; j++) {
            before[j] = sc[j];
            sc[j] = s[j] * swv;
        }
        swv = swp[min(b + 1, kb - 1)];
#pragma unroll
        for (int i = 0; i < TF; i++) {
            if (i + 1 < TF) {
                A[(i + 1) & 1] = operand(w0, w1, 2048 * (i + 1));
            } else {
                // every wave has the rest of block b in registers, and block b + 1 is there
                stage_barrier<0>();
                in.issue(lds_dyn, min(b + 2, kb - 1), b);
                // (past the last block: some block's codes, not used)
                A[(i + 1) & 1] = operand(lds_dyn + noff + wlo, lds_dyn + noff + (wlo ^ 16), 0);
            }
            // (in program order: the compiler would read all operands at once, for which
            // it has no registers)
            {
                constexpr int n = TF * TT;
                auto old = [&](int j) -> v4f & { return acc[(i * TT + n - 1 - LAG - j) % n / TT][(i * TT + n - 1 - LAG - j) % TT]; };
                asm volatile("" : "+v"(A[i & 1].w), "+v"(old(0)), "+v"(old(1)), "+v"(old(2)), "+v"(old(3))::"memory");
            }
#pragma unroll
            for (int j = 0; j < TT; j++) {
                const int q = i * TT + j, p = (q + TF * TT - LAG) % (TF * TT);
                t[q % (LAG + 1)] = block_sum(A[i & 1], B[j]);
                if (i + 1 == TF) {
                    B[j] = operand(lds_dyn + noff + xlo, lds_dyn + noff + (xlo ^ 16), 2048 * j);
                    s[j] = *(const float *)(lds_dyn + noff + slo + 64 * j);
                }
                // the tile three before, of the block before where this one begins
#pragma unroll
                for (int e = 0; e < 4; e++)
                    acc[p / TT][p % TT][e] = __fmaf_rn(t[p % (LAG + 1)][e], q < LAG ? before[p % TT] : sc[p % TT], acc[p / TT][p % TT][e]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
#pragma unroll
    for (int p = TF * TT - LAG; p < TF * TT; p++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            acc[p / TT][p % TT][e] = __fmaf_rn(t[p % (LAG + 1)][e], sc[p % TT], acc[p / TT][p % TT][e]);
    stage_barrier<0>();        // (the loads past the last block)
    const bool words = N % 4 == 0 && n0 + BF <= N;           // whole tiles, rows on 16 (8) bytes
#pragma unroll
    for (int j = 0; j < TT; j++) {
        const int tok = m0 + xrow + 16 * j + r;
        if (tok >= M)
            continue;
#pragma unroll
        for (int i = 0; i < TF; i++) {
            const int n = n0 + wf * TF * 16 + 16 * i + 4 * g;
            store_y<YB>(Y, (size_t)tok * N + n, N - n, words, acc[i][j]);
        }
    }
}

// The largest of each half of a wave, in its last lane.
template <int N>
__device__ __forceinline__ void half_max(float (&v)[N])
{
    auto step = [&](auto ctrl, auto rows) {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] = fmaxf(v[i], dpp_mov<decltype(ctrl)::value, decltype(rows)::value>(0.0f, v[i]));
    };
    using All = std::integral_constant<int, 0xF>;
    step(std::integral_constant<int, 0x111>(), All());
    step(std::integral_constant<int, 0x112>(), All());
    step(std::integral_constant<int, 0x114>(), All());
    step(std::integral_constant<int, 0x118>(), All());
    step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xA>());
}

// Up to 16 tokens: HBM bound.  A workgroup of eight waves takes 16 features; the waves
// take the blocks of 128 in turn, every load of a wave's next kAhead blocks in flight,
// and their sums are added up in LDS in their order.  Exact sums (bf16 products) cost
// nothing here.  With XT (0: codes; fp32, bf16) the activations' codes are formed by the
// wave that needs them, for one or two tokens.  Every workgroup does that for all of
// them, 2 us of its time, as long as there is one a CU no more than a launch of its own
// takes (fp32, calls: 4096 x 4096 8.8 us, in two launches 10.5; 14336 x 4096 20 - 25 and
// 20).  4096 x 4096 from codes 5.1 us, 3.3 TB/s.
template <bool YB, int XT>
__global__ __launch_bounds__(512) void k_block_few(void *__restrict__ Y, const void *__restrict__ X, const float *__restrict__ sx,
                                                   const uint8_t *__restrict__ W, const float *__restrict__ sw, int M, int N, int K,
                                                   size_t x_stride)
{
    constexpr int NW = 8, kAhead = 4, kCoded = 2;
    __shared__ float sum[NW][16][17];
    __shared__ __align__(16) uint32_t own[XT ? NW : 1][XT ? kAhead : 1][kCoded][kBlock / 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16;
    const int kb = (K + kBlock - 1) / kBlock;
    const uint8_t *wp = W + (size_t)min(n0 + r, N - 1) * K + 16 * g;
    const size_t tok = min(r, M - 1);
    const float *swp = sw + (size_t)(n0 / kBlock) * kb;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    // codes 16 g .. and 64 + 16 g .. of a block
    auto load = [&](const uint8_t *p, int b) {
        const int k = b * kBlock + 16 * g;
        const v4i zero = {0, 0, 0, 0};
        const v4i lo = k < K ? *(const v4i *)(p + (size_t)b * kBlock) : zero;
        const v4i hi = k + 64 < K ? *(const v4i *)(p + (size_t)b * kBlock + 64) : zero;
        return Codes{v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
    };
    // four elements of token `row` of a block
    auto activations = [&](int row, int b) {
        const int k = b * kBlock + 4 * (lane & 31);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < K) {
            const size_t at = (size_t)min(row, M - 1) * x_stride + k;
            if constexpr (XT == 2) {
                uint16_t u[4];
                __builtin_memcpy(u, (const uint16_t *)X + at, 8);
                v = make_float4(bf16_to_f32(u[0]), bf16_to_f32(u[1]), bf16_to_f32(u[2]), bf16_to_f32(u[3]));
            } else {
                __builtin_memcpy(&v, (const float *)X + at, 16);
            }
        }
        return v;
    };
    for (int b0 = wave; b0 < kb; b0 += NW * kAhead) {
        Codes w[kAhead], x[XT ? 1 : kAhead];
        float s[kAhead];
        float4 v[XT ? kAhead : 1];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int b = min(b0 + NW * i, kb - 1);
            w[i] = load(wp, b);
            s[i] = swp[b];
            if constexpr (XT) {
                v[i] = activations(lane >> 5, b);
            } else {
                x[i] = load((const uint8_t *)X + tok * K + 16 * g, b);
                s[i] *= sx[tok * kb + b];
            }
        }
        if constexpr (XT) {
            // half a wave a token; all blocks beside each other
            float top[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                top[i] = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
            half_max(top);
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(top[i]), 31));
                const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(top[i]), 63));
                const float m = lane < 32 ? a : c, scale = m > 0.0f ? m / 224.0f : 1.0f, inv = m > 0.0f ? 1.0f / scale : 1.0f;
                const float mine = r ? c : a;                   // the token of the lane's column
                s[i] *= mine > 0.0f ? mine / 224.0f : 1.0f;
                const float e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                own[wave][i][lane >> 5][lane & 31] = scaled_to_fp8(e, inv);
            }
            // (the wave's own: what it wrote is there once its writes are)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (b0 + NW * i >= kb)
                break;
            Codes xc;
            if constexpr (XT) {
                const uint32_t *o = own[wave][i][min(r, kCoded - 1)];
                const v4i lo = *(const v4i *)(o + 4 * g), hi = *(const v4i *)(o + 16 + 4 * g);
                xc.w = v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            } else {
                xc = x[i];
            }
            Wide a, c;
            widen(w[i], a);
            widen(xc, c);
            const v4f t = block_sum(a, c);
#pragma unroll
            for (int e = 0; e < 4; e++)
                acc[e] = __fmaf_rn(t[e], s[i], acc[e]);
        }
        asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        sum[wave][r][4 * g + e] = acc[e];
    __syncthreads();
    if (threadIdx.x < 256) {
        const int t = threadIdx.x >> 4, f = threadIdx.x & 15, n = n0 + f;
        float v = sum[0][t][f];
#pragma unroll
        for (int w = 1; w < NW; w++)
            v += sum[w][t][f];
        if (t < M && n < N) {
            if (YB)
                ((uint16_t *)Y)[(size_t)t * N + n] = f32_to_bf16(v);
            else
                ((float *)Y)[(size_t)t * N + n] = v;
        }
    }
}

struct BlockArgs {
    void *y;
    const uint8_t *xq;
    const float *sx;
    const uint8_t *wq;
    const float *sw;
    int m, n, k;
    float *part;              // [parts][m][n] where there are several
    int parts, n0;            // n0: the first feature of the launch
    hipStream_t s;
};

template <bool F8, bool YB, int WF, int WT, int TF, int TT, int NS>
static void launch_dma(const BlockArgs &a)
{
    constexpr int BF = WF * TF * 16, BT = WT * TT * 16;
    constexpr int lds = NS * Loader<BT, BF, WF * WT, NS, false>::SBYTES;
    static_assert(lds <= 160 * 1024, "LDS budget");
    const int tm = (a.m + BT - 1) / BT, tn = (a.n - a.n0 + BF - 1) / BF;
    auto go = [&](auto *fn) {
        (void)hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(fn, dim3((unsigned)tm * tn, a.parts), dim3(WF * WT * 64), lds, a.s, a.parts > 1 ? a.part : a.y, a.xq, a.sx, a.wq,
                           a.sw, a.m, a.n, a.k, tm, tn, a.n0 / BF);
    };
    auto of_k = [&](auto part) {
        constexpr bool PART = decltype(part)::value;
        a.k % kBlock ? go(k_block_dma<F8, YB, WF, WT, TF, TT, NS, true, PART>) : go(k_block_dma<F8, YB, WF, WT, TF, TT, NS, false, PART>);
    };
    a.parts > 1 ? of_k(std::true_type()) : of_k(std::false_type());
    if (a.parts > 1) {
        const size_t all = (size_t)a.m * a.n;
        hipLaunchKernelGGL(k_block_join<YB>, dim3((unsigned)((all + 1023) / 1024)), dim3(256), 0, a.s, a.y, a.part, all, a.parts);
    }
}

template <bool YB>
static void launch_big(void *y, const uint8_t *xq, const float *sx, const uint8_t *wq, const float *sw, int m, int n, int k, int tn,
                       hipStream_t s)
{
    constexpr int lds = 2 * Loader<256, 256, 8, 2, false>::SBYTES;
    const int tm = (m + 255) / 256;
    auto go = [&](auto *fn) {
        (void)hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(fn, dim3((unsigned)tm * tn), dim3(512), lds, s, y, xq, sx, wq, sw, m, n, k, tm, tn);
    };
    k % kBlock ? go(k_block_big<YB, true>) : go(k_block_big<YB, false>);
}

// Tiles (tokens x features; places of the ring) and what a block of 128 takes, in us,
// where a CU has one workgroup of theirs and where it has two (0: LDS holds one), for
// fp32 and bf16 outputs.  From 261 x 2064 x 14352, 1024 x 4096 x 4096 and 8192^3.
enum Tile { kTile64, kTile64x128, kTile128, kTile128Deep, kTile256, kTiles };
struct TileTime {
    int bt, bf;
    float one[2], two[2];
};
constexpr TileTime kTileTime[kTiles] = {
    {64, 64, {0.50f, 0.42f}, {0.74f, 0.61f}},      // NS 4
    {64, 128, {0.78f, 0.57f}, {1.13f, 0.81f}},     // NS 3
    {128, 128, {1.23f, 1.04f}, {1.90f, 1.27f}},    // NS 2
    {128, 128, {1.25f, 0.80f}, {0.0f, 0.0f}},      // NS 4
    {256, 256, {0.0f, 2.09f}, {0.0f, 0.0f}},       // NS 2, bf16 outputs
};
struct Plan {
    Tile tile;
    int parts;                // of the blocks, joined by a launch of their own
    int front;                // tiles of 256 features that a launch of 256 x 256 takes before
};

// The tile, and the parts that the blocks are cut into where there are few tiles, that
// take the least time, with 3 us for a launch and 5 TB/s for the parts' sums.  (bf16
// outputs, by the tile that it takes and by others, in us: 64 x 4096 x 4096 in 4 parts
// 10.7, in one 13.2; 261 x 2064 x 14352 30.9 in 3 parts of 64 x 128, 52.6 in one of 64 x
// 64, 67.5 in 2 of 128 x 128; 512 x 4096 x 4096 19.4, 26.4 in 128 x 128; 1024 30.0 in
// deep 128 x 128, 34.9 in 64 x 128; 2048 x 14336 x 4096 141 in 256 x 256, 168 in 128 x
// 128; 8192^3 532, 648; 4096 x 14336 x 4096 272, with the codes, in three rounds of 256 x
// 256 and 2048 features in 128 x 128, all in 256 x 256 283.)
static Plan plan_block(long m, long n, long k, bool yb)
{
    const long blocks = (k + kBlock - 1) / kBlock;
    Plan best = {kTile64, 1, 0};
    double least = 1e30;
    for (int t = 0; t < kTiles; t++) {
        const TileTime &x = kTileTime[t];
        if (!(x.one[yb] > 0.0f))
            continue;
        const long tiles = ((m + x.bt - 1) / x.bt) * ((n + x.bf - 1) / x.bf);
        for (int parts = 1; parts <= 8 && parts * 4 <= std::max(blocks, 4L); parts++) {
            if (t == kTile256 && parts > 1)
                break;
            const long wgs = tiles * parts, each = (blocks + parts - 1) / parts;
            double us;
            if (wgs <= 256 || !(x.two[yb] > 0.0f))
                us = (double)((wgs + 255) / 256) * each * x.one[yb];
            else
                us = std::max(1.0, (double)((wgs + 511) / 512)) * each * x.two[yb];
            us += 3.0;
            if (parts > 1)
                us += 3.0 + 8.0 * parts * m * n / 5e6;
            if (us < least) {
                least = us;
                best = {(Tile)t, parts, 0};
            }
        }
    }
    if (best.tile != kTile256)
        return best;
    // whole rounds of the 256 CUs, and what is left of the features in smaller tiles
    const long tm = (m + 255) / 256, tn = (n + 255) / 256, rounds = (tm * tn + 255) / 256;
    for (long r = rounds - 1; r > 0 && r > rounds - 3; r--) {
        const long front = std::min<long>(256 * r / tm, tn - 1);
        if (front <= 0)
            break;
        const double before = 3.0 + (double)((tm * front + 255) / 256) * blocks * kTileTime[kTile256].one[yb];
        for (int t = 0; t < kTile256; t++) {
            const TileTime &x = kTileTime[t];
            const long wgs = ((m + x.bt - 1) / x.bt) * ((n - 256 * front + x.bf - 1) / x.bf);
            const bool two = wgs > 256 && x.two[yb] > 0.0f;
            const double us = before + 3.0 + (double)((wgs + (two ? 511 : 255)) / (two ? 512 : 256)) * blocks * (two ? x.two : x.one)[yb];
            if (us < least) {
                least = us;
                best = {(Tile)t, 1, (int)front};
            }
        }
    }
    return best;
}

constexpr int kFew = 16;      // tokens of k_block_few
static bool few_coded(long m, long n) { return m <= 2 && n <= 16 * 256; }      // and their codes formed there

static size_t parts_bytes(long m, long n, long k, bool yb)
{
    const Plan p = plan_block(m, n, k, yb);
    return m > kFew && p.parts > 1 ? (size_t)p.parts * m * n * sizeof(float) : 0;
}

template <bool YB, int XT>
static void launch_few(const BlockArgs &a, const void *x, size_t x_stride)
{
    hipLaunchKernelGGL((k_block_few<YB, XT>), dim3((unsigned)((a.n + 15) / 16)), dim3(512), 0, a.s, a.y, x, a.sx, a.wq, a.sw, a.m, a.n, a.k,
                       x_stride);
}

template <bool YB>
static void block_gemm_of(BlockArgs a, void *workspace)
{
    if (a.m <= kFew) {
        launch_few<YB, 0>(a, a.xq, 0);
        return;
    }
    constexpr bool F8 = YB;
    Plan p = plan_block(a.m, a.n, a.k, YB);
    a.parts = p.parts;
    a.part = (float *)workspace;
    a.n0 = 256 * p.front;
    if constexpr (YB)
        if (p.front || p.tile == kTile256)
            launch_big<true>(a.y, a.xq, a.sx, a.wq, a.sw, a.m, a.n, a.k, p.front ? p.front : (a.n + 255) / 256, a.s);
    switch (p.tile) {
    case kTile64: launch_dma<F8, YB, 2, 2, 2, 2, 4>(a); break;
    case kTile64x128: launch_dma<F8, YB, 2, 2, 4, 2, 3>(a); break;
    case kTile128: launch_dma<F8, YB, 2, 2, 4, 4, 2>(a); break;
    case kTile128Deep: launch_dma<F8, YB, 2, 2, 4, 4, 4>(a); break;
    default: break;
    }
}

static void block_gemm(void *y, bool yb, const uint8_t *xq, const float *sx, const uint8_t *wq, const float *sw, int m, int n,
                       int k, void *workspace, hipStream_t s)
{
    const BlockArgs a = {y, xq, sx, wq, sw, m, n, k, nullptr, 1, 0, s};
    yb ? block_gemm_of<true>(a, workspace) : block_gemm_of<false>(a, workspace);
}

// Codes [m][k], then scales [m][blocks], of a call's activations; none where the product
// forms them.
static size_t codes_bytes(long m, long n, long k)
{
    const size_t codes = ((size_t)m * k + 15) / 16 * 16;
    return few_coded(m, n) ? 0 : (codes + (size_t)m * ((k + kBlock - 1) / kBlock) * sizeof(float) + 15) / 16 * 16;
}

// The workspace that a call takes, or the library's.
static int take_workspace(const char *who, void *&workspace, size_t bytes, size_t need, hipStream_t s)
{
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && bytes >= need),
               "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", who, bytes, need);
    // (whether or not these sizes use it)
    BE42_CHECK(workspace || !captured(s), "%s: a captured call needs a workspace of the caller's", who);
    if (!workspace && need > 16 && !(workspace = be42::workspace(need, s)))
        return BE42_ENOMEM;
    return BE42_OK;
}

static int check_shape(const char *who, long m, long n, long k)
{
    BE42_CHECK(m >= 0 && n > 0 && k > 0 && k % 16 == 0 && k <= kMaxK, "%s: m %ld, n %ld, k %ld (k a multiple of 16, at most 2^22)", who, m, n, k);
    // (workgroups of up to 512 threads)
    BE42_CHECK(((m + 31) / 32) * ((n + 15) / 16) <= kMaxBlocks / 2, "%s: m %ld, n %ld", who, m, n);
    return BE42_OK;
}

}  // namespace be42

using namespace be42;

extern "C" size_t be42_gemm_fp8_block_workspace_bytes(int m, int n, int k, int y_bf16)
{
    if (m <= 0 || n <= 0 || k <= 0 || k % 16 || k > kMaxK)
        return 0;
    return 16 + parts_bytes(m, n, k, y_bf16);
}

extern "C" int be42_gemm_fp8_block(void *y, int y_bf16, const uint8_t *xq, const float *sx, const uint8_t *wq,
                                   const float *sw, int m, int n, int k, void *workspace, size_t workspace_bytes, void *stream)
{
    BE42_CHECK(m == 0 || (y && xq && sx && wq && sw), "be42_gemm_fp8_block: null pointer");
    if (const int rc = check_shape("be42_gemm_fp8_block", m, n, k))
        return rc;
    BE42_CHECK(!(((uintptr_t)xq | (uintptr_t)wq | (uintptr_t)y) & 15) && !(((uintptr_t)sx | (uintptr_t)sw) & 3),
               "be42_gemm_fp8_block: unaligned pointer");
    if (m == 0)
        return BE42_OK;
    hipStream_t s = as_stream(stream);
    if (const int rc = take_workspace("be42_gemm_fp8_block", workspace, workspace_bytes,
                                      be42_gemm_fp8_block_workspace_bytes(m, n, k, y_bf16), s))
        return rc;
    block_gemm(y, y_bf16, xq, sx, wq, sw, m, n, k, workspace, s);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

extern "C" size_t be42_linear_fp8_block_workspace_bytes(int m, int n, int k, int y_bf16)
{
    const size_t product = be42_gemm_fp8_block_workspace_bytes(m, n, k, y_bf16);
    return product ? product + codes_bytes(m, n, k) : 0;
}

extern "C" int be42_linear_fp8_block(void *y, int y_bf16, const void *x, int x_bf16, int x_stride, const uint8_t *wq,
                                     const float *sw, int m, int n, int k, void *workspace, size_t workspace_bytes,
                                     void *stream)
{
    BE42_CHECK(m == 0 || (y && x && wq && sw), "be42_linear_fp8_block: null pointer");
    if (const int rc = check_shape("be42_linear_fp8_block", m, n, k))
        return rc;
    BE42_CHECK(x_stride >= k, "be42_linear_fp8_block: rows of %d at stride %d", k, x_stride);
    BE42_CHECK(!(((uintptr_t)wq | (uintptr_t)y) & 15) && !((uintptr_t)sw & 3) && !((uintptr_t)x & (x_bf16 ? 1 : 3)),
               "be42_linear_fp8_block: unaligned pointer");
    if (m == 0)
        return BE42_OK;
    hipStream_t s = as_stream(stream);
    if (const int rc = take_workspace("be42_linear_fp8_block", workspace, workspace_bytes,
                                      be42_linear_fp8_block_workspace_bytes(m, n, k, y_bf16), s))
        return rc;
    if (few_coded(m, n)) {
        int dev = 0;
        BE42_HIP(hipGetDevice(&dev));
        if (const int rc = upload_fp8_thresholds(dev))
            return rc;
        const BlockArgs a = {y, nullptr, nullptr, wq, sw, m, n, k, nullptr, 1, 0, s};
        if (y_bf16)
            x_bf16 ? launch_few<true, 2>(a, x, x_stride) : launch_few<true, 1>(a, x, x_stride);
        else
            x_bf16 ? launch_few<false, 2>(a, x, x_stride) : launch_few<false, 1>(a, x, x_stride);
        BE42_LAUNCH_CHECK();
        return BE42_OK;
    }
    uint8_t *q = (uint8_t *)workspace;
    float *scales = (float *)(q + ((size_t)m * k + 15) / 16 * 16);
    if (const int rc = be42_quant_blocks_fp8(q, scales, x, x_bf16, x_stride, m, k, stream))
        return rc;
    block_gemm(y, y_bf16, q, scales, wq, sw, m, n, k, q + codes_bytes(m, n, k), s);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
