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

namespace be42 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 128;

// eight E4M3 codes as bf16 (exact)
__device__ __forceinline__ bf16x8 codes_bf16(uint2 c)
{
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, 1.0f, true);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, 1.0f, false), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// A tile of 64 tokens x 64 features, a wave 32 x 32 of them: rows of the product are
// features, columns tokens, so that a lane has one token and its scale.
template <bool YB>
__global__ __launch_bounds__(256) void k_block_mm(void *__restrict__ Y, const uint8_t *__restrict__ X, const float *__restrict__ sx,
                                                  const uint8_t *__restrict__ W, const float *__restrict__ sw, int M, int N, int K,
                                                  int tiles_m)
{
    constexpr int LD = kBlock + 16;
    __shared__ __align__(16) uint8_t lx[64 * LD], lw[64 * LD];
    const int m0 = (int)(blockIdx.x % (unsigned)tiles_m) * 64, n0 = (int)(blockIdx.x / (unsigned)tiles_m) * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1, kb = (K + kBlock - 1) / kBlock;
    const int tok = min(m0 + 32 * wm + r, M - 1);
    v16f acc = {};
    for (int b = 0; b < kb; b++) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 8; i += 256) {
            const int row = i >> 3, col = b * kBlock + (i & 7) * 16;
            const v4i zero = {0, 0, 0, 0};
            *(v4i *)(lx + row * LD + (i & 7) * 16) = col < K ? *(const v4i *)(X + (size_t)min(m0 + row, M - 1) * K + col) : zero;
            *(v4i *)(lw + row * LD + (i & 7) * 16) = col < K ? *(const v4i *)(W + (size_t)min(n0 + row, N - 1) * K + col) : zero;
        }
        __syncthreads();
        v16f t = {};
#pragma unroll
        for (int s = 0; s < 8; s++) {
            const bf16x8 w = codes_bf16(*(const uint2 *)(lw + (32 * wn + r) * LD + 16 * s + 8 * h));
            const bf16x8 x = codes_bf16(*(const uint2 *)(lx + (32 * wm + r) * LD + 16 * s + 8 * h));
            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, t, 0, 0, 0);
        }
        const float sc = sx[(size_t)tok * kb + b] * sw[(size_t)(n0 / kBlock) * kb + b];
#pragma unroll
        for (int i = 0; i < 16; i++)
            acc[i] = __fmaf_rn(t[i], sc, acc[i]);
    }
    if (m0 + 32 * wm + r >= M)
        return;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int n = n0 + 32 * wn + 8 * (i / 4) + 4 * h + i % 4;
        if (n < N) {
            if (YB)
                ((uint16_t *)Y)[(size_t)tok * N + n] = f32_to_bf16(acc[i]);
            else
                ((float *)Y)[(size_t)tok * N + n] = acc[i];
        }
    }
}

static void block_gemm(void *y, bool yb, const uint8_t *xq, const float *sx, const uint8_t *wq, const float *sw, int m, int n,
                       int k, hipStream_t s)
{
    const int tm = (m + 63) / 64, tn = (n + 63) / 64;
    if (yb)
        hipLaunchKernelGGL(k_block_mm<true>, dim3((unsigned)tm * tn), dim3(256), 0, s, y, xq, sx, wq, sw, m, n, k, tm);
    else
        hipLaunchKernelGGL(k_block_mm<false>, dim3((unsigned)tm * tn), dim3(256), 0, s, y, xq, sx, wq, sw, m, n, k, tm);
}

// Codes [m][k], then scales [m][blocks], of a call's activations.
static size_t codes_bytes(long m, long k) { return ((size_t)m * k + 15) / 16 * 16; }

static int check_shape(const char *who, long m, long n, long k)
{
    BE42_CHECK(m >= 0 && n > 0 && k > 0 && k % 16 == 0, "%s: m %ld, n %ld, k %ld (k a multiple of 16)", who, m, n, k);
    BE42_CHECK(((m + 63) / 64) * ((n + 63) / 64) <= kMaxBlocks, "%s: m %ld, n %ld", who, m, n);
    return BE42_OK;
}

}  // namespace be42

using namespace be42;

extern "C" int be42_gemm_fp8_block(void *y, int y_bf16, const uint8_t *xq, const float *sx, const uint8_t *wq,
                                   const float *sw, int m, int n, int k, void *stream)
{
    BE42_CHECK(m == 0 || (y && xq && sx && wq && sw), "be42_gemm_fp8_block: null pointer");
    if (const int rc = check_shape("be42_gemm_fp8_block", m, n, k))
        return rc;
    BE42_CHECK(!(((uintptr_t)xq | (uintptr_t)wq | (uintptr_t)y) & 15) && !(((uintptr_t)sx | (uintptr_t)sw) & 3),
               "be42_gemm_fp8_block: unaligned pointer");
    if (m == 0)
        return BE42_OK;
    block_gemm(y, y_bf16, xq, sx, wq, sw, m, n, k, as_stream(stream));
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

extern "C" size_t be42_linear_fp8_block_workspace_bytes(int m, int n, int k)
{
    if (m <= 0 || n <= 0 || k <= 0 || k % 16)
        return 0;
    return 16 + codes_bytes(m, k) + (size_t)m * ((k + kBlock - 1) / kBlock) * sizeof(float);
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
    const size_t need = be42_linear_fp8_block_workspace_bytes(m, n, k);
    BE42_CHECK(!workspace || (!((uintptr_t)workspace & 15) && workspace_bytes >= need),
               "be42_linear_fp8_block: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    hipStream_t s = as_stream(stream);
    BE42_CHECK(workspace || !captured(s), "be42_linear_fp8_block: a captured call needs a workspace of the caller's");
    if (!workspace)
        workspace = be42::workspace(need, s);
    if (!workspace)
        return BE42_ENOMEM;
    uint8_t *q = (uint8_t *)workspace;
    float *scales = (float *)(q + codes_bytes(m, k));
    if (const int rc = be42_quant_blocks_fp8(q, scales, x, x_bf16, x_stride, m, k, stream))
        return rc;
    block_gemm(y, y_bf16, q, scales, wq, sw, m, n, k, s);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
