// quant.hip -- INT8 / FP8 E4M3 codecs of the reference, row-wise, on gfx950.
//
// quant_f32_to_int8  src/compute/ops_quant.c:229-270
// quant_f32_to_fp8   src/compute/ops_quant.c:103-136 (float_to_fp8 :68-98)
// g_fp8_lut          src/compute/ops_quant.c:18-63
//
// Codes and scales are bit-identical to the reference: the absmax is an exact
// max reduction, the divisions are IEEE divisions, roundf rounds half away
// from zero, and the FP8 exponent reproduces glibc's floorf(log2f(a)) through
// a per-binade threshold table measured on the host at init.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "be42_common.h"

namespace be42 {

__constant__ float c_fp8_thr[kFp8ThrN];

// Reference E4M3 encoder (ops_quant.c:68-98) on the device.
__device__ __forceinline__ uint8_t f32_to_fp8(float v)
{
    if (v == 0.0f)
        return 0;
    const uint32_t sign = v < 0.0f ? 0x80u : 0u;
    float a = fabsf(v);
    if (a > 448.0f)
        a = 448.0f;
    int ex = (int)((__float_as_uint(a) >> 23) & 0xFF) - 127;   // floor(log2 a), a normal
    if ((__float_as_uint(a) >> 23) == 0)
        ex = -127;                                            // subnormal: far below e = 0
    const int up = ex + 1;
    // a threshold lies at most 64 ulps below its power of two
    // (host_fp8_thresholds), so the table is read for such values only
    if ((__float_as_uint(a) & 0x7FFFFFu) >= 0x7FFFC0u && up >= kFp8ThrE0 && up < kFp8ThrE0 + kFp8ThrN &&
        a >= c_fp8_thr[up - kFp8ThrE0])
        ex = up;                                              // log2f rounded up to an integer
    int e = ex + 7;
    e = e < 0 ? 0 : (e > 15 ? 15 : e);
    const float frac = (e == 0) ? a * 64.0f
                                : a * __uint_as_float((uint32_t)(127 + 7 - e) << 23) - 1.0f;
    int m = (int)__fmaf_rn(frac, 8.0f, 0.5f);
    if (m > 7)
        m = 7;
    return (uint8_t)(sign | ((uint32_t)e << 3) | (uint32_t)m);
}

// f32_to_fp8 of a finite value in half the instructions: the kept mantissa bits
// are counted up by the next bit unless they are all ones (8 frac + 0.5 is exact
// in fp32, so its integer part is that).  Compared with it over all fp32 values;
// the pass over 300 x 14336 fp32 15.3 -> 14.7 us.
__device__ __forceinline__ uint8_t finite_to_fp8(float v)
{
    const float a = fminf(fabsf(v), 448.0f);
    const uint32_t u = __float_as_uint(a);
    int ex = (int)(u >> 23) - 127;
    uint32_t c = (u >> 20) - ((127u - 7u) << 3) + ((u & 0x700000u) != 0x700000u ? u >> 19 & 1u : 0u);
    if ((u & 0x7FFFFFu) >= 0x7FFFC0u && ex + 1 >= kFp8ThrE0 && ex + 1 < kFp8ThrE0 + kFp8ThrN &&
        a >= c_fp8_thr[ex + 1 - kFp8ThrE0]) {
        ex++;                                              // log2f rounded up to an integer
        c = (uint32_t)(ex + 7) << 3;
    }
    if (ex < -6)                                           // multiples of 2^-9
        c = (uint32_t)min((int)__fmaf_rn(a, 512.0f, 0.5f), 7);
    return (uint8_t)(a == 0.0f ? 0u : c | (__float_as_uint(v) >> 24 & 0x80u));
}

// quant_f32_to_int8's code of one element (ops_quant.c:262-267)
__device__ __forceinline__ int8_t f32_to_int8(float v, float inv)
{
    const int c = (int)roundf(v * inv);
    return (int8_t)(c > 127 ? 127 : (c < -127 ? -127 : c));
}

// block-wide absmax of one row (256 threads)
__device__ __forceinline__ float row_absmax(const float *x, int cols, float *red)
{
    float m = 0.0f;
    for (int i = threadIdx.x; i < cols; i += blockDim.x)
        m = fmaxf(m, fabsf(x[i]));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = m;
    __syncthreads();
    float r = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); w++)
        r = fmaxf(r, red[w]);
    return r;
}

__global__ __launch_bounds__(256) void k_quant_rows_int8(int8_t *q, float *scales, const float *x,
                                                         int cols)
{
    __shared__ float red[4];
    const size_t row = blockIdx.x;
    const float *xr = x + row * cols;
    const float amax = row_absmax(xr, cols, red);
    float scale = 1.0f, inv = 1.0f;
    if (amax > 0.0f) {
        scale = amax / 127.0f;
        inv = 127.0f / amax;
    }
    if (threadIdx.x == 0)
        scales[row] = scale;
    for (int i = threadIdx.x; i < cols; i += blockDim.x)
        q[row * cols + i] = f32_to_int8(xr[i], inv);
}

__global__ __launch_bounds__(256) void k_quant_rows_fp8(uint8_t *q, float *scales, const float *x,
                                                        int cols)
{
    __shared__ float red[4];
    const size_t row = blockIdx.x;
    const float *xr = x + row * cols;
    const float amax = row_absmax(xr, cols, red);
    float scale = 1.0f, inv = 1.0f;
    if (amax > 0.0f) {
        scale = amax / 224.0f;
        inv = 1.0f / scale;
    }
    if (threadIdx.x == 0)
        scales[row] = scale;
    for (int i = threadIdx.x; i < cols; i += blockDim.x)
        q[row * cols + i] = f32_to_fp8(xr[i] * inv);
}

// Both codecs on rows whose elements come four to an aligned word.  HBM bound
// (4 bytes in, 1 out per element): a block keeps its row in registers between
// the absmax and the codes, so the row is read once, by NV 16-byte loads per
// thread that are all in flight together, and leaves as 4-byte stores; the
// one-element loops above read it twice, a round trip per element.  A pass of
// quantize + product: FP8 8192 x 4096 x 14336 616 -> 559 us, INT8 500 x 4096 x
// 4096 29.3 -> 24.3 us (the product alone 22).
template <bool FP8, int NV>
__global__ __launch_bounds__(256) void k_quant_rows_vec(uint8_t *__restrict__ q, float *__restrict__ scales,
                                                        const float *__restrict__ x, int cols)
{
    __shared__ float red[4];
    const size_t row = blockIdx.x;
    const float4 *xr = (const float4 *)(x + row * cols);
    const int n4 = cols / 4;
    float4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = threadIdx.x + 256 * j;
        v[j] = i < n4 ? xr[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
        m = fmaxf(fmaxf(fmaxf(m, fabsf(v[j].x)), fmaxf(fabsf(v[j].y), fabsf(v[j].z))), fabsf(v[j].w));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = m;
    __syncthreads();
    const float amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float scale = 1.0f, inv = 1.0f;
    if (amax > 0.0f) {
        scale = amax / (FP8 ? 224.0f : 127.0f);
        inv = FP8 ? 1.0f / scale : 127.0f / amax;
    }
    if (threadIdx.x == 0)
        scales[row] = scale;
    uint32_t *qr = (uint32_t *)(q + row * cols);
    auto code = [&](float e) {
        return FP8 ? (uint32_t)f32_to_fp8(e * inv) : (uint32_t)(uint8_t)f32_to_int8(e, inv);
    };
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = threadIdx.x + 256 * j;
        if (i < n4)
            qr[i] = code(v[j].x) | code(v[j].y) << 8 | code(v[j].z) << 16 | code(v[j].w) << 24;
    }
}

// Rows of up to 16384 elements (16 words per thread) in 16-byte words; longer,
// odd or unaligned ones take the one-element kernels.
template <bool FP8>
static bool launch_quant_vec(uint8_t *q, float *scales, const float *x, int rows, int cols, hipStream_t s)
{
    const int nv = (cols / 4 + 255) / 256;
    if (cols % 4 || nv > 16 || (uintptr_t)x % 16 || (uintptr_t)q % 4)
        return false;
    const dim3 g(rows), b(256);
    if (nv <= 1)
        hipLaunchKernelGGL((k_quant_rows_vec<FP8, 1>), g, b, 0, s, q, scales, x, cols);
    else if (nv <= 4)
        hipLaunchKernelGGL((k_quant_rows_vec<FP8, 4>), g, b, 0, s, q, scales, x, cols);
    else if (nv <= 8)
        hipLaunchKernelGGL((k_quant_rows_vec<FP8, 8>), g, b, 0, s, q, scales, x, cols);
    else
        hipLaunchKernelGGL((k_quant_rows_vec<FP8, 16>), g, b, 0, s, q, scales, x, cols);
    return true;
}

// ---- residual + RMS norm + codes -----------------------------------------------
// h = x + residual in the stream's type, y = fp32(h / sqrt(mean h^2 + eps) * w)
// and the codec's code of y.  The sum of squares and the product are formed in
// 64 bits and rounded once to fp32, so y does not depend on how the row is split
// over threads, but where the product falls within 2^-50 of the middle between
// two fp32 values.

// element i of a row of the residual stream (fp32 or bf16) as fp32
template <bool BF16>
__device__ __forceinline__ float act_load(const void *p, size_t i)
{
    return BF16 ? bf16_to_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}

template <bool BF16>
__device__ __forceinline__ void act_store(void *p, size_t i, float v)
{
    if (BF16)
        ((uint16_t *)p)[i] = f32_to_bf16(v);
    else
        ((float *)p)[i] = v;
}

// x + r as the stream holds it
template <bool BF16>
__device__ __forceinline__ float act_add(float x, float r)
{
    return BF16 ? bf16_to_f32(f32_to_bf16(x + r)) : x + r;
}

__device__ __forceinline__ float norm_value(float h, double r, uint16_t w)
{
    return (float)((double)h * r * (double)bf16_to_f32(w));
}

// Any row: three passes over it, one element a thread (whose place passes 2^31
// behind the longest rows).  (1024 threads: one row of
// 70000 fp32 46 us, 2000 rows 629; 256 threads 156 and 752.)
template <bool FP8, bool BF16>
__global__ __launch_bounds__(1024) void k_norm_quant_rows(uint8_t *q, float *scales, void *sum, const void *x,
                                                          size_t x_stride, const void *res, size_t res_stride,
                                                          const uint16_t *w, int cols, float eps)
{
    __shared__ double redd[16];
    __shared__ float red[16];
    const size_t row = blockIdx.x;
    auto load = [&](unsigned i) {
        const float v = act_load<BF16>(x, row * x_stride + i);
        return res ? act_add<BF16>(v, act_load<BF16>(res, row * res_stride + i)) : v;
    };
    // after the first pass the new stream is read where it was written (it may
    // have replaced x or the residual)
    auto again = [&](unsigned i) { return sum ? act_load<BF16>(sum, row * cols + i) : load(i); };
    double ss = 0.0;
    for (unsigned i = threadIdx.x; i < (unsigned)cols; i += 1024) {
        const float h = load(i);
        if (sum)
            act_store<BF16>(sum, row * cols + i, h);
        ss = fma((double)h, (double)h, ss);
    }
    ss = wave_sum_d(ss);
    if ((threadIdx.x & 63) == 0)
        redd[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = redd[0];
#pragma unroll
    for (int x = 1; x < 16; x++)
        ss += redd[x];
    const double r = 1.0 / sqrt(ss / cols + (double)eps);
    float m = 0.0f;
    for (unsigned i = threadIdx.x; i < (unsigned)cols; i += 1024)
        m = fmaxf(m, fabsf(norm_value(again(i), r, w[i])));
    m = wave_top(m);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = m;
    __syncthreads();
    float amax = red[0];
#pragma unroll
    for (int x = 1; x < 16; x++)
        amax = fmaxf(amax, red[x]);
    float scale = 1.0f, inv = 1.0f;
    if (amax > 0.0f) {
        scale = amax / (FP8 ? 224.0f : 127.0f);
        inv = FP8 ? 1.0f / scale : 127.0f / amax;
    }
    if (threadIdx.x == 0)
        scales[row] = scale;
    for (unsigned i = threadIdx.x; i < (unsigned)cols; i += 1024) {
        const float y = norm_value(again(i), r, w[i]);
        q[row * cols + i] = FP8 ? finite_to_fp8(y * inv) : (uint8_t)f32_to_int8(y, inv);
    }
}

// A row of up to NV words of VE elements a thread (16 bytes of fp32 or of bf16)
// is held in registers from the sum to the codes, so that x, the residual and w
// are read once, all in flight together.  TPR threads a row, 256 / TPR rows a
// block; threads of one wave need no barrier.
template <int TPR>
__device__ __forceinline__ double row_sum(double v, double *red)
{
    v = wave_sum_d(v);
    if constexpr (TPR > kWave) {
        if ((threadIdx.x & 63) == 0)
            red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TPR / kWave; w++)
            v += red[w];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float *red)
{
    v = wave_top(v);
    if constexpr (TPR > kWave) {
        if ((threadIdx.x & 63) == 0)
            red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TPR / kWave; w++)
            v = fmaxf(v, red[w]);
    }
    return v;
}

template <bool BF16, int VE>
struct Word {
    float v[VE];
    __device__ __forceinline__ void load(const void *p, size_t at)
    {
        if constexpr (VE == 1) {
            v[0] = act_load<BF16>(p, at);
        } else {
            const uint4 w = *(const uint4 *)((const char *)p + at * (BF16 ? 2 : 4));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < VE; j++)
                v[j] = __uint_as_float(!BF16 ? u[j % 4] : j & 1 ? u[j / 2] & 0xFFFF0000u : u[j / 2] << 16);
        }
    }
    __device__ __forceinline__ void store(void *p, size_t at) const
    {
        if constexpr (VE == 1) {
            act_store<BF16>(p, at, v[0]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                u[j] = !BF16 ? __float_as_uint(v[j])
                             : __float_as_uint(v[2 * j % VE]) >> 16 | (__float_as_uint(v[(2 * j + 1) % VE]) & 0xFFFF0000u);
            *(uint4 *)((char *)p + at * (BF16 ? 2 : 4)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
};

template <bool FP8, bool BF16, int VE, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_quant_vec(uint8_t *__restrict__ q, float *__restrict__ scales,
                                                                          void *sum, const void *x, size_t x_stride,
                                                                          const void *res, size_t res_stride,
                                                                          const uint16_t *__restrict__ w, int rows, int cols,
                                                                          float eps)
{
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    __shared__ double redd[TPR > kWave ? TPR / kWave : 1];
    __shared__ float red[TPR > kWave ? TPR / kWave : 1];
    const int t = threadIdx.x % TPR;
    const size_t row = (size_t)blockIdx.x * kRows + threadIdx.x / TPR;
    if (kRows > 1 && row >= (size_t)rows)
        return;                            // (whole waves, and no barrier follows)
    Word<BF16, VE> h[NV], r[NV];
    uint16_t wt[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = (t + TPR * j) * VE;
#pragma unroll
        for (int e = 0; e < VE; e++)
            h[j].v[e] = r[j].v[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < VE; e++)
            wt[j][e] = 0;
        if (i < cols) {
            h[j].load(x, row * x_stride + i);
            if (res)
                r[j].load(res, row * res_stride + i);
            __builtin_memcpy(wt[j], __builtin_assume_aligned(w + i, 2 * VE), 2 * VE);
        }
    }
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = (t + TPR * j) * VE;
        if (res)
#pragma unroll
            for (int e = 0; e < VE; e++)
                h[j].v[e] = act_add<BF16>(h[j].v[e], r[j].v[e]);
        if (sum && i < cols)
            h[j].store(sum, row * cols + i);
#pragma unroll
        for (int e = 0; e < VE; e++)
            ss = fma((double)h[j].v[e], (double)h[j].v[e], ss);
    }
    const double f = 1.0 / sqrt(row_sum<TPR>(ss, redd) / cols + (double)eps);
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < VE; e++) {
            h[j].v[e] = norm_value(h[j].v[e], f, wt[j][e]);
            m = fmaxf(m, fabsf(h[j].v[e]));
        }
    m = row_max<TPR>(m, red);
    float scale = 1.0f, inv = 1.0f;
    if (m > 0.0f) {
        scale = m / (FP8 ? 224.0f : 127.0f);
        inv = FP8 ? 1.0f / scale : 127.0f / m;
    }
    if (t == 0)
        scales[row] = scale;
    auto code = [&](float y) { return FP8 ? (uint32_t)finite_to_fp8(y * inv) : (uint32_t)(uint8_t)f32_to_int8(y, inv); };
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = (t + TPR * j) * VE;
        if constexpr (VE == 1) {
            if (i < cols)
                q[row * cols + i] = (uint8_t)code(h[j].v[0]);
        } else {
            uint32_t c[VE / 4];
#pragma unroll
            for (int e = 0; e < VE; e += 4)
                c[e / 4] = code(h[j].v[e]) | code(h[j].v[e + 1]) << 8 | code(h[j].v[e + 2]) << 16 | code(h[j].v[e + 3]) << 24;
            if (i < cols)
                __builtin_memcpy(__builtin_assume_aligned(q + row * cols + i, VE), c, VE);
        }
    }
}

// Rows of up to 32768 elements go in 16-byte words where every row of x, the
// residual, w and the outputs begins on one and has whole ones, and else, up to
// 16384, an element at a time; longer ones take the three passes above.
// The fewest threads that hold the row in four words each (a wave two, 512 eight):
// few large loads a thread and as many rows a CU as fit.  Measured, fp32 with a
// residual (the bytes of 8192 x 4096 at the rate of a large copy: 84 us):
//   1 x 4096 3.5 us, 2048 x 4096 18.6 (1024 threads the same and 22.1), 8192 x 4096 81
//   30000 x 512 35.9 (256 threads 49.9), 30000 x 256 18.4 (44.1)
//   2000 x 8192 to E4M3 40.8 (256 threads of eight words 48.8)
//   2000 x 12288 to E4M3 75.2 (1024 threads 81.2), 300 x 12288 14.1 (15.8)
//   2000 x 28672 158 (the three passes 295), one such row 9.2 (65)
//   3000 x 4099, element at a time, 45.6 (the three passes 63.3), 300 x 12289 18.7
//   (47.7)
// A few hundred rows are bound by one row's way through load, sum and maximum
// (1 x 8192: 4.5 us), very wide ones to E4M3 by the codec's instructions.
template <bool FP8, bool BF16>
static bool launch_norm_vec(uint8_t *q, float *scales, void *sum, const void *x, size_t x_stride, const void *res,
                            size_t res_stride, const uint16_t *w, int rows, int cols, float eps, hipStream_t s)
{
    constexpr int VE = BF16 ? 8 : 4;
    using std::integral_constant;
    constexpr integral_constant<int, VE> vec;
    constexpr integral_constant<int, 1> one;
    constexpr integral_constant<int, 2> two;
    constexpr integral_constant<int, 4> four;
    constexpr integral_constant<int, 8> eight;
    constexpr integral_constant<int, 64> wave;
    constexpr integral_constant<int, 256> some;
    constexpr integral_constant<int, 512> more;
    constexpr integral_constant<int, 1024> most;
    auto go = [&](auto ve, auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value;
        constexpr int per = TPR < 256 ? 256 / TPR : 1;
        hipLaunchKernelGGL((k_norm_quant_vec<FP8, BF16, decltype(ve)::value, TPR, decltype(nv)::value>),
                           dim3((rows + per - 1) / per), dim3(TPR < 256 ? 256 : TPR), 0, s, q, scales, sum, x, x_stride, res,
                           res_stride, w, rows, cols, eps);
        return true;
    };
    if (cols % VE || x_stride % VE || (res && res_stride % VE) ||
        (((uintptr_t)x | (uintptr_t)res | (uintptr_t)sum) & 15) || (uintptr_t)w % (2 * VE) || (uintptr_t)q % VE) {
        if (cols <= 64)
            return go(one, wave, one);
        if (cols <= 512)
            return go(one, some, two);
        if (cols <= 2048)
            return go(one, some, eight);
        if (cols <= 8192)
            return go(one, most, eight);
        return cols <= 16384 && go(one, most, integral_constant<int, 16>());
    }
    const int words = cols / VE;
    if (words <= 64)
        return go(vec, wave, one);
    if (words <= 128)
        return go(vec, wave, two);
    if (words <= 256)
        return go(vec, some, one);
    if (words <= 512)
        return go(vec, some, two);
    if (words <= 1024)
        return go(vec, some, four);
    if (words <= 2048)
        return go(vec, most, two);
    if (words <= 4096)
        return go(vec, more, eight);
    return !BF16 && words <= 8192 && go(vec, most, eight);
}

template <bool FP8>
static void launch_norm_quant(uint8_t *q, float *scales, void *sum, const void *x, size_t x_stride, const void *res,
                              size_t res_stride, bool bf16, const uint16_t *w, int rows, int cols, float eps,
                              hipStream_t s)
{
    const dim3 g(rows), b(1024);
    if (bf16 ? launch_norm_vec<FP8, true>(q, scales, sum, x, x_stride, res, res_stride, w, rows, cols, eps, s)
             : launch_norm_vec<FP8, false>(q, scales, sum, x, x_stride, res, res_stride, w, rows, cols, eps, s))
        return;
    if (bf16)
        hipLaunchKernelGGL((k_norm_quant_rows<FP8, true>), g, b, 0, s, q, scales, sum, x, x_stride, res, res_stride,
                           w, cols, eps);
    else
        hipLaunchKernelGGL((k_norm_quant_rows<FP8, false>), g, b, 0, s, q, scales, sum, x, x_stride, res, res_stride,
                           w, cols, eps);
}

__global__ void k_dequant_rows_int8(float *out, const int8_t *q, const float *scales, int cols,
                                    size_t total)
{
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (size_t)gridDim.x * blockDim.x)
        out[i] = (float)q[i] * scales[i / cols];
}

__global__ void k_fp8_decode(float *out, const uint8_t *q, size_t n)
{
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
         i += (size_t)gridDim.x * blockDim.x)
        out[i] = fp8_to_f32(q[i]);
}

// Threshold table of glibc's log2f: smallest float in [2^(E-1), 2^E) whose
// floorf(log2f()) is E (log2f rounds up within a few ulps of 2^E).
static void host_fp8_thresholds(float *thr)
{
    for (int i = 0; i < kFp8ThrN; i++) {
        const int E = kFp8ThrE0 + i;
        float a = ldexpf(1.0f, E);
        for (int step = 0; step < 64; step++) {
            const float b = nextafterf(a, 0.0f);
            if ((int)floorf(log2f(b)) != E)
                break;
            a = b;
        }
        thr[i] = a;
    }
}

static int g_thr_ready[64];

int upload_fp8_thresholds(int device)
{
    if (device < 0 || device >= 64)
        return BE42_EINVAL;
    if (g_thr_ready[device])
        return BE42_OK;
    float thr[kFp8ThrN];
    host_fp8_thresholds(thr);
    BE42_HIP(hipMemcpyToSymbol(HIP_SYMBOL(c_fp8_thr), thr, sizeof thr));
    g_thr_ready[device] = 1;
    return BE42_OK;
}

int fp8_thresholds_ready(int device) { return device >= 0 && device < 64 && g_thr_ready[device]; }

}  // namespace be42

using namespace be42;

static int ensure_thresholds()
{
    int dev = 0;
    BE42_HIP(hipGetDevice(&dev));
    if (!fp8_thresholds_ready(dev))
        return upload_fp8_thresholds(dev);
    return BE42_OK;
}

extern "C" int be42_quant_rows_int8(int8_t *q, float *scales, const float *x, int rows, int cols,
                                    void *stream)
{
    BE42_CHECK(q && scales && x, "be42_quant_rows_int8: null pointer");
    BE42_CHECK(rows >= 0 && cols > 0, "be42_quant_rows_int8: bad shape %d x %d", rows, cols);
    if (rows == 0)
        return BE42_OK;
    if (!launch_quant_vec<false>((uint8_t *)q, scales, x, rows, cols, as_stream(stream)))
        hipLaunchKernelGGL(k_quant_rows_int8, dim3(rows), dim3(256), 0, as_stream(stream), q, scales, x, cols);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

extern "C" int be42_quant_rows_fp8(uint8_t *q, float *scales, const float *x, int rows, int cols,
                                   void *stream)
{
    BE42_CHECK(q && scales && x, "be42_quant_rows_fp8: null pointer");
    BE42_CHECK(rows >= 0 && cols > 0, "be42_quant_rows_fp8: bad shape %d x %d", rows, cols);
    int rc = ensure_thresholds();
    if (rc)
        return rc;
    if (rows == 0)
        return BE42_OK;
    if (!launch_quant_vec<true>(q, scales, x, rows, cols, as_stream(stream)))
        hipLaunchKernelGGL(k_quant_rows_fp8, dim3(rows), dim3(256), 0, as_stream(stream), q, scales, x, cols);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

static int norm_quant_rows(const char *name, bool fp8, uint8_t *q, float *scales, void *sum, const void *x,
                           int x_stride, const void *residual, int residual_stride, int act_bf16, const uint16_t *w,
                           int rows, int cols, float eps, void *stream)
{
    BE42_CHECK(rows >= 0 && cols > 0, "%s: bad shape %d x %d", name, rows, cols);
    BE42_CHECK(x_stride >= cols && (!residual || residual_stride >= cols), "%s: rows of %d at strides %d, %d", name,
               cols, x_stride, residual_stride);
    BE42_CHECK(eps >= 0.0f, "%s: eps %g", name, (double)eps);
    if (rows == 0)
        return BE42_OK;
    BE42_CHECK(q && scales && x && w, "%s: null pointer", name);
    // a row is written where it was read only if both lie at the same place
    BE42_CHECK(!sum || ((sum != x || x_stride == cols) && (sum != residual || residual_stride == cols)),
               "%s: sum replaces rows that are not contiguous", name);
    const uintptr_t unit = act_bf16 ? 1 : 3;
    BE42_CHECK(!(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum) & unit) && !((uintptr_t)w & 1) &&
                   !((uintptr_t)scales & 3), "%s: unaligned pointer", name);
    if (fp8) {
        const int rc = ensure_thresholds();
        if (rc)
            return rc;
    }
    // a launch has less than 2^32 threads
    constexpr int kMost = 1 << 21;
    const size_t sz = act_bf16 ? 2 : 4;
    for (size_t r = 0; r < (size_t)rows; r += kMost) {
        const int some = (int)std::min((size_t)rows - r, (size_t)kMost);
        auto at = [&](const void *p, size_t stride) { return p ? (const char *)p + r * stride * sz : nullptr; };
        auto go = fp8 ? launch_norm_quant<true> : launch_norm_quant<false>;
        go(q + r * cols, scales + r, (void *)at(sum, cols), at(x, x_stride), x_stride, at(residual, residual_stride),
           residual_stride, act_bf16 != 0, w, some, cols, eps, as_stream(stream));
        BE42_LAUNCH_CHECK();
    }
    return BE42_OK;
}

extern "C" int be42_norm_quant_rows_int8(int8_t *q, float *scales, void *sum, const void *x, int x_stride,
                                         const void *residual, int residual_stride, int act_bf16, const uint16_t *w,
                                         int rows, int cols, float eps, void *stream)
{
    return norm_quant_rows("be42_norm_quant_rows_int8", false, (uint8_t *)q, scales, sum, x, x_stride, residual,
                           residual_stride, act_bf16, w, rows, cols, eps, stream);
}

extern "C" int be42_norm_quant_rows_fp8(uint8_t *q, float *scales, void *sum, const void *x, int x_stride,
                                        const void *residual, int residual_stride, int act_bf16, const uint16_t *w,
                                        int rows, int cols, float eps, void *stream)
{
    return norm_quant_rows("be42_norm_quant_rows_fp8", true, q, scales, sum, x, x_stride, residual, residual_stride,
                           act_bf16, w, rows, cols, eps, stream);
}

extern "C" int be42_dequant_rows_int8(float *out, const int8_t *q, const float *scales, int rows,
                                      int cols, void *stream)
{
    BE42_CHECK(out && q && scales, "be42_dequant_rows_int8: null pointer");
    BE42_CHECK(rows >= 0 && cols > 0, "be42_dequant_rows_int8: bad shape");
    size_t total = (size_t)rows * cols;
    if (total == 0)
        return BE42_OK;
    int blocks = (int)((total + 255) / 256);
    if (blocks > 8192)
        blocks = 8192;
    hipLaunchKernelGGL(k_dequant_rows_int8, dim3(blocks), dim3(256), 0, as_stream(stream), out, q, scales,
                       cols, total);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}

extern "C" int be42_fp8_decode(float *out, const uint8_t *q, size_t n, void *stream)
{
    BE42_CHECK(out && q, "be42_fp8_decode: null pointer");
    if (n == 0)
        return BE42_OK;
    int blocks = (int)((n + 255) / 256);
    if (blocks > 8192)
        blocks = 8192;
    hipLaunchKernelGGL(k_fp8_decode, dim3(blocks), dim3(256), 0, as_stream(stream), out, q, n);
    BE42_LAUNCH_CHECK();
    return BE42_OK;
}
