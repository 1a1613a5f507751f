// linear_i8.hip -- Linear over 8-bit weights: O = s * epi(x_m w_n sum_k a_mk
// b_nk + bias) (+R), a the rows of X rounded to 8-bit integers with one scale
// x_m each, b the weight's integers with one scale w_n per output channel.
//
// The sums are 32-bit integers (exact: K <= 131072), so nothing depends on
// how K is split or in which order the parts meet.
#include <algorithm>

#include "device_common.h"
#include "kernels.h"
#include "launch_once.h"

#define LDS_AS __attribute__((address_space(3)))

namespace vai_dev {

typedef int int4v __attribute__((ext_vector_type(4)));

namespace {

// The row's scale from the largest |x| as bits (NaN and infinity sort above
// every finite value): max / 127 rounded to fp32; NaN for a row that holds
// something not finite; 0, all codes 0, for a row below fp32's normal range.
__device__ __forceinline__ float row_scale(uint32_t amax)
{
    if (amax >= 0x7f800000u) return __builtin_nanf("");
    const float s = __builtin_bit_cast(float, amax) / 127.0f;
    return s < 1.17549435e-38f ? 0.f : s;
}

// x / s rounded to the nearest integer, halves to even, from the remainder
// x - n s, which one fma gives exactly: a product with 1 / s alone would round
// quotients next to a half either way. inv = 1 / s; inv = 0 gives 0.
__device__ __forceinline__ int code_of(float x, float s, float inv)
{
    float n = rintf(x * inv);
    const float r = 2.0f * fmaf(-n, s, x);
    if (r > s || (r == s && ((int)n & 1))) n += 1.f;
    else if (r < -s || (r == -s && ((int)n & 1))) n -= 1.f;
    return (int)n;
}

}   // namespace

// One workgroup per row; rows of `stride` bytes, zeros past K.
__global__ __launch_bounds__(256) void quantize_i8_kernel(int8_t* out, float* scale, const void* in, int in_dt,
                                                          uint32_t K, uint32_t stride)
{
    __shared__ uint32_t red[4];
    const size_t row = blockIdx.x;
    uint32_t amax = 0;
    for (uint32_t k = threadIdx.x; k < K; k += 256)
        amax = std::max(amax, __builtin_bit_cast(uint32_t, ld(in, in_dt, row * K + k)) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = std::max(amax, (uint32_t)__shfl_xor((int)amax, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = std::max(std::max(red[0], red[1]), std::max(red[2], red[3]));
    const float s = row_scale(amax), inv = s > 0.f ? 1.0f / s : 0.f;
    if (threadIdx.x == 0) scale[row] = s;
    for (uint32_t k = threadIdx.x; k < stride; k += 256)
        out[row * stride + k] = k < K && inv > 0.f ? (int8_t)code_of(ld(in, in_dt, row * K + k), s, inv) : 0;
}

hipError_t quantize_i8_launch(void* out, float* scale, const void* in, int in_dtype, uint32_t rows, uint32_t K,
                              uint32_t stride, hipStream_t s)
{
    hipLaunchKernelGGL(quantize_i8_kernel, dim3(rows), dim3(256), 0, s, (int8_t*)out, scale, in, in_dtype, K, stride);
    return hipGetLastError();
}

__device__ __forceinline__ OutputSpec i8_output(const LinearI8Params& p)
{
    return OutputSpec{p.out, p.bias, p.residual, p.o_dtype, p.b_dtype, p.bias_repeat, p.residual_repeat,
                      p.epilogue, p.residual_order, p.scalar_scale};
}

// A workgroup's tile is 16 NT weight rows by 16 MT rows of X; its 4 waves take
// 128-byte blocks of K in turn and their sums meet in LDS.
template <int MT, int NT>
__global__ __launch_bounds__(256) void linear_i8_tile_kernel(LinearI8Params p)
{
    constexpr int NW = 4;
    __shared__ int4v part[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int8_t* wr[NT];
    const int8_t* xr[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wr[j] = p.weight + (size_t)std::min(n0 + 16 * j + c16, p.N - 1) * p.w_stride;
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = p.x + (size_t)std::min(m0 + 16 * i + c16, p.M - 1) * p.x_stride;
    int4v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (int4v)0;
    // (X rows are whole 128-byte blocks, zero past K: what stands in W's place
    // there does not count, and W's last block is read from its row's start)
    for (uint32_t k0 = wave * 128; k0 < p.x_stride; k0 += NW * 128) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t k = k0 + 32 * g + 16 * h, kw = k < p.w_stride ? k : 0u;
            int4v a[NT], b[MT];
#pragma unroll
            for (int j = 0; j < NT; ++j) a[j] = *(const int4v*)(wr[j] + kw);
#pragma unroll
            for (int i = 0; i < MT; ++i) b[i] = *(const int4v*)(xr[i] + k);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[i], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    // lane (c16, g) of fragment (i, j) holds row m = 16 i + c16, columns 16 j + 4 g ..+3
    for (int f = wave; f < MT * NT; f += NW) {
        int4v v = part[0][f][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w][f][lane];
        const uint32_t m = m0 + 16 * (f / NT) + c16, n = n0 + 16 * (f % NT) + 4 * g;
        if (m >= p.M) continue;
        const float xs = p.x_scale[m];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N)
                store_output(i8_output(p), (size_t)m * p.N + n + e, (float)v[e] * xs * p.w_scale[n + e]);
    }
}

hipError_t linear_i8_launch(const LinearI8Params& p, hipStream_t s)
{
    const dim3 grid((p.N + 31) / 32, (p.M + 31) / 32);
    hipLaunchKernelGGL((linear_i8_tile_kernel<2, 2>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
