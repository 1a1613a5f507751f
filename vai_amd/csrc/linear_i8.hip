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
    const float q = rintf(x * inv), r = 2.0f * fmaf(-q, s, x);
    const int n = (int)q;
    const bool odd = n & 1, up = r > s || (r == s && odd), down = r < -s || (r == -s && odd);
    return n + (int)up - (int)down;
}

}   // namespace

// 16 values of a row from k on, zeros past its end, kept in the row's type
template <typename T> struct Raw16 {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 a, b;
    __device__ __forceinline__ void load(const T* row, uint32_t k, uint32_t K)
    {
        typedef t8 t8u __attribute__((aligned(sizeof(T))));
        a = b = (t8)(T)0;
        if (k + 16 <= K) {
            a = *(const t8u*)(row + k);
            b = *(const t8u*)(row + k + 8);
        } else if (k < K) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const T v = k + e < K ? row[k + e] : (T)0;
                if (e < 8) a[e] = v;
                else b[e - 8] = v;
            }
        }
    }
    __device__ __forceinline__ void values(float (&x)[16]) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (float)a[e];
            x[8 + e] = (float)b[e];
        }
    }
};
template <typename T>
__device__ __forceinline__ void row16(const T* row, uint32_t k, uint32_t K, float (&x)[16])
{
    Raw16<T> r;
    r.load(row, k, K);
    r.values(x);
}

__device__ __forceinline__ uint32_t abs_max16(const float (&x)[16], uint32_t m)
{
#pragma unroll
    for (int e = 0; e < 16; ++e) m = std::max(m, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    return m;
}

// N codes as bytes. x / s is taken as x * inv, and the sum with 1.5 * 2^23
// leaves its nearest integer in the low bits (one fma); that quotient is off by
// 127 * 2^-23 at most, so only where it comes within 2^-13 of a half are the
// codes taken from the exact remainder (one wave of 1024 values in five).
template <int N>
__device__ __forceinline__ void codes_of(const float (&x)[N], float s, float inv, uint32_t (&w)[N / 4])
{
    float far = 0.f;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = x[4 * q + e], f = fmaf(v, inv, 12582912.0f);
            b[e] = __builtin_bit_cast(uint32_t, f);
            far = fmaxf(far, __builtin_fabsf(fmaf(v, inv, -(f - 12582912.0f))));
        }
        // byte 0 of each, one above the other
        w[q] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u),
                                     __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
    }
    if (far > 0.5f - 1.f / 8192) {
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            w[q] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[q] |= ((uint32_t)code_of(x[4 * q + e], s, inv) & 255u) << (8 * e);
        }
    }
}

__device__ __forceinline__ int4v codes16(const float (&x)[16], float s, float inv)
{
    uint32_t w[4];
    codes_of(x, s, inv, w);
    return int4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// One workgroup per row; rows of `stride` bytes (a multiple of 16), zeros past
// K. The row is read once: the first 8192 values stay in registers (16 and 16 a
// thread) until its scale is known, what lies past them is read again.
template <typename T>
__global__ __launch_bounds__(256) void quantize_i8_kernel(int8_t* out, float* scale, const T* in, uint32_t K,
                                                          uint32_t stride)
{
    constexpr uint32_t C = 256 * 16;
    __shared__ uint32_t red[4];
    const T* row = in + (size_t)blockIdx.x * K;
    int8_t* dst = out + (size_t)blockIdx.x * stride;
    const uint32_t k0 = threadIdx.x * 16;
    float x[2][16];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i * C < K) row16(row, k0 + i * C, K, x[i]);
        else
#pragma unroll
            for (int e = 0; e < 16; ++e) x[i][e] = 0.f;
        amax = abs_max16(x[i], amax);
    }
    for (uint32_t k = k0 + 2 * C; k < K; k += C) {
        float y[16];
        row16(row, k, K, y);
        amax = abs_max16(y, amax);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = std::max(amax, (uint32_t)__shfl_xor((int)amax, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = std::max(std::max(red[0], red[1]), std::max(red[2], red[3]));
    const float s = row_scale(amax), inv = s > 0.f ? 1.0f / s : 0.f;
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    const bool some = inv > 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (k0 + i * C < stride) *(int4v*)(dst + k0 + i * C) = some ? codes16(x[i], s, inv) : (int4v)0;
    for (uint32_t k = k0 + 2 * C; k < stride; k += C) {
        float y[16];
        row16(row, k, K, y);
        *(int4v*)(dst + k) = some ? codes16(y, s, inv) : (int4v)0;
    }
}

hipError_t quantize_i8_launch(void* out, float* scale, const void* in, int in_dtype, uint32_t rows, uint32_t K,
                              uint32_t stride, hipStream_t s)
{
    if (in_dtype == DT_F16)
        hipLaunchKernelGGL(quantize_i8_kernel<half_t>, dim3(rows), dim3(256), 0, s, (int8_t*)out, scale, (const half_t*)in, K, stride);
    else
        hipLaunchKernelGGL(quantize_i8_kernel<float>, dim3(rows), dim3(256), 0, s, (int8_t*)out, scale, (const float*)in, K, stride);
    return hipGetLastError();
}

__device__ __forceinline__ OutputSpec i8_output(const LinearI8Params& p)
{
    return OutputSpec{p.out, p.bias, p.residual, p.o_dtype, p.b_dtype, p.bias_repeat, p.residual_repeat,
                      p.epilogue, p.residual_order, p.scalar_scale};
}

template <int N>
__device__ __forceinline__ void few_wait()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
// all but the copies of the blocks behind this one (`behind` of them, N counted) have landed
template <int N, int COPIES>
__device__ __forceinline__ void few_wait_behind(int behind)
{
    if constexpr (N == 0) few_wait<0>();
    else if (behind >= N) few_wait<N * COPIES>();
    else few_wait_behind<N - 1, COPIES>(behind);
}
__device__ __forceinline__ void few_wait_lds() { __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14)); }

// Few rows of X (16 MT at most): bound by reading W once. A workgroup takes 16 NT
// weight rows and its NW waves 128-byte blocks of K in turn, each through a ring
// of its own in LDS: blocks are copied straight there (eight lanes to a row's 128
// bytes; lanes that loaded fragments would each touch another row), D of them in
// flight, and no wave waits for another until the sums meet. Chunk c of slab row
// r stands at chunk c ^ (r / 2 % 8): fragment reads hit every bank group once.
// FUSED (MT = 1): X is rounded here, under the first copies of W, by every
// workgroup for itself; else its codes come from the workspace, through the ring
// like W.
template <int MT, int NT, int NW, int D, bool FUSED> struct FewCfg {
    static constexpr int BLOCK = (NT + (FUSED ? 0 : MT)) * 2048;   // a block of K in LDS: 16-row slabs
    static constexpr int COPIES = BLOCK / 1024;
    static constexpr int RING = NW * D * BLOCK;
    static_assert(RING >= NW * MT * NT * 1024, "the sums' exchange takes the ring's place");
};

template <int MT, int NT, int NW, int D, typename TX, bool FUSED>
__global__ __launch_bounds__(64 * NW) void linear_i8_few_kernel(LinearI8Params p, const TX* in)
{
    typedef FewCfg<MT, NT, NW, D, FUSED> C;
    static_assert(!FUSED || MT == 1, "one slab of rounded rows");
    extern __shared__ int4v few_lds[];
    LDS_AS char* lds = (LDS_AS char*)(LDS_AS void*)few_lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT, blocks = p.x_stride / 128;
    const int mine = ((int)blocks - wave + NW - 1) / NW;   // blocks of this wave
    LDS_AS char* ring = lds + wave * D * C::BLOCK;

    // Copy i of a block fills slab rows 8 (i % 2) ..+7 of slab i / 2 (W's, then
    // X's). Rows past the operands' ends read as zero: the resources end there.
    const uint32_t rows_w = std::min<uint32_t>(p.N - n0, 16 * NT), rows_x = std::min<uint32_t>(p.M - m0, 16 * MT);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(p.weight + (size_t)n0 * p.w_stride), (short)0,
                                                                        (int)(rows_w * p.w_stride), 0x00020000);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(FUSED ? nullptr : p.x + (size_t)m0 * p.x_stride), (short)0, FUSED ? 0 : (int)(rows_x * p.x_stride), 0x00020000);
    const uint32_t cr = lane >> 3;
    const auto copy = [&](int i) __attribute__((always_inline)) {   // the wave's i-th block
        const uint32_t k = (wave + NW * (uint32_t)i) * 128;
        LDS_AS char* dst = ring + (i % D) * C::BLOCK;
#pragma unroll
        for (int c = 0; c < C::COPIES; ++c) {
            const uint32_t row = 8 * (c & 1) + cr, ch = (lane & 7) ^ (row / 2 % 8);
            const bool w = c < 2 * NT;
            const uint32_t slab_row = (w ? c / 2 : c / 2 - NT) * 16 + row;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(w ? rw : rx, (LDS_AS void*)(dst + c * 1024), 16,
                                                     (int)(slab_row * (w ? p.w_stride : p.x_stride) + ch * 16 + k), 0, 0, 0);
        }
    };
    // FUSED (M <= 4, M K <= 8192): NW / M waves share a row of X, 1024 values at a
    // time each, 3 times at most (X before W: loads and copies are waited for in
    // their order)
    constexpr int KEEP = FUSED ? 3 : 1;
    const uint32_t share = std::max<uint32_t>(NW / p.M, 1), part = wave % share, row = wave / share;
    Raw16<TX> kept[KEEP];
    if constexpr (FUSED)
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            kept[i].load(in + (size_t)std::min<uint32_t>(row, p.M - 1) * p.K, (i * share + part) * 1024 + lane * 16, p.K);
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < mine) copy(i);

    const uint32_t ls = p.x_stride + 16;   // a row of codes in LDS (16 more: rows start in different banks)
    LDS_AS int8_t* xl = (LDS_AS int8_t*)(lds + C::RING);
    LDS_AS float* sl = (LDS_AS float*)(xl + p.M * ls);
    if constexpr (FUSED) {
        LDS_AS uint32_t* ml = (LDS_AS uint32_t*)(sl + p.M);   // largest values, a part each
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
            float y[16];
            kept[i].values(y);
            amax = abs_max16(y, amax);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) amax = std::max(amax, (uint32_t)__shfl_xor((int)amax, o));
        if (lane == 0) ml[wave] = amax;
        __syncthreads();
        for (uint32_t w = 0; w < share; ++w) amax = std::max(amax, (uint32_t)ml[wave / share * share + w]);
        if (row < p.M) {
            const float s = row_scale(amax), inv = s > 0.f ? 1.0f / s : 0.f;
            if (part == 0 && lane == 0) sl[row] = s;
#pragma unroll
            for (int i = 0; i < KEEP; ++i) {
                const uint32_t k = (i * share + part) * 1024 + lane * 16;
                if (k >= p.x_stride) continue;
                float y[16];
                kept[i].values(y);
                *(LDS_AS int4v*)(xl + row * ls + k) = inv > 0.f ? codes16(y, s, inv) : (int4v)0;
            }
        }
        __syncthreads();
    }
    const uint32_t xrow = std::min<uint32_t>(c16, p.M - 1);   // (FUSED: columns past M repeat the last row)
    int4v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (int4v)0;
    const int swz = c16 / 2 % 8;
    for (int i = 0; i < mine; ++i) {
        few_wait_behind<D - 1, C::COPIES>(mine - 1 - i);   // block i has landed; those after it may be in flight
        LDS_AS const char* src = ring + (i % D) * C::BLOCK + c16 * 128;
        int4v a[2][NT], b[2][MT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = ((4 * h + g) ^ swz) * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j) a[h][j] = *(LDS_AS const int4v*)(src + j * 2048 + at);
#pragma unroll
            for (int m = 0; m < MT; ++m)
                b[h][m] = FUSED ? *(LDS_AS const int4v*)(xl + xrow * ls + (wave + NW * i) * 128 + 64 * h + 16 * g)
                                : *(LDS_AS const int4v*)(src + (NT + m) * 2048 + at);
        }
        few_wait_lds();                    // read before the block is copied over
        if (i + D < mine) copy(i + D);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[m][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h][j], b[h][m], acc[m][j], 0, 0, 0);
    }

    // the waves' sums, then lane (c16, g) of fragment (m, j) holds row 16 m + c16, columns 16 j + 4 g ..+3
    __syncthreads();
    LDS_AS int4v* sums = (LDS_AS int4v*)lds;
#pragma unroll
    for (int f = 0; f < MT * NT; ++f) sums[(wave * MT * NT + f) * 64 + lane] = acc[f / NT][f % NT];
    __syncthreads();
    const OutputSpec q = i8_output(p);
    for (int f = wave; f < MT * NT; f += NW) {
        int4v v = sums[f * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += sums[(w * MT * NT + f) * 64 + lane];
        const uint32_t m = m0 + 16 * (f / NT) + c16, n = n0 + 16 * (f % NT) + 4 * g;
        if (m >= p.M) continue;
        // (a sum, below 2^31, times a row's scale up to 2^64 stays within fp32; what a larger
        // scale has above it follows the column's)
        const float xs = FUSED ? sl[m] : p.x_scale[m];
        const float lift = xs > 0x1p64f ? 0x1p64f : 1.0f, xr = xs > 0x1p64f ? xs * 0x1p-64f : xs;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N) store_output(q, (size_t)m * p.N + n + e, (float)v[e] * xr * p.w_scale[n + e] * lift);
    }
}

template <int MT, int NT, int NW, int D, typename TX, bool FUSED>
static hipError_t few_launch_t(const LinearI8Params& p, const void* in, hipStream_t s)
{
    typedef FewCfg<MT, NT, NW, D, FUSED> C;
    static PerDevice once;
    auto kern = linear_i8_few_kernel<MT, NT, NW, D, TX, FUSED>;
    constexpr int xmax = FUSED ? 9 * 1024 : 0;   // more than linear_i8_fused allows
    if constexpr (C::RING + xmax > 64 * 1024) {
        const hipError_t e = set_max_lds(once, (const void*)kern, C::RING + xmax);
        if (e != hipSuccess) return e;
    }
    const dim3 grid((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT));
    const size_t lds = C::RING + (FUSED ? (size_t)p.M * (p.x_stride + 16 + sizeof(float)) + NW * 4 : 0);
    hipLaunchKernelGGL(kern, grid, dim3(64 * NW), lds, s, p, (const TX*)in);
    return hipGetLastError();
}

// One launch in place of two where every workgroup can round X for itself at no
// cost: the kernels' times are then alike and a launch's host time is saved
// (one / two launches, us: 1 x 8192 x 2048 8.2 / 8.2, 1 x 16384 x 2048 8.8 / 9.3,
// 4 x 16384 x 2048 8.2 / 10.0). Not with a wave for more than one row (8 x 4096 x
// 1024 8.8 / 6.9, 16 x 4096 x 512 10.7 / 7.6), longer rows (4 x 4096 x 8192 13.6 /
// 10.8), more workgroups than one round of the chip (1 x 32768 x 2048 19 / 16) or
// weights from 64 MB on, which the 64-wide tiles read faster (below; 1 x 16384 x
// 8192 33 / 27, 1 x 8192 x 8192 22.9 / 21.2).
bool linear_i8_fused(uint32_t M, uint32_t N, uint32_t K)
{
    return M <= 4 && (uint64_t)M * K <= 8192 && N <= 16384 && (uint64_t)N * K < 1u << 26;
}

// Wider workgroups where there are enough of them (M = 1, K = 2048, N = 8192, us:
// 32 columns 7.7, 16 8.5; K = N = 4096: 8.9, 8.0).
hipError_t linear_i8_fused_launch(const LinearI8Params& p, const void* in, int in_dtype, hipStream_t s)
{
    if (p.N <= 4096)
        return in_dtype == DT_F16 ? few_launch_t<1, 1, 4, 8, half_t, true>(p, in, s) : few_launch_t<1, 1, 4, 8, float, true>(p, in, s);
    return in_dtype == DT_F16 ? few_launch_t<1, 2, 4, 4, half_t, true>(p, in, s) : few_launch_t<1, 2, 4, 4, float, true>(p, in, s);
}

// Up to 32 rows over up to 8192 columns, and 64 over 5120, the wave rings, whose
// workgroups are then one round (us, rings / 64-wide tiles: 8 x 4096 x 8192 6.5 / 16,
// 16 x 8192 x 4096 7.2 / 10.5, 32 x 4096 x 4096 7.0 / 10.2, 61 x 5003 x 1999 8.2 /
// 9.1, 64 x 8192 x 2048 9.1 / 7.1; 16 and 64 x 16384 x 4096 13.5 and 25 / 12.2), and
// weights that the L2s hold or nearly (16 x 6144 x 8192 16.2 / 15.9, 8 x 8192 x 8192
// 20.0 / 16.5, 64 x 8192 x 8192 24.6 / 17.0). Past that the
// tile whose modelled time is least: kt stages of 128 bytes of K, c tiles a CU.
// Measured, us, 64-wide / 128-wide / 256-wide: 500 x 2048 x 2048 7.9 / 14.7 /
// 32.7, 1000 x 4096 x 4096 28 / 25 / 57, 2048 x 4096 x 11008 137 / 90 / 135,
// 4096^3 103 / 77 / 67.
hipError_t linear_i8_launch(const LinearI8Params& p, hipStream_t s)
{
    if (p.N <= 8192 && (uint64_t)p.N * p.K < 1u << 26) {
        if (p.M <= 16)
            return p.N <= 4096 ? few_launch_t<1, 1, 4, 4, half_t, false>(p, nullptr, s)
                               : few_launch_t<1, 2, 4, 4, half_t, false>(p, nullptr, s);
        if (p.M <= 32) return few_launch_t<2, 2, 4, 3, half_t, false>(p, nullptr, s);
        if (p.M <= 64 && p.N <= 5120) return few_launch_t<4, 2, 4, 3, half_t, false>(p, nullptr, s);
    }
    int cus = 0;
    const hipError_t e = device_cus(&cus);
    if (e != hipSuccess) return e;
    const auto per_cu = [&](uint32_t b) {
        const uint64_t tiles = (uint64_t)((p.M + b - 1) / b) * ((p.N + b - 1) / b);
        return (float)((tiles + cus - 1) / cus);
    };
    const float kt = (float)(p.x_stride / 128);
    const float t1 = 3.f + kt * (.1f + .2f * per_cu(64)), t2 = 3.f + kt * (.2f + .5f * per_cu(128)),
                t4 = 4.f + kt * 2.f * per_cu(256);
    return linear_i8_big_launch(p, t4 <= t2 && t4 <= t1 ? 4 : t2 <= t1 ? 2 : 1, s);
}

}   // namespace vai_dev
