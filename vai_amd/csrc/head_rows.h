// head_rows.h -- the parts of the head norms and the position rotation that the
// kernels over rows of heads share: the angles, the root of the norm, and loads
// and stores of up to four values of a head.
#pragma once
#include <cmath>

#include "device_common.h"

namespace vai_dev {

// cos and sin of position * f_i. The angle is taken in turns, in 64 bits (at
// position 100000 the fastest pair has made 16000 turns, of which fp32 would
// keep three digits), and only its fraction goes on in fp32. From there the
// nearest quarter turn is taken off and the rest, at most pi / 4, put into the
// power series: the first term left out is below 2^-25 for the cosine (x^10 /
// 10!) and 2^-28 of the sine (x^10 / 11!).
template <class P>
__device__ __forceinline__ void turn_of(const P& p, uint32_t pos, uint32_t i, float& c, float& s)
{
    const double f = p.inv_freq ? (double)p.inv_freq[i] * 0.15915494309189533577 : p.turn_hi[i >> 4] * p.turn_lo[i & 15];
    const double t = (double)pos * f;
    const float fr = (float)(t - rint(t)), q = rintf(4.0f * fr);
    const float x = 6.2831853071795865f * fmaf(-0.25f, q, fr), x2 = x * x;
    const float sx = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cx = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.0f);
    const int k = (int)q & 3;
    const float a = k & 1 ? cx : sx, b = k & 1 ? sx : cx;
    s = k & 2 ? -a : a;
    c = k == 1 || k == 2 ? -b : b;
}

// 1 / sqrt(sq / D + eps) of a head, from the sum of its squares: as far as that
// number lies well inside fp32's range (no square that counts has then under- or
// overflowed).
__device__ __forceinline__ bool rms_in_range(float v) { return v > 0x1p-80f && v < 0x1p100f; }
__device__ __forceinline__ float inv_root(float v) { return 1.0f / sqrtf(v); }

// Else the head is taken in units of 2^e, 2^e the larger of its largest |x|
// and sqrt(eps), rounded up: the squares then lie in range, and x and the root
// lose the same factor. (A head with an infinity or a NaN stays as it is; one of
// zeros with eps = 0 is 0 / 0.)
__device__ __forceinline__ int rms_unit(float amax, float eps)
{
    if (!(amax < __builtin_inff())) return 0;
    const int a = amax > 0.f ? __builtin_amdgcn_frexp_expf(amax) : -200;
    const int b = eps > 0.f ? (__builtin_amdgcn_frexp_expf(eps) + 1) >> 1 : -200;
    return a > b ? a : b;
}

// op(x, what another lane holds) until every lane of a group of L (a power of two) has the group's result
template <int L, class Op>
__device__ __forceinline__ float group_reduce(float x, Op op)
{
    const auto moved = [](float v, auto ctrl) __attribute__((always_inline)) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (L >= 2) x = op(x, moved(x, std::integral_constant<int, 0xB1>{}));    // lane ^ 1
    if constexpr (L >= 4) x = op(x, moved(x, std::integral_constant<int, 0x4E>{}));    // lane ^ 2
    if constexpr (L >= 8) x = op(x, moved(x, std::integral_constant<int, 0x141>{}));   // the other 4 of 8 (mirrored)
    if constexpr (L >= 16) x = op(x, moved(x, std::integral_constant<int, 0x140>{}));  // the other 8 of 16
    if constexpr (L >= 32) x = op(x, __shfl_xor(x, 16));
    if constexpr (L >= 64) x = op(x, __shfl_xor(x, 32));
    return x;
}
template <int L>
__device__ __forceinline__ float group_sum(float x) { return group_reduce<L>(x, [](float a, float b) { return a + b; }); }
template <int L>
__device__ __forceinline__ float group_max(float x) { return group_reduce<L>(x, [](float a, float b) { return fmaxf(a, b); }); }

// n of 4 values at any alignment of their type, zeros for the rest (FULL: 4)
template <bool FULL, typename T>
__device__ __forceinline__ float4v some4(const T* p, uint32_t n)
{
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef t4 t4u __attribute__((aligned(sizeof(T))));
    if (FULL || n == 4) return __builtin_convertvector(*(const t4u*)p, float4v);
    float4v v = (float4v)0.f;
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if ((uint32_t)e < n) v[e] = (float)p[e];
    return v;
}
template <bool FULL, typename T>
__device__ __forceinline__ void put4(T* p, uint32_t n, float4v v)
{
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef t4 t4u __attribute__((aligned(sizeof(T))));
    if (FULL || n == 4) *(t4u*)p = __builtin_convertvector(v, t4);
    else
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if ((uint32_t)e < n) p[e] = (T)v[e];
}
__device__ __forceinline__ float4v weight4(const void* w, int dt, uint32_t d, uint32_t n)
{
    return dt == DT_F16 ? some4<false>((const half_t*)w + d, n) : some4<false>((const float*)w + d, n);
}

// f_i = theta^(-2i / rot) in turns, i = 16 a + b, as a product of two short
// tables: 32 powers on the host for up to 256 pairs
template <class P>
inline void rope_tables(P& p, float theta)
{
    if (p.rot_dim && !p.inv_freq) {
        const double step = -2.0 * std::log2((double)theta) / (double)p.rot_dim;
        for (uint32_t a = 0; 16 * a < p.rot_dim / 2; ++a) p.turn_hi[a] = std::exp2(16.0 * a * step);
        for (uint32_t b = 0; b < 16; ++b) p.turn_lo[b] = std::exp2(b * step) * 0.15915494309189533577;
    }
}

}   // namespace vai_dev
