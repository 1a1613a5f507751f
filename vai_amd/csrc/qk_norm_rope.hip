// qk_norm_rope.hip -- from the fused query / key / value projection to the
// planes attention reads: RMS norm of each query and key head, the position
// rotation, and token-major rows to head-major planes, in one pass.
//
//   y_d = x_d / sqrt(mean_d x_d^2 + eps) * (w_d + offset)
//   (a, e) -> (a cos t - e sin t, e cos t + a sin t), t = position * f_i
//
// for the rot_dim / 2 pairs (a, e) = (y_i, y_{i + rot/2}) or (y_2i, y_2i+1).
// Bound by memory: each value is read once and written once.
#include <algorithm>
#include <cmath>

#include "device_common.h"
#include "kernels.h"

namespace vai_dev {

// cos and sin of position * f_i. The angle is taken in turns, in 64 bits (at
// position 100000 the fastest pair has made 16000 turns, of which fp32 would
// keep three digits), and only its fraction goes on in fp32. From there the
// nearest quarter turn is taken off and the rest, at most pi / 4, put into the
// power series: the first term left out is below 2^-25 for the cosine (x^10 /
// 10!) and 2^-28 of the sine (x^10 / 11!).
__device__ __forceinline__ void turn_of(const QkNormRopeParams& p, uint32_t pos, uint32_t i, float& c, float& s)
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

// Larger head dims: a wave takes one head at a time, in LDS as fp32.
__global__ __launch_bounds__(64) void qk_norm_rope_any_kernel(QkNormRopeParams p)
{
    __shared__ float y[QkNormRopeParams::MAX_DIM];
    const uint32_t D = p.head_dim, heads = p.hq + 2 * p.hkv, lane = threadIdx.x;
    const uint64_t total = (uint64_t)p.batch * p.tokens * heads;
    const uint32_t first = p.count ? *p.count : 0u;
    for (uint64_t u = blockIdx.x; u < total; u += gridDim.x) {
        const uint64_t bt = u / heads;
        const uint32_t h = (uint32_t)(u - bt * heads), b = (uint32_t)(bt / p.tokens), t = (uint32_t)(bt - (uint64_t)b * p.tokens);
        const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
        if (is_v && !p.v_out) continue;
        const size_t src = bt * p.row_stride + (size_t)h * D;
        float sq = 0.f;
        for (uint32_t d = lane; d < D; d += 64) {
            const float x = ld(p.qkv, p.i_dtype, src + d);
            y[d] = x;
            sq += x * x;
        }
        void* out = is_q ? p.q_out : is_v ? p.v_out : p.k_out;
        const uint32_t oh = is_q ? h : is_v ? h - p.hq - p.hkv : h - p.hq, nh = is_q ? p.hq : p.hkv;
        const size_t dst = (((size_t)b * nh + oh) * p.tokens + t) * D;
        if (p.norm && !is_v) {
            float v = wave_sum(sq) / (float)D + p.eps;
            int e = 0;
            if (!rms_in_range(v)) {   // (the same in every lane)
                float amax = 0.f, sum = 0.f;
                for (uint32_t d = lane; d < D; d += 64) amax = fmaxf(amax, __builtin_fabsf(y[d]));
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
                e = rms_unit(amax, p.eps);
                for (uint32_t d = lane; d < D; d += 64) {
                    const float x = ldexpf(y[d], -e);
                    sum += x * x;
                }
                v = wave_sum(sum) / (float)D + ldexpf(p.eps, -2 * e);
            }
            const float inv = inv_root(v);
            const void* w = is_q ? p.q_weight : p.k_weight;
            for (uint32_t d = lane; d < D; d += 64)
                y[d] = ldexpf(y[d], -e) * inv * (w ? ld(w, p.w_dtype, d) + p.weight_offset : 1.0f);
        }
        __syncthreads();
        const uint32_t rot = is_v ? 0u : p.rot_dim, half = rot / 2;
        const uint32_t pos = p.positions ? p.positions[bt] : first + t;
        for (uint32_t d = lane; d < D; d += 64) {
            float v = y[d];
            if (d < rot) {
                const bool second = p.neighbours ? (d & 1) : d >= half;
                const uint32_t i = p.neighbours ? d / 2 : second ? d - half : d;
                const float o = y[p.neighbours ? d ^ 1 : second ? d - half : d + half];
                float c, s;
                turn_of(p, pos, i, c, s);
                v = second ? v * c + o * s : v * c - o * s;
            }
            st(out, p.o_dtype, dst + d, v);
        }
        __syncthreads();   // y is rewritten by the next head
    }
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

// Head dims up to 512: L lanes share a head, 8 values each, cut so that a lane
// holds both values of its four pairs: with halves values 4 j ..+3 and the same of
// the other half, else (and past the rotated values) 8 neighbouring ones. Where a
// half is no multiple of 4, or what is left none of 8, a lane's last values do not
// exist (na, nb of its two groups of four do; FULL: all). A lane's four angles
// serve every head of the token. A wave takes a token's heads 64 / L at a time,
// its share of them (blockIdx.y of `shares`). One step's loads at a time: 94
// registers, five waves a SIMD, which hide the loads better than the three that
// four steps at a time leave (143 registers). 4096 tokens of 32 + 8 + 8 fp16 heads
// of 128: 21.3 us (23.8 with four steps at a time), 4.7 TB/s, where a large copy
// makes 5.2; a single token's 4.1 us are latency (the smallest kernels here take
// 2.3).
template <typename TI, typename TO, int L, bool FULL>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeParams p, uint32_t shares, uint32_t steps)
{
    constexpr int HPW = 64 / L;
    const uint32_t D = p.head_dim, heads = p.hq + 2 * p.hkv, nk = p.hq + p.hkv, lane = threadIdx.x & 63;
    const uint32_t j = lane % L, sub = lane / L, half = p.rot_dim / 2;
    const uint32_t turners = (p.neighbours ? p.rot_dim + 7 : 2 * half + 6) / 8;   // lanes with pairs
    const bool turned = j < turners, split = turned && !p.neighbours;
    // (neighbours: 8 values a lane throughout, pairs past rot_dim stay)
    const uint32_t base = p.neighbours || turned ? 8 * j : p.rot_dim + 8 * (j - turners);
    const uint32_t oa = split ? 4 * j : base, ob = split ? oa + half : base + 4, lim = split ? half : D;
    const uint32_t na = oa < lim ? min(4u, lim - oa) : 0u, nb = split ? na : ob < D ? min(4u, D - ob) : 0u;
    const bool on = na != 0;   // (a lane past the head's last value loads its first ones where FULL, and drops them)
    const uint32_t first_pos = p.count ? *p.count : 0u, rows = p.batch * p.tokens;
    const float inv_d = 1.0f / (float)D;
    float4v wq[2] = {(float4v)1.0f, (float4v)1.0f}, wk[2] = {(float4v)1.0f, (float4v)1.0f};
    if (p.q_weight) {
        wq[0] = weight4(p.q_weight, p.w_dtype, oa, na) + p.weight_offset;
        wq[1] = weight4(p.q_weight, p.w_dtype, ob, nb) + p.weight_offset;
    }
    if (p.k_weight) {
        wk[0] = weight4(p.k_weight, p.w_dtype, oa, na) + p.weight_offset;
        wk[1] = weight4(p.k_weight, p.w_dtype, ob, nb) + p.weight_offset;
    }
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t s0 = steps * blockIdx.y / shares, s1 = steps * (blockIdx.y + 1) / shares;
    for (uint32_t bt = blockIdx.x * 4 + wave; bt < rows; bt += gridDim.x * 4) {
        const uint32_t b = bt / p.tokens, t = bt - b * p.tokens;
        const TI* row = (const TI*)p.qkv + (size_t)bt * p.row_stride;
        float c[4], s[4];
        bool angles = false;
        for (uint32_t it = s0; it < s1; ++it) {
            const uint32_t h = it * HPW + sub, hc = min(h, heads - 1);
            const float4v xa = some4<FULL>(row + (size_t)hc * D + (FULL && !on ? 0u : oa), na);
            const float4v xb = some4<FULL>(row + (size_t)hc * D + (FULL && !on ? 0u : ob), nb);
            if (!angles) {   // (under the first loads)
                angles = true;
                const uint32_t pos = p.positions ? p.positions[bt] : first_pos + t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = 1.f;
                    s[i] = 0.f;
                    if (2 * (4 * j + i) < p.rot_dim) turn_of(p, pos, 4 * j + i, c[i], s[i]);
                }
            }
            float y[8], sq = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = xa[e];
                y[4 + e] = xb[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sq = fmaf(y[e], y[e], sq);
            sq = group_sum<L>(FULL && !on ? 0.f : sq);
            const bool is_q = h < p.hq, is_v = h >= nk;
            if (p.norm && !is_v) {
                float v = sq * inv_d + p.eps;
                if (__builtin_expect(__any(!rms_in_range(v)), 0)) {   // (whole groups of lanes hold the same v)
                    float amax = 0.f, sum = 0.f;
                    if (!FULL || on)
#pragma unroll
                        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, __builtin_fabsf(y[e]));
                    amax = group_max<L>(amax);
                    const int e2 = rms_in_range(v) ? 0 : rms_unit(amax, p.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y[e] = ldexpf(y[e], -e2);
                        sum = fmaf(y[e], y[e], sum);
                    }
                    sum = group_sum<L>(FULL && !on ? 0.f : sum);
                    v = sum * inv_d + ldexpf(p.eps, -2 * e2);
                }
                const float inv = inv_root(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= inv * (is_q ? wq[e >> 2][e & 3] : wk[e >> 2][e & 3]);
            }
            if (turned && !is_v) {
                const auto turn = [&](float& a, float& e, int i) __attribute__((always_inline)) {
                    const float x = a;
                    a = x * c[i] - e * s[i];
                    e = e * c[i] + x * s[i];
                };
                if (p.neighbours)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // (pairs past rot_dim are not turned by 0: an infinity times its sine would reach the other value)
                        if (FULL || 2 * (4 * j + i) < p.rot_dim) turn(y[2 * i], y[2 * i + 1], i);
                    }
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) turn(y[i], y[4 + i], i);
            }
            TO* out = (TO*)(is_q ? p.q_out : is_v ? p.v_out : p.k_out);
            const uint32_t oh = is_q ? h : is_v ? h - nk : h - p.hq, nh = is_q ? p.hq : p.hkv;
            if (on && h < heads && out) {
                TO* dst = out + (((size_t)b * nh + oh) * p.tokens + t) * D;
                put4<FULL>(dst + oa, na, float4v{y[0], y[1], y[2], y[3]});
                put4<FULL>(dst + ob, nb, float4v{y[4], y[5], y[6], y[7]});
            }
        }
    }
}

template <typename TI, typename TO, int L, bool FULL>
static hipError_t launch_vec(const QkNormRopeParams& p, hipStream_t s)
{
    // tokens whose waves alone fill the chip are not shared out: each share takes
    // the angles again (4096 tokens: one share 20.4 us, two 22.6)
    const uint32_t steps = (p.hq + 2 * p.hkv + 64 / L - 1) / (64 / L);
    const uint32_t rows = p.batch * p.tokens;
    const uint32_t shares = std::min(steps, std::max(1u, 4096 / rows));
    hipLaunchKernelGGL((qk_norm_rope_kernel<TI, TO, L, FULL>), dim3(std::min((rows + 3) / 4, 1u << 20), shares), dim3(256), 0, s,
                       p, shares, steps);
    return hipGetLastError();
}

template <typename TI, typename TO, bool FULL>
static hipError_t launch_lanes(const QkNormRopeParams& p, hipStream_t s)
{
    const uint32_t l = p.neighbours || !p.rot_dim ? (p.head_dim + 7) / 8
                                                  : (p.rot_dim + 6) / 8 + (p.head_dim - p.rot_dim + 7) / 8;
    if (l <= 4) return launch_vec<TI, TO, 4, FULL>(p, s);
    if (l <= 8) return launch_vec<TI, TO, 8, FULL>(p, s);
    if (l <= 16) return launch_vec<TI, TO, 16, FULL>(p, s);
    if (l <= 32) return launch_vec<TI, TO, 32, FULL>(p, s);
    return launch_vec<TI, TO, 64, FULL>(p, s);
}

hipError_t qk_norm_rope_launch(QkNormRopeParams p, float theta, hipStream_t s)
{
    // f_i = theta^(-2i / rot) in turns, i = 16 a + b, as a product of two short
    // tables: 32 powers on the host for up to 256 pairs
    if (p.rot_dim && !p.inv_freq) {
        const double step = -2.0 * std::log2((double)theta) / (double)p.rot_dim;
        for (uint32_t a = 0; 16 * a < p.rot_dim / 2; ++a) p.turn_hi[a] = std::exp2(16.0 * a * step);
        for (uint32_t b = 0; b < 16; ++b) p.turn_lo[b] = std::exp2(b * step) * 0.15915494309189533577;
    }
    // whole groups of four values everywhere (the tests for others cost a third:
    // 4096 tokens 33.7 us with them, 23.3 without)
    const bool full = p.head_dim % 8 == 0 && p.rot_dim % 8 == 0;
    if (p.head_dim <= (full ? 512 : 496)) {   // 64 lanes hold a head (with one more where both parts are odd)
        const auto go = [&](auto in, auto out) {
            typedef decltype(in) TI;
            typedef decltype(out) TO;
            return full ? launch_lanes<TI, TO, true>(p, s) : launch_lanes<TI, TO, false>(p, s);
        };
        if (p.i_dtype == DT_F16) return p.o_dtype == DT_F16 ? go(half_t{}, half_t{}) : go(half_t{}, float{});
        return p.o_dtype == DT_F16 ? go(float{}, half_t{}) : go(float{}, float{});
    }
    const uint64_t units = (uint64_t)p.batch * p.tokens * (p.hq + 2 * p.hkv);
    hipLaunchKernelGGL(qk_norm_rope_any_kernel, dim3((uint32_t)std::min<uint64_t>(units, 65536)), dim3(64), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
