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

// Any head dim: a wave takes one head at a time, in LDS as fp32.
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
            const float inv = 1.0f / sqrtf(wave_sum(sq) / (float)D + p.eps);
            const void* w = is_q ? p.q_weight : p.k_weight;
            for (uint32_t d = lane; d < D; d += 64)
                y[d] = y[d] * inv * (w ? ld(w, p.w_dtype, d) + p.weight_offset : 1.0f);
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

// x summed over each group of L lanes (a power of two), in every lane
template <int L>
__device__ __forceinline__ float group_sum(float x)
{
    const auto moved = [](float v, auto ctrl) __attribute__((always_inline)) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (L >= 2) x += moved(x, std::integral_constant<int, 0xB1>{});    // lane ^ 1
    if constexpr (L >= 4) x += moved(x, std::integral_constant<int, 0x4E>{});    // lane ^ 2
    if constexpr (L >= 8) x += moved(x, std::integral_constant<int, 0x141>{});   // the other 4 of 8 (mirrored)
    if constexpr (L >= 16) x += moved(x, std::integral_constant<int, 0x140>{});  // the other 8 of 16
    if constexpr (L >= 32) x += __shfl_xor(x, 16);
    if constexpr (L >= 64) x += __shfl_xor(x, 32);
    return x;
}

// Head dims that are a multiple of 8, up to 512, rotated in whole groups of 8:
// L lanes (D / 8 rounded up to a power of two) share a head, 8 values each, cut
// so that a lane holds both values of its four pairs: with halves values 4 j ..
// +3 and the same of the other half, else 8 neighbouring ones. A lane's four
// angles then serve every head of the token. A wave takes a token's heads 64 / L
// at a time, its share of them (blockIdx.y of `shares`). One step's loads at a
// time and 44 registers: eight waves a SIMD hide the loads better than four
// steps at a time in 72 registers do. 4096 tokens of 32 + 8 + 8 fp16 heads of
// 128: 20.4 us (23.8 with four steps at a time), 4.9 TB/s, where a large copy
// makes 5.2; a single token's 3.9 us are latency (the smallest kernels here take 2.3).
__device__ __forceinline__ float4v weight4(const void* w, int dt, uint32_t d)
{
    typedef half4 half4u __attribute__((aligned(2)));
    if (dt == DT_F16) return __builtin_convertvector(*(const half4u*)((const half_t*)w + d), float4v);
    return load4f((const float*)w + d);
}

template <typename TI, typename TO, int L>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormRopeParams p, uint32_t shares, uint32_t steps)
{
    typedef TI in4 __attribute__((ext_vector_type(4)));
    typedef TO out4 __attribute__((ext_vector_type(4)));
    constexpr int HPW = 64 / L;
    const uint32_t D = p.head_dim, heads = p.hq + 2 * p.hkv, nk = p.hq + p.hkv, lane = threadIdx.x & 63;
    const uint32_t j = lane % L, sub = lane / L, half = p.rot_dim / 2;
    const bool on = 8 * j < D, turned = 8 * j < p.rot_dim, split = turned && !p.neighbours;
    const uint32_t oa = !on ? 0u : split ? 4 * j : 8 * j, ob = split ? oa + half : on ? oa + 4 : 0u;
    const uint32_t first_pos = p.count ? *p.count : 0u, rows = p.batch * p.tokens;
    const float inv_d = 1.0f / (float)D;
    float4v wq[2] = {(float4v)1.0f, (float4v)1.0f}, wk[2] = {(float4v)1.0f, (float4v)1.0f};
    if (p.q_weight) {
        wq[0] = weight4(p.q_weight, p.w_dtype, oa) + p.weight_offset;
        wq[1] = weight4(p.q_weight, p.w_dtype, ob) + p.weight_offset;
    }
    if (p.k_weight) {
        wk[0] = weight4(p.k_weight, p.w_dtype, oa) + p.weight_offset;
        wk[1] = weight4(p.k_weight, p.w_dtype, ob) + p.weight_offset;
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
            const in4 xa = *(const in4*)(row + (size_t)hc * D + oa), xb = *(const in4*)(row + (size_t)hc * D + ob);
            if (!angles) {   // (under the first loads)
                angles = true;
                const uint32_t pos = p.positions ? p.positions[bt] : first_pos + t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = 1.f;
                    s[i] = 0.f;
                    if (turned) turn_of(p, pos, 4 * j + i, c[i], s[i]);
                }
            }
            float y[8], sq = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = (float)xa[e];
                y[4 + e] = (float)xb[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sq = fmaf(y[e], y[e], sq);
            sq = group_sum<L>(on ? sq : 0.f);
            const bool is_q = h < p.hq, is_v = h >= nk;
            if (p.norm && !is_v) {
                const float inv = __builtin_amdgcn_rsqf(sq * inv_d + p.eps);
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
                    for (int i = 0; i < 4; ++i) turn(y[2 * i], y[2 * i + 1], i);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) turn(y[i], y[4 + i], i);
            }
            TO* out = (TO*)(is_q ? p.q_out : is_v ? p.v_out : p.k_out);
            const uint32_t oh = is_q ? h : is_v ? h - nk : h - p.hq, nh = is_q ? p.hq : p.hkv;
            if (on && h < heads && out) {
                TO* dst = out + (((size_t)b * nh + oh) * p.tokens + t) * D;
                *(out4*)(dst + oa) = __builtin_convertvector((float4v{y[0], y[1], y[2], y[3]}), out4);
                *(out4*)(dst + ob) = __builtin_convertvector((float4v{y[4], y[5], y[6], y[7]}), out4);
            }
        }
    }
}

template <typename TI, typename TO, int L>
static hipError_t launch_vec(const QkNormRopeParams& p, hipStream_t s)
{
    // tokens whose waves alone fill the chip are not shared out: each share takes
    // the angles again (4096 tokens: one share 20.4 us, two 22.6)
    const uint32_t steps = (p.hq + 2 * p.hkv + 64 / L - 1) / (64 / L);
    const uint32_t rows = p.batch * p.tokens;
    const uint32_t shares = std::min(steps, std::max(1u, 4096 / rows));
    hipLaunchKernelGGL((qk_norm_rope_kernel<TI, TO, L>), dim3(std::min((rows + 3) / 4, 1u << 20), shares), dim3(256), 0, s,
                       p, shares, steps);
    return hipGetLastError();
}

template <typename TI, typename TO>
static hipError_t launch_lanes(const QkNormRopeParams& p, hipStream_t s)
{
    const uint32_t l = p.head_dim / 8;
    if (l <= 4) return launch_vec<TI, TO, 4>(p, s);
    if (l <= 8) return launch_vec<TI, TO, 8>(p, s);
    if (l <= 16) return launch_vec<TI, TO, 16>(p, s);
    if (l <= 32) return launch_vec<TI, TO, 32>(p, s);
    return launch_vec<TI, TO, 64>(p, s);
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
    // four values at a time from every row of every plane
    const size_t isz = p.i_dtype == DT_F16 ? 8 : 16, osz = p.o_dtype == DT_F16 ? 8 : 16;
    const uintptr_t outs = (uintptr_t)p.q_out | (uintptr_t)p.k_out | (uintptr_t)p.v_out;
    if (p.head_dim % 8 == 0 && p.head_dim <= 512 && p.rot_dim % 8 == 0 && p.row_stride % 4 == 0 &&
        (uintptr_t)p.qkv % isz == 0 && outs % osz == 0) {
        if (p.i_dtype == DT_F16)
            return p.o_dtype == DT_F16 ? launch_lanes<half_t, half_t>(p, s) : launch_lanes<half_t, float>(p, s);
        return p.o_dtype == DT_F16 ? launch_lanes<float, half_t>(p, s) : launch_lanes<float, float>(p, s);
    }
    const uint64_t units = (uint64_t)p.batch * p.tokens * (p.hq + 2 * p.hkv);
    hipLaunchKernelGGL(qk_norm_rope_any_kernel, dim3((uint32_t)std::min<uint64_t>(units, 65536)), dim3(64), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
