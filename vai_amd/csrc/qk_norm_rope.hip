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
// keep three digits), and only its fraction goes on in fp32.
__device__ __forceinline__ void turn_of(const QkNormRopeParams& p, uint32_t pos, uint32_t i, float& c, float& s)
{
    const double f = p.inv_freq ? (double)p.inv_freq[i] * 0.15915494309189533577 : p.turn_hi[i >> 4] * p.turn_lo[i & 15];
    const double t = (double)pos * f;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
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

hipError_t qk_norm_rope_launch(QkNormRopeParams p, float theta, hipStream_t s)
{
    // f_i = theta^(-2i / rot) in turns, i = 16 a + b, as a product of two short
    // tables: 32 powers on the host for up to 256 pairs
    if (p.rot_dim && !p.inv_freq) {
        const double step = -2.0 * std::log2((double)theta) / (double)p.rot_dim;
        for (uint32_t a = 0; 16 * a < p.rot_dim / 2; ++a) p.turn_hi[a] = std::exp2(16.0 * a * step);
        for (uint32_t b = 0; b < 16; ++b) p.turn_lo[b] = std::exp2(b * step) * 0.15915494309189533577;
    }
    const uint64_t units = (uint64_t)p.batch * p.tokens * (p.hq + 2 * p.hkv);
    hipLaunchKernelGGL(qk_norm_rope_any_kernel, dim3((uint32_t)std::min<uint64_t>(units, 65536)), dim3(64), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
