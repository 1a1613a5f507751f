// paged_append.hip -- from the fused query / key / value projection of a ragged
// batch to the KV cache's pages: RMS norm of each query and key head, the
// position rotation, queries to token-major rows, keys and values to the slot of
// their position, in one pass.
//
//   y_d = x_d / sqrt(mean_d x_d^2 + eps) * (w_d + offset)
//   (a, e) -> (a cos t - e sin t, e cos t + a sin t), t = position * f_i
//
// for the rot_dim / 2 pairs (a, e) = (y_i, y_{i + rot/2}) or (y_2i, y_2i+1).
// Bound by memory: each value is read once and written once.
#include <algorithm>

#include "head_rows.h"
#include "pages.h"

namespace vai_dev {

namespace {

// Where a token's keys and values go: its position, and the slot (slot < 0: none)
struct Place {
    uint32_t pos;
    int64_t slot;      // element of the pages where head 0's values of the position start
    bool row;          // whether the token is a sequence's
};
__device__ __forceinline__ Place place_of(const PagedAppendParams& p, uint32_t token)
{
    Place r{0, -1, false};
    const KvPages& g = p.pages;
    // (the same in every lane: scalar registers)
    const auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); };
    const uint32_t s = wave_last_le(g.start, g.sequences, token);
    if (s == g.sequences || token >= uniform(g.start[s + 1])) return r;
    r.row = true;
    const uint64_t pos = (uint64_t)uniform(g.counts[s]) + (token - uniform(g.start[s]));
    r.pos = (uint32_t)pos;
    if (pos < (uint64_t)g.max_pages * g.page_size) {
        const uint32_t i = r.pos / g.page_size, page = uniform(g.table[(size_t)s * g.max_pages + i]);
        if (page < g.num_pages) r.slot = (int64_t)(page * g.stride + (uint64_t)(r.pos - i * g.page_size) * p.head_dim);
    }
    return r;
}

template <bool FULL>
__device__ __forceinline__ void put4_as(void* base, int dt, size_t i, uint32_t n, float4v v)
{
    if (dt == DT_F16) put4<FULL>((half_t*)base + i, n, v);
    else put4<FULL>((float*)base + i, n, v);
}

}   // namespace

// Larger head dims: a wave takes one head at a time, in LDS as fp32.
__global__ __launch_bounds__(64) void paged_append_any_kernel(PagedAppendParams p)
{
    __shared__ float y[PagedAppendParams::MAX_DIM];
    const uint32_t D = p.head_dim, first = p.q_out ? 0u : p.hq, heads = p.hq + 2 * p.hkv - first, lane = threadIdx.x;
    const uint64_t total = (uint64_t)p.tokens * heads;
    for (uint64_t u = blockIdx.x; u < total; u += gridDim.x) {
        const uint32_t token = (uint32_t)(u / heads), h = first + (uint32_t)(u - (uint64_t)token * heads);
        const Place at = place_of(p, token);
        const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
        if (!at.row || (!is_q && at.slot < 0)) continue;
        const size_t src = (size_t)token * p.row_stride + (size_t)h * D;
        float sq = 0.f;
        for (uint32_t d = lane; d < D; d += 64) {
            const float x = ld(p.qkv, p.i_dtype, src + d);
            y[d] = x;
            sq += x * x;
        }
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
        void* out = is_q ? p.q_out : is_v ? p.pages.v : p.pages.k;
        const int dt = is_q ? p.o_dtype : p.pages.dtype;
        const uint32_t kh = is_v ? h - p.hq - p.hkv : h - p.hq;
        const size_t dst = is_q ? ((size_t)token * p.hq + h) * D : (size_t)at.slot + (size_t)kh * p.pages.page_size * D;
        for (uint32_t d = lane; d < D; d += 64) {
            float v = y[d];
            if (d < rot) {
                const bool second = p.neighbours ? (d & 1) : d >= half;
                const uint32_t i = p.neighbours ? d / 2 : second ? d - half : d;
                const float o = y[p.neighbours ? d ^ 1 : second ? d - half : d + half];
                float c, s;
                turn_of(p, at.pos, i, c, s);
                v = second ? v * c + o * s : v * c - o * s;
            }
            st(out, dt, dst + d, v);
        }
        __syncthreads();   // y is rewritten by the next head
    }
}

// Head dims up to 512, as qk_norm_rope_kernel cuts them: L lanes share a head, 8
// values each, so that a lane holds both values of its four pairs (FULL: of all
// its groups of four). A wave takes a token's heads 64 / L at a time, its share of
// them (blockIdx.y of `shares`), the next heads' values in flight. 4098 tokens in
// three sequences, 32 + 8 + 8 fp16 heads of 128: 24 us, 4.2 TB/s (with one step's
// loads at a time and the weights in registers, four waves a SIMD, 33); a single
// token's 5 us are latency.
template <typename TI, int L, bool FULL>
__global__ __launch_bounds__(256, 5) void paged_append_kernel(PagedAppendParams p, uint32_t shares, uint32_t steps)
{
    constexpr int HPW = 64 / L;
    const uint32_t D = p.head_dim, heads = p.hq + 2 * p.hkv, nk = p.hq + p.hkv, lane = threadIdx.x & 63;
    const uint32_t h0 = p.q_out ? 0u : p.hq;
    const uint32_t j = lane % L, sub = lane / L, half = p.rot_dim / 2;
    const uint32_t turners = (p.neighbours ? p.rot_dim + 7 : 2 * half + 6) / 8;   // lanes with pairs
    const bool turned = j < turners, split = turned && !p.neighbours;
    const uint32_t base = p.neighbours || turned ? 8 * j : p.rot_dim + 8 * (j - turners);
    const uint32_t oa = split ? 4 * j : base, ob = split ? oa + half : base + 4, lim = split ? half : D;
    const uint32_t na = oa < lim ? min(4u, lim - oa) : 0u, nb = split ? na : ob < D ? min(4u, D - ob) : 0u;
    const bool on = na != 0;   // (a lane past the head's last value loads its first ones where FULL, and drops them)
    const float inv_d = 1.0f / (float)D;
    // a lane's weights wait in LDS, not in registers: five waves a SIMD instead of four (for
    // which 8 to 32 lanes a head of whole groups still keep 4 or 5 registers in scratch)
    __shared__ float4v weights[4][4][64];
    float4v w4[4] = {(float4v)1.0f, (float4v)1.0f, (float4v)1.0f, (float4v)1.0f};
    if (p.q_weight) {
        w4[0] = weight4(p.q_weight, p.w_dtype, oa, na);
        w4[1] = weight4(p.q_weight, p.w_dtype, ob, nb);
    }
    if (p.k_weight) {
        w4[2] = weight4(p.k_weight, p.w_dtype, oa, na);
        w4[3] = weight4(p.k_weight, p.w_dtype, ob, nb);
    }
    bool kept = false;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t s0 = steps * blockIdx.y / shares, s1 = steps * (blockIdx.y + 1) / shares;
    for (uint32_t token = blockIdx.x * 4 + wave; token < p.tokens; token += gridDim.x * 4) {
        const TI* row = (const TI*)p.qkv + (size_t)token * p.row_stride;
        Place at{};
        float c[4], s[4];
        bool angles = false;
        typedef TI t4 __attribute__((ext_vector_type(4)));
        typedef t4 t4u __attribute__((aligned(sizeof(TI))));
        t4 ra, rb;               // (FULL: the next step's values, as they are)
        const auto read = [&](uint32_t it) __attribute__((always_inline)) {
            const TI* src = row + (size_t)min(h0 + it * HPW + sub, heads - 1) * D;
            ra = *(const t4u*)(src + (on ? oa : 0u));
            rb = *(const t4u*)(src + (on ? ob : 0u));
        };
        if constexpr (FULL) read(s0);
        for (uint32_t it = s0; it < s1; ++it) {
            const uint32_t h = h0 + it * HPW + sub;
            float4v xa, xb;
            if constexpr (FULL) {
                xa = __builtin_convertvector(ra, float4v);
                xb = __builtin_convertvector(rb, float4v);
                if (it + 1 < s1) read(it + 1);
            } else {
                const TI* src = row + (size_t)min(h, heads - 1) * D;
                xa = some4<false>(src + oa, na);
                xb = some4<false>(src + ob, nb);
            }
            if (!angles) {   // (under the first loads)
                angles = true;
                at = place_of(p, token);
                if (!kept) {
                    kept = true;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        weights[wave][i][lane] = w4[i] + ((i < 2 ? p.q_weight : p.k_weight) ? p.weight_offset : 0.f);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = 1.f;
                    s[i] = 0.f;
                    if (2 * (4 * j + i) < p.rot_dim) turn_of(p, at.pos, 4 * j + i, c[i], s[i]);
                }
            }
            if (!at.row) break;
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
                const float4v wa = weights[wave][is_q ? 0 : 2][lane], wb = weights[wave][is_q ? 1 : 3][lane];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= inv * (e < 4 ? wa[e & 3] : wb[e & 3]);
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
            if (!on || h >= heads || (!is_q && at.slot < 0)) continue;
            void* out = is_q ? p.q_out : is_v ? p.pages.v : p.pages.k;
            const int dt = is_q ? p.o_dtype : p.pages.dtype;
            const uint32_t kh = is_v ? h - nk : h - p.hq;
            const size_t dst = is_q ? ((size_t)token * p.hq + h) * D : (size_t)at.slot + (size_t)kh * p.pages.page_size * D;
            put4_as<FULL>(out, dt, dst + oa, na, float4v{y[0], y[1], y[2], y[3]});
            put4_as<FULL>(out, dt, dst + ob, nb, float4v{y[4], y[5], y[6], y[7]});
        }
    }
}

template <typename TI, int L, bool FULL>
static hipError_t launch_vec(const PagedAppendParams& p, hipStream_t s)
{
    // tokens whose waves alone fill the chip are not shared out: each share takes the
    // place and the angles again, as long as one and a half of its steps (32 + 8 + 8
    // heads of 128, 12 steps; tokens: us with 1, 2, 4, 12 shares: 64: 12.8, 9.0, 7.3, 6.4;
    // 1000: 15.1, 11.8, 11.7, 18.6; 2500: 19.3, 17.5; 3000: 19.6, 23.6. Other numbers of
    // steps take the line that these draw.)
    const uint32_t steps = ((p.q_out ? p.hq : 0u) + 2 * p.hkv + 64 / L - 1) / (64 / L);
    const uint32_t shares = std::min(steps, std::max(1u, (3800 + p.tokens / 2) / p.tokens));
    hipLaunchKernelGGL((paged_append_kernel<TI, L, FULL>), dim3(std::min((p.tokens + 3) / 4, 1u << 20), shares), dim3(256), 0,
                       s, p, shares, steps);
    return hipGetLastError();
}

template <typename TI, bool FULL>
static hipError_t launch_lanes(const PagedAppendParams& p, hipStream_t s)
{
    const uint32_t l = p.neighbours || !p.rot_dim ? (p.head_dim + 7) / 8
                                                  : (p.rot_dim + 6) / 8 + (p.head_dim - p.rot_dim + 7) / 8;
    if (l <= 4) return launch_vec<TI, 4, FULL>(p, s);
    if (l <= 8) return launch_vec<TI, 8, FULL>(p, s);
    if (l <= 16) return launch_vec<TI, 16, FULL>(p, s);
    if (l <= 32) return launch_vec<TI, 32, FULL>(p, s);
    return launch_vec<TI, 64, FULL>(p, s);
}

hipError_t paged_append_launch(PagedAppendParams p, float theta, hipStream_t s)
{
    rope_tables(p, theta);
    const bool full = p.head_dim % 8 == 0 && p.rot_dim % 8 == 0;   // whole groups of four values everywhere
    if (p.head_dim <= (full ? 512 : 496)) {   // 64 lanes hold a head (with one more where both parts are odd)
        if (p.i_dtype == DT_F16) return full ? launch_lanes<half_t, true>(p, s) : launch_lanes<half_t, false>(p, s);
        return full ? launch_lanes<float, true>(p, s) : launch_lanes<float, false>(p, s);
    }
    const uint64_t units = (uint64_t)p.tokens * ((p.q_out ? p.hq : 0u) + 2 * p.hkv);
    hipLaunchKernelGGL(paged_append_any_kernel, dim3((uint32_t)std::min<uint64_t>(units, 65536)), dim3(64), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
