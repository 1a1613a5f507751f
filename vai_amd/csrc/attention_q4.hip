// attention_q4.hip -- the KV cache in 4 bits (q4_cache.h): appending a call's
// rows, reading rows back, and attention over the values as stored.
//
// A call's new rows are rounded into the cache first and then attended like
// every other cached row, so the result does not depend on how a sequence was
// cut into calls.
#include <algorithm>

#include "kernels.h"
#include "launch_once.h"
#include "q4_cache.h"

namespace vai_dev {

// dp / 8 lanes to a row of one plane, 8 values each; a workgroup takes 2048 / dp
// rows of K and of V at a time.
__global__ __launch_bounds__(256) void q4_append_kernel(AttnParams p, uint32_t dp)
{
    const uint32_t HD = p.head_dim, hk = blockIdx.y, lanes = dp / 8, c = threadIdx.x % lanes, plane = blockIdx.z;
    const uint32_t cached = *p.cache_count, step = 256 / lanes;
    uint8_t* head = (plane ? p.v4 : p.k4) + (size_t)hk * q4::head_bytes(p.kv_rows, dp);
    const void* src = plane ? p.v_new : p.k_new;
    // (whole workgroups of rows: the exchanges between a group's lanes need them all)
    for (uint64_t t0 = (uint64_t)blockIdx.x * step; t0 < p.tkv; t0 += (uint64_t)gridDim.x * step) {
        const uint64_t t = t0 + threadIdx.x / lanes;
        const uint32_t tok = (uint32_t)std::min<uint64_t>(t, p.tkv - 1), pos = cached + tok;
        half_t s, m;
        const uint32_t values = 8 * c < HD ? HD - 8 * c : 0u;
        const half8 h = q4::row8(src, p.new_dtype, ((size_t)hk * p.tkv + tok) * HD, 8 * c, HD);
        const uint32_t codes = q4::encode8(h, values, s, m);
        // positions past a plane are dropped (a ring's rows all differ: Tkv <= its size)
        if (t >= p.tkv || !(p.ring || (pos < p.kv_rows && pos >= cached))) continue;
        const uint32_t row = p.ring ? pos % p.kv_rows : pos, j = row % q4::KT;
        uint8_t* tile = head + (size_t)(row / q4::KT) * q4::tile_bytes(dp);
        if (plane == 0) q4::put_k(tile, dp, j, c, codes, s, m);
        else q4::put_v(tile, dp, j, c, codes, s, m);
    }
}

// The value stored at position row, value d of a head's plane.
__device__ __forceinline__ float q4_value(const uint8_t* head, uint32_t dp, uint32_t row, uint32_t d, bool is_v)
{
    const uint32_t j = row % q4::KT;
    const uint8_t* tile = head + (size_t)(row / q4::KT) * q4::tile_bytes(dp);
    const half_t* sm = (const half_t*)(tile + (is_v ? q4::v_scale(dp, j, d) : q4::k_scale(dp, j, d)));
    const uint32_t n = is_v ? (tile[q4::v_byte(dp, j, d)] >> (4 * (d & 1))) & 15u
                            : (*(const uint32_t*)(tile + q4::k_word(dp, j, d)) >> (4 * q4::nibble_of(d & 7))) & 15u;
    return fmaf((float)sm[0], (float)n, (float)sm[is_v ? 8 : 1]);
}

// The live rows of the cache as fp16 copies for the kernels that read fp16:
// from the 64-position tile the first query's window starts in. Each wave takes
// a row of one head. A hidden position must not reach a query through a NaN
// (0 * NaN in P V), so a row with a NaN in V is copied as V = 0 and K = NaN:
// the score is masked where the position is hidden and NaN where it is not.
__global__ __launch_bounds__(256) void q4_copy_kernel(AttnParams p, uint32_t dp, half_t* k16, half_t* v16)
{
    const uint32_t HD = p.head_dim, hk = blockIdx.y, lane = threadIdx.x & 63;
    const uint32_t cached = *p.cache_count;
    const uint64_t end = (uint64_t)cached + p.tkv;
    uint64_t beg = (uint64_t)p.mask.key_start_cached(0, cached) / 64 * 64;
    // (a ring holds the last kv_rows positions)
    if (p.ring && end > p.kv_rows && beg < end - p.kv_rows) beg = end - p.kv_rows;
    const uint64_t live = p.ring ? end : std::min<uint64_t>(end, p.kv_rows);
    const size_t hb = q4::head_bytes(p.kv_rows, dp);
    const uint8_t* kh = p.k4 + hk * hb;
    const uint8_t* vh = p.v4 + hk * hb;
    for (uint64_t pos = beg + blockIdx.x * 4 + (threadIdx.x >> 6); pos < live; pos += (uint64_t)gridDim.x * 4) {
        const uint32_t row = p.ring ? (uint32_t)(pos % p.kv_rows) : (uint32_t)pos;
        const size_t dst = ((size_t)hk * p.kv_rows + row) * HD;
        bool bad = false;
        for (uint32_t d = lane; d < HD; d += 64) {
            const float v = q4_value(vh, dp, row, d, true);
            bad |= v != v;
            v16[dst + d] = v != v ? (half_t)0.f : (half_t)v;
        }
        bad = __any(bad);
        for (uint32_t d = lane; d < HD; d += 64)
            k16[dst + d] = bad ? (half_t)__builtin_nanf("") : (half_t)q4_value(kh, dp, row, d, false);
    }
}

__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadParams p, uint32_t dp)
{
    const uint32_t hk = blockIdx.y, plane = blockIdx.z, HD = p.head_dim;
    const size_t total = (size_t)p.n * HD;
    void* out = plane ? p.v_out : p.k_out;
    const void* src = plane ? p.v : p.k;
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (size_t)gridDim.x * 256) {
        const uint32_t i = (uint32_t)(e / HD), d = (uint32_t)(e % HD);
        const uint32_t row = (uint32_t)(((uint64_t)p.first + i) % p.rows);
        const float v = p.cache_dtype == DT_Q4
                            ? q4_value((const uint8_t*)src + hk * q4::head_bytes(p.rows, dp), dp, row, d, plane != 0)
                            : ld(src, p.cache_dtype, ((size_t)hk * p.rows + row) * HD + d);
        st(out, p.o_dtype, (size_t)hk * total + e, v);
    }
}

uint32_t q4_dp(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : head_dim <= 256 ? 256 : 0; }

size_t q4_plane_bytes(uint32_t hkv, uint32_t rows, uint32_t head_dim)
{
    return hkv * q4::head_bytes(rows, q4_dp(head_dim));
}

hipError_t cache_read_launch(const CacheReadParams& p, hipStream_t s)
{
    const size_t blocks = ((size_t)p.n * p.head_dim + 255) / 256;
    hipLaunchKernelGGL(cache_read_kernel, dim3((uint32_t)std::min<size_t>(blocks, 4096), p.hkv, 2), dim3(256), 0, s, p,
                       q4_dp(p.head_dim));
    return hipGetLastError();
}

static size_t copy_bytes(const AttnParams& p)
{
    return (2 * (size_t)p.hkv * p.kv_rows * p.head_dim * sizeof(half_t) + 255) & ~(size_t)255;
}

void attention_q4_plan(AttnParams& p, uint32_t cus)
{
    if (q4_few_rows(p)) {
        p.q4 = 2;
        q4_decode_plan(p, cus);
    } else {
        p.q4 = 1;
        attention_plan(p, cus);
    }
}

size_t attention_q4_workspace(const AttnParams& p)
{
    return p.q4 == 2 ? q4_decode_workspace(p) : copy_bytes(p) + attention_workspace_bytes(p);
}

void attention_q4_set_workspace(AttnParams& p, void* ws)
{
    p.ws4 = ws;
    if (p.q4 == 2) return;
    p.k = ws;
    p.v = (half_t*)ws + (size_t)p.hkv * p.kv_rows * p.head_dim;
    attention_set_workspace(p, (char*)ws + copy_bytes(p));
}

hipError_t attention_q4_launch(const AttnParams& p, hipStream_t s)
{
    if (p.q4 == 2) return q4_decode_launch(p, p.ws4, s);
    const uint32_t dp = q4_dp(p.head_dim);
    if (p.tkv > 0) {
        const uint32_t blocks = (p.tkv + 2048 / dp - 1) / (2048 / dp);
        hipLaunchKernelGGL(q4_append_kernel, dim3(std::min(blocks, 4096u), p.hkv, 2), dim3(256), 0, s, p, dp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(q4_copy_kernel, dim3(std::min<uint32_t>((p.kv_rows + 3) / 4, 2048), p.hkv), dim3(256), 0, s, p, dp,
                       (half_t*)p.k, (half_t*)p.v);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return attention_launch(p, s);
}

}   // namespace vai_dev
