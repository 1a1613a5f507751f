// attention_q4.hip -- the KV cache in 4 bits (q4_cache.h): appending a call's
// rows, reading rows back, and attention over the values as stored.
//
// A call's new rows are rounded into the cache first and then attended like
// every other cached row, so what the cache holds does not depend on how a sequence
// was cut into calls. Results do in their last places: calls of many rows
// (q4_few_rows is false) read the cache as fp16 copies.
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

// 8 values of a row from value 8 c on, in fp32
__device__ __forceinline__ void q4_values8(const uint8_t* head, uint32_t dp, uint32_t row, uint32_t c, bool is_v, float (&x)[8])
{
    const uint32_t j = row % q4::KT, d = 8 * c;
    const uint8_t* tile = head + (size_t)(row / q4::KT) * q4::tile_bytes(dp);
    const float s = (float)*(const half_t*)(tile + (is_v ? q4::v_scale(dp, j, d) : q4::k_step(dp, j, d)));
    const float m = (float)*(const half_t*)(tile + (is_v ? q4::v_scale(dp, j, d) + 16 : q4::k_min(dp, j, d)));
    uint32_t w = 0;
    if (is_v) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w |= (uint32_t)tile[q4::v_byte(dp, j, d + 2 * i)] << (8 * i);
    } else {
        w = *(const uint32_t*)(tile + q4::k_word(dp, j, d));
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) x[e] = fmaf(s, (float)(w >> (4 * (is_v ? e : q4::nibble_of(e))) & 15u), m);
}

// The live rows of the cache as copies for the kernels that read rows of values
// (T: fp16 for the flash kernel, fp32, exact, for the plain one): from the
// 64-position tile the first query's window starts in. K and V rounded to fp16 are
// what the flash kernel's matrix products take, as of an fp16 cache: a result is
// then off by 3.4e-4 to 4.1e-4 of its norm (1.9e-4 from the codes; with fp16 output
// and channels of K that stand out 5.8e-4), and a prompt of 512 tokens over 7001
// cached positions takes 98 us where the codes, unpacked for every 32 rows, take 173.
//
// A workgroup takes a 32-position tile of one head at a time: half its threads V
// (a slice of 4 positions each, so that a row's values leave in wide stores), half
// K (a word of 8 values each). A hidden position must not reach a query through a NaN (0 *
// NaN in P V), so a row with a NaN in V is copied as V = 0 and K = NaN: the score
// is masked where the position is hidden and NaN where it is not.
// 7513 positions of 8 heads of 128: 16 us (25 with a wave to a row).
template <int DP, typename T>
__global__ __launch_bounds__(256) void q4_copy_kernel(AttnParams p, T* k_out, T* v_out)
{
    constexpr int G = DP / 32, ND = DP / 16;
    __shared__ uint32_t bad[2][q4::KT];
    const uint32_t HD = p.head_dim, hk = blockIdx.y, t = threadIdx.x;
    const uint32_t cached = *p.cache_count;
    const uint64_t end = (uint64_t)cached + p.tkv;
    uint64_t beg = (uint64_t)p.mask.key_start_cached(0, cached) / 64 * 64;
    // (a ring holds the last kv_rows positions)
    if (p.ring && end > p.kv_rows && beg < end - p.kv_rows) beg = end - p.kv_rows;
    const uint64_t live = p.ring ? end : std::min<uint64_t>(end, p.kv_rows);
    const size_t hb = q4::head_bytes(p.kv_rows, DP);
    const uint8_t* kh = p.k4 + hk * hb;
    const uint8_t* vh = p.v4 + hk * hb;
    const uint32_t wrap = p.ring ? p.kv_rows / q4::KT : 0xffffffffu;
    if (t < 2 * q4::KT) bad[t / q4::KT][t % q4::KT] = 0;
    __syncthreads();
    uint32_t round = 0;
    for (uint64_t tile = beg / q4::KT + blockIdx.x; tile * q4::KT < live; tile += gridDim.x, round ^= 1) {
        const uint32_t place = (uint32_t)(p.ring ? tile % wrap : tile), row0 = place * q4::KT;
        const uint8_t* kt = kh + (size_t)place * q4::tile_bytes(DP);
        const uint8_t* vt = vh + (size_t)place * q4::tile_bytes(DP);
        const size_t dst = ((size_t)hk * p.kv_rows + row0) * HD;
        // rows of this tile that are copied (of a ring also those a full turn older: not before beg)
        const auto copied = [&](uint32_t j) { return tile * q4::KT + j >= beg && tile * q4::KT + j < live; };
        for (uint32_t e = t; e < q4::KT * G; e += 256) {
            const uint32_t j = e % q4::KT;
            const half_t m = *(const half_t*)(vt + q4::v_scale(DP, j, e / q4::KT * 32) + 16);
            if (m != m) bad[round][j] = 1;
        }
        __syncthreads();
        if (t < 128) {
            const uint32_t slice = t % 16, b = t / 32, h = t / 16 % 2, d0 = slice * ND;   // positions 8 b + 4 h ..+3
            uint32_t w[ND / 2];
#pragma unroll
            for (int i = 0; i < ND / 2; ++i)
                w[i] = *(const uint32_t*)(vt + b * (DP * 4) + slice * (DP / 4) + i * 8 + h * 4);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t j = 8 * b + 4 * h + r;
                const half_t* sm = (const half_t*)(vt + q4::v_scale(DP, j, d0));
                const float s = (float)sm[0], m = (float)sm[8];
                typedef T out_t __attribute__((ext_vector_type(ND)));
                typedef out_t out_u __attribute__((aligned(sizeof(T))));
                out_t x;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    const float v = fmaf(s, (float)(w[i / 2] >> (8 * r + 4 * (i & 1)) & 15u), m);
                    x[i] = v != v ? (T)0.f : (T)v;
                }
                T* o = v_out + dst + (size_t)j * HD + d0;
                if (!copied(j)) continue;
                if (d0 + ND <= HD) *(out_u*)o = x;
                else
#pragma unroll
                    for (int i = 0; i < ND; ++i)
                        if (d0 + i < HD) o[i] = x[i];
            }
        } else {
            for (uint32_t e = t - 128; e < q4::KT * DP / 8; e += 128) {
                const uint32_t j = e / (DP / 8), c = e % (DP / 8);
                const uint32_t w = *(const uint32_t*)(kt + q4::k_word(DP, j, 8 * c));
                const float s = bad[round][j] ? __builtin_nanf("") : (float)*(const half_t*)(kt + q4::k_step(DP, j, 8 * c));
                const float m = (float)*(const half_t*)(kt + q4::k_min(DP, j, 8 * c));
                typedef T out8 __attribute__((ext_vector_type(8)));
                typedef out8 out8u __attribute__((aligned(sizeof(T))));
                out8 x;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) x[i] = (T)fmaf(s, (float)(w >> (4 * q4::nibble_of(i)) & 15u), m);
                T* o = k_out + dst + (size_t)j * HD + 8 * c;
                if (!copied(j)) continue;
                if (8 * c + 8 <= HD) *(out8u*)o = x;
                else
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (8 * c + i < HD) o[i] = x[i];
            }
        }
        // (the other round's flags, which every thread is done with)
        if (t < q4::KT) bad[round ^ 1][t] = 0;
        __syncthreads();
    }
}

// 8 values a thread
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadParams p, uint32_t dp)
{
    const uint32_t hk = blockIdx.y, plane = blockIdx.z, HD = p.head_dim, C = (HD + 7) / 8;
    const uint64_t total = (uint64_t)p.n * C;
    void* out = plane ? p.v_out : p.k_out;
    const void* src = plane ? p.v : p.k;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint32_t i = (uint32_t)(e / C), c = (uint32_t)(e % C);
        const uint32_t row = (uint32_t)(((uint64_t)p.first + i) % p.rows);
        float x[8];
        if (p.cache_dtype == DT_Q4)
            q4_values8((const uint8_t*)src + hk * q4::head_bytes(p.rows, dp), dp, row, c, plane != 0, x);
        else
#pragma unroll
            for (uint32_t d = 0; d < 8; ++d)
                x[d] = 8 * c + d < HD ? ld(src, p.cache_dtype, ((size_t)hk * p.rows + row) * HD + 8 * c + d) : 0.f;
        const size_t o = ((size_t)hk * p.n + i) * HD + 8 * c;
        if (8 * c + 8 <= HD && p.o_dtype == DT_F32) {
            typedef float4v float4u __attribute__((aligned(4)));
            *(float4u*)((float*)out + o) = float4v{x[0], x[1], x[2], x[3]};
            *(float4u*)((float*)out + o + 4) = float4v{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (uint32_t d = 0; d < 8; ++d)
                if (8 * c + d < HD) st(out, p.o_dtype, o + d, x[d]);
        }
    }
}

uint32_t q4_dp(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : head_dim <= 256 ? 256 : 0; }

size_t q4_plane_bytes(uint32_t hkv, uint32_t rows, uint32_t head_dim)
{
    return hkv * q4::head_bytes(rows, q4_dp(head_dim));
}

hipError_t cache_read_launch(const CacheReadParams& p, hipStream_t s)
{
    const size_t blocks = ((size_t)p.n * ((p.head_dim + 7) / 8) + 255) / 256;
    hipLaunchKernelGGL(cache_read_kernel, dim3((uint32_t)std::min<size_t>(blocks, 4096), p.hkv, 2), dim3(256), 0, s, p,
                       q4_dp(p.head_dim));
    return hipGetLastError();
}

static size_t copy_bytes(const AttnParams& p)
{
    const size_t value = p.kv_dtype == DT_F32 ? sizeof(float) : sizeof(half_t);
    return (2 * (size_t)p.hkv * p.kv_rows * p.head_dim * value + 255) & ~(size_t)255;
}

void attention_q4_plan(AttnParams& p, uint32_t cus)
{
    if (q4_few_rows(p)) {
        p.q4 = 2;
        q4_decode_plan(p, cus);
    } else {
        p.q4 = 1;
        attention_plan(p, cus);
        if (!p.dp) p.kv_dtype = DT_F32;   // the plain kernel takes values as they are
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
    const size_t n = (size_t)p.hkv * p.kv_rows * p.head_dim;
    p.v = p.kv_dtype == DT_F32 ? (void*)((float*)ws + n) : (void*)((half_t*)ws + n);
    attention_set_workspace(p, (char*)ws + copy_bytes(p));
}

hipError_t attention_q4_launch(const AttnParams& p, hipStream_t s)
{
    const uint32_t dp = q4_dp(p.head_dim);
    if (p.tkv > 0 && (p.q4 == 1 || q4_append_apart(p))) {
        const uint32_t blocks = (p.tkv + 2048 / dp - 1) / (2048 / dp);
        hipLaunchKernelGGL(q4_append_kernel, dim3(std::min(blocks, 4096u), p.hkv, 2), dim3(256), 0, s, p, dp);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.q4 == 2) return q4_decode_launch(p, p.ws4, s);
    const dim3 grid(std::min<uint32_t>((p.kv_rows + q4::KT - 1) / q4::KT, 1024), p.hkv);
    const auto copy = [&](auto value) {
        typedef decltype(value) T;
        T *k = (T*)p.k, *v = (T*)p.v;
        if (dp == 64) hipLaunchKernelGGL((q4_copy_kernel<64, T>), grid, dim3(256), 0, s, p, k, v);
        else if (dp == 128) hipLaunchKernelGGL((q4_copy_kernel<128, T>), grid, dim3(256), 0, s, p, k, v);
        else hipLaunchKernelGGL((q4_copy_kernel<256, T>), grid, dim3(256), 0, s, p, k, v);
    };
    if (p.kv_dtype == DT_F32) copy(float{});
    else copy(half_t{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return attention_launch(p, s);
}

}   // namespace vai_dev
