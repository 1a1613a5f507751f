// paged_plan.h -- how the attention kernels over pages deal their work out, and
// what they share at the end of a piece of it.
//
// A unit is RB query rows (token-major: row r is token r / g, head r % g of the KV
// head's g) of one sequence and KV head. Its keys are the 32-position tiles that
// some row of the sequence sees. All units' tiles form one line, sequence by
// sequence, which the workgroups cut into equal shares: however different the
// lengths, each walks as many tiles as the next, and the host, which does not know
// the lengths, need not. Beginning and ending a unit takes as long as `lead` tiles,
// which therefore stand before its own in the line (64 sequences of 64 to 8192
// positions, where a share without them could hold 25 short units: 123 us, with
// them 87). A unit that a cut runs through leaves partial results (its rows'
// maximum, sum and weighted values, fp32) in the workspace, at most two a
// workgroup, which paged_merge_kernel joins in a fixed order.
#pragma once
#include <algorithm>

#include "head_rows.h"
#include "pages.h"

namespace vai_dev {
namespace pg {

constexpr int KT = 32;                 // positions a tile

// The tiles [tb, te) that a sequence's rows see (at least one), and its blocks of rows.
struct Span {
    uint32_t tb, te, blocks;
};
// The positions [first_key, end_key) that row t of a sequence sees: held + t itself may
// lie past what the table holds, and past 32 bits, and its window with it (2^30 then:
// no position).
__device__ __forceinline__ uint32_t first_key(const PagedAttnParams& p, uint32_t held, uint32_t t)
{
    const uint64_t end = (uint64_t)held + t + 1;
    return p.span && end > p.span ? (uint32_t)std::min<uint64_t>(end - p.span, KvPages::MAX_POSITIONS) : 0u;
}
__device__ __forceinline__ uint32_t end_key(const PagedAttnParams& p, uint32_t held, uint32_t live, uint32_t t)
{
    return p.causal && held < live ? std::min(held + t + 1, live) : live;
}
__device__ __forceinline__ Span span_of(const PagedAttnParams& p, const Sequence& q, uint32_t rb)
{
    Span r;
    r.tb = first_key(p, q.held, 0) / KT;
    r.te = std::max(r.tb + 1, (q.live + KT - 1) / KT);
    r.blocks = (q.n * (p.hq / p.hkv) + rb - 1) / rb;
    return r;
}

// The first sequences of a batch, kept in LDS by plan_line: walk need not load them again.
constexpr uint32_t KEPT = 128;

// pre[s] = the line's tiles before sequence s, pre[sequences] all. LDS, as `kept`
// [KEPT]; every thread of the workgroup's NW waves calls.
template <int NW>
__device__ __forceinline__ void plan_line(const PagedAttnParams& p, uint32_t rb, uint32_t* pre, Sequence* kept)
{
    __shared__ uint32_t wave_sum_[NW];
    const uint32_t n = p.pages.sequences, per = (n + 64 * NW - 1) / (64 * NW), lane = threadIdx.x & 63;
    const uint32_t s0 = std::min(threadIdx.x * per, n), s1 = std::min(s0 + per, n);
    uint32_t sum = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        const Sequence q = sequence_of(p.pages, s, p.tokens);
        if (s < KEPT) kept[s] = q;
        uint32_t w = 0;
        if (q.n && q.n * (p.hq / p.hkv) <= p.few_rows) {
            const Span r = span_of(p, q, rb);
            w = (r.te - r.tb + p.lead) * r.blocks * p.hkv;
        }
        pre[s] = w;
        sum += w;
    }
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(scan, o);
        if (lane >= (uint32_t)o) scan += x;
    }
    if (lane == 63) wave_sum_[threadIdx.x >> 6] = scan;
    __syncthreads();
    uint32_t at = scan - sum;
    for (uint32_t w = 0; w < threadIdx.x >> 6; ++w) at += wave_sum_[w];
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t w = pre[s];
        pre[s] = at;
        at += w;
    }
    if (s1 == n && (s0 < n || threadIdx.x == 0)) pre[n] = at;   // (thread 0 where there is none: n >= 1)
    __syncthreads();
}

// The sequence that position f of the line is in.
__device__ __forceinline__ uint32_t line_sequence(const uint32_t* pre, uint32_t n, uint32_t f)
{
    uint32_t lo = 0, hi = n;           // pre[lo] <= f < pre[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (pre[mid] <= f) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A share's piece of a unit.
struct Piece {
    Sequence q;
    uint32_t s, hk, rb;        // sequence, KV head, block of rows
    uint32_t t0, t1;           // tiles
    bool whole;
    uint32_t slot;             // of the partial results: 2 w for a unit that an earlier
};                             // workgroup began, 2 w + 1 for one that a later one ends

// A unit to merge, left in ws_plan by the second of the workgroups that share it.
struct Joint {
    uint32_t parts;            // 0: none
    uint32_t wg;               // the first part's workgroup
    uint32_t first, hk, row0, rows;   // the sequence's first row; rows row0 .. + rows - 1 of the KV head
    uint32_t pad[2];
};

// Rows of a unit as partial results or output: acc / sum of 4 values from value d on.
__device__ __forceinline__ void put_row(const PagedAttnParams& p, uint32_t first, uint32_t hk, uint32_t row, uint32_t d,
                                        float4v acc, float sum)
{
    const uint32_t group = p.hq / p.hkv, token = first + row / group, h = hk * group + row % group;
    acc *= sum != 0.f ? 1.0f / sum : 0.f;     // (a NaN sum divides)
    const size_t at = ((size_t)token * p.hq + h) * p.head_dim + d;
    const uint32_t n = std::min(4u, p.head_dim - d);
    if (p.o_dtype == DT_F16) put4<false>((half_t*)p.out + at, n, acc);
    else put4<false>((float*)p.out + at, n, acc);
}

template <int DP> constexpr int orow() { return DP * 4 + 16; }   // bytes of an fp32 row in LDS
template <int DP, int NQ, int NW> constexpr int finish_bytes() { return NW * NQ * 16 * (orow<DP>() + 8); }

// The waves' sums meet in LDS (`lds`, finish_bytes(); what it held is done with
// once every wave is here) and leave as rows or partial results. Lane (c16, g) of
// a wave holds row c16 of each 16: m (log2 units), l, and in o[d][r] value 16 d + 4 g
// + r (ACROSS: (4 g + r) DP / 16 + d).
template <int DP, int NQ, int NW, bool ACROSS = false>
__device__ __forceinline__ void finish_piece(const PagedAttnParams& p, const Piece& u, char* lds, const float (&m)[NQ],
                                             const float (&l)[NQ], const float4v (&o)[NQ][DP / 16])
{
    constexpr int RB = NQ * 16, C4 = DP / 4;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
    float* ml = (float*)(lds + NW * RB * orow<DP>());
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint32_t r = wave * RB + q * 16 + c16;
        if (g == 0) {
            ml[2 * r] = m[q];
            ml[2 * r + 1] = l[q];
        }
        if constexpr (ACROSS) {
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
#pragma unroll
                for (int d = 0; d < DP / 16; d += 4)
                    *(float4v*)(lds + r * orow<DP>() + ((4 * g + rr) * (DP / 16) + d) * 4) =
                        float4v{o[q][d][rr], o[q][d + 1][rr], o[q][d + 2][rr], o[q][d + 3][rr]};
        } else {
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) *(float4v*)(lds + r * orow<DP>() + (16 * d + 4 * g) * 4) = o[q][d];
        }
    }
    __syncthreads();
    const uint32_t rows = std::min<uint32_t>(RB, u.q.n * (p.hq / p.hkv) - u.rb * RB);
    for (uint32_t e = threadIdx.x; e < rows * C4; e += 64 * NW) {
        const uint32_t r = e / C4, d = 4 * (e % C4);
        float mw[NW], M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            mw[w] = ml[2 * (w * RB + r)];
            M = fmaxf(M, mw[w]);
        }
        const float ref = M == -__builtin_inff() ? 0.f : M;
        float4v acc = (float4v)0.f;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float a = __builtin_amdgcn_exp2f(mw[w] - ref);
            acc += a * *(const float4v*)(lds + (w * RB + r) * orow<DP>() + d * 4);
            sum += a * ml[2 * (w * RB + r) + 1];
        }
        if (u.whole) {
            if (d < p.head_dim) put_row(p, u.q.first, u.hk, u.rb * RB + r, d, acc, sum);
        } else {
            const size_t at = (size_t)u.slot * RB + r;
            *(float4v*)(p.ws_o + at * DP + d) = acc;
            if (d == 0) {
                p.ws_ml[2 * at] = M;
                p.ws_ml[2 * at + 1] = sum;
            }
        }
    }
    __syncthreads();
}

// Calls f for each piece of this workgroup's share; pre: plan_line's.
template <int RB, class F>
__device__ __forceinline__ void walk(const PagedAttnParams& p, const uint32_t* pre, const Sequence* kept, F&& f)
{
    const uint32_t n = p.pages.sequences, total = __builtin_amdgcn_readfirstlane(pre[n]), wg = blockIdx.x;
    const uint32_t share = std::max(p.min_share, (total + p.wgs - 1) / p.wgs);
    const uint64_t begin = (uint64_t)wg * share;
    Joint joint{};
    const uint32_t end = (uint32_t)std::min<uint64_t>(begin + share, total);
    for (uint32_t at = (uint32_t)std::min<uint64_t>(begin, total); at < end;) {
        Piece u;
        u.s = __builtin_amdgcn_readfirstlane(line_sequence(pre, n, at));
        u.q = uniform(u.s < KEPT ? kept[u.s] : sequence_of(p.pages, u.s, p.tokens));
        const Span r = span_of(p, u.q, RB);
        const uint32_t tiles = r.te - r.tb, len = tiles + p.lead;
        const uint32_t off = at - __builtin_amdgcn_readfirstlane(pre[u.s]), unit = off / len, o0 = off - unit * len;
        const uint32_t o1 = std::min(len, o0 + (end - at));
        if (unit >= r.blocks * p.hkv) break;   // (starts that do not increase)
        u.hk = unit / r.blocks;
        u.rb = unit - u.hk * r.blocks;
        const uint32_t t0 = o0 > p.lead ? o0 - p.lead : 0u, t1 = o1 > p.lead ? o1 - p.lead : 0u;
        if (at == begin && t0 > 0) {
            const uint32_t a = at - o0 + p.lead, wg0 = a / share;    // (the unit's first tile)
            if (wg0 + 1 == wg)
                joint = Joint{std::min((a + tiles - 1) / share + 1, p.wgs) - wg0, wg0, u.q.first, u.hk, u.rb * RB,
                              std::min<uint32_t>(RB, u.q.n * (p.hq / p.hkv) - u.rb * RB), {0, 0}};
        }
        at += o1 - o0;
        if (t1 == t0) continue;
        u.t0 = r.tb + t0;
        u.t1 = r.tb + t1;
        u.whole = t1 - t0 == tiles;
        u.slot = 2 * wg + (t0 == 0 ? 1u : 0u);
        f(u);
    }
    if (threadIdx.x == 0) ((Joint*)p.ws_plan)[wg] = joint;
}

}   // namespace pg

hipError_t paged_merge_launch(const PagedAttnParams& p, hipStream_t s);

}   // namespace vai_dev
