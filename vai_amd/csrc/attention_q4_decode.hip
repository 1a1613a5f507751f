// attention_q4_decode.hip -- up to 128 or 256 query rows of a KV head over a 4-bit
// cache: append and attention in one launch (and a merge where the keys are split;
// an append before it where the call brings many rows).
//
// What bounds it: reading the cache once, 5 bits a value. The query rows of a KV
// head are the columns of one matrix tile (16 or 32), as in attention_decode.hip;
// a workgroup is a share of the head's 32-position tiles, which its 4 waves take
// in turn, each through a ring of its own in LDS: a tile's 20 dp bytes of K and of
// V are copied there as they lie, D tiles in flight, and no wave waits for another
// until the share ends. 120001 positions, 32 heads over 8 of 128: 37.5 us, 4.1 TB/s,
// where a large copy makes 5.2 (fp32 queries: 1.5 us more a pass); waves wait for memory a quarter of their time, and
// for an issue slot, the unpacking of each other's codes, a third.
//
// The codes enter the matrix cores as they are. An fp16 whose bits are a code n of
// 0 .. 15 is n * 2^-24, and the cores multiply such numbers exactly, so one step
// of 32 head-dim values (a group) gives 2^-24 sum n q from masked nibbles alone,
// and a score is
//   scale * (sum over groups of s * sum n q + sum over groups of m * sum q):
// the first sum in fp32, the second a product of its own of the minima with the
// groups' sums of q (as two fp16 numbers each): K is never rounded. Nibbles that
// stand 4 bits up are 16 n; their q is taken as q / 16. For that every row of q is
// scaled by a power of two, so that its largest value lies in [512, 1024) and none
// that counts is lost (fp16 holds what is 2^-25 of it). An fp32 q enters as two
// fp16 numbers. V enters as s n + m rounded to fp16 (one packed fma from the exact
// n; as two numbers it would double both the unpacking, which the waves wait for,
// and the products), the probabilities as two fp16 numbers (the second the rest
// that the first leaves) and times 2^14, so that those far below the row's largest
// keep their bits too (fp16 holds 2^-38 of it; unscaled, a key of 2^-25 was lost,
// and with thousands of them what they bring): V's and the result's are then the
// only roundings to fp16: error against 64 bits 2.9e-4 of the result, of which the
// rounding of the result is 2.1e-4 (3.6e-4 with the probabilities in one number).
//
// A few rows that the call brings are rounded by the wave whose tile they are in,
// into that tile in LDS (and into the cache): nothing waits for an append.
#include <algorithm>
#include <type_traits>

#include "decode_range.h"
#include "kernels.h"
#include "launch_once.h"
#include "q4_cache.h"

#define LDS_AS __attribute__((address_space(3)))

namespace vai_dev {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));

namespace {

template <int DP> struct Q4Lds {
    static constexpr int TILE = (int)q4::tile_bytes(DP);      // one plane's tile
    static constexpr int COPIES = (TILE + 1023) / 1024;       // 1 KB copies, the last one partly
    // tiles in flight a wave: what a CU's waves have in flight together hides the
    // latency. A pass over 120000 positions, us, two / three / four tiles: 128, 32 heads
    // over 8, one token 38.3 / 44.1 / 45.2 (three workgroups a CU with two tiles, two
    // with four), fp32 queries 40.3 / 41.2 / 42.2, 8 tokens in blocks of 32 rows 74.3 /
    // 75.1 / 76.2; 64, three / four tiles 29.3 / 30.0; 256, two / three 36.7 / 37.9
    static constexpr int D = DP == 256 ? 3 : DP == 128 ? 2 : 4;
    static constexpr int WAVE = D * 2 * TILE;
    static constexpr int OROW = DP * 4 + 16;                  // bytes of an fp32 O row in the final exchange
    template <int NQ> static constexpr int bytes()
    {
        const int o = fd::NW * NQ * 16 * OROW + fd::NW * NQ * 16 * 8;   // (m, l) per wave and row after it
        return fd::NW * WAVE > o ? fd::NW * WAVE : o;
    }
};

template <int N>
__device__ __forceinline__ void q4_wait()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
// all but the copies of the tiles behind this one (`behind` of them, N counted) have landed
template <int N, int COPIES>
__device__ __forceinline__ void q4_wait_behind(int behind)
{
    if constexpr (N == 0) q4_wait<0>();
    else if (behind >= N) q4_wait<N * COPIES>();
    else q4_wait_behind<N - 1, COPIES>(behind);
}
__device__ __forceinline__ void q4_wait_lds() { __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14)); }

__device__ __forceinline__ float swap_max16(float x)
{
    float y = x;
    lane_swap<16>(x, y);
    return fmaxf(x, y);
}

}   // namespace

// workgroups a CU, as registers allow
constexpr int q4_resident(uint32_t dp, uint32_t nq, bool q32)
{
    return dp == 256 ? 1 : dp == 128 && nq == 1 && !q32 ? 3 : 2;
}

// DP: the padded head dim; NQ: 16-row query blocks. Grid: (units, row blocks x
// hkv). p.k / p.v are the 4-bit planes.
template <int DP, int NQ, bool Q32>
__global__ __launch_bounds__(256, q4_resident(DP, NQ, Q32)) void attention_q4_decode_kernel(AttnDecodeParams p)
{
    using namespace fd;
    using L = Q4Lds<DP>;
    constexpr int G = DP / 32, ND = DP / 16, D = L::D;   // groups; values of a lane's V slice
    constexpr uint32_t NIB = 0x000f000fu, NIB16 = 0x00f000f0u;
    constexpr float LIFT = 14.f, SLACK = 1.f;
    extern __shared__ uint4v q4_lds[];
    LDS_AS uint8_t* lds = (LDS_AS uint8_t*)(LDS_AS void*)q4_lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const uint32_t HD = p.head_dim, unit = blockIdx.x, hk = blockIdx.y % p.hkv, rb = blockIdx.y / p.hkv;

    // query rows: row r of the KV head is query head hk g + r / tq, token r % tq
    // (loaded before the first copies: both are waited for in order)
    const uint32_t rows = p.rows, row0 = rb * p.rpb, rend = std::min(row0 + p.rpb, rows);
    typedef typename std::conditional<Q32, float8v, half8>::type q8;
    q8 qraw[NQ][G];
    uint32_t tok[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint32_t r = std::min(row0 + q * 16 + c16, rend - 1);
        tok[q] = r % p.tq;
        const size_t base = ((size_t)hk * rows + r) * HD;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t d = 32 * i + 8 * g;   // (HD is a multiple of 8)
            typedef q8 q8u __attribute__((aligned(sizeof(qraw[0][0][0]))));
            qraw[q][i] = 0;
            if (d < HD) qraw[q][i] = *(const q8u*)((const typename std::conditional<Q32, float, half_t>::type*)p.q + base + d);
        }
    }
    const Range R = range_of(p);
    if (unit >= R.used) return;

    const size_t hb = q4::head_bytes(p.kv_rows, DP);
    uint8_t* kh = uniform_ptr((uint8_t*)p.k + hk * hb);
    uint8_t* vh = uniform_ptr((uint8_t*)p.v + hk * hb);
    LDS_AS uint8_t* ring = lds + wave * L::WAVE;
    // the tokens of the block's rows (all of them where it is the only one or goes over a head's end)
    uint32_t tok0 = 0, tok1 = p.tq - 1;
    if (rows > p.rpb && (rend - 1) / p.tq == row0 / p.tq) {
        tok0 = row0 % p.tq;
        tok1 = (rend - 1) % p.tq;
    }
    // this wave's tiles: first, first + step, .., and their places in the planes
    // (a ring's size is a multiple of 64: no tile wraps)
    const uint32_t step = p.units * NW, wrap = p.ring ? p.kv_rows / KT : 0xffffffffu;
    int64_t first = R.tb + unit * NW + wave, last = R.te;
    if (p.n_new == 0 && rows > p.rpb) {   // only tiles that some row of the block sees (both bounds grow with the token)
        const int64_t beg = p.mask.key_start_cached(tok0, R.cached) / KT;
        last = std::min<int64_t>(last, (p.mask.key_end_cached(tok1, R.cached) + KT - 1) / KT);
        if (beg > first) first += ((uint32_t)(beg - first) + step - 1) / step * step;
    }
    const int mine = __builtin_amdgcn_readfirstlane((int)(last > first ? ((uint32_t)(last - first) + step - 1) / step : 0));
    const uint32_t place0 = __builtin_amdgcn_readfirstlane((uint32_t)(p.ring ? first % wrap : first));
    const uint32_t hop = __builtin_amdgcn_readfirstlane(p.ring ? step % wrap : step);
    const auto next_place = [&](uint32_t t) __attribute__((always_inline)) {
        t += hop;
        return t >= wrap ? t - wrap : t;
    };
    uint32_t ahead = place0;   // the next copy's place, and how many were made
    int copied = 0;
    const auto copy = [&](int slot) __attribute__((always_inline)) {
        LDS_AS uint8_t* dst = ring + slot * 2 * L::TILE;
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                (void*)((plane ? vh : kh) + (size_t)ahead * L::TILE), (short)0, L::TILE, 0x00020000);
#pragma unroll
            for (int c = 0; c < L::COPIES; ++c)
                if ((c + 1) * 1024 <= L::TILE || c * 1024 + lane * 16 < L::TILE)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_AS void*)(dst + plane * L::TILE + c * 1024), 16,
                                                             c * 1024 + lane * 16, 0, 0, 0);
        }
        ++copied;
        ahead = next_place(ahead);
    };
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < mine) copy(i);

    // the rows as the cores take them: qf (and ql, what fp16 leaves of an fp32 q),
    // and the groups' sums in two numbers (quarter 0 the first, quarter 1 the second)
    half8 qf[NQ][G], ql[Q32 ? NQ : 1][Q32 ? G : 1], qsum[NQ];
    float down[NQ];   // undoes the row's power of two
    int64_t kbeg[NQ], kend[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        kend[q] = std::min<int64_t>(p.mask.key_end_cached(tok[q], R.cached), R.live);
        kbeg[q] = p.mask.key_start_cached(tok[q], R.cached);
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf((float)qraw[q][i][e]));
        top = swap_max32(swap_max16(top));
        const int ex = top > 0.f && top < __builtin_inff() ? 10 - __builtin_amdgcn_frexp_expf(top) : 0;
        down[q] = ldexpf(1.f, -ex);
        qsum[q] = (half8)(half_t)0;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float8v x = __builtin_convertvector(qraw[q][i], float8v);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = ldexpf(x[e], ex);
                sum += x[e];
            }
            const float8v part = {1.f, 1.f, .0625f, .0625f, 1.f, 1.f, .0625f, .0625f};
            qf[q][i] = __builtin_convertvector(x * part, half8);
            if constexpr (Q32) {
                const float8v rest = x * part - __builtin_convertvector(qf[q][i], float8v);
                ql[q][i] = __builtin_convertvector(rest, half8);
            }
            sum = swap_sum<16>(sum, sum);
            sum = swap_sum<32>(sum, sum);
            const half_t hi = (half_t)sum;
            qsum[q][i] = g == 0 ? hi : g == 1 ? (half_t)(sum - (float)hi) : (half_t)0.f;
        }
    }
    const int64_t kfirst = p.mask.key_start_cached(0, R.cached);   // no query sees a position before it
    // what every row of this wave sees: tiles inside need no mask
    const int64_t all_beg = p.mask.key_start_cached(tok1, R.cached);
    const int64_t all_end = std::min<int64_t>(p.mask.key_end_cached(tok0, R.cached), R.live);
    const float sl2 = p.scale * 1.4426950408889634f;   // scores in log2 units

    float m[NQ], l[NQ];
    float4v o[NQ][ND];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q] = -__builtin_inff();
        l[q] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[q][d] = (float4v)0.f;
    }

    uint32_t place = place0;
    int slot = 0;
    for (int it = 0; it < mine; ++it) {
        // its copies have landed; the next tiles' may be in flight
        q4_wait_behind<D - 1, 2 * L::COPIES>(mine - 1 - it);
        const int64_t j0 = (first + (int64_t)it * step) * KT;
        LDS_AS uint8_t* kt = ring + slot * 2 * L::TILE;
        LDS_AS uint8_t* vt = kt + L::TILE;

        // the call's own rows in this tile, 256 / DP at a time: DP / 8 lanes to a row of
        // K, as many to V's, 8 values each
        if (p.n_new != 0 && j0 + KT > R.cached) {
            constexpr uint32_t LR = DP / 8, RP = 32 / LR;
            const uint32_t ja = R.cached > j0 ? (uint32_t)(R.cached - j0) : 0u;
            const uint32_t je = (uint32_t)std::min<int64_t>(KT, R.live - j0);
            const uint32_t c = lane % LR, jr = lane / LR % RP, values = 8 * c < HD ? HD - 8 * c : 0u;
            const bool is_v = lane >= 32;
            const void* rows_new = is_v ? p.v_new : p.k_new;
            const size_t at = (size_t)place * L::TILE;
            for (uint32_t ju = ja; ju < je; ju += RP) {
                const uint32_t j = ju + jr, jc = std::min(j, je - 1);
                const size_t row = ((size_t)hk * p.n_new + (uint32_t)(j0 + jc - R.cached)) * HD;
                half_t s, m;
                const uint32_t codes = q4::encode8(q4::row8(rows_new, p.new_dtype, row, 8 * c, HD), values, s, m);
                if (j < je) {
                    if (is_v) q4::put_v(vt, DP, j, c, codes, s, m);
                    else q4::put_k(kt, DP, j, c, codes, s, m);
                    if (rb == 0) {
                        if (is_v) q4::put_v(vh + at, DP, j, c, codes, s, m);
                        else q4::put_k(kh + at, DP, j, c, codes, s, m);
                    }
                }
            }
            q4_wait_lds();
        }
        place = next_place(place);

        // what the score product reads of the tile: codes, steps and minima
        uint32_t kw[2][G];
        half8 ma[2];
        half4 ks[2][G];        // rows 4 g ..+3
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            LDS_AS const uint8_t* a = kt + ((t * 4 + g) * 16 + c16) * (G * 4);
            if constexpr (G == 2) {
                const uint2v w = *(LDS_AS const uint2v*)a;
                kw[t][0] = w.x;
                kw[t][1] = w.y;
            } else {
#pragma unroll
                for (int i = 0; i < G; i += 4) {
                    const uint4v w = *(LDS_AS const uint4v*)(a + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kw[t][i + e] = w[e];
                }
            }
            typedef half_t halfg __attribute__((ext_vector_type(G)));
            const halfg mg = *(LDS_AS const halfg*)(kt + q4::k_min_offset(DP) + (t * 16 + c16) * (G * 2));
            ma[t] = (half8)(half_t)0;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                ma[t][i] = mg[i];
                ks[t][i] = *(LDS_AS const half4*)(kt + q4::scale_offset(DP) + ((i * 2 + t) * 16 + 4 * g) * 2);
            }
        }
        uint32_t vw[ND];       // V's words 2 i, 2 i + 1: the two halves of the block's positions, values 2 i and 2 i + 1
        half8 vs, vm;
        uint32_t bad = 0;      // of the lane's 8 positions, those whose V holds a NaN
        bool any_bad = false;  // (of the wave's)
        half8 ph[NQ], pl[NQ];   // P^T: positions 0 2 1 3 4 6 5 7 of the lane's 8, and what fp16 leaves of them
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            // S^T: lane (c16, g) holds query row c16 and positions 8 g + 4 t ..+3
            float4v x[2], y[2];   // 2^-24 sum s sum n q, sum m sum q
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                x[t] = (float4v)0.f;
                y[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ma[t], qsum[q], (float4v)0.f, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const uint32_t w = kw[t][i], u = w >> 8;
                    const half8 n8 = __builtin_bit_cast(half8, uint4v{w & NIB, w & NIB16, u & NIB, u & NIB16});
                    float4v n = __builtin_amdgcn_mfma_f32_16x16x32_f16(n8, qf[q][i], (float4v)0.f, 0, 0, 0);
                    if constexpr (Q32) n = __builtin_amdgcn_mfma_f32_16x16x32_f16(n8, ql[q][i], n, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[t][r] = fmaf((float)ks[t][i][r], n[r], x[t][r]);
                }
            }
            if (q == 0) {   // V's share of the tile, under the first rows' products
                LDS_AS const uint8_t* a = vt + g * (DP * 4) + c16 * (DP / 4);
#pragma unroll
                for (int i = 0; i < ND; i += 4) {
                    const uint4v w = *(LDS_AS const uint4v*)(a + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) vw[i + e] = w[e];
                }
                LDS_AS const uint8_t* va = vt + q4::scale_offset(DP) + ((c16 * ND / 32) * 4 + g) * 32;
                vs = *(LDS_AS const half8*)va;
                vm = *(LDS_AS const half8*)(va + 16);
                q4_wait_lds();         // read before the slot is copied over
                if (copied < mine) copy(slot);
                slot = slot + 1 == D ? 0 : slot + 1;

                // Positions that no query sees (stale rows, rows past the count) may hold
                // anything: their V is zero here, their scores are masked below.
                if (j0 < kfirst || j0 + KT > R.live) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int64_t j = j0 + 8 * g + q4::order_of(e);
                        if (j < kfirst || j >= R.live) vs[e] = vm[e] = (half_t)0.f;
                    }
                }
                // A row with a NaN in V must not reach a query it is hidden from through 0 *
                // NaN: its V is zero and its score NaN, which the mask replaces. (The sum of
                // the minima is NaN if one is, and at worst also where they overflow.)
                const half2v z = half2v{vm[0], vm[1]} + half2v{vm[2], vm[3]} + half2v{vm[4], vm[5]} + half2v{vm[6], vm[7]};
                if (__builtin_expect(__any(z.x != z.x || z.y != z.y), 0)) {
                    any_bad = true;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (vm[e] != vm[e]) {
                            vs[e] = vm[e] = (half_t)0.f;
                            bad |= 1u << q4::order_of(e);
                        }
                    bad |= q4::moved<q4::XOR1>(bad);
                    bad |= q4::moved<q4::XOR2>(bad);
                    bad |= q4::moved<q4::MIRROR8>(bad);
                    bad |= q4::moved<q4::MIRROR16>(bad);
                }
            }
            if (__builtin_expect(any_bad, 0))
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (bad >> (4 * t + r) & 1) x[t][r] = __builtin_nanf("");
            float v[8];
            const float sc = sl2 * down[q];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(x[i >> 2][i & 3], 16777216.f, y[i >> 2][i & 3]) * sc;
            if (j0 < all_beg || j0 + KT > all_end) {
                const int lo = (int)std::min<int64_t>(std::max<int64_t>(kbeg[q] - j0, -1), KT + 1);
                const int hi = (int)std::min<int64_t>(std::max<int64_t>(kend[q] - j0, -1), KT + 1);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (8 * g + i >= hi || 8 * g + i < lo) v[i] = -__builtin_inff();
            }
            float tmax = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
            tmax = swap_max32(swap_max16(tmax));
            // the row's reference m moves only when the max exceeds it by more than
            // SLACK (P stays below 2^(SLACK + LIFT), in fp16's range), for the whole
            // wave at once
            if (__any(tmax > m[q] + SLACK)) {
                const float mnew = fmaxf(m[q], tmax);
                const float alpha = __builtin_amdgcn_exp2f(m[q] - (mnew == -__builtin_inff() ? 0.f : mnew));
                l[q] *= alpha;
                m[q] = mnew;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[q][d] *= alpha;
            }
            const float mref = (m[q] == -__builtin_inff() ? 0.f : m[q]) - LIFT;   // (l and o carry 2^LIFT alike)
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(v[i] - mref);
            l[q] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));   // (this lane's positions)
            const float8v f = {e[0], e[2], e[1], e[3], e[4], e[6], e[5], e[7]};
            ph[q] = __builtin_convertvector(f, half8);
            pl[q] = __builtin_convertvector(f - __builtin_convertvector(ph[q], float8v), half8);
        }

        // O^T += V^T P^T: value c16 ND + 2 i + h in row c16 of the product's A
#pragma unroll
        for (int i = 0; i < ND / 2; ++i) {
            const uint32_t w0 = vw[2 * i], w1 = vw[2 * i + 1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // 1024 + n or (high nibbles where they stand) 1024 + 16 n as bits, then n: exact
                const uint32_t mask = h ? NIB16 : NIB;
                const uint4v b = uint4v{w0 & mask, (w0 >> 8) & mask, w1 & mask, (w1 >> 8) & mask} | (uint4v)0x64006400u;
                const half8 k = __builtin_bit_cast(half8, b);
                const half8 n = h ? __builtin_elementwise_fma(k, (half8)(half_t)0.0625f, (half8)(half_t)-64.f)
                                  : k - (half8)(half_t)1024.f;
                const half8 a = __builtin_elementwise_fma(n, vs, vm);
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    o[q][2 * i + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[q], o[q][2 * i + h], 0, 0, 0);
                    o[q][2 * i + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[q], o[q][2 * i + h], 0, 0, 0);
                }
            }
        }
    }

    // the waves' sums meet in LDS (the rings are done with); o[q][d] register r is
    // row c16, value (4 g + r) ND + d
    __syncthreads();
    LDS_AS uint8_t* ml = lds + NW * NQ * 16 * L::OROW;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int r = q * 16 + c16;
        float s = l[q];
        s = swap_sum<16>(s, s);
        s = swap_sum<32>(s, s);
        if (g == 0) *(LDS_AS float2v*)(ml + (wave * NQ * 16 + r) * 8) = float2v{m[q], s};
        LDS_AS uint8_t* orow = lds + (wave * NQ * 16 + r) * L::OROW;
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
            for (int d = 0; d < ND; d += 4)
                *(LDS_AS float4v*)(orow + ((4 * g + rr) * ND + d) * 4) =
                    float4v{o[q][d][rr], o[q][d + 1][rr], o[q][d + 2][rr], o[q][d + 3][rr]};
    }
    __syncthreads();
    const bool whole = R.used == 1;
    constexpr int C4 = DP / 4;
    for (uint32_t e = threadIdx.x; e < (rend - row0) * C4; e += 256) {
        const uint32_t r = e / C4, c = e % C4;
        float mw[NW], lw[NW], M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2v y = *(LDS_AS const float2v*)(ml + (w * NQ * 16 + r) * 8);
            mw[w] = y.x;
            lw[w] = y.y;
            M = fmaxf(M, y.x);
        }
        const float mref = M == -__builtin_inff() ? 0.f : M;
        float4v acc = (float4v)0.f;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float a = __builtin_amdgcn_exp2f(mw[w] - mref);
            acc += a * *(LDS_AS const float4v*)(lds + (w * NQ * 16 + r) * L::OROW + c * 16);
            sum += a * lw[w];
        }
        const uint32_t row = row0 + r;
        if (whole) {
            // (no key: zeros; a NaN stays one)
            acc *= sum == 0.f ? 0.f : 1.0f / sum;
            const uint32_t h = hk * (p.hq / p.hkv) + row / p.tq, t = row % p.tq;
            const size_t out = ((size_t)t * p.hq + h) * HD + 4 * c;
            if (4 * c < HD) {
                typedef half4 half4u __attribute__((aligned(2)));
                typedef float4v float4u __attribute__((aligned(4)));
                if (p.o_dtype == DT_F16) *(half4u*)((half_t*)p.out + out) = __builtin_convertvector(acc, half4);
                else *(float4u*)((float*)p.out + out) = acc;
            }
        } else {
            const size_t part = ((size_t)hk * p.units + unit) * rows + row;
            *(float4v*)(p.ws_o + part * DP + 4 * c) = acc;
            if (c == 0) {
                p.ws_ml[2 * part] = M;
                p.ws_ml[2 * part + 1] = sum;
            }
        }
    }
}

template <int DP, int NQ, bool Q32>
static hipError_t q4_decode_launch_t(const AttnDecodeParams& p, hipStream_t s)
{
    constexpr int bytes = Q4Lds<DP>::template bytes<NQ>();
    static PerDevice lds_once;
    if constexpr (bytes > 64 * 1024) {
        const hipError_t e = set_max_lds(lds_once, (const void*)attention_q4_decode_kernel<DP, NQ, Q32>, bytes);
        if (e != hipSuccess) return e;
    }
    const dim3 grid(p.units, (p.rows + p.rpb - 1) / p.rpb * p.hkv);
    hipLaunchKernelGGL((attention_q4_decode_kernel<DP, NQ, Q32>), grid, dim3(256), bytes, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.units == 1) return e;
    return attention_decode_merge_launch(p, DP, 1, s);
}

// Up to 128 query rows of a KV head, 256 over a cache of 4096 positions and more:
// past them the copies for the flash kernel cost less than unpacking the codes for
// 16 or 32 rows at a time. One pass, us, this way / over the copies, at 1000, 8000
// and 120000 positions (8 KV heads, fp16 queries):
//   D = 128, 68 rows   16.8 / 20.3   27.3 / 46.5   133 / 426
//           128        18.9 / 21.9   31.4 / 46.5   170 / 426
//           192        23.0 / 22.4   37.4 / 46.0   260 / 427
//           256        24.2 / 22.0   41.0 / 45.8   321 / 427
//           384        27.4 / 26.3   55.4 / 46.1   498 / 429
//   D = 64, 128        16.1 / 17.4   23.2 / 37.8   122 / 255
//           256        19.5 / 17.5   30.8 / 38.0   228 / 255
//   D = 256, 128       21.6 / 33.8   48.1 / 75.7   471 / 989
//           256        27.6 / 34.6   78.9 / 75.4   920 / 989
// fp32 queries: D = 128, 256 rows 20.9 / 22.9, 43.7 / 47.0, 428 / 428. One or two
// KV heads: faster this way at 256 rows throughout (2 of 128, 120000: 95.3 / 116).
bool q4_few_rows(const AttnParams& p)
{
    return p.head_dim % 8 == 0 && (uint64_t)(p.hq / p.hkv) * p.tq <= (p.kv_rows < 4096 ? 128 : 256) &&
           (uint64_t)p.hq * p.tq <= 65535;
}

// The call's rows are rounded where their tiles are attended, 256 / DP of them
// at a time and by every row block, or before, by a launch of their own: its 2 us
// against 0.4-1.4 a step. 3000 positions, us, in the walk / apart: D = 64, 8 rows
// 13.4 / 14.0, 16 15.4 / 16.7 (in four row blocks 16.1 / 13.4), 32 22.4 / 19.5; D =
// 128, 4 12.7 / 13.4, 5 17.0 / 15.9, 8 18.9 / 16.7; D = 256, 2 15.7 / 16.2, 4 19.3 /
// 16.9. (And apart where a window leaves rows of the call out of every query's sight.)
bool q4_append_apart(const AttnParams& p)
{
    return p.tkv > 512 / q4_dp(p.head_dim) || (p.span != 0 && p.tkv >= p.tq + p.span);
}

void q4_decode_plan(AttnParams& p, uint32_t cus)
{
    const uint32_t dp = q4_dp(p.head_dim);
    const bool q32 = p.q_dtype == DT_F32;
    p.dp = dp;
    p.dec_rows = p.hq / p.hkv * p.tq;
    // 32 rows a workgroup where the registers hold them for two workgroups a CU (fp32
    // queries at D = 128, 32 and 16 rows: 128 rows over 120000 positions 252, 223 us)
    p.dec_rpb = std::min<uint32_t>(p.dec_rows, dp == 256 || (dp == 128 && q32) ? 16 : 32);
    const uint32_t keys = p.span ? std::min<uint64_t>(p.kv_rows, (uint64_t)p.span + p.tq + 2 * fd::KT) : p.kv_rows;
    const uint32_t tiles = (keys + fd::KT - 1) / fd::KT, most = std::max<uint32_t>((tiles + fd::NW - 1) / fd::NW, 1);
    const uint32_t blocks = p.hkv * ((p.dec_rows + p.dec_rpb - 1) / p.dec_rpb);
    // shares in one round of the chip: one more and its last workgroups run alone, 68
    // rows over 120000 positions 141 us instead of 132
    const uint32_t chip = cus * q4_resident(dp, p.dec_rpb > 16 ? 2 : 1, q32);
    uint32_t units = std::max(chip / blocks, 1u);
    // 17 to 32 rows: a second workgroup a CU only where each wave still has four tiles
    // (32 rows of D = 128, one / two: 8000 positions 18.3 / 20.3 us, 16000 22.7 / 24.4,
    // 30000 31.0 / 30.5, 120000 74 / 58)
    if (p.dec_rpb > 16) units = std::min(units, std::max(std::max(cus / blocks, 1u), tiles / (4 * fd::NW)));
    p.dec_units = std::min(std::min(units, most), AttnDecodeParams::MAX_UNITS);
}

size_t q4_decode_workspace(const AttnParams& p) { return attention_decode_workspace(p, p.dec_units); }

hipError_t q4_decode_launch(const AttnParams& a, void* ws, hipStream_t s)
{
    AttnDecodeParams p{};
    p.out = a.out; p.q = a.q; p.k = a.k4; p.v = a.v4;
    p.o_dtype = a.o_dtype; p.q_dtype = a.q_dtype;
    p.hq = a.hq; p.hkv = a.hkv; p.tq = a.tq; p.tkv = a.tkv; p.head_dim = a.head_dim;
    p.cache_count = a.cache_count; p.kv_rows = a.kv_rows; p.ring = a.ring;
    p.k_new = a.k_new; p.v_new = a.v_new; p.n_new = q4_append_apart(a) ? 0u : a.tkv; p.new_dtype = a.new_dtype;
    p.scale = a.scale;
    p.mask = a.mask;
    p.rows = a.dec_rows; p.rpb = a.dec_rpb; p.units = a.dec_units;
    p.ws_o = (float*)ws;
    p.ws_ml = (float*)ws + (size_t)a.hkv * a.dec_units * a.dec_rows * a.dp;
    const bool one = p.rpb <= 16;
    if (a.q_dtype == DT_F32) {
        switch (a.dp) {
        case 64: return one ? q4_decode_launch_t<64, 1, true>(p, s) : q4_decode_launch_t<64, 2, true>(p, s);
        case 128: return q4_decode_launch_t<128, 1, true>(p, s);
        default: return q4_decode_launch_t<256, 1, true>(p, s);
        }
    }
    switch (a.dp) {
    case 64: return one ? q4_decode_launch_t<64, 1, false>(p, s) : q4_decode_launch_t<64, 2, false>(p, s);
    case 128: return one ? q4_decode_launch_t<128, 1, false>(p, s) : q4_decode_launch_t<128, 2, false>(p, s);
    default: return q4_decode_launch_t<256, 1, false>(p, s);
    }
}

}   // namespace vai_dev
