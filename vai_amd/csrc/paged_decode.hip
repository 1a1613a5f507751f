// paged_decode.hip -- attention of a ragged batch over fp16 pages whose sizes are
// whole 16s, head dims whole 8s.
//
// What bounds it: reading each sequence's K and V once. A workgroup's share of the
// line (paged_plan.h) is walked by its waves a 32-position tile in turn, each
// through a ring of D tiles in LDS of its own: the copies (K and V as they lie, 16
// positions of one page at a time, 16-byte chunks XOR-swizzled by row) of the next
// tiles are in flight during a tile, and no wave waits for another until the piece
// of the share ends. Where their pages lie is looked up for a wave's next 32 tiles
// at once, a lane for each 16 positions; the wave waits for that, and for the copies
// before it, once in 32 tiles.
//
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, the query rows of a KV
// head the columns: lane (c16, g) gets row c16's scores of keys 16 k + 4 g ..+3,
// which are P^T's operand as they stand when V^T is read (transposed, from LDS) in
// that order of keys. K and V are exact; an fp32 q enters as two fp16 numbers,
// after a power of two that puts the row's largest value into [512, 1024), and the
// probabilities as two, times 2^14 so that those far below the row's largest keep
// their bits.
#include <algorithm>
#include <type_traits>

#include "paged_plan.h"

#include "launch_once.h"

#define LDS_AS __attribute__((address_space(3)))

namespace vai_dev {

namespace {

template <int DP> struct Ring {
    static constexpr int ROWB = DP * 2;                      // bytes of a K or V row in LDS
    static constexpr int BLOCK = 16 * ROWB;                  // 16 positions of K or V
    static constexpr int TILE = 4 * BLOCK;                   // K's two blocks, V's two
    static constexpr int COPIES = BLOCK / 1024;              // 1 KB copies a block
    static constexpr int NW = DP == 64 ? 4 : 2;              // waves
    static constexpr int D = 2;                              // tiles
    static constexpr int RES = DP == 256 ? 1 : 2;            // workgroups a CU, as LDS allows
    static constexpr int BYTES = NW * D * TILE;
};

// Physical 16-byte chunk of logical chunk c in row r: what one pass of 16 lanes
// reads, K's 16 rows at a chunk or V's 4 rows at two, lies in different banks (for
// 64-wide rows K's in half of them).
__host__ __device__ constexpr int swz_f(int r) { return 2 * (r & 3) + ((r >> 2) & 1); }
template <int DP> __host__ __device__ constexpr int swz_row(int r) { return DP == 64 ? swz_f(r & 7) : swz_f(r & 7) | (r & 8); }

// LDS reads in asm, waited for in the same block: the compiler's own would wait for
// every copy in flight.
template <int O0, int O1, int O2, int O3>
__device__ __forceinline__ void read4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, half8 (&x)[4])
{
    asm volatile("ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%9\n\t"
                 "ds_read_b128 %2, %6 offset:%10\n\tds_read_b128 %3, %7 offset:%11\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(O0), "n"(O1), "n"(O2), "n"(O3)
                 : "memory");
}
// V^T of 4 output blocks, 4 keys of each half a lane (ds_read_b64_tr_b16: per 16-lane
// group, result lane j element k is element j % 4 of what source lane 4 k + j / 4
// points at)
template <int OFF, int HALF>
__device__ __forceinline__ void read_tr4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, half4 (&x)[8])
{
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF), "n"(OFF + HALF)
                 : "memory");
}
// all but the last N vector memory operations have ended
template <int N>
__device__ __forceinline__ void wait_vm()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int N, int COPIES>
__device__ __forceinline__ void wait_behind(int behind)
{
    if constexpr (N == 0) wait_vm<0>();
    else if (behind >= N) wait_vm<N * COPIES>();
    else wait_behind<N - 1, COPIES>(behind);
}

__device__ __forceinline__ float swap_max16(float x)
{
    float y = x;
    lane_swap<16>(x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ bool finite(half_t x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) != 0x7c00u; }

}   // namespace

template <int DP, int NQ, bool Q32>
__global__ __launch_bounds__(64 * Ring<DP>::NW, Ring<DP>::RES) void paged_decode_kernel(PagedAttnParams p, uint32_t ring_at)
{
    using namespace pg;
    using R = Ring<DP>;
    constexpr int NW = R::NW, D = R::D, RB = 16 * NQ, KS = DP / 32, DB = DP / 16;
    constexpr float LIFT = 14.f, SLACK = 1.f;
    constexpr uint32_t OUT = 0x7fffff00u;      // an offset past any page
    extern __shared__ __attribute__((aligned(256))) float4v paged_decode_lds[];   // (the reads' XORs: tiles start on 256 bytes)
    uint32_t* pre = (uint32_t*)paged_decode_lds;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c16 = lane & 15, g = lane >> 4, HD = p.head_dim, group = p.hq / p.hkv;
    const KvPages& pgs = p.pages;
    LDS_AS char* ring = (LDS_AS char*)(LDS_AS void*)paged_decode_lds + ring_at + wave * (D * R::TILE);
    const uint32_t ring0 = (uint32_t)(uintptr_t)ring;

    // the lane's 16 bytes of each of a block's copies: row and logical chunk
    uint32_t voff[R::COPIES];
#pragma unroll
    for (int i = 0; i < R::COPIES; ++i) {
        constexpr uint32_t CH = DP / 8;
        const uint32_t at = i * 64 + lane, r = at / CH, pc = at % CH;
        const uint32_t c = (pc & ~15u) | ((pc & 15u) ^ (uint32_t)swz_row<DP>(r));
        voff[i] = 8 * c < HD ? r * HD * 2 + c * 16 : OUT;
    }
    // where the lane's reads start in a tile; a step of the head dim is an XOR away
    const uint32_t kread = c16 * R::ROWB + ((g ^ (uint32_t)swz_row<DP>(c16)) << 4);
    const uint32_t vrow = 4 * g + (c16 >> 2);
    const uint32_t vread = 2 * R::BLOCK + vrow * R::ROWB + ((((c16 >> 1) & 1u) ^ (uint32_t)swz_row<DP>(vrow)) << 4) + (c16 & 1) * 8;

    __shared__ Sequence kept[KEPT];
    plan_line<NW>(p, RB, pre, kept);
    walk<RB>(p, pre, kept, [&](const Piece& u) __attribute__((always_inline)) {
        const uint32_t rows = u.q.n * group, row0 = u.rb * RB, rend = min(row0 + RB, rows);
        typedef typename std::conditional<Q32, float, half_t>::type qt;
        typedef qt q8 __attribute__((ext_vector_type(8)));
        typedef q8 q8u __attribute__((aligned(sizeof(qt))));
        q8 qraw[NQ][KS];
        int kbeg[NQ], kend[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const uint32_t r = min(row0 + q * 16 + c16, rend - 1), tok = r / group;
            kbeg[q] = (int)first_key(p, u.q.held, tok);
            kend[q] = (int)end_key(p, u.q.held, u.q.live, tok);
            const qt* src = (const qt*)p.q + (size_t)(u.q.first + tok) * p.q_stride + (size_t)(u.hk * group + r % group) * HD;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint32_t d = 32 * s + 8 * g;
                qraw[q][s] = (q8)(qt)0;
                if (d < HD) qraw[q][s] = *(const q8u*)(src + d);
            }
        }
        // what every row of the block sees
        const uint32_t tok0 = row0 / group, tok1 = (rend - 1) / group;
        const int all_beg = (int)first_key(p, u.q.held, tok1);
        const int all_end = (int)end_key(p, u.q.held, u.q.live, tok0);

        const uint32_t first = u.t0 + wave;
        const int mine = first < u.t1 ? (int)((u.t1 - first + NW - 1) / NW) : 0;
        // lane i's 16 positions of the 32 tiles from `it` on: their page's entry (none: the
        // last), and the byte where they start in a head's part of it
        uint32_t entry = 0xffffffffu, start = 0;
        const auto look_up = [&](int it) __attribute__((always_inline)) {
            const uint64_t pos = (uint64_t)(first + (uint32_t)(it + (int)(lane >> 1)) * NW) * KT + 16 * (lane & 1);
            entry = 0xffffffffu;
            start = 0;
            if (pos < u.q.live) {
                const uint32_t i = (uint32_t)pos / pgs.page_size;
                entry = pgs.table[(size_t)u.s * pgs.max_pages + i];
                start = ((uint32_t)pos - i * pgs.page_size) * HD * 2;
            }
        };
        const auto copy = [&](int it) __attribute__((always_inline)) {
            LDS_AS char* dst = ring + (it % D) * R::TILE;
            const uint32_t j0 = (first + (uint32_t)it * NW) * KT;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int l = 2 * (it & 31) + b;
                const uint32_t e = __builtin_amdgcn_readlane(entry, l), at = __builtin_amdgcn_readlane(start, l);
                const uint32_t pos = j0 + 16 * b;
                // positions that are not there, and rows past the last one, read as zeros
                const uint32_t n = e < pgs.num_pages && pos < u.q.live ? min(16u, u.q.live - pos) * HD * 2 : 0u;
                const size_t byte = n ? (e * pgs.stride + (uint64_t)u.hk * pgs.page_size * HD) * 2 + at : 0u;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                        (void*)(uniform_ptr((char*)(v ? pgs.v : pgs.k)) + byte), (short)0, (int)n, 0x00020000);
#pragma unroll
                    for (int i = 0; i < R::COPIES; ++i)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(
                            r, (LDS_AS void*)(dst + v * 2 * R::BLOCK + b * R::BLOCK + i * 1024), 16, (int)voff[i], 0, 0, 0);
                }
            }
        };
        // bit b: the tile's block b is a page's
        const auto there = [&](int it) __attribute__((always_inline)) {
            const uint32_t a = __builtin_amdgcn_readlane(entry, 2 * (it & 31)), c = __builtin_amdgcn_readlane(entry, 2 * (it & 31) + 1);
            return (a < pgs.num_pages ? 1u : 0u) | (c < pgs.num_pages ? 2u : 0u);
        };
        uint32_t have = 0;                     // two bits a ring tile
        look_up(0);
#pragma unroll
        for (int i = 0; i < D; ++i)
            if (i < mine) {
                copy(i);
                have |= there(i) << (2 * i);
            }

        half8 qf[NQ][KS], ql[Q32 ? NQ : 1][Q32 ? KS : 1];
        float sc[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            sc[q] = p.scale * 1.4426950408889634f;   // scores in log2 units
            if constexpr (Q32) {
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(qraw[q][s][e]));
                top = swap_max32(swap_max16(top));
                const int ex = top > 0.f && top < __builtin_inff() ? 10 - __builtin_amdgcn_frexp_expf(top) : 0;
                sc[q] = ldexpf(sc[q], -ex);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    float8v x;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = ldexpf(qraw[q][s][e], ex);
                    qf[q][s] = __builtin_convertvector(x, half8);
                    ql[q][s] = __builtin_convertvector(x - __builtin_convertvector(qf[q][s], float8v), half8);
                }
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[q][s] = qraw[q][s];
            }
        }

        float m[NQ], l[NQ];
        float4v o[NQ][DB];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            m[q] = -__builtin_inff();
            l[q] = 0.f;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[q][d] = (float4v)0.f;
        }

        for (int it = 0; it < mine; ++it) {
            wait_behind<D - 1, 4 * R::COPIES>(mine - 1 - it);
            const int j0 = (int)((first + (uint32_t)it * NW) * KT);
            const uint32_t slot = ring0 + (uint32_t)(it % D) * R::TILE;
            float4v sa[2][NQ];
            {
                half8 kf[2][KS];
                const uint32_t a = slot + kread;
                if constexpr (DP == 64) {
                    half8 x[4];
                    read4<0, 0, R::BLOCK, R::BLOCK>(a, a ^ 64, a, a ^ 64, x);
                    kf[0][0] = x[0]; kf[0][1] = x[1]; kf[1][0] = x[2]; kf[1][1] = x[3];
                } else {
                    static_for<2 * KS / 4>([&](auto idx) __attribute__((always_inline)) {
                        constexpr int k = decltype(idx)::value / (KS / 4), h = decltype(idx)::value % (KS / 4), OFF = k * R::BLOCK + h * 256;
                        half8 x[4];
                        read4<OFF, OFF, OFF, OFF>(a, a ^ 64, a ^ 128, a ^ 192, x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) kf[k][4 * h + e] = x[e];
                    });
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        sa[k][q] = (float4v)0.f;
#pragma unroll
                        for (int s = 0; s < KS; ++s) {
                            sa[k][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k][s], qf[q][s], sa[k][q], 0, 0, 0);
                            if constexpr (Q32) sa[k][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k][s], ql[q][s], sa[k][q], 0, 0, 0);
                        }
                    }
            }
            // whether some row does not see some position (uniform)
            const uint32_t blocks = have >> (2 * (it % D)) & 3u;
            const bool edge = j0 < all_beg || j0 + KT > all_end || blocks != 3u;
            half8 ph[NQ], pl[NQ], seen[NQ];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = sa[i >> 2][q][i & 3] * sc[q];
                if (edge) {
                    const int lo = kbeg[q] - j0, hi = kend[q] - j0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = 16 * (i >> 2) + 4 * (int)g + (i & 3);
                        const bool see = key >= lo && key < hi && (blocks >> (i >> 2) & 1u);
                        v[i] = see ? v[i] : -__builtin_inff();
                        seen[q][i] = see ? (half_t)1.f : (half_t)0.f;
                    }
                }
                float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
                top = swap_max32(swap_max16(top));
                // the row's reference m moves only when the maximum exceeds it by more than
                // SLACK (P stays below 2^(SLACK + LIFT), in fp16's range), for the whole wave at once
                if (__any(top > m[q] + SLACK)) {
                    const float mnew = fmaxf(m[q], top);
                    const float alpha = __builtin_amdgcn_exp2f(m[q] - (mnew == -__builtin_inff() ? 0.f : mnew));
                    l[q] *= alpha;
                    m[q] = mnew;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[q][d] *= alpha;
                }
                const float ref = (m[q] == -__builtin_inff() ? 0.f : m[q]) - LIFT;   // (l and o carry 2^LIFT alike)
                float8v e;
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(v[i] - ref);
                l[q] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));   // (the lane's positions)
                ph[q] = __builtin_convertvector(e, half8);
                pl[q] = __builtin_convertvector(e - __builtin_convertvector(ph[q], float8v), half8);
            }
            // O^T += V^T P^T
            const uint32_t a = slot + vread;
            static_for<DB / 4>([&](auto idx) __attribute__((always_inline)) {
                constexpr int d0 = 4 * decltype(idx)::value, X = (d0 & 7) << 5;
                half4 x[8];
                read_tr4<(d0 >> 3) * 256, R::BLOCK>(a ^ X, a ^ (X + 32), a ^ (X + 64), a ^ (X + 96), x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    half8 va = __builtin_shufflevector(x[2 * i], x[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    if (edge) {
                        // a value that is not finite: 0 times it would reach rows that do not see it
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < 8; ++e) odd = odd || !finite(va[e]);
                        if (__builtin_expect(__any(odd), 0)) {
                            half8 is;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                is[e] = finite(va[e]) ? (half_t)0.f : (half_t)1.f;
                                va[e] = finite(va[e]) ? va[e] : (half_t)0.f;
                            }
#pragma unroll
                            for (int q = 0; q < NQ; ++q) {
                                const float4v bad = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, seen[q], (float4v)0.f, 0, 0, 0);
#pragma unroll
                                for (int r = 0; r < 4; ++r) o[q][d0 + i][r] = bad[r] > 0.f ? __builtin_nanf("") : o[q][d0 + i][r];
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        o[q][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[q], o[q][d0 + i], 0, 0, 0);
                        o[q][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[q], o[q][d0 + i], 0, 0, 0);
                    }
                }
            });
            if (it + D < mine) {
                if (((it + D) & 31) == 0) look_up(it + D);
                copy(it + D);
                have = (have & ~(3u << (2 * (it % D)))) | there(it + D) << (2 * (it % D));
            }
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            l[q] = swap_sum<16>(l[q], l[q]);
            l[q] = swap_sum<32>(l[q], l[q]);
        }
        finish_piece<DP, NQ, NW>(p, u, (char*)paged_decode_lds + ring_at, m, l, o);
    });
}

bool paged_decode_ok(const PagedAttnParams& p)
{
    return p.pages.dtype == DT_F16 && p.head_dim % 8 == 0 && p.pages.page_size % 16 == 0 && p.pages.stride % 8 == 0 &&
           (uintptr_t)p.pages.k % 16 == 0 && (uintptr_t)p.pages.v % 16 == 0 &&
           (uint64_t)p.pages.page_size * p.head_dim * 2 < 1ull << 32;   // (offsets in a head's part of a page)
}

void paged_decode_plan(PagedAttnParams& p, uint32_t* resident)
{
    // (32 rows of 256-wide heads would spill)
    p.rb = p.dp == 256 || (uint64_t)p.max_new * (p.hq / p.hkv) <= 16 ? 16 : 32;
    // (shares of 1, 2, 4, 8 tiles, one token over 500 positions of heads of 64: 9.7, 9.7,
    // 10.1, 10.7 us; over 3000 of 128: 11.5, 11.5, 12.1, 13.9)
    p.min_share = 2;
    // (64 sequences of up to 8192 positions, heads of 128, with 1, 2, 3, 4, 6, 9: 104, 100,
    // 92, 88, 87, 88 us; of 64, 1, 3, 6, 9, 12, 16: 66, 58, 52, 48.5, 48.7, 49.6)
    p.lead = p.dp == 64 ? 10 : 6;
    *resident = p.dp == 256 ? Ring<256>::RES : Ring<128>::RES;
}

template <int DP, int NQ, bool Q32>
static hipError_t decode_launch(const PagedAttnParams& p, hipStream_t s)
{
    using R = Ring<DP>;
    static_assert(R::BYTES >= pg::finish_bytes<DP, NQ, R::NW>(), "the waves' sums meet where the rings were");
    const uint32_t at = ((p.pages.sequences + 1) * 4 + 255) / 256 * 256;
    static PerDevice once;
    const hipError_t e = set_max_lds(once, (const void*)paged_decode_kernel<DP, NQ, Q32>, R::BYTES + (KvPages::MAX_SEQUENCES + 64) * 4);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_decode_kernel<DP, NQ, Q32>), dim3(p.wgs), dim3(64 * R::NW), at + R::BYTES, s, p, at);
    return hipGetLastError();
}

hipError_t paged_decode_launch(const PagedAttnParams& p, hipStream_t s)
{
    const auto rows = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        if constexpr (DP < 256)
            if (p.rb == 32) return p.q_dtype == DT_F16 ? decode_launch<DP, 2, false>(p, s) : decode_launch<DP, 2, true>(p, s);
        return p.q_dtype == DT_F16 ? decode_launch<DP, 1, false>(p, s) : decode_launch<DP, 1, true>(p, s);
    };
    if (p.dp == 64) return rows(std::integral_constant<int, 64>{});
    return p.dp == 128 ? rows(std::integral_constant<int, 128>{}) : rows(std::integral_constant<int, 256>{});
}

}   // namespace vai_dev
