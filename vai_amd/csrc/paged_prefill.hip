// paged_prefill.hip -- attention of the sequences of a ragged batch that bring
// many rows (chunks of prompts), over fp16 pages whose sizes are whole 16s, head
// dims whole 8s.
//
// What bounds it: the matrix cores (4 D operations a query and position). A unit is
// 128 query rows of a sequence and KV head, token-major, so that the heads of a
// group share the tiles; a workgroup walks 64-position tiles of K and V, copied to
// LDS while the tile before is multiplied, each wave one page's 16 positions of
// them (attention.hip's tile and fragment order: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16_f16, the scores of a row in a lane and its partner). Two
// workgroups a CU (D = 256: one, by registers): one's softmax, and its beginning
// and end of a unit, under the other's products. (One of two groups of waves that
// take the tiles in turn halves the partial results, but 8192 tokens of a prompt
// took 823 us so where two workgroups took 700, with probabilities in one number
// each; 888 by now, with two.)
// All units' tiles form a line that the workgroups cut into equal shares, head by
// head on one XCD, as paged_plan.h does for few rows; a unit's tiles are those its
// own rows see. An fp32 q enters as two fp16 numbers (Q2), and so do the
// probabilities, whatever the output's type: one number alone leaves 2^-11 of sum p
// |v| in the result, as much as an fp16 output's own rounding, and would cost a
// sequence's single token bits where a prompt joins its batch. (A chunk of 512
// beside 8 single tokens, 32 heads over 8 of 128: 128 us, with one number 106.)
// Registers are short: heads of 128 keep 43 of a lane's in scratch (an fp32 q 85),
// heads of 256 25 (80). With an fp16 q they come back once a piece, or where V is not
// finite; with an fp32 q in the tile loop, behind the copies in flight (the chunk
// 161 us; 512 beside 8 with heads of 256 263 and 547).
#include "attention_tile.h"
#include "paged_plan.h"

#include "launch_once.h"

namespace vai_dev {

namespace pp {
constexpr int RB = 128, KT = 64;

// The tiles [tb, te) that block rb of a sequence's rows sees (at least one).
struct Tiles {
    uint32_t tb, te;
};
__device__ __forceinline__ Tiles tiles_of(const PagedAttnParams& p, uint32_t held, uint32_t live, uint32_t rows, uint32_t rb)
{
    const uint32_t group = p.hq / p.hkv, tok0 = rb * RB / group, tok1 = (min((rb + 1) * RB, rows) - 1) / group;
    const uint32_t end = pg::end_key(p, held, live, tok1);
    Tiles t;
    t.tb = pg::first_key(p, held, tok0) / KT;
    t.te = max(t.tb + 1, (end + KT - 1) / KT);
    return t;
}
__device__ __forceinline__ uint32_t wave_add(uint32_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// pre[s] = the line's tiles before sequence s (few rows: none of its own), pre[n] all.
template <int NWAVES>
__device__ __forceinline__ void plan_line(const PagedAttnParams& p, uint32_t* pre)
{
    __shared__ uint32_t sums[NWAVES];
    const uint32_t n = p.pages.sequences, per = (n + 64 * NWAVES - 1) / (64 * NWAVES), lane = threadIdx.x & 63;
    const uint32_t s0 = min(threadIdx.x * per, n), s1 = min(s0 + per, n), group = p.hq / p.hkv;
    uint32_t sum = 0;
    for (uint32_t i = 0; i < per; ++i) {
        Sequence q{};
        const uint32_t s = s0 + i;
        if (s < s1) q = sequence_of(p.pages, s, p.tokens);
        const uint32_t rows = q.n * group, nb = rows > p.few_rows ? (rows + RB - 1) / RB : 0u;
        uint32_t w = 0;
        if (nb <= 8)
            for (uint32_t b = 0; b < nb; ++b) {
                const Tiles t = tiles_of(p, q.held, q.live, rows, b);
                w += t.te - t.tb + p.lead;
            }
        // (many blocks: the wave's lanes take them together)
        for (uint64_t many = __ballot(nb > 8); many; many &= many - 1) {
            const int l = __builtin_ctzll(many);
            const uint32_t held = __shfl(q.held, l), live = __shfl(q.live, l), r = __shfl(rows, l), m = __shfl(nb, l);
            uint32_t x = 0;
            for (uint32_t b = lane; b < m; b += 64) {
                const Tiles t = tiles_of(p, held, live, r, b);
                x += t.te - t.tb + p.lead;
            }
            x = wave_add(x);
            if (lane == (uint32_t)l) w = x;
        }
        w *= p.hkv;
        if (s < s1) pre[s] = w;
        sum += w;
    }
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(scan, o);
        if (lane >= (uint32_t)o) scan += x;
    }
    if (lane == 63) sums[threadIdx.x >> 6] = scan;
    __syncthreads();
    uint32_t at = scan - sum;
    for (uint32_t w = 0; w < threadIdx.x >> 6; ++w) at += sums[w];
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t w = pre[s];
        pre[s] = at;
        at += w;
    }
    if (s1 == n && s0 < n) pre[n] = at;
    __syncthreads();
}

struct Piece {
    Sequence q;
    uint32_t s, hk, rb, t0, t1;
    bool whole;
    uint32_t slot;
};

// Calls f for each piece of share `me` of the line.
template <class F>
__device__ __forceinline__ void walk(const PagedAttnParams& p, const uint32_t* pre, uint32_t me, F&& f)
{
    const uint32_t n = p.pages.sequences, total = __builtin_amdgcn_readfirstlane(pre[n]), lane = threadIdx.x & 63;
    const uint32_t share = max(p.min_share, (total + p.wgs - 1) / p.wgs), group = p.hq / p.hkv;
    const uint64_t begin = (uint64_t)me * share;
    pg::Joint joint{};
    const uint32_t end = (uint32_t)std::min<uint64_t>(begin + share, total);
    for (uint32_t at = (uint32_t)std::min<uint64_t>(begin, total); at < end;) {
        Piece u;
        u.s = __builtin_amdgcn_readfirstlane(pg::line_sequence(pre, n, at));
        u.q = sequence_of(p.pages, u.s, p.tokens);
        const uint32_t base = __builtin_amdgcn_readfirstlane(pre[u.s]), all = __builtin_amdgcn_readfirstlane(pre[u.s + 1]) - base;
        const uint32_t rows = u.q.n * group, nb = (rows + RB - 1) / RB, head = all / p.hkv;
        if (rows <= p.few_rows || head == 0) break;      // (starts that do not increase)
        u.hk = (at - base) / head;
        // the block that `off` of the head's stretch is in, 64 at a time
        uint32_t off = at - base - u.hk * head, b0 = 0, len = 0, tb = 0;
        for (;; b0 += 64) {
            const uint32_t b = b0 + lane;
            Tiles t{0, 0};
            uint32_t x = 0;
            if (b < nb) {
                t = tiles_of(p, u.q.held, u.q.live, rows, b);
                x = t.te - t.tb + p.lead;
            }
            uint32_t scan = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(scan, o);
                if (lane >= (uint32_t)o) scan += y;
            }
            const uint64_t past = __ballot(scan > off);
            if (past) {
                const int l = __builtin_ctzll(past);
                len = __builtin_amdgcn_readlane(x, l);
                off -= __builtin_amdgcn_readlane(scan, l) - len;
                tb = __builtin_amdgcn_readlane(t.tb, l);
                u.rb = b0 + l;
                break;
            }
            if (b0 + 64 >= nb) break;
            off -= __builtin_amdgcn_readlane(scan, 63);
        }
        if (len == 0 || u.hk >= p.hkv) break;            // (the same)
        const uint32_t o0 = off, o1 = min(len, o0 + (end - at)), tiles = len - p.lead;
        const uint32_t t0 = o0 > p.lead ? o0 - p.lead : 0u, t1 = o1 > p.lead ? o1 - p.lead : 0u;
        if (at == begin && t0 > 0) {
            const uint32_t a = at - o0 + p.lead, wg0 = a / share;    // (the unit's first tile)
            if (wg0 + 1 == me)
                joint = pg::Joint{min((a + tiles - 1) / share + 1, p.wgs) - wg0, wg0, u.q.first, u.hk, u.rb * RB,
                                  min((uint32_t)RB, rows - u.rb * RB), {0, 0}};
        }
        at += o1 - o0;
        if (t1 == t0) continue;
        u.t0 = tb + t0;
        u.t1 = tb + t1;
        u.whole = t1 - t0 == tiles;
        u.slot = 2 * me + (t0 == 0 ? 1u : 0u);
        f(u);
    }
    if (threadIdx.x == 0) ((pg::Joint*)p.ws_plan)[me] = joint;
}

// fa_vfrag, waited for
template <int D, int KK, int DD>
__device__ __forceinline__ half8 vfrag_now(const uint32_t (&vaddr)[2])
{
    half4 a, b;
    asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b)
                 : "v"(vaddr[DD & 1]), "n"(fa_voff<D, KK, DD, 0>()), "n"(fa_voff<D, KK, DD, 1>()));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ bool finite(half_t x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) != 0x7c00u; }

}   // namespace pp

template <int D, bool Q2>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_prefill_kernel(PagedAttnParams p, uint32_t tiles_at)
{
    using namespace fa;
    using pp::Piece;
    using pp::RB;
    using L = Lds<D>;
    constexpr int KS = D / 16, DF = D / 32, CR = D / 4;
    // P stays below 2^15, and of those far below the row's largest two fp16 numbers hold
    // what lies above 2^-25, which is 2^-39 of the largest. (8 and 7, with fewer changes of
    // the reference, take 125 us of a chunk's 128, and hold 2^-32 of it.)
    constexpr float SLACK = 1.f, LIFT = 14.f;
    extern __shared__ __attribute__((aligned(1024))) float4v paged_prefill_lds[];
    uint32_t* pre = (uint32_t*)paged_prefill_lds;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    LDS_AS char* lds = (LDS_AS char*)(LDS_AS void*)paged_prefill_lds + tiles_at;
    const int ql = lane & 31, hf = lane >> 5;
    const uint32_t HD = p.head_dim, group = p.hq / p.hkv;
    const KvPages& pgs = p.pages;

    // copy j of the wave's 16 positions: the lane's row of them and logical chunk (past the head dim: no byte)
    uint32_t coff[L::COPIES];
#pragma unroll
    for (int j = 0; j < L::COPIES; ++j) {
        const int byte = (wave * L::COPIES + j) * 1024 + lane * 16;
        const int r = byte / L::ROWB, pc = (byte % L::ROWB) / 16, lc = swz<D>(r, pc);
        coff[j] = 8u * lc < HD ? (uint32_t)((r & 15) * HD * 2 + lc * 16) : 0x7fffff00u;
    }
    // lane parts of the fragment addresses, of the stage in use
    const int g = lane >> 4, s16 = lane & 15;
    const int vrow = s16 >> 2, vcol = 16 * (g & 1) + 4 * (s16 & 3), vkey = 4 * (g >> 1);
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
    constexpr int NK = fa_nk<D>;
    uint32_t kaddr[NK], vaddr[2];
#pragma unroll
    for (int j = 0; j < NK; ++j)
        kaddr[j] = lds0 + ql * L::ROWB +
                  (((2 * (j & 3) + hf) ^ swz_f(ql & 7)) + (D >= 128 ? (8 * (j >> 2)) ^ (ql & 8) : 0)) * 16;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        vaddr[j] = lds0 + (vkey + vrow) * L::ROWB + ((4 * j + (vcol >> 3)) ^ swz_f((vkey + vrow) & 7)) * 16 +
                  (vcol & 7) * 2;

    pp::plan_line<NW>(p, pre);
    pp::walk(p, pre, fa_xcd_block(blockIdx.x, gridDim.x), [&](const Piece& u) __attribute__((always_inline)) {
        const uint32_t rows = u.q.n * group, row = min(u.rb * RB + wave * QW + ql, rows - 1);
        const uint32_t tok = row / group;
        const int kbeg = (int)pg::first_key(p, u.q.held, tok), kend = (int)pg::end_key(p, u.q.held, u.q.live, tok);

        // query rows: lane l holds query l % 32, values 16 s + 8 (l / 32) ..+7
        half8 qf[KS], q2[Q2 ? KS : 1];
        float sc = p.scale * 1.4426950408889634f;        // scores in log2 units
        {
            const size_t at = (size_t)(u.q.first + tok) * p.q_stride + (size_t)(u.hk * group + row % group) * HD;
            if constexpr (Q2) {
                typedef float8v float8u __attribute__((aligned(4)));
                float8v x[KS];
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const uint32_t d = 16 * s + 8 * hf;
                    x[s] = (float8v)0.f;
                    if (d < HD) x[s] = *(const float8u*)((const float*)p.q + at + d);
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[s][e]));
                }
                top = swap_max32(top);
                const int ex = top > 0.f && top < __builtin_inff() ? 10 - __builtin_amdgcn_frexp_expf(top) : 0;
                sc = ldexpf(sc, -ex);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[s][e] = ldexpf(x[s][e], ex);
                    qf[s] = __builtin_convertvector(x[s], half8);
                    q2[s] = __builtin_convertvector(x[s] - __builtin_convertvector(qf[s], float8v), half8);
                }
            } else {
                typedef half8 half8u __attribute__((aligned(2)));
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const uint32_t d = 16 * s + 8 * hf;
                    qf[s] = (half8)(half_t)0;
                    if (d < HD) qf[s] = *(const half8u*)((const half_t*)p.q + at + d);
                }
            }
        }

        // where the 16 tiles of a batch lie, four blocks of 16 positions each: lane 4 i + b holds
        // tile i's block b
        const int mine = (int)(u.t1 - u.t0);
        uint32_t entry, start, entry2 = 0xffffffffu, start2 = 0;
        const auto look_up = [&](int t, uint32_t& e, uint32_t& st) __attribute__((always_inline)) {
            const uint64_t at = (uint64_t)(u.t0 + (uint32_t)(t + (int)(lane >> 2))) * pp::KT + 16 * (lane & 3);
            e = 0xffffffffu;
            st = 0;
            if (at < u.q.live) {
                const uint32_t i = (uint32_t)at / pgs.page_size;
                e = pgs.table[(size_t)u.s * pgs.max_pages + i];
                st = ((uint32_t)at - i * pgs.page_size) * HD * 2;
            }
        };
        look_up(0, entry, start);
        const auto rsrc = [&](int t, const void* pool) __attribute__((always_inline)) {
            const int l = 4 * (t & 15) + (int)wave;
            const uint32_t e = __builtin_amdgcn_readlane(entry, l), at = __builtin_amdgcn_readlane(start, l);
            const uint32_t ps = (u.t0 + (uint32_t)t) * pp::KT + 16 * wave;
            // positions that are not there, and rows past the last one, read as zeros
            const uint32_t n = t < mine && e < pgs.num_pages && ps < u.q.live ? min(16u, u.q.live - ps) * HD * 2 : 0u;
            const size_t byte = n ? (e * pgs.stride + (uint64_t)u.hk * pgs.page_size * HD) * 2 + at : 0u;
            return __builtin_amdgcn_make_buffer_rsrc((void*)(uniform_ptr((char*)pool) + byte), (short)0, (int)n, 0x00020000);
        };
        fa_issue<D>(rsrc(0, pgs.k), rsrc(0, pgs.v), lds, coff, 0, wave);

        float m = -__builtin_inff(), l = 0.f;
        float16v o[DF];
#pragma unroll
        for (int d = 0; d < DF; ++d) o[d] = (float16v)0.f;

        // A wave without rows (a sequence's last unit, one of few rows) only copies: a chunk
        // of 512 tokens beside 32 single ones takes 165 us, 178 where it multiplies too.
        const bool idle = u.rb * RB + wave * QW >= rows;
        if (idle) {
            for (int t = 0; t < mine; ++t) {
                fa_wait_vmcnt<0>();
                __builtin_amdgcn_s_barrier();
                if ((t & 15) == 14) look_up(t + 2, entry2, start2);
                if ((t & 15) == 15) {
                    entry = entry2;
                    start = start2;
                }
                if (t + 1 < mine) fa_issue<D>(rsrc(t + 1, pgs.k), rsrc(t + 1, pgs.v), lds, coff, (t + 1) & 1, wave);
                __builtin_amdgcn_s_barrier();
            }
        }
        for (int t = 0; t < mine && !idle; ++t) {
            // tile t is in stage t % 2; the next one's copies go out during its S^T products
            fa_wait_vmcnt<0>();
            __builtin_amdgcn_s_barrier();
            const uint32_t blocks = (uint32_t)(__ballot(entry < pgs.num_pages) >> (4 * (t & 15))) & 15u;
            if ((t & 15) == 14) look_up(t + 2, entry2, start2);
            if ((t & 15) == 15) {
                entry = entry2;
                start = start2;
            }
            const int j0 = (int)((u.t0 + (uint32_t)t) * pp::KT);

            // step i of the 2 KS products is key block i % 2, head-dim step i / 2; K fragments are
            // read G at a time, the next group's behind this one's products
            constexpr int NS = 2 * KS, G = D == 64 ? 8 : 4;
            constexpr int OPG = 2 * L::COPIES / (NS / G);
            static_assert(OPG * (NS / G) == 2 * L::COPIES, "copies spread evenly over the groups");
            const bool next = t + 1 < mine;
            const __amdgpu_buffer_rsrc_t rkn = rsrc(t + 1, pgs.k), rvn = rsrc(t + 1, pgs.v);
            LDS_AS char* nst = lds + ((t + 1) & 1) * L::STAGE + wave * L::COPIES * 1024;
            float16v sacc[2] = {(float16v)0.f, (float16v)0.f};
            half8 ka[2][G];
            static_for<G>([&](auto I) __attribute__((always_inline)) { ka[0][I] = fa_kfrag<D, I>(kaddr); });
            static_for<NS / G>([&](auto GI) __attribute__((always_inline)) {
                constexpr int gi = GI, cur = gi & 1;
                if constexpr (gi + 1 < NS / G) {
                    static_for<G>([&](auto I) __attribute__((always_inline)) {
                        ka[cur ^ 1][I] = fa_kfrag<D, (gi + 1) * G + I>(kaddr);
                    });
                    fa_lgkm_wait<G>();
                } else {
                    fa_lgkm_wait<0>();
                }
#pragma unroll
                for (int i = 0; i < G; ++i) fa_pin(ka[cur][i]);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const int idx = gi * G + i;
                    sacc[idx & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[cur][i], qf[idx >> 1], sacc[idx & 1], 0, 0, 0);
                    if constexpr (Q2)
                        sacc[idx & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[cur][i], q2[idx >> 1], sacc[idx & 1], 0, 0, 0);
                }
                if (next) {
                    static_for<OPG>([&](auto I) __attribute__((always_inline)) {
                        constexpr int op = gi * OPG + I;   // K copies, then V copies
                        constexpr int j = op % L::COPIES;
                        if constexpr (op < L::COPIES)
                            __builtin_amdgcn_raw_ptr_buffer_load_lds(rkn, (LDS_AS void*)(nst + j * 1024), 16, (int)coff[j], 0, 0, 0);
                        else
                            __builtin_amdgcn_raw_ptr_buffer_load_lds(rvn, (LDS_AS void*)(nst + L::TILE + j * 1024), 16,
                                                                     (int)coff[j], 0, 0, 0);
                    });
                }
            });

            // Softmax in log2 units. Keys of the tile: kb*32 + 8 (rr / 4) + 4 hf + rr % 4. Where every
            // row of the wave sees the whole tile: the maximum over the raw scores, then 2^(fma(s, scale, -m)).
            const int lo = kbeg - j0, hi = kend - j0;
            const bool edge = !(__all(lo <= 0 && hi >= pp::KT) && blocks == 15u);
            const bool fast = !edge && sc >= 0.f;     // (the scale's sign is every lane's)
            // A position whose V holds a value that is not finite must not reach rows that do not
            // see it through 0 times that value: its V is 0 here and its score NaN, which the mask
            // replaces. Bit 8 kk + i of a lane is the position of its probability i of step kk.
            bool odd = false;
            if (edge) {
                uint32_t bad = 0;
                static_for<4>([&](auto KK) __attribute__((always_inline)) {
                    static_for<DF>([&](auto DD) __attribute__((always_inline)) {
                        const half8 v = pp::vfrag_now<D, KK, DD>(vaddr);
#pragma unroll
                        for (int i = 0; i < 8; ++i) bad |= pp::finite(v[i]) ? 0u : 1u << (8 * KK + i);
                    });
                });
                odd = __any(bad != 0);
                if (__builtin_expect(odd, 0)) {
#pragma unroll
                    for (int x = 1; x < 32; x <<= 1) bad |= __shfl_xor(bad, x);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (bad >> i & 1u) sacc[i >> 4][i & 15] = __builtin_nanf("");
                }
            }
            if (!fast) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int rr = 0; rr < 16; ++rr) {
                        const int kl = kb * 32 + 8 * (rr >> 2) + 4 * hf + (rr & 3);
                        sacc[kb][rr] = kl < hi && kl >= lo ? sacc[kb][rr] * sc : -__builtin_inff();
                    }
                if (blocks != 15u) {
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (!(blocks >> b & 1u))
#pragma unroll
                            for (int i = 0; i < 8; ++i) sacc[b >> 1][8 * (b & 1) + i] = -__builtin_inff();
                }
            }
            float tm[10];
#pragma unroll
            for (int i = 0, j = 0; i < 10; ++i, j += 3)
                tm[i] = fa_max3(sacc[j >> 4][j & 15], sacc[(j + 1) >> 4][(j + 1) & 15], sacc[(j + 2) >> 4][(j + 2) & 15]);
            float tmax = fa_max3(fa_max3(tm[0], tm[1], tm[2]), fa_max3(tm[3], tm[4], tm[5]),
                                 fa_max3(fa_max3(tm[6], tm[7], tm[8]), tm[9], fa_max3(sacc[1][14], sacc[1][15], sacc[1][15])));
            if (fast) tmax *= sc;
            tmax = swap_max32(tmax);
            // the row's reference moves only when the maximum exceeds it by more than SLACK, for the
            // whole wave at once
            if (__builtin_expect(__any(tmax > m + SLACK), 0)) {
                const float mnew = fmaxf(m, tmax);
                const float alpha = __builtin_amdgcn_exp2f(m - (mnew == -__builtin_inff() ? 0.f : mnew));
                l *= alpha;
                m = mnew;
                if (t > 0) {
#pragma unroll
                    for (int d = 0; d < DF; ++d) o[d] *= alpha;
                }
            }
            const float ref = (m == -__builtin_inff() ? 0.f : m) - LIFT;    // (l and o carry 2^LIFT alike)
            half8 pb[4], p2[4];
            const float esc = fast ? sc : 1.f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                float8v e;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[kk >> 1][8 * (kk & 1) + i], esc, -ref));
                pb[kk] = __builtin_convertvector(e, half8);
                p2[kk] = __builtin_convertvector(e - __builtin_convertvector(pb[kk], float8v), half8);
                l += ((e[0] + e[4]) + (e[1] + e[5])) + ((e[2] + e[6]) + (e[3] + e[7]));   // (the lane's positions)
            }

            {
                // O^T += V^T P^T, the next step's V^T fragments in flight behind this one's products
                half8 vb[2][DF];
                static_for<DF>([&](auto DD) __attribute__((always_inline)) { vb[0][DD] = fa_vfrag<D, 0, DD>(vaddr); });
                static_for<4>([&](auto KK) __attribute__((always_inline)) {
                    constexpr int kk = KK, cur = kk & 1;
                    if constexpr (kk + 1 < 4) {
                        static_for<DF>([&](auto DD) __attribute__((always_inline)) {
                            vb[cur ^ 1][DD] = fa_vfrag<D, kk + 1, DD>(vaddr);
                        });
                        fa_lgkm_wait<(2 * DF < 15 ? 2 * DF : 15)>();
                    } else {
                        fa_lgkm_wait<0>();
                    }
#pragma unroll
                    for (int d = 0; d < DF; ++d) fa_pin(vb[cur][d]);
                    if (__builtin_expect(odd, 0)) {
#pragma unroll
                        for (int d = 0; d < DF; ++d)
#pragma unroll
                            for (int i = 0; i < 8; ++i) vb[cur][d][i] = pp::finite(vb[cur][d][i]) ? vb[cur][d][i] : (half_t)0.f;
                    }
#pragma unroll
                    for (int d = 0; d < DF; ++d) {
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb[cur][d], pb[kk], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb[cur][d], p2[kk], o[d], 0, 0, 0);
                    }
                });
            }
            const int32_t flip = t & 1 ? -L::STAGE : L::STAGE;    // the other stage
#pragma unroll
            for (int j = 0; j < NK; ++j) kaddr[j] += flip;
#pragma unroll
            for (int j = 0; j < 2; ++j) vaddr[j] += flip;
            // every wave is done reading stage t % 2 before tile t + 2 overwrites it
            __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));   // lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
        }

        if ((mine & 1) && !idle) {
#pragma unroll
            for (int j = 0; j < NK; ++j) kaddr[j] -= L::STAGE;
#pragma unroll
            for (int j = 0; j < 2; ++j) vaddr[j] -= L::STAGE;
        }

        // The wave's rows go out through LDS (chunk c of row r at slot c ^ (r % 16)), as
        // partial results or as rows of the output. Fragment d: values 32 d + 8 q4 + 4 hf ..+3.
        l = swap_sum<32>(l, l);
        const float inv = u.whole ? (l != 0.f ? 1.0f / l : 0.f) : 1.0f;
        LDS_AS float4v* ob = (LDS_AS float4v*)(lds + wave * QW * D * 4);
#pragma unroll
        for (int d = 0; d < DF; ++d)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                ob[ql * CR + ((8 * d + 2 * q4 + hf) ^ (ql & 15))] = float4v{o[d][4 * q4] * inv, o[d][4 * q4 + 1] * inv,
                                                                          o[d][4 * q4 + 2] * inv, o[d][4 * q4 + 3] * inv};
        constexpr int NJ = QW * CR / 64;
        if (idle) {
        } else if (u.whole) {
            const uint32_t row0 = u.rb * RB + wave * QW;
#pragma unroll 4
            for (int j = 0; j < NJ; ++j) {
                const uint32_t e = j * 64 + lane, r = e / CR, c = e % CR, rr = row0 + r;
                const float4v v = ob[r * CR + (c ^ (r & 15))];
                if (rr < rows && 4 * c < HD) {
                    const uint32_t tk = rr / group;
                    const size_t at = ((size_t)(u.q.first + tk) * p.hq + u.hk * group + (rr - tk * group)) * HD + 4 * c;
                    if (p.o_dtype == DT_F16) put4<true>((half_t*)p.out + at, 4, v);
                    else put4<true>((float*)p.out + at, 4, v);
                }
            }
        } else {
            const size_t at = (size_t)u.slot * RB + wave * QW;
            if (hf == 0) {
                p.ws_ml[2 * (at + ql)] = m;
                p.ws_ml[2 * (at + ql) + 1] = l;
            }
            float* dst = uniform_ptr(p.ws_o + at * D);
#pragma unroll 4
            for (int j = 0; j < NJ; ++j) {
                const uint32_t e = j * 64 + lane, r = e / CR, c = e % CR;
                const float4v v = ob[r * CR + (c ^ (r & 15))];
                if (u.rb * RB + wave * QW + r < rows) *(float4v*)(dst + r * D + 4 * c) = v;
            }
        }
        __syncthreads();     // the next piece's copies go where these were
    });
}

// Joins the parts of the units that a cut runs through, four values a thread: few
// parts of many rows. Grid: (cuts, shares of the unit's values).
template <int D>
__global__ __launch_bounds__(256) void paged_merge_rows_kernel(PagedAttnParams p)
{
    constexpr uint32_t C4 = D / 4, AHEAD = 8;
    const pg::Joint x = ((const pg::Joint*)p.ws_plan)[blockIdx.x + 1];
    const uint32_t e = blockIdx.y * 256 + threadIdx.x, row = e / C4, c = e % C4;
    if (x.parts == 0 || row >= x.rows || 4 * c >= p.head_dim) return;
    const auto at = [&](uint32_t i) { return (size_t)(2 * (x.wg + i) + (i == 0 ? 1u : 0u)) * pp::RB + row; };
    float M = -__builtin_inff(), sum = 0.f;
    float4v acc = (float4v)0.f;
    for (uint32_t i = 0; i < x.parts; i += AHEAD) {      // (all their loads in flight)
        float m[AHEAD], l[AHEAD], top = M;
        float4v v[AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            const size_t a = at(min(i + k, x.parts - 1));
            m[k] = p.ws_ml[2 * a];
            l[k] = p.ws_ml[2 * a + 1];
            v[k] = *(const float4v*)(p.ws_o + a * D + 4 * c);
        }
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) top = fmaxf(top, m[k]);
        const float ref = top == -__builtin_inff() ? 0.f : top, w0 = __builtin_amdgcn_exp2f(M - ref);
        acc *= w0;
        sum *= w0;
        M = top;
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            if (i + k >= x.parts) break;
            const float w = __builtin_amdgcn_exp2f(m[k] - ref);
            acc += w * v[k];
            sum += w * l[k];
        }
    }
    pg::put_row(p, x.first, x.hk, x.row0 + row, 4 * c, acc, sum);
}

void paged_prefill_plan(PagedAttnParams& p, uint32_t cus)
{
    p.rb = pp::RB;
    p.lead = 6;
    p.min_share = 4;
    p.wgs = std::min<uint32_t>(p.dp == 256 ? cus : 2 * cus, PagedAttnParams::MAX_WGS);
}

template <int D, bool Q2>
static hipError_t prefill_launch(const PagedAttnParams& p, hipStream_t s)
{
    constexpr int bytes = fa::Lds<D>::BYTES;
    const uint32_t at = ((p.pages.sequences + 1) * 4 + 1023) / 1024 * 1024;
    static PerDevice once;
    const hipError_t e = set_max_lds(once, (const void*)paged_prefill_kernel<D, Q2>, bytes + KvPages::MAX_SEQUENCES * 4 + 1024);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_prefill_kernel<D, Q2>), dim3(p.wgs), dim3(256), at + bytes, s, p, at);
    return hipGetLastError();
}

template <int D>
static hipError_t prefill_launch_d(const PagedAttnParams& p, hipStream_t s)
{
    const hipError_t e = p.q_dtype == DT_F32 ? prefill_launch<D, true>(p, s) : prefill_launch<D, false>(p, s);
    if (e != hipSuccess || p.wgs == 1) return e;
    hipLaunchKernelGGL(paged_merge_rows_kernel<D>, dim3(p.wgs - 1, pp::RB * (D / 4) / 256), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t paged_prefill_launch(const PagedAttnParams& p, hipStream_t s)
{
    return p.dp == 64 ? prefill_launch_d<64>(p, s) : p.dp == 128 ? prefill_launch_d<128>(p, s) : prefill_launch_d<256>(p, s);
}

}   // namespace vai_dev
