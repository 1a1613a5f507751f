// paged_attention.hip -- attention of a ragged batch over a KV cache in pages:
// the fp32 kernel for any head dim, page size and dtype, the merge of partial
// results, and which kernel a call takes.
//
// The fp32 kernel: v_mfma_f32_16x16x4_f32 throughout, operands from memory to
// registers. S^T = K Q^T over 16 keys x 16 query rows: lane (c16, g) reads 4
// neighbouring values of key c16 at a time, which are its k's of four steps, and
// gets the scores of row c16 with keys 4 g ..+3. Those are, as they stand, the
// lane's P^T operands of O^T += V^T P^T when step r of it takes key 4 g + r; of that
// key's V the lane reads DP / 16 neighbouring values, one for each output block (so
// that O^T's row i of block b is value i DP / 16 + b). No value moves between lanes
// but for where the keys lie and the row's maximum and sum. Where the next 16 keys'
// K and V lie is looked up, and what the next ones hold is read, while 16 are
// multiplied: 64 sequences of up to 8192 positions of fp32 pages, 8 heads of 128,
// take 182 us (409 with one load after the other).
#include "paged_plan.h"

#include "launch_once.h"

namespace vai_dev {

// Rows a KV head up to which a sequence is paged_decode.hip's, whose units of 32 (D =
// 256: 16) rows read the keys once each. 8 sequences of 4000 positions, 32 heads over
// 8 of 128, us there / in paged_prefill.hip: 32 rows 37 / 42, 64 rows 55 / 48, where one
// sequence of 16000 takes 28 / 47, 35 / 50; of 64, 64 rows 33 / 32, one 23 / 38; of 256
// (16 over 4), 32 rows 55 / 52, one 35 / 47, 64 rows 90 / 55, one 50 / 51.
static uint32_t few_most(uint32_t dp) { return dp <= 128 ? 64 : 32; }

// Values d ..+3 of a row of D, as they are, zeros past its end or where there is no row
// (any row that is), W at a time: D is a multiple of W (1, 2 or 4). Without branches,
// what is not wanted is read from the row's own values. That is not for speed alone: a
// form whose loads stood behind divergent branches gave wrong scores for head dims up
// to 48, for a reason that was not found.
template <int W, typename T>
__device__ __forceinline__ auto raw4(const T* row, uint32_t d, uint32_t D, bool there)
{
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    if constexpr (W == 4) {
        typedef t4 t4u __attribute__((aligned(sizeof(T))));
        const t4 v = *(const t4u*)(row + (d < D ? d : 0u));
        return there && d < D ? v : (t4)(T)0;
    } else if constexpr (W == 2) {
        typedef t2 t2u __attribute__((aligned(sizeof(T))));
        t2 a = *(const t2u*)(row + (d < D ? d : 0u)), b = *(const t2u*)(row + (d + 2 < D ? d + 2 : 0u));
        a = there && d < D ? a : (t2)(T)0;
        b = there && d + 2 < D ? b : (t2)(T)0;
        return (t4)__builtin_shufflevector(a, b, 0, 1, 2, 3);
    } else {
        t4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T x = row[min(d + e, D - 1)];
            v[e] = there && d + e < D ? x : (T)0;
        }
        return v;
    }
}

template <int DP, typename T, int W>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void paged_attention_any_kernel(PagedAttnParams p)
{
    using namespace pg;
    constexpr int KB = DP / 16, RB = 16, NW = 4;
    constexpr bool AHEAD = DP < 256;       // (of 256-wide heads two steps' values would not fit the registers)
    extern __shared__ float4v paged_lds[];
    __shared__ uint32_t pre[KvPages::MAX_SEQUENCES + 1];
    __shared__ Sequence kept[KEPT];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c16 = lane & 15, g = lane >> 4, D = p.head_dim, group = p.hq / p.hkv;
    const KvPages& pgs = p.pages;
    const float sl2 = p.scale * 1.4426950408889634f;   // scores in log2 units
    typedef T t4 __attribute__((ext_vector_type(4)));
    struct Step {                          // 16 keys
        t4 k[KB], v[4][KB / 4];            // key c16's values 16 b + 4 g ..+3; keys 4 g + r's values c16 KB ..
        uint32_t there;                    // bit r: key 4 g + r is there
    };
    plan_line<NW>(p, RB, pre, kept);
    walk<RB>(p, pre, kept, [&](const Piece& u) {
        const uint32_t rows = u.q.n * group, row = min(u.rb * RB + c16, rows - 1);
        const uint32_t tok = row / group;
        const uint32_t kbeg = first_key(p, u.q.held, tok), kend = end_key(p, u.q.held, u.q.live, tok);
        const size_t qat = (size_t)(u.q.first + tok) * p.q_stride + (size_t)(u.hk * group + row % group) * D;
        const uint32_t see = first_key(p, u.q.held, 0);     // no row sees a position before it
        const uint32_t first = u.t0 + wave;
        const int steps = first < u.t1 ? 2 * (int)((u.t1 - first + NW - 1) / NW) : 0;
        const auto j0_of = [&](int i) __attribute__((always_inline)) { return (first + (uint32_t)(i >> 1) * NW) * KT + 16 * (i & 1); };
        // where the lane's key of step i starts (in both pools), -1: it is not there
        const auto locate = [&](int i) __attribute__((always_inline)) {
            const uint32_t j = j0_of(i) + c16, n = j / pgs.page_size;
            if (i >= steps || j < see || j >= u.q.live) return (int64_t)-1;
            const uint32_t page = pgs.table[(size_t)u.s * pgs.max_pages + n];
            if (page >= pgs.num_pages) return (int64_t)-1;
            return (int64_t)(page * pgs.stride + ((uint64_t)u.hk * pgs.page_size + (j - n * pgs.page_size)) * D);
        };
        const auto load = [&](int64_t at, Step& x) __attribute__((always_inline)) {
            const T* k = (const T*)pgs.k + (at < 0 ? 0 : at);
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                x.k[b] = raw4<W>(k, 16 * b + 4 * g, D, at >= 0);
            }
            x.there = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t vat = __shfl(at, 4 * g + r);
                x.there |= vat >= 0 ? 1u << r : 0u;
                const T* v = (const T*)pgs.v + (vat < 0 ? 0 : vat);
#pragma unroll
                for (int b = 0; b < KB / 4; ++b) x.v[r][b] = raw4<W>(v, c16 * KB + 4 * b, D, vat >= 0);
            }
        };
        Step cur, nxt;
        int64_t at = locate(0);
        if constexpr (AHEAD) {
            load(at, cur);
            at = locate(1);
        }
        float4v qf[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = 16 * b + 4 * g + i;
                qf[b][i] = d < D ? ld(p.q, p.q_dtype, qat + d) : 0.f;
            }
        float m[1] = {-__builtin_inff()}, l[1] = {0.f};
        float4v o[1][KB];
#pragma unroll
        for (int d = 0; d < KB; ++d) o[0][d] = (float4v)0.f;
        for (int i = 0; i < steps; ++i) {
            if constexpr (AHEAD) {
                load(at, nxt);
                at = locate(i + 2);
            } else {
                load(at, cur);
                at = locate(i + 1);
            }
            if (__any(cur.there != 0)) {
                const uint32_t j0 = j0_of(i);
                float4v sa = (float4v)0.f;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sa = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur.k[b][e], qf[b][e], sa, 0, 0, 0);
                // scores of the lane's row with keys 4 g + r
                float v[4], top = -__builtin_inff();
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t key = j0 + 4 * g + r;
                    v[r] = key >= kbeg && key < kend && (cur.there >> r & 1u) ? sa[r] * sl2 : -__builtin_inff();
                    top = fmaxf(top, v[r]);
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mnew = fmaxf(m[0], top), ref = mnew == -__builtin_inff() ? 0.f : mnew;
                const float alpha = __builtin_amdgcn_exp2f(m[0] - ref);
                m[0] = mnew;
                float e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(v[r] - ref);
                l[0] = l[0] * alpha + ((e[0] + e[1]) + (e[2] + e[3]));    // (the lane's keys)
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    float x[4];
                    bool odd = false;       // a value that is not finite: 0 times it would reach rows that do not see it
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = (float)cur.v[r][b >> 2][b & 3];
                        odd = odd || !(__builtin_fabsf(x[r]) < __builtin_inff());
                    }
                    o[0][b] *= alpha;
                    if (__builtin_expect(__any(odd), 0)) {
                        float4v bad = (float4v)0.f;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool is = !(__builtin_fabsf(x[r]) < __builtin_inff());
                            bad = __builtin_amdgcn_mfma_f32_16x16x4f32(is ? 1.f : 0.f, v[r] != -__builtin_inff() ? 1.f : 0.f, bad, 0, 0, 0);
                            x[r] = is ? 0.f : x[r];
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[0][b][r] = bad[r] > 0.f ? __builtin_nanf("") : o[0][b][r];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[0][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], e[r], o[0][b], 0, 0, 0);
                }
            }
            if constexpr (AHEAD) cur = nxt;
        }
        l[0] += __shfl_xor(l[0], 16);
        l[0] += __shfl_xor(l[0], 32);
        finish_piece<DP, 1, NW, true>(p, u, (char*)paged_lds, m, l, o);
    });
}

// Joins the partial results of the units that a cut of the line runs through:
// O = sum_u 2^(m_u - M) O_u / sum_u 2^(m_u - M) l_u. Grid: (cuts, rows), a Joint a cut.
// WAVES: (cuts, rows / 4), a row a wave where a unit has up to 64 parts, which needs
// neither barriers nor, for the cuts without a Joint, as many workgroups.
template <int DP, bool WAVES>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnParams p)
{
    constexpr uint32_t C4 = DP / 4, UG = 256 / C4, AHEAD = 8;     // lanes to a part's row; parts at a time; loads in flight
    constexpr uint32_t MAXP = PagedAttnParams::MAX_WGS;
    __shared__ float wgt[MAXP];
    __shared__ float4v part[256];
    __shared__ float red[8];
    const pg::Joint x = ((const pg::Joint*)p.ws_plan)[blockIdx.x + 1];
    if (x.parts == 0) return;
    const uint32_t t = threadIdx.x, c = t % C4, ug = t / C4;
    const auto at = [&](uint32_t i, uint32_t row) { return (size_t)(2 * (x.wg + i) + (i == 0 ? 1u : 0u)) * p.rb + row; };
    if (WAVES && x.parts <= 64) {
        // a row a wave: lane i makes part i's weight
        constexpr uint32_t WG = 64 / C4;
        const uint32_t lane = t & 63, wu = lane / C4;
        for (uint32_t row = 4 * blockIdx.y + (t >> 6); row < x.rows; row += 4 * gridDim.y) {
            float4v v[AHEAD];
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                v[i] = *(const float4v*)(p.ws_o + at(min(wu + i * WG, x.parts - 1), row) * DP + 4 * c);
            const float* ml = p.ws_ml + 2 * at(min(lane, x.parts - 1), row);
            const float m = lane < x.parts ? ml[0] : -__builtin_inff(), l = ml[1];
            float M = m;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
            const float w = lane < x.parts ? __builtin_amdgcn_exp2f(m - (M == -__builtin_inff() ? 0.f : M)) : 0.f;
            const float sum = wave_sum(lane < x.parts ? w * l : 0.f);
            float4v acc = (float4v)0.f;
            for (uint32_t u = 0; u < x.parts; u += AHEAD * WG) {
                if (u > 0) {
#pragma unroll
                    for (uint32_t i = 0; i < AHEAD; ++i)
                        v[i] = *(const float4v*)(p.ws_o + at(min(u + wu + i * WG, x.parts - 1), row) * DP + 4 * c);
                }
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    const uint32_t k = u + wu + i * WG;
                    const float wk = __shfl(w, k & 63);
                    if (k < x.parts) acc += wk * v[i];
                }
            }
#pragma unroll
            for (uint32_t o = C4; o < 64; o <<= 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
            if (lane < C4 && 4 * c < p.head_dim) pg::put_row(p, x.first, x.hk, x.row0 + row, 4 * c, acc, sum);
        }
        return;
    }
    for (uint32_t row = blockIdx.y; row < x.rows; row += gridDim.y) {
        // the first loads of values are in flight while the weights are made
        float4v v[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            v[i] = *(const float4v*)(p.ws_o + at(min(ug + i * UG, x.parts - 1), row) * DP + 4 * c);
        float m[MAXP / 256], l[MAXP / 256], M = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < MAXP / 256; ++i) {
            m[i] = -__builtin_inff();
            l[i] = 0.f;
            if (t + 256 * i < x.parts) {
                const float* ml = p.ws_ml + 2 * at(t + 256 * i, row);
                m[i] = ml[0];
                l[i] = ml[1];
            }
            M = fmaxf(M, m[i]);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
        if ((t & 63) == 0) red[t >> 6] = M;
        __syncthreads();
        M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float ref = M == -__builtin_inff() ? 0.f : M;
#pragma unroll
        for (uint32_t i = 0; i < MAXP / 256; ++i) {
            const float w = __builtin_amdgcn_exp2f(m[i] - ref);
            wgt[t + 256 * i] = w;
            sum += w * l[i];
        }
        sum = wave_sum(sum);
        if ((t & 63) == 0) red[4 + (t >> 6)] = sum;
        __syncthreads();
        float4v acc = (float4v)0.f;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            if (ug + i * UG < x.parts) acc += wgt[ug + i * UG] * v[i];
        for (uint32_t u = ug + AHEAD * UG; u < x.parts; u += AHEAD * UG) {
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                v[i] = *(const float4v*)(p.ws_o + at(min(u + i * UG, x.parts - 1), row) * DP + 4 * c);
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                if (u + i * UG < x.parts) acc += wgt[u + i * UG] * v[i];
        }
        part[t] = acc;
        __syncthreads();
        if (t < C4 && 4 * c < p.head_dim) {
#pragma unroll
            for (uint32_t i = 1; i < UG; ++i) acc += part[i * C4 + c];
            sum = (red[4] + red[5]) + (red[6] + red[7]);
            pg::put_row(p, x.first, x.hk, x.row0 + row, 4 * c, acc, sum);
        }
        __syncthreads();
    }
}

template <int DP>
static hipError_t merge_launch(const PagedAttnParams& p, hipStream_t s)
{
    // (a unit's rows, as far as the hint knows: more take turns)
    const uint32_t rows = (uint32_t)std::min<uint64_t>(p.rb, (uint64_t)p.max_new * (p.hq / p.hkv));
    // Rows a wave where there are rows and, on average, at most 32 parts to a unit: 7
    // sequences of 30 rows 17.9 us so (with the attention), 20.2 with a workgroup a row;
    // 64 of 12 rows 49, 52; but one of 16 over 60000 positions, 4 heads of 256, 65, 62.
    if (rows < 8 || (uint64_t)p.pages.sequences * p.hkv * 32 < p.wgs)
        hipLaunchKernelGGL((paged_merge_kernel<DP, false>), dim3(p.wgs - 1, rows), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((paged_merge_kernel<DP, true>), dim3(p.wgs - 1, (rows + 3) / 4), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t paged_merge_launch(const PagedAttnParams& p, hipStream_t s)
{
    if (p.wgs == 1) return hipSuccess;
    return p.dp == 64 ? merge_launch<64>(p, s) : p.dp == 128 ? merge_launch<128>(p, s) : merge_launch<256>(p, s);
}

bool paged_attention_plan(const PagedAttnParams& call, PagedAttnPlan& plan, uint32_t cus)
{
    PagedAttnParams& p = plan.few;
    p = call;
    p.dp = p.head_dim <= 64 ? 64 : p.head_dim <= 128 ? 128 : 256;
    const uint32_t group = p.hq / p.hkv;
    const uint64_t blocks = (uint64_t)p.tokens * group / 16 + std::min(p.tokens, p.pages.sequences);
    const uint64_t tiles = ((uint64_t)p.pages.max_pages * p.pages.page_size + pg::KT - 1) / pg::KT + 1;
    uint32_t resident = 2;
    p.rb = 16;
    p.min_share = 4;
    // the fp32 kernel's: fp32 pages, 64 sequences of up to 8192 positions, 8 heads of 128,
    // 64 and 50 (fp16) with 2, 4, 6, 10: 204, 185, 182, 185 us; 109, 96, 99, 102; 120, 106,
    // 100, 104; 4 heads of 256 257, 261, 279, 284
    p.lead = p.dp == 256 ? 2 : 5;
    p.few_rows = 0xffffffffu;
    p.decode = paged_decode_ok(p);
    if (p.decode) paged_decode_plan(p, &resident);
    const uint64_t unit = tiles + p.lead;
    p.wgs = (uint32_t)std::min<uint64_t>({(uint64_t)resident * cus, (blocks * p.hkv * unit + p.min_share - 1) / p.min_share,
                                          (uint64_t)PagedAttnParams::MAX_WGS});
    plan.many = p;
    plan.many.wgs = 0;
    if (p.decode && (uint64_t)p.max_new * group > few_most(p.dp)) {
        p.few_rows = plan.many.few_rows = few_most(p.dp);
        paged_prefill_plan(plan.many, cus);
        // One launch takes them all where the units of the sequences with few rows are not
        // many: it fills 4 of 128 rows then, but is bound by memory like the other, whose
        // launch and merge are saved. A chunk of 512 tokens beside 8, 32, 64, 128 (and of
        // half the length 256) single ones, 32 heads over 8 of 128: 136, 175, 223, 308, 238
        // us so, 146, 182, 221, 292, 230 apart. Beside 32, 64, 128: with an fp32 q 220, 280,
        // 386 and 220, 264, 339; 16 over 2 85, 97, 121 and 96, 112, 135; 16 over 4 of 256
        // 197, 271, 335 and 199, 239, 310.
        if ((uint64_t)p.pages.sequences * p.hkv <= plan.many.wgs) {
            plan.many.few_rows = 0;
            p.wgs = 0;
        }
    }
    // a line's length, and the shares' sum rounded up, stay below 2^32
    const uint64_t seqs = std::min(p.tokens, p.pages.sequences), rows = (uint64_t)p.tokens * group;
    const uint64_t most = 0xffffffffull - PagedAttnParams::MAX_WGS;
    const uint64_t few = std::min(rows / p.rb + seqs, seqs * ((p.few_rows + (uint64_t)p.rb - 1) / p.rb));
    if (p.wgs && few * p.hkv > most / unit) return false;
    return !plan.many.wgs || (rows / plan.many.rb + seqs) * p.hkv <= most / (tiles / 2 + 2 + plan.many.lead);
}

static size_t part_bytes(const PagedAttnParams& p)
{
    return p.wgs * (sizeof(pg::Joint) + (size_t)2 * p.rb * (p.dp + 2) * sizeof(float));
}

size_t paged_attention_workspace(const PagedAttnPlan& plan) { return part_bytes(plan.few) + part_bytes(plan.many); }

static void set_workspace(PagedAttnParams& p, char* ws)
{
    p.ws_plan = (uint32_t*)ws;
    p.ws_o = (float*)(ws + p.wgs * sizeof(pg::Joint));
    p.ws_ml = p.ws_o + (size_t)2 * p.wgs * p.rb * p.dp;
}

template <int DP, typename T, int W>
static hipError_t any_launch(const PagedAttnParams& p, hipStream_t s)
{
    constexpr int bytes = pg::finish_bytes<DP, 1, 4>();
    static PerDevice once;
    const hipError_t e = set_max_lds(once, (const void*)paged_attention_any_kernel<DP, T, W>, bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_attention_any_kernel<DP, T, W>), dim3(p.wgs), dim3(256), bytes, s, p);
    return hipGetLastError();
}

template <typename T, int W>
static hipError_t any_launch_d(const PagedAttnParams& p, hipStream_t s)
{
    return p.dp == 64 ? any_launch<64, T, W>(p, s) : p.dp == 128 ? any_launch<128, T, W>(p, s) : any_launch<256, T, W>(p, s);
}

hipError_t paged_attention_launch(PagedAttnPlan& plan, void* ws, hipStream_t s)
{
    set_workspace(plan.few, (char*)ws);
    set_workspace(plan.many, (char*)ws + part_bytes(plan.few));
    const PagedAttnParams& p = plan.few;
    const auto go = [&](auto t) {
        typedef decltype(t) T;
        return p.head_dim % 4 == 0 ? any_launch_d<T, 4>(p, s) : p.head_dim % 2 == 0 ? any_launch_d<T, 2>(p, s) : any_launch_d<T, 1>(p, s);
    };
    hipError_t e = plan.many.wgs ? paged_prefill_launch(plan.many, s) : hipSuccess;
    if (e != hipSuccess || p.wgs == 0) return e;
    e = p.decode ? paged_decode_launch(p, s) : p.pages.dtype == DT_F16 ? go(half_t{}) : go(float{});
    return e != hipSuccess ? e : paged_merge_launch(p, s);
}

}   // namespace vai_dev
