// paged_attention.hip -- attention of a ragged batch over a KV cache in pages:
// the fp32 kernel for any head dim, page size and dtype, the merge of partial
// results, and which kernel a call takes.
//
// The fp32 kernel: v_mfma_f32_16x16x4_f32 throughout, operands from memory to
// registers. S^T = K Q^T over 16 keys x 16 query rows: lane (c16, g) reads 4
// neighbouring values of key c16 at a time, which are its k's of four steps, and
// gets the scores of row c16 with keys 4 g ..+3. Those are, as they stand, the
// lane's P^T operands of O^T += V^T P^T when step r of it takes key 4 g + r. No
// value moves between lanes but for the row's maximum and sum.
#include "paged_plan.h"

#include "launch_once.h"

namespace vai_dev {

// Rows a KV head up to which a sequence is paged_decode.hip's, whose units of 32 (D =
// 256: 16) rows read the keys once each. 8 sequences of 4000 positions, 32 heads over
// 8 of 128, us there / in paged_prefill.hip: 32 rows 40 / 55, 48 rows 61 / 55, 64 rows
// 63 / 55, where one sequence of 16000 takes 28 / 52, 35 / 52, 35 / 53; of 64, 64 rows
// 40 / 30; of 256 (16 over 4), 32 rows 56 / 53, 64 rows 93 / 54.
static uint32_t few_most(uint32_t dp) { return dp == 128 ? 64 : 32; }

template <int DP, typename T>
__global__ __launch_bounds__(256) void paged_attention_any_kernel(PagedAttnParams p)
{
    using namespace pg;
    constexpr int KB = DP / 16, RB = 16, NW = 4;
    extern __shared__ float4v paged_lds[];
    __shared__ uint32_t pre[KvPages::MAX_SEQUENCES + 1];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c16 = lane & 15, g = lane >> 4, D = p.head_dim, group = p.hq / p.hkv;
    const KvPages& pgs = p.pages;
    const float sl2 = p.scale * 1.4426950408889634f;   // scores in log2 units
    plan_line<NW>(p, RB, pre);
    walk<RB>(p, pre, [&](const Piece& u) {
        const uint32_t rows = u.q.n * group, row = min(u.rb * RB + c16, rows - 1);
        const uint32_t tok = row / group, pos = u.q.held + tok;
        const uint32_t kbeg = first_key(p, pos), kend = p.causal ? min(pos + 1, u.q.live) : u.q.live;
        const size_t qat = (size_t)(u.q.first + tok) * p.q_stride + (size_t)(u.hk * group + row % group) * D;
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
        const uint32_t see = first_key(p, u.q.held);     // no row sees a position before it
        for (uint32_t t = u.t0 + wave; t < u.t1; t += NW)
            for (uint32_t j0 = t * KT; j0 < (t + 1) * KT; j0 += 16) {
                // the lane's key: where its K and V start, if it is there
                const uint32_t j = j0 + c16, i = j / pgs.page_size;
                int64_t at = -1;
                if (j >= see && j < u.q.live) {
                    const uint32_t page = pgs.table[(size_t)u.s * pgs.max_pages + i];
                    if (page < pgs.num_pages)
                        at = (int64_t)(page * pgs.stride + ((uint64_t)u.hk * pgs.page_size + (j - i * pgs.page_size)) * D);
                }
                if (!__any(at >= 0)) continue;
                float4v sa = (float4v)0.f;
                const T* k = (const T*)pgs.k + (at < 0 ? 0 : at);
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const uint32_t d = 16 * b + 4 * g;
                    const float4v x = some4<false>(k + d, at >= 0 && d < D ? min(4u, D - d) : 0u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sa = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[b][e], sa, 0, 0, 0);
                }
                // scores of the lane's row with keys 4 g + r
                float v[4], top = -__builtin_inff();
                int64_t vat[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t key = j0 + 4 * g + r;
                    vat[r] = __shfl(at, 4 * g + r);
                    const bool seen = key >= kbeg && key < kend && vat[r] >= 0;
                    v[r] = seen ? sa[r] * sl2 : -__builtin_inff();
                    top = fmaxf(top, v[r]);
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mnew = fmaxf(m[0], top), ref = mnew == -__builtin_inff() ? 0.f : mnew;
                const float alpha = __builtin_amdgcn_exp2f(m[0] - ref);
                m[0] = mnew;
                float e[4], sum = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[r] = __builtin_amdgcn_exp2f(v[r] - ref);
                    sum += e[r];
                }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                l[0] = l[0] * alpha + sum;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const uint32_t d = 16 * b + c16;
                    float x[4];
                    bool odd = false;       // a value that is not finite: 0 times it would reach rows that do not see it
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = vat[r] >= 0 && d < D ? (float)((const T*)pgs.v)[vat[r] + d] : 0.f;
                        odd = odd || !(__builtin_fabsf(x[r]) < __builtin_inff());
                    }
                    o[0][b] *= alpha;
                    if (__any(odd)) {
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
        finish_piece<DP, 1, NW>(p, u, (char*)paged_lds, m, l, o);
    });
}

// Joins the partial results of the units that a cut of the line runs through:
// O = sum_u 2^(m_u - M) O_u / sum_u 2^(m_u - M) l_u. Grid: (cuts, rows), a Joint a cut.
template <int DP>
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

hipError_t paged_merge_launch(const PagedAttnParams& p, hipStream_t s)
{
    if (p.wgs == 1) return hipSuccess;
    // (a unit's rows, as far as the hint knows: more take turns)
    const uint32_t rows = (uint32_t)std::min<uint64_t>(p.rb, (uint64_t)p.max_new * (p.hq / p.hkv));
    const dim3 grid(p.wgs - 1, rows);
    if (p.dp == 64) hipLaunchKernelGGL(paged_merge_kernel<64>, grid, dim3(256), 0, s, p);
    else if (p.dp == 128) hipLaunchKernelGGL(paged_merge_kernel<128>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(paged_merge_kernel<256>, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

bool paged_attention_plan(const PagedAttnParams& call, PagedAttnPlan& plan, uint32_t cus)
{
    PagedAttnParams& p = plan.few;
    p = call;
    p.dp = p.head_dim <= 64 ? 64 : p.head_dim <= 128 ? 128 : 256;
    const uint32_t group = p.hq / p.hkv;
    // the lines' lengths stay below 2^32
    const uint64_t blocks = (uint64_t)p.tokens * group / 16 + std::min(p.tokens, p.pages.sequences);
    const uint64_t tiles = ((uint64_t)p.pages.max_pages * p.pages.page_size + pg::KT - 1) / pg::KT + 1;
    uint32_t resident = 2;
    p.rb = 16;
    p.min_share = 4;
    p.lead = 2;
    p.few_rows = 0xffffffffu;
    p.decode = paged_decode_ok(p);
    if (p.decode) paged_decode_plan(p, &resident);
    const uint64_t unit = tiles + p.lead;
    if (blocks * p.hkv > 0xffffffffull / unit) return false;
    p.wgs = (uint32_t)std::min<uint64_t>({(uint64_t)resident * cus, (blocks * p.hkv * unit + p.min_share - 1) / p.min_share,
                                          (uint64_t)PagedAttnParams::MAX_WGS});
    plan.many = p;
    plan.many.wgs = 0;
    if (p.decode && (uint64_t)p.max_new * group > few_most(p.dp)) {
        p.few_rows = plan.many.few_rows = few_most(p.dp);
        paged_prefill_plan(plan.many, cus);
        // One launch takes them all where the units of the sequences with few rows are not
        // many: it fills 4 of 128 rows then, but is bound by memory like the other, whose
        // launch and merge are saved. A chunk of 512 tokens beside 8, 32, 64 and 128 single
        // ones, 8 KV heads: 112, 147, 195, 276 us so, 134, 161, 215, 274 apart.
        if ((uint64_t)p.pages.sequences * p.hkv <= plan.many.wgs * 3 / 2) {
            plan.many.few_rows = 0;
            p.wgs = 0;
        }
    }
    return true;
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

template <int DP, typename T>
static hipError_t any_launch(const PagedAttnParams& p, hipStream_t s)
{
    constexpr int bytes = pg::finish_bytes<DP, 1, 4>();
    static PerDevice once;
    const hipError_t e = set_max_lds(once, (const void*)paged_attention_any_kernel<DP, T>, bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_attention_any_kernel<DP, T>), dim3(p.wgs), dim3(256), bytes, s, p);
    return hipGetLastError();
}

hipError_t paged_attention_launch(PagedAttnPlan& plan, void* ws, hipStream_t s)
{
    set_workspace(plan.few, (char*)ws);
    set_workspace(plan.many, (char*)ws + part_bytes(plan.few));
    const PagedAttnParams& p = plan.few;
    const auto go = [&](auto t) {
        typedef decltype(t) T;
        return p.dp == 64 ? any_launch<64, T>(p, s) : p.dp == 128 ? any_launch<128, T>(p, s) : any_launch<256, T>(p, s);
    };
    hipError_t e = plan.many.wgs ? paged_prefill_launch(plan.many, s) : hipSuccess;
    if (e != hipSuccess || p.wgs == 0) return e;
    e = p.decode ? paged_decode_launch(p, s) : p.pages.dtype == DT_F16 ? go(half_t{}) : go(float{});
    return e != hipSuccess ? e : paged_merge_launch(p, s);
}

}   // namespace vai_dev
