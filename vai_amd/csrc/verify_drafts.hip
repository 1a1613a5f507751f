// verify_drafts.hip -- drafted tokens against the target's probabilities.
//
//   p = softmax(target / T), q = softmax(draft / T); draft x is kept if u q(x) < p(x);
//   the first that is not is replaced by the lowest j whose running sum of
//   max(p - q, 0) exceeds u' times the whole sum; after the last, p's.
//
// Three passes, as which row is drawn from is known only when all are judged:
// every row's maximum and sum of powers, CH logits a workgroup; the judged row's
// max(p - q, 0) summed over the same parts; the part and place where the running
// sum passes. Sums and powers are fp64: the running sum passes a token of
// probability 1e-5 in steps that fp32 does not tell apart. The first pass is bound
// by reading the logits, the others by latency: loads that do not wait for the
// judgement are issued before it.
#include <algorithm>

#include "pages.h"

namespace vai_dev {

namespace {

constexpr uint32_t CH = 4096, NT = 256, PT = CH / NT;   // logits a workgroup, threads, logits a thread
constexpr uint32_t NO_TOKEN = 0xffffffffu;

// A part of a row: its largest logit (NaN: one that is NaN or +infinity is there),
// where that is first, and the sum of exp((x - largest) / T).
struct Stat {
    float top;
    uint32_t at;
    double sum;
};

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// e^y for y <= 0, within 2e-14 of it: 2^n e^r, n = y / ln 2 rounded and |r| <= ln 2 / 2
// (ln 2 in two parts, the first short enough that n times it is exact), e^r its power
// series up to r^11 (the next term is below 7e-15). Below -800, and where the logit
// is -infinity, nothing is left. Sixteen fp64 operations: 46 M logits take 19 us of
// them where they take 36 to read; the library's exp takes three times as many.
__device__ __forceinline__ double power(double y)
{
    y = fmax(y, -800.0);
    const double n = rint(y * 1.4426950408889634074);
    const double r = fma(-n, 0x1.9ef35793c7673p-41, fma(-n, 0x1.62e42fefa2p-1, y));
    double p = 1.0 / 39916800;
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// exp((x - top) / T)
__device__ __forceinline__ double power(float x, float top, double inv_t) { return power(((double)x - (double)top) * inv_t); }

// 8 logits of a row from j on, -infinity past its end
__device__ __forceinline__ void logits8(const void* rows, int dt, size_t row, uint32_t j, uint32_t vocab, float (&x)[8])
{
    if (j + 8 <= vocab) {
        if (dt == DT_F16) {
            typedef half8 half8u __attribute__((aligned(2)));
            const half8 v = *(const half8u*)((const half_t*)rows + row + j);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
        } else {
            const float4v a = load4f((const float*)rows + row + j), b = load4f((const float*)rows + row + j + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                x[4 + i] = b[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = j + i < vocab ? ld(rows, dt, row + j + i) : -__builtin_inff();
    }
}

__device__ __forceinline__ double wave_sum64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// the larger top (NaN above all), the lower place among equals
__device__ __forceinline__ void take_larger(float& top, uint32_t& at, float top2, uint32_t at2)
{
    const bool nan = top != top, nan2 = top2 != top2;
    if (nan2 ? !nan || at2 < at : !nan && (top2 > top || (top2 == top && at2 < at))) {
        top = top2;
        at = at2;
    }
}
__device__ __forceinline__ void wave_larger(float& top, uint32_t& at)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) take_larger(top, at, __shfl_xor(top, o), __shfl_xor(at, o));
}

__device__ __forceinline__ uint32_t parts_of(uint32_t vocab) { return (vocab + CH - 1) / CH; }
__device__ __forceinline__ Stat* stats_of(const VerifyParams& p, uint32_t which, uint32_t row)
{
    return (Stat*)p.workspace + ((size_t)which * p.rows + row) * parts_of(p.vocab);
}
__device__ __forceinline__ double* weights_of(const VerifyParams& p, uint32_t s)
{
    return (double*)((Stat*)p.workspace + (size_t)(p.draft ? 2 : 1) * p.rows * parts_of(p.vocab)) + (size_t)s * parts_of(p.vocab);
}
__device__ __forceinline__ float logit(const VerifyParams& p, uint32_t which, uint32_t row, uint32_t j)
{
    return which ? ld(p.draft, p.draft_dtype, (size_t)row * p.draft_stride + j)
                 : ld(p.target, p.target_dtype, (size_t)row * p.target_stride + j);
}
__device__ __forceinline__ float temperature_of(const VerifyParams& p, uint32_t s)
{
    const float t = p.temperature ? p.temperature[s] : 1.f;
    return t > 0.f ? t : 0.f;
}
__device__ __forceinline__ double inverse_of(float t) { return t > 0.f ? 1.0 / (double)t : 0.0; }

}   // namespace

// Grid: (parts x rows, target and draft).
__global__ __launch_bounds__(NT) void verify_rows_kernel(VerifyParams p)
{
    __shared__ float tops[4];
    __shared__ uint32_t ats[4];
    __shared__ double sums[4];
    const uint32_t parts = parts_of(p.vocab), row = blockIdx.x / parts, part = blockIdx.x - row * parts;
    const uint32_t which = blockIdx.y, t = threadIdx.x, j0 = part * CH + 8 * t;
    float x[PT / 8][8];
    const auto read = [&] {
#pragma unroll
        for (uint32_t k = 0; k < PT / 8; ++k)
            logits8(which ? p.draft : p.target, which ? p.draft_dtype : p.target_dtype,
                    (size_t)row * (which ? p.draft_stride : p.target_stride), j0 + k * NT * 8, p.vocab, x[k]);
    };
    if (!which) read();          // (a row of no sequence in vain: the loads do not wait for the search)
    const uint32_t s = wave_last_le(p.start, p.sequences, row);
    if (s == p.sequences || row >= p.start[s + 1]) return;
    if (which) {
        if (row + 1 >= min(p.start[s + 1], p.rows)) return;      // no draft follows
        read();
    }
    const float T = temperature_of(p, s);
    float top = neg_inf();
    bool odd = false;
#pragma unroll
    for (uint32_t k = 0; k < PT / 8; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = fmaxf(top, x[k][i]);
            odd = odd || !(x[k][i] < __builtin_inff());
        }
    if (odd) top = __builtin_inff();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((t & 63) == 0) tops[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0;
    uint32_t at = 0xffffffffu;
    if (top < __builtin_inff() && top > neg_inf()) {
        if (T > 0.f) {
            const double inv_t = inverse_of(T);
#pragma unroll
            for (uint32_t k = 0; k < PT / 8; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += power(x[k][i], top, inv_t);
            sum = wave_sum64(sum);
        } else {
            // the lowest index of the largest
#pragma unroll
            for (uint32_t k = 0; k < PT / 8; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (x[k][i] == top) at = min(at, j0 + k * NT * 8 + i);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
        }
    }
    if ((t & 63) == 0) {
        sums[t >> 6] = sum;
        ats[t >> 6] = at;
    }
    __syncthreads();
    if (t != 0) return;
    if (top == __builtin_inff()) top = __builtin_nanf("");
    stats_of(p, which, row)[part] = Stat{top, min(min(ats[0], ats[1]), min(ats[2], ats[3])), (sums[0] + sums[1]) + (sums[2] + sums[3])};
}

namespace {

// A whole row, from its parts' (a wave).
struct Row {
    float top;         // NaN or -infinity: no distribution
    uint32_t at;
    double sum;
};
__device__ __forceinline__ Row row_of(const VerifyParams& p, uint32_t which, uint32_t row, float T)
{
    const double inv_t = inverse_of(T);
    const Stat* st = stats_of(p, which, row);
    const uint32_t parts = parts_of(p.vocab), lane = threadIdx.x & 63;
    Row r{neg_inf(), 0xffffffffu, 0.0};
    const Stat mine = lane < parts ? st[lane] : Stat{neg_inf(), 0xffffffffu, 0.0};
    take_larger(r.top, r.at, mine.top, mine.at);
    for (uint32_t i = lane + 64; i < parts; i += 64) take_larger(r.top, r.at, st[i].top, st[i].at);
    wave_larger(r.top, r.at);
    if (T > 0.f && r.top > neg_inf()) {
        if (mine.top > neg_inf()) r.sum = mine.sum * power(mine.top, r.top, inv_t);
        for (uint32_t i = lane + 64; i < parts; i += 64)
            if (st[i].top > neg_inf()) r.sum += st[i].sum * power(st[i].top, r.top, inv_t);
        r.sum = wave_sum64(r.sum);
    }
    return r;
}

// What becomes of a sequence: the row it ends at, and what its last token is drawn from.
struct Verdict {
    uint32_t first, last, stop;    // rows
    uint32_t mode;                 // 0: w = p; 1: w = max(p - q, 0); 2: no distribution; 3: the largest logit
    float T;
    Row p, q;
    uint32_t x;                    // the draft that was not kept
};

// The judgement of row r (a wave): 0 kept, else what it ends with as 1 + mode
__device__ __forceinline__ uint32_t judge_row(const VerifyParams& p, uint32_t r, bool draft_follows, float T, Row& a, Row& b, uint32_t& x)
{
    const double inv_t = inverse_of(T);
    // (loads first)
    x = draft_follows ? p.tokens[r + 1] : NO_TOKEN;
    const bool in = x < p.vocab;
    const float lp = in ? logit(p, 0, r, x) : neg_inf(), lq = in && p.draft ? logit(p, 1, r, x) : neg_inf();
    const double u = (double)p.uniform[r];
    a = row_of(p, 0, r, T);
    b = Row{0.f, 0, 1.0};
    if (p.draft && draft_follows) b = row_of(p, 1, r, T);
    if (!(a.top > neg_inf()) || !(b.top > neg_inf())) return 3;
    if (!draft_follows) return T > 0.f ? 1 : 4;
    double px, qx;
    if (T > 0.f) {
        px = in ? power(lp, a.top, inv_t) / a.sum : 0.0;
        qx = !p.draft ? 1.0 : in ? power(lq, b.top, inv_t) / b.sum : 0.0;
    } else {
        px = x == a.at ? 1.0 : 0.0;
        qx = !p.draft || x == b.at ? 1.0 : 0.0;
    }
    if (u * qx < px) return 0;
    return T > 0.f ? 2 : 4;
}

// Judges a sequence, a row a wave; every thread of the workgroup gets the verdict.
template <uint32_t NW>
__device__ __forceinline__ Verdict judge(const VerifyParams& p, uint32_t s)
{
    __shared__ Verdict out;
    __shared__ uint32_t ends[NW];
    const uint32_t wave = threadIdx.x >> 6;
    Verdict v{};
    v.first = min(p.start[s], p.rows);
    v.last = min(p.start[s + 1], p.rows);
    v.T = temperature_of(p, s);
    if (v.last <= v.first) {
        v.stop = v.last = v.first;
        v.mode = 4;                // no rows
        return v;
    }
    v.last -= 1;
    for (uint32_t r0 = v.first;; r0 += NW) {
        const uint32_t r = r0 + wave;
        Row a, b;
        uint32_t x = NO_TOKEN;
        const uint32_t end = r <= v.last ? judge_row(p, r, r < v.last, v.T, a, b, x) : 0u;
        if ((threadIdx.x & 63) == 0) ends[wave] = end;
        __syncthreads();
        uint32_t w = 0;
        while (w < NW && ends[w] == 0) ++w;
        if (w < NW) {               // (the last row always ends)
            if (wave == w && (threadIdx.x & 63) == 0) {
                v.stop = r;
                v.mode = end - 1;
                v.p = a;
                v.q = b;
                v.x = x;
                out = v;
            }
            __syncthreads();
            return out;
        }
        __syncthreads();
    }
}

// w of 8 tokens from j on: max(p - q, 0) or p. (No fused multiply-add: p and q that
// are equal leave 0, not the rounding of one of them.)
__device__ __forceinline__ void weights8(const VerifyParams& p, const Verdict& v, bool rest, double inv_t, uint32_t j, double (&w)[8])
{
#pragma clang fp contract(off)
    float x[8], y[8];
    logits8(p.target, p.target_dtype, (size_t)v.stop * p.target_stride, j, p.vocab, x);
    if (rest && p.draft) logits8(p.draft, p.draft_dtype, (size_t)v.stop * p.draft_stride, j, p.vocab, y);
    const double a = 1.0 / v.p.sum, b = 1.0 / v.q.sum;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        w[i] = power(x[i], v.p.top, inv_t) * a;
        if (rest) w[i] = fmax(w[i] - (p.draft ? power(y[i], v.q.top, inv_t) * b : j + i == v.x ? 1.0 : 0.0), 0.0);
    }
}
__device__ __forceinline__ Verdict* verdict_of(const VerifyParams& p, uint32_t s)
{
    return (Verdict*)(weights_of(p, p.sequences)) + s;
}

}   // namespace

// Grid: (parts, sequences): the judged row's max(p - q, 0), summed over the part.
__global__ __launch_bounds__(512) void verify_weights_kernel(VerifyParams p)
{
    __shared__ double sums[8];
    const uint32_t part = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const Verdict v = judge<8>(p, s);
    if (part == 0 && t == 0) *verdict_of(p, s) = v;
    if (v.mode != 1) return;
    double w[8], sum = 0;
    weights8(p, v, true, inverse_of(v.T), part * CH + 8 * t, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += w[i];
    sum = wave_sum64(sum);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0)
        weights_of(p, s)[part] = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
}

namespace {

// The sum of the values of the threads before this one, and the whole sum.
__device__ __forceinline__ double before_me(double v, double& whole)
{
    __shared__ double sums[4];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double scan = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(scan, o);
        if (lane >= (uint32_t)o) scan += x;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    double at = scan - v;
    for (uint32_t w = 0; w < wave; ++w) at += sums[w];
    whole = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    return at;
}
__device__ __forceinline__ uint32_t smallest(uint32_t v)
{
    __shared__ uint32_t all[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = v;
    __syncthreads();
    return min(min(all[0], all[1]), min(all[2], all[3]));
}

}   // namespace

// One workgroup a sequence: the last token, and what is reported.
__global__ __launch_bounds__(NT) void verify_draw_kernel(VerifyParams p)
{
    const uint32_t s = blockIdx.x, t = threadIdx.x;
    const Verdict v = *verdict_of(p, s);
    if (v.mode == 4) {
        if (t == 0) {
            p.accepted[s] = 0;
            if (p.new_counts) p.new_counts[s] = p.counts[s];
        }
        return;
    }
    uint32_t token = v.mode == 3 ? v.p.at : NO_TOKEN;
    if (v.mode < 2) {
        const double inv_t = inverse_of(v.T), u = (double)p.uniform[v.last];
        const uint32_t parts = parts_of(p.vocab), per = (parts + NT - 1) / NT;
        const uint32_t i0 = min(t * per, parts), i1 = min(i0 + per, parts);
        bool rest = v.mode == 1;
        const auto part_sum = [&](uint32_t i) {
            if (rest) return weights_of(p, s)[i];
            const Stat st = stats_of(p, 0, v.stop)[i];
            return st.top > neg_inf() ? st.sum * power(st.top, v.p.top, inv_t) / v.p.sum : 0.0;
        };
        double own, whole, at;
        for (;;) {
            own = 0;
            for (uint32_t i = i0; i < i1; ++i) own += part_sum(i);
            at = before_me(own, whole);
            if (whole > 0 || !rest) break;
            rest = false;          // nothing is left: from p
        }
        // the part where the running sum passes u * whole, and what comes before it
        __shared__ double before;
        double run = at;
        uint32_t pass = 0xffffffffu, filled = 0xffffffffu;
        double start = 0, start_filled = 0;
        for (uint32_t i = i0; i < i1; ++i) {
            const double w = part_sum(i);
            if (w > 0) {
                filled = i;
                start_filled = run;
            }
            if (pass == 0xffffffffu && w > 0 && run + w > u * whole) {
                pass = i;
                start = run;
            }
            run += w;
        }
        uint32_t part = smallest(pass);
        if (part == 0xffffffffu) {   // (rounding: the last part that holds anything)
            part = ~smallest(filled == 0xffffffffu ? filled : ~filled);
            if (filled == part) before = start_filled;
        } else if (pass == part) {
            before = start;
        }
        __syncthreads();
        const double goal = u * whole - before;
        // the same inside the part: thread t has PT neighbouring logits
        const uint32_t j0 = part * CH + t * PT;
        double w[PT];
        own = 0;
#pragma unroll
        for (uint32_t k = 0; k < PT; k += 8) {
            double y[8];
            weights8(p, v, rest, inv_t, j0 + k, y);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                w[k + i] = y[i];
                own += y[i];
            }
        }
        run = before_me(own, whole);
        uint32_t found = 0xffffffffu, last = 0xffffffffu;
#pragma unroll
        for (uint32_t i = 0; i < PT; ++i) {
            run += w[i];
            if (w[i] > 0) last = j0 + i;
            if (found == 0xffffffffu && w[i] > 0 && run > goal) found = j0 + i;
        }
        token = smallest(found);
        if (token == 0xffffffffu) token = ~smallest(last == 0xffffffffu ? last : ~last);
    }
    const uint32_t kept = v.stop - v.first;
    for (uint32_t r = v.first + t; r <= v.last; r += NT)
        p.out_tokens[r] = r < v.stop ? p.tokens[r + 1] : r == v.stop ? token : NO_TOKEN;
    if (t == 0) {
        p.accepted[s] = kept;
        if (p.new_counts) p.new_counts[s] = p.counts[s] + kept + 1;
    }
}

size_t verify_workspace(const VerifyParams& p)
{
    const size_t parts = (p.vocab + CH - 1) / CH;
    return (size_t)(p.draft ? 2 : 1) * p.rows * parts * sizeof(Stat) + (size_t)p.sequences * (parts * sizeof(double) + sizeof(Verdict));
}

hipError_t verify_launch(const VerifyParams& p, hipStream_t s)
{
    const uint32_t parts = (p.vocab + CH - 1) / CH;
    hipLaunchKernelGGL(verify_rows_kernel, dim3(parts * p.rows, p.draft ? 2 : 1), dim3(NT), 0, s, p);
    hipLaunchKernelGGL(verify_weights_kernel, dim3(parts, p.sequences), dim3(512), 0, s, p);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(p.sequences), dim3(NT), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
