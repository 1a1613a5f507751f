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
#include <cmath>
#include <type_traits>

#include "pages.h"

namespace vai_dev {

namespace {

constexpr uint32_t CH = 4096;                           // logits a workgroup
constexpr uint32_t NT = 256, PT = CH / NT;              // threads of the first pass, logits a thread
constexpr uint32_t NO_TOKEN = 0xffffffffu;

// A part of a row: its largest logit (infinity: one that is NaN or +infinity is
// there), where that is first (T = 0), and the sum of exp((x - largest) / T).
struct Stat {
    float top;
    uint32_t at;
    double sum;
};

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// e^y for y <= 0, within 2e-14 of it: 2^n e^r, n = y / ln 2 rounded and |r| <= ln 2 / 2
// (ln 2 in two parts, the first short enough that n times it is exact), e^r its power
// series up to r^11 (the next term is below 7e-15). Below -800, and where the logit
// is -infinity, nothing is left.
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
// The same for the first pass, where every logit needs one: n = 32 y / ln 2 rounded,
// |r| <= ln 2 / 64, the power series up to r^5 (the next term is below 3e-15) and
// 2^(n % 32 / 32) from `table`, whose 32 entries lie in as many pairs of LDS banks. A
// third fewer operations: 46 M logits, 184 MB, take 45 us, with the long series 51.
__device__ __forceinline__ double power(double y, const double* table)
{
    y = fmax(y, -800.0);
    const double n = rint(y * 46.16624130844682904);
    const double r = fma(-n, 0x1.9ef35793c7673p-46, fma(-n, 0x1.62e42fefa2p-6, y));
    double p = 1.0 / 120;
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const int i = (int)n;
    return ldexp(p * table[i & 31], i >> 5);
}
// exp((x - top) / T)
__device__ __forceinline__ double power(float x, float top, double inv_t) { return power(((double)x - (double)top) * inv_t); }

// Which logits a thread of N takes as its 8: neighbouring ones of fp16, two times 4 of
// fp32, 16 bytes a lane and load
template <uint32_t N>
__device__ __forceinline__ uint32_t nth(int dt, uint32_t t, uint32_t i)
{
    return dt == DT_F16 ? 8 * t + i : (i >> 2) * (4 * N) + 4 * t + (i & 3);
}
template <uint32_t N>
__device__ __forceinline__ void logits8_apart(const void* rows, int dt, size_t row, uint32_t j, uint32_t t, uint32_t vocab, float (&x)[8])
{
    if (j + 8 * N <= vocab) {
        if (dt == DT_F16) {
            typedef half8 half8u __attribute__((aligned(2)));
            const half8 v = *(const half8u*)((const half_t*)rows + row + j + 8 * t);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
        } else {
            const float* at = (const float*)rows + row + j + 4 * t;
            const float4v a = load4f(at), b = load4f(at + 4 * N);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                x[4 + i] = b[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t k = j + nth<N>(dt, t, i);
            x[i] = k < vocab ? ld(rows, dt, row + k) : -__builtin_inff();
        }
    }
}

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

// op over the wave's lanes: within rows of 16 lanes by DPP, the four rows' by reading
// their first lanes. The order is fixed.
template <class T, class Op>
__device__ __forceinline__ T wave_reduce(T v, Op op)
{
    constexpr int N = sizeof(T) / 4;
    struct Words { int w[N]; };
    const auto moved = [](T x, auto ctrl) __attribute__((always_inline)) {
        Words a = __builtin_bit_cast(Words, x);
#pragma unroll
        for (int i = 0; i < N; ++i) a.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], decltype(ctrl)::value, 0xf, 0xf, true);
        return __builtin_bit_cast(T, a);
    };
    const auto lane = [](T x, int l) __attribute__((always_inline)) {
        Words a = __builtin_bit_cast(Words, x);
#pragma unroll
        for (int i = 0; i < N; ++i) a.w[i] = __builtin_amdgcn_readlane(a.w[i], l);
        return __builtin_bit_cast(T, a);
    };
    v = op(v, moved(v, std::integral_constant<int, 0xB1>{}));     // lane ^ 1
    v = op(v, moved(v, std::integral_constant<int, 0x4E>{}));     // lane ^ 2
    v = op(v, moved(v, std::integral_constant<int, 0x141>{}));    // the other 4 of 8 (mirrored)
    v = op(v, moved(v, std::integral_constant<int, 0x140>{}));    // the other 8 of 16
    return op(op(lane(v, 0), lane(v, 16)), op(lane(v, 32), lane(v, 48)));
}
__device__ __forceinline__ double wave_sum64(double v) { return wave_reduce(v, [](double a, double b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float v) { return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ uint32_t wave_min(uint32_t v) { return wave_reduce(v, [](uint32_t a, uint32_t b) { return min(a, b); }); }

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
    const uint32_t which = blockIdx.y, t = threadIdx.x;
    const int dt = which ? p.draft_dtype : p.target_dtype;
    __shared__ double table[32];
    if (t < 32) table[t] = p.powers[t];
    float x[PT / 8][8];
    const auto read = [&] {
#pragma unroll
        for (uint32_t k = 0; k < PT / 8; ++k)
            logits8_apart<NT>(which ? p.draft : p.target, dt, (size_t)row * (which ? p.draft_stride : p.target_stride),
                              part * CH + k * NT * 8, t, p.vocab, x[k]);
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
    top = wave_max(top);
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
                for (int i = 0; i < 8; ++i) sum += power(((double)x[k][i] - (double)top) * inv_t, table);
            sum = wave_sum64(sum);
        } else {
            // the lowest index of the largest
#pragma unroll
            for (uint32_t k = 0; k < PT / 8; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (x[k][i] == top) at = min(at, part * CH + k * NT * 8 + nth<NT>(dt, t, i));
            at = wave_min(at);
        }
    }
    if ((t & 63) == 0) {
        sums[t >> 6] = sum;
        ats[t >> 6] = at;
    }
    __syncthreads();
    if (t != 0) return;
    stats_of(p, which, row)[part] = Stat{top, min(min(ats[0], ats[1]), min(ats[2], ats[3])), (sums[0] + sums[1]) + (sums[2] + sums[3])};
}

namespace {

// A whole row, from its parts' (a wave).
struct Row {
    float top;         // infinite: no distribution
    uint32_t at;
    double sum;
    __device__ bool good() const { return top < __builtin_inff() && top > neg_inf(); }
};
__device__ __forceinline__ Row row_of(const VerifyParams& p, uint32_t which, uint32_t row, float T)
{
    const double inv_t = inverse_of(T);
    const Stat* st = stats_of(p, which, row);
    const uint32_t parts = parts_of(p.vocab), lane = threadIdx.x & 63;
    Row r{neg_inf(), 0xffffffffu, 0.0};
    const Stat mine = lane < parts ? st[lane] : Stat{neg_inf(), 0xffffffffu, 0.0};
    r.top = mine.top;
    for (uint32_t i = lane + 64; i < parts; i += 64) r.top = fmaxf(r.top, st[i].top);
    r.top = wave_max(r.top);
    if (!r.good()) return r;
    if (T > 0.f) {
        if (mine.top > neg_inf()) r.sum = mine.sum * power(mine.top, r.top, inv_t);
        for (uint32_t i = lane + 64; i < parts; i += 64)
            if (st[i].top > neg_inf()) r.sum += st[i].sum * power(st[i].top, r.top, inv_t);
        r.sum = wave_sum64(r.sum);
    } else {
        if (mine.top == r.top) r.at = mine.at;
        for (uint32_t i = lane + 64; i < parts; i += 64)
            if (st[i].top == r.top) r.at = min(r.at, st[i].at);
        r.at = wave_min(r.at);
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
    if (!a.good() || !b.good()) return 3;
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

// Grid: (shares of the parts, sequences): the judged row's max(p - q, 0), summed over
// each part. (Every workgroup judges for itself: with one a part, 32 sequences of 32
// parts, that took 22 us.)
__global__ __launch_bounds__(512) void verify_weights_kernel(VerifyParams p)
{
    __shared__ double sums[2][8];
    const uint32_t s = blockIdx.y, t = threadIdx.x, parts = parts_of(p.vocab);
    const Verdict v = judge<8>(p, s);
    if (blockIdx.x == 0 && t == 0) *verdict_of(p, s) = v;
    if (v.mode != 1) return;
    uint32_t turn = 0;
    for (uint32_t part = blockIdx.x; part < parts; part += gridDim.x, turn ^= 1) {
        double sum = 0;
#pragma unroll
        for (uint32_t k = 0; k < CH / 4096; ++k) {
            double w[8];
            weights8(p, v, true, inverse_of(v.T), part * CH + k * 4096 + 8 * t, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += w[i];
        }
        sum = wave_sum64(sum);
        double* all = sums[turn];    // (the other turn's may still be read)
        if ((t & 63) == 0) all[t >> 6] = sum;
        __syncthreads();
        if (t == 0) weights_of(p, s)[part] = ((all[0] + all[1]) + (all[2] + all[3])) + ((all[4] + all[5]) + (all[6] + all[7]));
    }
}

namespace {

constexpr uint32_t DT = 512;       // threads of the last pass, 8 logits each
static_assert(DT * 8 == CH);

// The sum of the values of the threads before this one, and the whole sum.
__device__ __forceinline__ double before_me(double v, double& whole)
{
    __shared__ double sums[DT / 64];
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
    whole = 0;
    for (uint32_t w = 0; w < DT / 64; ++w) {
        if (w < wave) at += sums[w];
        whole += sums[w];
    }
    return at;
}
__device__ __forceinline__ uint32_t smallest(uint32_t v)
{
    __shared__ uint32_t all[DT / 64];
    v = wave_min(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = v;
    __syncthreads();
    v = all[0];
    for (uint32_t w = 1; w < DT / 64; ++w) v = min(v, all[w]);
    return v;
}

}   // namespace

// One workgroup a sequence: the last token, and what is reported.
__global__ __launch_bounds__(DT) void verify_draw_kernel(VerifyParams p)
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
        const uint32_t parts = parts_of(p.vocab), per = (parts + DT - 1) / DT;
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
        // the same inside the part: thread t has 8 neighbouring logits
        const uint32_t j0 = part * CH + t * 8;
        double w[8];
        weights8(p, v, rest, inv_t, j0, w);
        own = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) own += w[i];
        run = before_me(own, whole);
        uint32_t found = 0xffffffffu, last = 0xffffffffu;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            run += w[i];
            if (w[i] > 0) last = j0 + i;
            if (found == 0xffffffffu && w[i] > 0 && run > goal) found = j0 + i;
        }
        token = smallest(found);
        if (token == 0xffffffffu) token = ~smallest(last == 0xffffffffu ? last : ~last);
    }
    const uint32_t kept = v.stop - v.first;
    for (uint32_t r = v.first + t; r <= v.last; r += DT)
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

hipError_t verify_launch(VerifyParams p, hipStream_t s)
{
    for (int i = 0; i < 32; ++i) p.powers[i] = std::exp2(i / 32.0);
    const uint32_t parts = (p.vocab + CH - 1) / CH;
    hipLaunchKernelGGL(verify_rows_kernel, dim3(parts * p.rows, p.draft ? 2 : 1), dim3(NT), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;      // (the others would judge by what the workspace held)
    const uint32_t shares = std::max(1u, std::min(parts, 512 / p.sequences));
    hipLaunchKernelGGL(verify_weights_kernel, dim3(shares, p.sequences), dim3(512), 0, s, p);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(p.sequences), dim3(DT), 0, s, p);
    return hipGetLastError();
}

}   // namespace vai_dev
