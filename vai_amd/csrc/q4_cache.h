// q4_cache.h -- the KV cache in 4 bits: how a plane is laid out and how a
// group of values is rounded. Internal to the library (callers hold planes of
// vai_attention_cache_bytes() bytes and never look inside).
//
// A row of K or V (head_dim values, padded to dp = 64, 128 or 256) is cut into
// groups of 32 values. A group keeps its minimum m and its step s = (max - m) /
// 15 as fp16, and 4-bit codes n: the values stored are s n + m. Per KV head a
// plane is a run of tiles of 32 positions, each dp * 20 bytes: 16 dp of codes,
// then 4 dp of (s, m). A tile is copied into LDS as it lies, and there every lane
// of the attention kernel finds its share contiguous:
//   K: lane (r, q) of the score product takes row r of 16 and quarter q, the
//      values 32 i + 8 q ..+7 of each group i: dp / 32 words of 8 codes. Half t
//      of a tile's positions, quarter and row lead: [t][q][r][i]. Row r of half
//      t is position 8 (r / 4) + 4 t + r % 4, so that the scores a lane receives,
//      rows 4 g ..+3 of both halves, are 8 positions in a row. A word's nibbles 0,
//      4, 1, 5, 2, 6, 3, 7 are its values in order: masking every fourth nibble
//      gives the pairs of an fp16 operand. Then the steps as [i][t][r], as the
//      lanes that hold the product's results take them, and the minima as
//      [t][r][i], an operand of their own.
//   V: 4 blocks of 8 positions, each 16 slices (dp / 16 values): byte (i, j) of
//      a slice, 8 i + j, holds values 2 i (low) and 2 i + 1 (high) of position
//      j: a word is 4 positions of the same two values, as the transposed
//      operand needs it. Then for group i and block b 8 steps and 8 minima,
//      positions in the order 0 2 1 3 4 6 5 7 (the operand's).
// Groups past the head dim hold zeros.
#pragma once
#include "device_common.h"

namespace vai_dev {
namespace q4 {

constexpr uint32_t KT = 32;   // positions of a tile

__host__ __device__ constexpr uint32_t tile_bytes(uint32_t dp) { return dp * 20; }
__host__ __device__ constexpr uint32_t scale_offset(uint32_t dp) { return dp * 16; }
__host__ __device__ inline size_t head_bytes(uint32_t rows, uint32_t dp)
{
    return (size_t)((rows + KT - 1) / KT) * tile_bytes(dp);
}
__host__ __device__ constexpr uint32_t nibble_of(uint32_t v) { return (v & 1) * 4 + (v >> 1); }   // of value v % 8
__host__ __device__ constexpr uint32_t order_of(uint32_t j) { return (j & 4) | ((j & 1) << 1) | ((j >> 1) & 1); }

// Byte offsets in a tile of position j (0 .. 31) and value d.
__host__ __device__ constexpr uint32_t half_of(uint32_t j) { return (j >> 2) & 1; }
__host__ __device__ constexpr uint32_t row_of(uint32_t j) { return (j >> 3) * 4 + (j & 3); }
__host__ __device__ constexpr uint32_t k_word(uint32_t dp, uint32_t j, uint32_t d)
{
    return (((half_of(j) * 4 + ((d >> 3) & 3)) * 16 + row_of(j)) * (dp / 32) + (d >> 5)) * 4;
}
__host__ __device__ constexpr uint32_t k_step(uint32_t dp, uint32_t j, uint32_t d)
{
    return scale_offset(dp) + (((d >> 5) * 2 + half_of(j)) * 16 + row_of(j)) * 2;
}
__host__ __device__ constexpr uint32_t k_min_offset(uint32_t dp) { return scale_offset(dp) + dp * 2; }
__host__ __device__ constexpr uint32_t k_min(uint32_t dp, uint32_t j, uint32_t d)
{
    return k_min_offset(dp) + ((half_of(j) * 16 + row_of(j)) * (dp / 32) + (d >> 5)) * 2;
}
__host__ __device__ constexpr uint32_t v_byte(uint32_t dp, uint32_t j, uint32_t d)
{
    return (j >> 3) * (dp * 4) + d / (dp / 16) * (dp / 4) + (d % (dp / 16) / 2) * 8 + (j & 7);
}
__host__ __device__ constexpr uint32_t v_scale(uint32_t dp, uint32_t j, uint32_t d)   // the step; the minimum 16 bytes on
{
    return scale_offset(dp) + ((d >> 5) * 4 + (j >> 3)) * 32 + order_of(j & 7) * 2;
}

// A group's step from its extremes: (max - min) / 15 rounded to fp16 once. The
// fp32 quotient rounded again is next to it; the remainder, exact in 64 bits,
// against half the distance to the neighbours says which fp16 number it is. A
// group that holds something not finite in fp16 keeps m = NaN, s = 0: all its
// values are NaN; one without values (past the head dim, lo > hi) zeros.
__device__ __forceinline__ void step_of(float lo, float hi, bool finite, half_t& s, half_t& m)
{
    const bool some = finite && lo <= hi;
    const double d = (double)hi - (double)lo;
    uint16_t b = __builtin_bit_cast(uint16_t, (half_t)((float)d / 15.0f));
    const auto value = [](uint16_t x) { return (double)(float)__builtin_bit_cast(half_t, x); };
    const double r = fma(-15.0, value(b), d);
    const double up = 7.5 * (value(b + 1) - value(b)), down = 7.5 * (value(b - 1) - value(b));   // (b = 0: down is NaN)
    if (r > up || (r == up && (b & 1))) ++b;
    else if (r < down || (r == down && (b & 1))) --b;
    // (s rounded up near fp16's end: one below, so that 15 s + m is an fp16 number too)
    if (fma(15.0, value(b), (double)lo) > 65504.0) --b;
    s = some ? __builtin_bit_cast(half_t, b) : (half_t)0.f;
    m = some ? (half_t)lo : finite ? (half_t)0.f : (half_t)__builtin_nanf("");
}

// (x - m) / s to the nearest integer, halves to even, from the exact remainder
// (inv: 1 / s or next to it: the first guess is at most one off); s = 0 gives 0.
// x >= m, and s is rounded: the last code is 15 all the same. x - m = t + te (te
// what fp32 leaves of it); where te is not 0, s and 2 (t - q s) are multiples of
// t's last place, so that their difference is exact too.
__device__ __forceinline__ uint32_t code_of(float x, float m, float s, float inv)
{
    const float t = x - m, z = t - x, te = (x - (t - z)) - (m + z);
    const float q = rintf(t * inv), r = 2.0f * fmaf(-q, s, t), e = -2.0f * te, above = r - s, below = r + s;
    const int n = (int)q;
    const bool odd = n & 1, up = above > e || (above == e && odd), down = below < e || (below == e && odd);
    const int c = n + (int)up - (int)down;
    return s > 0.f ? (uint32_t)(c < 15 ? c : 15) : 0u;
}

// What lane ^ 1, ^ 2, and the mirror image in 8 and in 16 lanes hold: with an
// associative operation after each, every lane gets its 2, 4, 8, 16 lanes' result.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float moved(float x) { return __builtin_bit_cast(float, moved<CTRL>(__builtin_bit_cast(uint32_t, x))); }
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, MIRROR8 = 0x141, MIRROR16 = 0x140;

template <class T>
__device__ __forceinline__ void store(uint8_t* p, T v) { *(T*)p = v; }
template <class T>
__device__ __forceinline__ void store(__attribute__((address_space(3))) uint8_t* p, T v) { *(__attribute__((address_space(3))) T*)p = v; }

// 8 values of a row, from value 8 c on (c: the lane's place, 4 neighbouring lanes
// hold a group), already rounded to fp16; those from `values` on do not exist.
// Its group's step and minimum, and the codes, value e in nibble e.
__device__ __forceinline__ uint32_t encode8(const half8 h, uint32_t values, half_t& s, half_t& m)
{
    float x[8], lo = __builtin_inff(), hi = -__builtin_inff();
    uint32_t top = 0;   // the largest |x| as bits: NaN and infinity above all
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = (float)h[e];
        if ((uint32_t)e < values) {
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
            const uint32_t b = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
            top = b > top ? b : top;
        }
    }
    const auto step = [&](float l, float u, uint32_t t) __attribute__((always_inline)) {
        lo = fminf(lo, l);
        hi = fmaxf(hi, u);
        top = t > top ? t : top;
    };
    step(moved<XOR1>(lo), moved<XOR1>(hi), moved<XOR1>(top));
    step(moved<XOR2>(lo), moved<XOR2>(hi), moved<XOR2>(top));
    const bool finite = top < 0x7f800000u;
    step_of(lo, hi, finite, s, m);
    const float fs = (float)s, fm = (float)m, inv = fs > 0.f ? __builtin_amdgcn_rcpf(fs) : 0.f;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (finite && (uint32_t)e < values) w |= code_of(x[e], fm, fs, inv) << (4 * e);
    return w;
}

// Writes the 8 values from 8 c on of position j into a tile.
template <class P>   // a byte pointer, global or LDS
__device__ __forceinline__ void put_k(P tile, uint32_t dp, uint32_t j, uint32_t c, uint32_t codes, half_t s, half_t m)
{
    uint32_t w = 0;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) w |= (codes >> (4 * e) & 15u) << (4 * nibble_of(e));
    store<uint32_t>(tile + k_word(dp, j, 8 * c), w);
    if ((c & 3) == 0) {
        store<uint16_t>(tile + k_step(dp, j, 8 * c), __builtin_bit_cast(uint16_t, s));
        store<uint16_t>(tile + k_min(dp, j, 8 * c), __builtin_bit_cast(uint16_t, m));
    }
}
template <class P>
__device__ __forceinline__ void put_v(P tile, uint32_t dp, uint32_t j, uint32_t c, uint32_t codes, half_t s, half_t m)
{
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) store<uint8_t>(tile + v_byte(dp, j, 8 * c + 2 * i), (uint8_t)(codes >> (8 * i)));
    if ((c & 3) == 0) {
        store<uint16_t>(tile + v_scale(dp, j, 8 * c), __builtin_bit_cast(uint16_t, s));
        store<uint16_t>(tile + v_scale(dp, j, 8 * c) + 16, __builtin_bit_cast(uint16_t, m));
    }
}

// 8 values of a new row from value d on, as fp16
__device__ __forceinline__ half8 row8(const void* rows, int dt, size_t row, uint32_t d, uint32_t HD)
{
    half8 h = (half8)(half_t)0;
    if (d + 8 <= HD) h = dt == DT_F16 ? load8((const half_t*)rows + row + d) : load8((const float*)rows + row + d);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (d + e < HD) h[e] = (half_t)ld(rows, dt, row + d + e);
    return h;
}

}   // namespace q4
}   // namespace vai_dev
