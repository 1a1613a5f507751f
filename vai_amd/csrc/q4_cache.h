// q4_cache.h -- the KV cache in 4 bits: how a plane is laid out and how a
// group of values is rounded. Internal to the library (callers hold planes of
// vai_attention_cache_bytes() bytes and never look inside).
//
// A row of K or V (head_dim values, padded to dp = 64, 128 or 256) is cut into
// groups of 32 values. A group keeps its minimum m and its step s = (max - m) /
// 15 as fp16, and 4-bit codes n: the values stored are s n + m. Per KV head a
// plane is a run of tiles of 32 positions, each dp * 20 bytes: 16 dp of codes,
// then 4 dp of (s, m). Codes and steps of a tile lie together so that a walk
// over the keys reads one stream per plane, and inside a tile every lane of
// the decode kernel finds its share contiguous:
//   K: position j's row is dp / 8 words of 8 codes; the word of values 32 i +
//      8 q ..+7 is word q * (dp / 32) + i, so that quarter q's words of a row
//      are one load. A word's nibbles 0, 4, 1, 5, 2, 6, 3, 7 are its values in
//      order: masking alternate nibbles gives the pairs of an fp16 operand.
//      Then (s, m) of group i, position j: word 32 i + j.
//   V: 4 blocks of 8 positions, each 16 slices (dp / 16 values): byte (i, j) of
//      a slice, 8 i + j, holds values 2 i (low) and 2 i + 1 (high) of position
//      j: a word is 4 positions of the same two values, as the transposed
//      operand needs it. Then for group i and block b 8 steps and 8 minima,
//      positions in the order 0 2 1 3 4 6 5 7 (the operand's).
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
__host__ __device__ constexpr uint32_t k_word(uint32_t dp, uint32_t j, uint32_t d)
{
    return j * (dp / 2) + (((d >> 3) & 3) * (dp / 32) + (d >> 5)) * 4;
}
__host__ __device__ constexpr uint32_t k_scale(uint32_t dp, uint32_t j, uint32_t d)
{
    return scale_offset(dp) + ((d >> 5) * 32 + j) * 4;
}
__host__ __device__ constexpr uint32_t v_byte(uint32_t dp, uint32_t j, uint32_t d)
{
    return (j >> 3) * (dp * 4) + d / (dp / 16) * (dp / 4) + (d % (dp / 16) / 2) * 8 + (j & 7);
}
__host__ __device__ constexpr uint32_t v_scale(uint32_t dp, uint32_t j, uint32_t d)   // the step; the minimum 16 bytes on
{
    return scale_offset(dp) + ((d >> 5) * 4 + (j >> 3)) * 32 + order_of(j & 7) * 2;
}

// A group's step from its extremes. Both are fp16 values, so max - min is
// exact in fp32 but for the far ends of fp16's range. A group that holds
// something not finite in fp16 keeps m = NaN, s = 0: all its values are NaN.
__device__ __forceinline__ void step_of(float lo, float hi, bool finite, half_t& s, half_t& m)
{
    s = finite ? (half_t)((hi - lo) / 15.0f) : (half_t)0.f;
    // (s rounded up near fp16's end: one below, so that 15 s + m is an fp16 number too)
    if (fmaf(15.0f, (float)s, lo) > 65504.f) s = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, s) - 1));
    m = finite ? (half_t)lo : (half_t)__builtin_nanf("");
}

// (x - m) / s to the nearest integer, halves to even, from the exact remainder;
// s = 0 gives 0. x >= m, and s is rounded: the last code is 15 all the same.
__device__ __forceinline__ uint32_t code_of(float x, float m, float s)
{
    if (!(s > 0.f)) return 0;
    const float t = x - m;
    float n = rintf(t / s);
    const float r = 2.0f * fmaf(-n, s, t);
    const bool odd = (int)n & 1;
    if (r > s || (r == s && odd)) n += 1.f;
    else if (r < -s || (r == -s && odd)) n -= 1.f;
    return (uint32_t)fminf(n, 15.f);
}

}   // namespace q4
}   // namespace vai_dev
