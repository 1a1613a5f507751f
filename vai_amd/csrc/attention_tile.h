// attention_tile.h -- what the flash attention kernels share: 64-key tiles of K and
// V in LDS, read as matrix-core fragments.
#pragma once
#include <algorithm>

#include "device_common.h"

#define LDS_AS __attribute__((address_space(3)))

namespace vai_dev {

namespace fa {
constexpr int NW = 4, QW = 32, BQ = NW * QW, BKV = 64;
template <int D> struct Lds {
    static constexpr int ROWB = D * 2;                  // bytes per K or V row
    static constexpr int CH = D / 8;                    // 16-byte chunks per row
    static constexpr int TILE = BKV * ROWB;             // one operand, one tile
    static constexpr int STAGE = 2 * TILE;              // K then V
    static constexpr int BYTES = 2 * STAGE;             // double buffered
    static constexpr int COPIES = TILE / 1024 / NW;     // 1 KB copies per wave and operand
};
// Physical 16-byte chunk of logical chunk c in row r. LDS serves a 16-byte
// read for 16 lanes per pass from 64 banks (256 bytes), and K / V rows of
// D >= 128 are 256 or 512 bytes long, so every row starts at bank 0. With
// 16 or more chunks per row the low four chunk bits XOR h(r % 16) = f(r % 8)
// + (r & 8), f = 0 2 4 6 1 3 5 7: the 16 rows one K fragment read touches
// per pass (lanes 0-15: rows 0-15 at one logical chunk) land on 16 distinct
// chunks of a 256-byte window, and the four rows each 16-lane group of a
// transposed V^T read touches (two chunks each) on eight distinct chunks.
// Rows of D = 64 (128 bytes, 8 chunks) XOR f(r % 8) in the low three bits.
// The swizzle is its own inverse.
__host__ __device__ constexpr int swz_f(int r) { return 2 * (r & 3) + ((r >> 2) & 1); }
template <int D> __host__ __device__ constexpr int swz(int r, int c)
{
    return D >= 128 ? (c & ~15) | ((c & 15) ^ (swz_f(r & 7) | (r & 8))) : (c & ~7) | ((c & 7) ^ swz_f(r & 7));
}
}

// LDS fragment reads of the main loop, as inline asm. The compiler's wait
// insertion makes its ds_read_b64_tr_b16 builtin wait for every LDS DMA in
// flight (vmcnt(0)), which would hold each tile's V^T reads until the next
// tile's copies have landed, and with no registers to spare at D = 256 it
// sinks prefetched reads down to their MFMAs. The reads below are invisible
// to that pass: fa_lgkm_wait<N> (N = LDS operations issued since the reads
// needed) waits for them, and fa_pin ties each fragment to the wait so that
// its MFMA cannot be scheduled above it. LDS operations complete in order;
// the loop issues no scalar memory loads (which share the counter out of
// order). The compiler's own waits only count more operations than it knows
// of, which makes them stricter.
template <int OFF>
__device__ __forceinline__ half8 lds_read128(uint32_t addr)
{
    static_assert(OFF >= 0 && OFF < 65536, "ds offset range");
    half8 r;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
    return r;
}

// ds_read_b64_tr_b16 (gfx950): per 16-lane group, result lane j element k is
// element j % 4 of the 8 bytes that source lane 4 k + j / 4 points at.
template <int OFF>
__device__ __forceinline__ half4 lds_read_tr16(uint32_t addr)
{
    static_assert(OFF >= 0 && OFF < 65536, "ds offset range");
    half4 r;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
    return r;
}

// Maximum of three, as v_maximum3_f32 (fmaxf keeps a quieting v_max per operand
// that comes from a matrix core: 46 instructions for a tile's 32 scores instead
// of 16). A builtin and not inline asm: its operands are MFMA results, and only
// for an instruction that the compiler itself places does it insert the wait
// states between an MFMA and a vector read of its result. A NaN score gives a
// NaN maximum, which moves no reference below; the row is NaN through its
// exponential either way.
__device__ __forceinline__ float fa_max3(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

template <int N>
__device__ __forceinline__ void fa_lgkm_wait()
{
    static_assert(N >= 0 && N < 16, "lgkmcnt range");
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N));
}

__device__ __forceinline__ void fa_pin(half8& v) { asm volatile("" : "+v"(v)); }

// K fragment of S^T step IDX (key block IDX % 2, head-dim step S = IDX / 2):
// lane (ql, hf) reads key row 32 (IDX % 2) + ql, head-dim values 16 S + 8 hf
// .. +7, i.e. logical chunk c = 2 S + hf. D >= 128: the physical chunk is
// 16 (S / 8) + (((2 (S % 4) + hf) ^ f(ql % 8)) | (8 ((S / 4) % 2) ^ (ql & 8))),
// so the lane part is kaddr[S % 8] = stage + ql ROWB + that chunk without its
// first term, times 16, and the immediate adds 32 (IDX % 2) ROWB + 256 (S / 8).
// D = 64 (S < 4): kaddr[S] with the three-bit swizzle.
template <int D>
constexpr int fa_nk = D >= 128 ? 8 : 4;
template <int D, int IDX>
__device__ __forceinline__ half8 fa_kfrag(const uint32_t (&kaddr)[fa_nk<D>])
{
    constexpr int S = IDX >> 1;
    return lds_read128<32 * (IDX & 1) * fa::Lds<D>::ROWB + (S >> 3) * 256>(kaddr[S & (fa_nk<D> - 1)]);
}

// V^T fragment of key step KK, head-dim block DD: two transposed 8-byte reads
// of keys 16 KK + 8 part + lr (lr = vkey + vrow < 8), head-dim values 32 DD +
// vcol .. +3 (logical chunk c = 4 DD + vcol / 8). The row's swizzle is f(lr)
// plus 8 part, so the physical chunk is 16 (DD / 4) + ((4 (DD % 2) + vcol / 8)
// ^ f(lr)) + 8 ((DD / 2) % 2 ^ part) (D = 64: DD < 2, no bit 3). The lane part
// is vaddr[DD % 2] = stage + lr ROWB + ((4 (DD % 2) + vcol / 8) ^ f(lr)) 16 +
// (vcol % 8) 2; the immediate adds the V tile, (16 KK + 8 part) ROWB and the
// rest of the chunk.
template <int D, int KK, int DD, int PART>
constexpr int fa_voff()
{
    using L = fa::Lds<D>;
    return L::TILE + (16 * KK + 8 * PART) * L::ROWB + (DD >> 2) * 256 +
           (D >= 128 ? (((DD >> 1) & 1) ^ PART) * 128 : (DD >> 1) * 128);
}
template <int D, int KK, int DD>
__device__ __forceinline__ half8 fa_vfrag(const uint32_t (&vaddr)[2])
{
    const half4 h0 = lds_read_tr16<fa_voff<D, KK, DD, 0>()>(vaddr[DD & 1]);
    const half4 h1 = lds_read_tr16<fa_voff<D, KK, DD, 1>()>(vaddr[DD & 1]);
    return __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The dispatcher deals workgroups out to the 8 XCDs round-robin (linear
// workgroup w runs on XCD w % 8). Logical block of w: XCD x takes the
// contiguous range [x q + min(x, r), ..) of the n blocks (q = n / 8,
// r = n % 8), so that consecutive units -- one head's query tiles and key
// chunks, which read the same K, V and Q -- share one XCD's L2.
__host__ __device__ inline uint32_t fa_xcd_block(uint32_t w, uint32_t n)
{
    const uint32_t q = n / 8, r = n % 8, x = w % 8;
    return x * q + (x < r ? x : r) + w / 8;
}

// K / V tile copies into stage t % 2, through resources that start at the
// tile's first key row and end at the head's last: copy j of this wave fills
// tile bytes [(wave*COPIES + j) KB, +1 KB); rows past Tkv and the padding past
// the head dim read as zero (the range check, which sees the per-lane offset).
template <int D>
__device__ __forceinline__ void fa_issue(__amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv, LDS_AS char* lds,
                                         const uint32_t* coff, int t, int wave)
{
    using L = fa::Lds<D>;
    LDS_AS char* st = lds + (t & 1) * L::STAGE + wave * L::COPIES * 1024;
#pragma unroll
    for (int j = 0; j < L::COPIES; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (LDS_AS void*)(st + j * 1024), 16, (int)coff[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < L::COPIES; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (LDS_AS void*)(st + L::TILE + j * 1024), 16, (int)coff[j], 0, 0,
                                                 0);
}

template <int N>
__device__ __forceinline__ void fa_wait_vmcnt()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

}   // namespace vai_dev
