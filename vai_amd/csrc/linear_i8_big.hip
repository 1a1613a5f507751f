// linear_i8_big.hip -- the 8-bit Linear where the matrix cores, not memory, are
// the bound: workgroup tiles of 64 F x 64 F (F = 4: 256 x 256, F = 2: 128 x 128)
// on v_mfma_i32_32x32x32_i8, both operands through LDS.
//
//  * 4 waves, each a quadrant of F x F fragments of 32x32 (F = 4: 256 integer
//    accumulators a lane). Larger quadrants read less LDS per product: at F = 4 a
//    128-byte stage of K is 2048 MFMA clocks of a SIMD against 1024 clocks of
//    LDS reads and 512 of copies into it.
//  * K advances in stages of 128 bytes through two LDS slots, copied straight
//    from global memory one stage ahead; one barrier a stage. Chunk c (16
//    bytes) of slab row r stands at chunk c ^ (r / 2 % 8), so that the 16 lanes
//    an LDS cycle serves hit 16 different bank groups.
//  * Persistent: a workgroup walks its tiles as one stream of stages, the next
//    tile's first copies in flight while a finished one is written out.
//  * The tile list is cut into 8 runs, one for each XCD (workgroup b runs on XCD
//    b % 8), and goes down groups of 8 row tiles column by column, so that an
//    L2 holds the rows of X and W its workgroups share.
//
// 2048 x 4096 x 16384 (fp16 in and out, F = 4): 160 us in the middle of a run, 1.7
// POP/s at the clock under load (the fastest launch 138), where a plain library
// product of the integers takes 131; 500 x 2048 x 2048 (F = 1): 7.7 us to fp16, 10.6
// with fp32 output and residual.
#include <algorithm>

#include "device_common.h"
#include "kernels.h"
#include "launch_once.h"

#define LDS_AS __attribute__((address_space(3)))

namespace vai_dev {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

namespace {

constexpr int BK = 128, CH = BK / 16;

template <int F> struct Cfg {
    static constexpr int STAGES = F == 1 ? 4 : 2;             // LDS slots: 128 KB at F = 4, else 64
    static constexpr int B = 64 * F;                          // tile rows and columns
    static constexpr int SLAB = B * BK;                       // bytes of one operand's stage
    static constexpr int STAGE = 2 * SLAB;
    static constexpr int LOADS = STAGE / 4096;                // 1 KB copies a wave makes for a stage
    static constexpr int LDS = STAGES * STAGE;
};

// The i-th tile of workgroup b: XCD x takes run x of the list.
struct TileWalk {
    uint32_t tiles_m, first, count, step;   // the workgroup's: list index first + i * step
    __device__ __forceinline__ TileWalk(uint32_t tm, uint32_t tn, uint32_t b, uint32_t grid)
    {
        tiles_m = tm;
        const uint32_t total = tm * tn, x = b % 8, q = total / 8, r = total % 8;
        const uint32_t run = x * q + std::min(x, r), len = q + (x < r ? 1u : 0u);
        // (fewer than 8 workgroups leave XCDs without one: a single run then)
        if (grid < 8) {
            step = grid;
            first = b;
            count = (total - b + grid - 1) / grid;
            return;
        }
        step = (grid - x + 7) / 8;          // workgroups on this XCD
        first = run + b / 8;
        count = b / 8 < len ? (len - b / 8 + step - 1) / step : 0u;
    }
    __device__ __forceinline__ void of(uint32_t i, uint32_t tn, uint32_t& m, uint32_t& n) const
    {
        const uint32_t l = first + i * step, g = l / (8 * tn), in = l - g * 8 * tn;
        const uint32_t rows = std::min(8u, tiles_m - 8 * g);
        n = in / rows;
        m = 8 * g + in - n * rows;
    }
};

template <int N>
__device__ __forceinline__ void wait_vm()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14)); }

template <uint32_t EPI>
__device__ __forceinline__ float activate(float x, uint32_t epi) { return epilogue(x, EPI == 6 ? epi : EPI); }

// A sum times the scales of its row and column, in the order in
// which nothing leaves fp32's range that the result does not: a sum (below 2^31)
// times a row's scale up to 2^64 cannot, and past that the column's comes first.
__device__ __forceinline__ float i8_scaled(int sum, float row, float col)
{
    const bool far = row > 0x1p64f;
    return (float)sum * (far ? col : row) * (far ? row : col);
}

// The accumulators are read through this so that the register allocator keeps
// them in accumulation registers across the tile loop (a plain use of an MFMA
// result lets it move them into ordinary ones and spill). The compiler does not
// see through it: the caller pads the distance from the last MFMA.
__device__ __forceinline__ int acc_read(int a)
{
    int v;
    asm("s_nop 0\n\tv_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
    return v;
}

// Two rows of one fp16 column, as two fp16 columns of one row: even lanes get
// (own, right neighbour) of the first row, odd lanes (left neighbour, own) of
// the second.
__device__ __forceinline__ uint32_t pair_columns(float r0, float r1, bool odd)
{
    typedef half_t half2v __attribute__((ext_vector_type(2)));
    const uint32_t own = __builtin_bit_cast(uint32_t, half2v{(half_t)r0, (half_t)r1});
    const uint32_t nb = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xf, 0xf, true);
    // bytes: own is 0..3 of the second operand, nb 4..7 of the first
    return __builtin_amdgcn_perm(nb, own, odd ? 0x03020706u : 0x05040100u);
}

}   // namespace

// Writes a tile from the accumulators. The products' scales and the bias of a
// lane's columns come in registers (loaded under the tile's K loop). Columns
// inside the output, a bias that is one row and no residual: buffer stores whose
// range ends with the output's last row; anything else goes element by element.
template <int F, uint32_t EPI, bool HALF>
__device__ __forceinline__ void i8_store_fast(const LinearI8Params& p, int16v (&acc)[F][F], const float (&ws)[F],
                                              const float (&cb)[F], uint32_t row0, uint32_t col0, int wm, int wn, int fr,
                                              int fk)
{
    constexpr int ES = HALF ? 2 : 4;
    const uint32_t rows = std::min<uint32_t>(p.M - row0, 64 * F), N = p.N;
    const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((char*)p.out + (size_t)row0 * N * ES), (short)0, (int)(rows * N * ES), 0x00020000);
    const bool odd = HALF && (fr & 1);
    const uint32_t lane_row = wm * 32 * F + 4 * fk, col = col0 + wn * 32 * F + fr;
    // (half: an even lane writes its own row's pair, an odd one the row below's, from the left column on)
    const uint32_t lane_off = ((lane_row + (odd ? 1 : 0)) * N + col - (odd ? 1 : 0)) * ES;
    const float sc = p.scalar_scale;
    static_for<F>([&](auto I) __attribute__((always_inline)) {
        constexpr int i = I;
        float4v xs[4];   // row scales: rows 8 q + 4 fk ..+3 of the fragment
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                xs[q][e] = p.x_scale[std::min(row0 + lane_row + 32 * i + 8 * q + e, p.M - 1)];
        static_for<F>([&](auto J) __attribute__((always_inline)) {
            constexpr int j = J;
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                v[r] = sc * activate<EPI>(i8_scaled(acc_read(acc[i][j][r]), xs[r >> 2][r & 3], ws[j]) + cb[j], p.epilogue);
            if constexpr (HALF) {
#pragma unroll
                for (int r = 0; r < 16; r += 2)
                    __builtin_amdgcn_raw_buffer_store_b32(pair_columns(v[r], v[r + 1], odd), out,
                        (int)(lane_off + (uint32_t)(32 * i + (r & 3) + 8 * (r >> 2)) * N * ES + 32 * j * ES), 0, 0);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v[r]), out,
                        (int)(lane_off + (uint32_t)(32 * i + (r & 3) + 8 * (r >> 2)) * N * ES + 32 * j * ES), 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);   // 16 outputs at a time: few live registers
        });
    });
}

// 16 operands of a fragment's outputs (a bias or a residual), rows of N values
// that repeat after `repeat` (0: never; N: one row)
__device__ __forceinline__ void rows16(const void* src, int dt, uint32_t repeat, uint32_t N, const uint32_t (&row)[16],
                                       uint32_t col, float (&x)[16])
{
    size_t o[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) o[r] = repeat == N ? col : (size_t)row[r] * N + col;
    if (repeat != 0 && repeat != N)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] %= repeat;
    if (dt == DT_F16)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = (float)((const half_t*)src)[o[r]];
    else
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = ((const float*)src)[o[r]];
}

template <int F>
__device__ __forceinline__ void i8_store_any(const LinearI8Params& p, int16v (&acc)[F][F], const float (&ws)[F],
                                             uint32_t row0, uint32_t col0, int wm, int wn, int fr, int fk)
{
    static_for<F>([&](auto I) __attribute__((always_inline)) {
        static_for<F>([&](auto J) __attribute__((always_inline)) {
            constexpr int i = I, j = J;
            const uint32_t col = col0 + wn * 32 * F + 32 * j + fr, lane_row = row0 + wm * 32 * F + 32 * i + 4 * fk;
            const uint32_t cc = std::min(col, p.N - 1);
            // (the loads of the 16 outputs in flight together)
            uint32_t rows[16];
            float xs[16], bias[16], res[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                rows[r] = std::min(lane_row + (r & 3) + 8 * (r >> 2), p.M - 1);
                xs[r] = p.x_scale[rows[r]];
                bias[r] = res[r] = 0.f;
            }
            if (p.bias) rows16(p.bias, p.b_dtype, p.bias_repeat, p.N, rows, cc, bias);
            if (p.residual) rows16(p.residual, p.o_dtype, p.residual_repeat, p.N, rows, cc, res);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                res[r] = finish(i8_scaled(acc_read(acc[i][j][r]), xs[r], ws[j]) + bias[r], res[r], p.epilogue,
                                p.residual_order, p.scalar_scale);
            if (col < p.N) {
                if (p.o_dtype == DT_F16) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (lane_row + (r & 3) + 8 * (r >> 2) < p.M) ((half_t*)p.out)[(size_t)rows[r] * p.N + col] = (half_t)res[r];
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (lane_row + (r & 3) + 8 * (r >> 2) < p.M) ((float*)p.out)[(size_t)rows[r] * p.N + col] = res[r];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    });
}

template <int F>
__global__ __launch_bounds__(256, F == 4 ? 1 : 2) void linear_i8_big_kernel(LinearI8Params p)
{
    typedef Cfg<F> C;
    constexpr int LOADS = C::LOADS, STAGES = C::STAGES, KS = BK / 32;
    extern __shared__ int4v i8_lds[];
    LDS_AS char* lds = (LDS_AS char*)(LDS_AS void*)i8_lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, fr = lane & 31, fk = lane >> 5;
    const uint32_t tiles_m = (p.M + C::B - 1) / C::B, tiles_n = (p.N + C::B - 1) / C::B;
    const TileWalk walk(tiles_m, tiles_n, blockIdx.x, gridDim.x);
    const int my_tiles = __builtin_amdgcn_readfirstlane((int)walk.count);
    if (my_tiles == 0) return;
    const int ktiles = (int)(p.x_stride / BK);

    // Copies: waves 0-1 fill X's slab of a stage, waves 2-3 W's; copy i of wave w
    // fills chunks [(w % 2 * LOADS + i) * 64, +64). Rows past an operand's last
    // read as zero (past the resource's range), and what W's rows hold past K
    // meets X's zeros.
    const bool is_w = wave >= 2;
    const uint32_t stride = is_w ? p.w_stride : p.x_stride;
    uint32_t voff[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int slot = ((wave & 1) * LOADS + i) * 64 + lane, row = slot / CH, ch = (slot % CH) ^ (row / 2 % CH);
        voff[i] = row * stride + ch * 16;
    }
    const auto tile_at = [&](int r, uint32_t& tm, uint32_t& tn) __attribute__((always_inline)) {
        walk.of((uint32_t)r, tiles_n, tm, tn);
        tm = __builtin_amdgcn_readfirstlane(tm);
        tn = __builtin_amdgcn_readfirstlane(tn);
    };
    // The stream's next stage to copy: its tile's resource and its place in K,
    // carried along (finding them anew costs three divisions a stage). Past the
    // last stage it copies the last again (never read), so that every wait counts
    // the same copies.
    int it = 0, ik = 0;
    __amdgpu_buffer_rsrc_t rsrc;
    const auto open_tile = [&]() __attribute__((always_inline)) {
        uint32_t tm, tn;
        tile_at(it, tm, tn);
        const uint32_t row0 = (is_w ? tn : tm) * C::B, rows = std::min<uint32_t>((is_w ? p.N : p.M) - row0, C::B);
        rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((is_w ? p.weight : p.x) + (size_t)row0 * stride), (short)0,
                                                 (int)(rows * stride), 0x00020000);
    };
    open_tile();
    const auto issue = [&](int g) __attribute__((always_inline)) {
        LDS_AS char* dst = lds + (g % STAGES) * C::STAGE + wave * LOADS * 1024;
        const int k = ik * BK;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LDS_AS void*)(dst + i * 1024), 16, (int)(voff[i] + (uint32_t)k),
                                                     0, 0, 0);
        if (++ik == ktiles) {
            ik = ktiles - 1;
            if (it + 1 < my_tiles) {
                ++it;
                ik = 0;
                open_tile();
            }
        }
    };
    // A wave's fragment rows are fr + 32 i: all with the same chunk swizzle.
    const int swz = fr / 2 % CH;
    const auto read_frags = [&](int g, int ks, int4v* a, int4v* b) __attribute__((always_inline)) {
        const int ch = (ks * 2 + fk) ^ swz;
        LDS_AS const char* pa = lds + (g % STAGES) * C::STAGE + ((wm * 32 * F + fr) * CH + ch) * 16;
        LDS_AS const char* pb = lds + (g % STAGES) * C::STAGE + C::SLAB + ((wn * 32 * F + fr) * CH + ch) * 16;
#pragma unroll
        for (int i = 0; i < F; ++i) a[i] = *(LDS_AS const int4v*)(pa + i * 32 * BK);
#pragma unroll
        for (int j = 0; j < F; ++j) b[j] = *(LDS_AS const int4v*)(pb + j * 32 * BK);
    };

    // F = 4 copies stages two ahead and keeps the next substep's fragments in
    // flight; the smaller tiles read a stage's fragments at once behind its barrier
    // and leave the overlap to the CU's other workgroup.
    constexpr bool AHEAD = F == 4;
    int4v fa[2][F], fb[2][F];
#pragma unroll
    for (int st = 0; st < STAGES - (AHEAD ? 0 : 1); ++st) issue(st);
    if constexpr (AHEAD) {
        wait_vm<(STAGES - 1) * LOADS>();
        __builtin_amdgcn_s_barrier();
        read_frags(0, 0, fa[0], fb[0]);
    }

    int g = 0;
    for (int r = 0; r < my_tiles; ++r) {
        uint32_t tm, tn;
        tile_at(r, tm, tn);
        const uint32_t row0 = tm * C::B, col0 = tn * C::B;
        float ws[F], cb[F];
        const bool row_bias = p.bias && p.bias_repeat == p.N;
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const uint32_t col = std::min(col0 + wn * 32 * F + 32 * j + fr, p.N - 1);
            ws[j] = p.w_scale[col];
            cb[j] = row_bias ? ld(p.bias, p.b_dtype, col) : 0.f;
        }
        int16v acc[F][F];
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = (int16v)0;
        // half of a substep's products (F = 1: all of them first)
        const auto mfma_half = [&](const int4v* a, const int4v* b, int h) __attribute__((always_inline)) {
#pragma unroll
            for (int i = (h * F + 1) / 2; i < ((h + 1) * F + 1) / 2; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        };
        if constexpr (!AHEAD) {
            for (int kt = 0; kt < ktiles; ++kt, ++g) {
                wait_lds();                              // this wave's reads of stage g - 1 are done
                wait_vm<(STAGES - 2) * LOADS>();         // its copies of stage g have landed
                __builtin_amdgcn_s_barrier();
                issue(g + STAGES - 1);                   // into the slot of stage g - 1
                int4v a[KS][F], b[KS][F];
#pragma unroll
                for (int q = 0; q < KS; ++q) read_frags(g, q, a[q], b[q]);
                // (all reads first: left to itself the compiler waits for each pair in turn)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = 0; q < KS; ++q) {
                    mfma_half(a[q], b[q], 0);
                    mfma_half(a[q], b[q], 1);
                }
            }
        } else
        for (int kt = 0; kt < ktiles; ++kt, ++g) {
            static_for<KS>([&](auto Q) __attribute__((always_inline)) {
                constexpr int q = Q, cur = q & 1, nxt = cur ^ 1;
                if constexpr (q + 1 < KS) {
                    read_frags(g, q + 1, fa[nxt], fb[nxt]);
                    mfma_half(fa[cur], fb[cur], 0);
                    mfma_half(fa[cur], fb[cur], 1);
#pragma unroll
                    for (int u = 0; u < 2 * F; ++u) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // 1 MFMA
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // 1 LDS read
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, F * F, 0);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    // the last substep: half of it covers the barrier, after which this
                    // slot is free for stage g + 2 and stage g + 1 is read
                    mfma_half(fa[cur], fb[cur], 0);
                    __builtin_amdgcn_sched_barrier(0);
                    wait_lds();
                    wait_vm<(STAGES - 2) * LOADS>();
                    __builtin_amdgcn_s_barrier();
                    issue(g + STAGES);
                    read_frags(g + 1, 0, fa[nxt], fb[nxt]);
                    mfma_half(fa[cur], fb[cur], 1);
#pragma unroll
                    for (int u = 0; u < 2 * F; ++u) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
                        __builtin_amdgcn_sched_group_barrier(0x020, LOADS / (2 * F), 1);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
        }
        __builtin_amdgcn_sched_barrier(0);
        // every accumulator passes through an empty asm, so that no MFMA moves past
        // this point; the s_nops are the last one's result-to-read distance
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) asm volatile("" : "+a"(acc[i][j]));
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
        const bool half_out = p.o_dtype == DT_F16;
        if (col0 + C::B <= p.N && !p.residual && (!p.bias || row_bias) && (size_t)C::B * p.N * 4 < (1u << 31) &&
            (!half_out || (p.N % 2 == 0 && (uintptr_t)p.out % 4 == 0))) {
            if (half_out) {
                if (p.epilogue == 0) i8_store_fast<F, 0, true>(p, acc, ws, cb, row0, col0, wm, wn, fr, fk);
                else i8_store_fast<F, 6, true>(p, acc, ws, cb, row0, col0, wm, wn, fr, fk);
            } else {
                if (p.epilogue == 0) i8_store_fast<F, 0, false>(p, acc, ws, cb, row0, col0, wm, wn, fr, fk);
                else i8_store_fast<F, 6, false>(p, acc, ws, cb, row0, col0, wm, wn, fr, fk);
            }
        } else {
            i8_store_any<F>(p, acc, ws, row0, col0, wm, wn, fr, fk);
        }
    }
    wait_vm<0>();   // the copies past the last stage land before the workgroup retires
}

template <int F>
static hipError_t big_launch(const LinearI8Params& p, hipStream_t s)
{
    const uint32_t tiles = ((p.M + 64 * F - 1) / (64 * F)) * ((p.N + 64 * F - 1) / (64 * F));
    static PerDevice once;
    hipError_t e = set_max_lds(once, (const void*)linear_i8_big_kernel<F>, Cfg<F>::LDS);
    if (e != hipSuccess) return e;
    int cus = 0;
    if ((e = device_cus(&cus)) != hipSuccess) return e;
    const uint32_t grid = std::min<uint32_t>(tiles, (uint32_t)cus * (F == 4 ? 1 : 2));
    hipLaunchKernelGGL(linear_i8_big_kernel<F>, dim3(grid), dim3(256), Cfg<F>::LDS, s, p);
    return hipGetLastError();
}

hipError_t linear_i8_big_launch(const LinearI8Params& p, int f, hipStream_t s)
{
    return f == 4 ? big_launch<4>(p, s) : f == 2 ? big_launch<2>(p, s) : big_launch<1>(p, s);
}

}   // namespace vai_dev
