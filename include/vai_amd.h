/*
 * vai_amd.h -- C ABI of the MI355X (gfx950) kernels behind vAi's matmul hot path.
 *
 * Plain pointers and sizes only. Every buffer is device memory the caller owns
 * (hipMalloc'd, or any device-visible pointer); every launch is asynchronous on
 * the given stream and returns a vai_status (0 = success). Nothing throws
 * across this boundary. The library keeps no per-call state: besides its
 * kernels it holds only per-device launch settings made once (thread-safe),
 * and the scratch array of vai_linear_launch_noalloc.
 *
 * Callers: the C++ nodes in vai_amd/engine (Linear::run, Convolution::run,
 * AttentionScores::run, GatedMul::run), which replace the reference's
 * pipelinePool().request(...) + descriptor write + dispatch sequence.
 */
#ifndef VAI_AMD_H
#define VAI_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* vai_stream_t;   /* == hipStream_t */

/* Status codes. Values >= 1000 are the library's own argument checks; other
 * non-zero values are hipError_t codes passed through. */
typedef enum {
    VAI_OK = 0,
    VAI_ERR_INVALID_ARG = 1001,    /* null pointer, zero size, bad enum */
    VAI_ERR_SHAPE = 1002,          /* shapes that do not fit together */
    VAI_ERR_DTYPE = 1003,          /* a dtype combination the reference rejects */
    VAI_ERR_WORKSPACE = 1004,      /* workspace missing or too small */
    VAI_ERR_UNSUPPORTED = 1005,    /* valid, but not implemented here */
} vai_status;

/* Dtype codes: the reference's DTYPE_F32 / DTYPE_F16 / DTYPE_NONE
 * (/root/reference/vai/shaders/common/spec_constants.h:6-8). */
enum {
    VAI_DTYPE_F32 = 0,
    VAI_DTYPE_F16 = 1,
    VAI_DTYPE_NONE = 2,
    VAI_DTYPE_Q4 = 3,   /* a KV cache in 4 bits (vai_attention_args.cache_dtype only); not the reference's */
};

/* Epilogue codes in the order of vai::Epilogue
 * (/root/reference/vai/nodes/common.h:31-39). */
enum { VAI_EPI_NONE = 0, VAI_EPI_RELU, VAI_EPI_GELU, VAI_EPI_GELU_TANH, VAI_EPI_SILU, VAI_EPI_SIGMOID };

/* vai::ResidualOrder (/root/reference/vai/nodes/common.h:42-45). */
enum { VAI_RESIDUAL_AFTER_EPILOGUE = 0, VAI_RESIDUAL_BEFORE_EPILOGUE = 1 };

/* ---------------------------------------------------------------------------
 * Linear: O = s * epi(I . W^T + bias) + R        (residual_order AFTER)
 *         O = s * epi(I . W^T + bias + R)        (residual_order BEFORE)
 * I [M,K] (i_dtype), W [N,K] (w_dtype), O [M,N] (o_dtype), bias (b_dtype),
 * residual R (o_dtype). bias_repeat / residual_repeat: 0 when the operand
 * covers [M,N], else its element count, read modulo (a [N] row that repeats).
 * M <= 8 runs the HBM-streaming GEMV (fp32 math on the operands as stored,
 * the linear-slab contract); M > 8 runs the MFMA GEMM (fp16 staging unless I
 * and W are both fp32, then fp32 MFMA -- the linear-tile contract).
 * split_size > 0 forces split-K with K spans of that length (>= 32);
 * 0 lets the library choose. Split-K needs a workspace of
 * vai_linear_workspace_size() bytes.
 *
 * gated != 0 fuses the reference's GatedMul after this Linear
 * (/root/reference/vai/nodes/gated-mul.h:9-20): W holds [2H, K] rows (the
 * activated half first), O is [M, H] with
 *   O[m,j] = gate_epilogue(Y[m,j]) * Y[m,H+j],  Y = I . W^T + bias,
 * and epilogue must be NONE, scalar_scale 1, no residual.
 *
 * Replaces Linear::prepare/run's dispatches (/root/reference/vai/nodes/
 * linear.h:2291-2798): linear-slab, linear-tile / linear-cm, linear-reduce.
 * ------------------------------------------------------------------------- */
typedef struct {
    void* out;
    const void* in;
    const void* weight;
    const void* bias;        /* NULL: no bias (Linear::hasBias() false) */
    const void* residual;    /* NULL: no residual */
    void* workspace;         /* split-K partials; may be NULL when not needed */
    size_t workspace_bytes;
    uint32_t M, N, K;        /* N = outDim (= 2H when gated) */
    int32_t o_dtype, i_dtype, w_dtype, b_dtype;
    uint32_t epilogue;
    uint32_t residual_order;
    uint32_t bias_repeat;
    uint32_t residual_repeat;
    float scalar_scale;
    uint32_t split_size;
    uint32_t gated;
    uint32_t gate_epilogue;
    /* NULL, or vai_linear_pack_weight()'s output for this weight: fp16 I and W
     * with M >= 3 then read W from that fragment-major copy (256x256 tiles and 3-8
     * rows straight into the matrix cores' registers, the small tiles through
     * LDS; the other plans read W as stored). */
    const void* packed_weight;
    /* Accumulator dtype, Linear::setAccDtype (/root/reference/vai/nodes/
     * linear.h:289,2320): VAI_DTYPE_F32 (0, the default and the reference's
     * AMD default) or VAI_DTYPE_F16. F16 applies where the reference's tile
     * kernel honours it -- M > 8 with at least one fp16 operand -- and then
     * sums in fp16 in the order of linear-tile.comp:292-320 (4-wide k steps
     * from each split's start, k+3 first, every fma rounded to fp16), clamps
     * the sums to +-65504 and finishes in fp32. The GEMV (M <= 8) and fp32 x
     * fp32 products accumulate in fp32 whatever is asked, as the reference's
     * do. Split-K only when split_size asks for it. */
    int32_t acc_dtype;
} vai_linear_args;

vai_status vai_linear_launch(const vai_linear_args* args, vai_stream_t stream);
size_t vai_linear_workspace_size(const vai_linear_args* args);

/* vai_linear_launch for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * No counterpart in the reference. Same arguments, kernels and results as
 * vai_linear_launch, but args->workspace is ignored: the split-K partials and
 * the M <= 8 gated intermediate go to a device array inside the library
 * (VAI_NOALLOC_SCRATCH_BYTES = 64 MiB per GPU, held from the library's load until the
 * process ends). Returns VAI_ERR_WORKSPACE when the launch needs more than that
 * (vai_linear_workspace_size() tells in advance). Nothing is allocated. All
 * calls on one GPU share its array: calls that overlap in time on that GPU
 * (two streams, two threads) race on it and must be serialised by the caller. */
#define VAI_NOALLOC_SCRATCH_BYTES (64u << 20)
vai_status vai_linear_launch_noalloc(const vai_linear_args* args, vai_stream_t stream);

/* Size of, and the one-time fill of, the packed copy of args->weight that
 * packed_weight takes (0 / VAI_ERR_UNSUPPORTED when the shape or dtypes have
 * no packed path: fp16 I and W, K % 128 == 0, K >= 256). Depends on N, K,
 * the dtypes and `gated`, not on M. The weight-side counterpart of the
 * reference preparing a Linear's weights once at prepare time
 * (/root/reference/vai/nodes/linear.h:2291-2704). */
size_t vai_linear_packed_weight_size(const vai_linear_args* args);
vai_status vai_linear_pack_weight(const vai_linear_args* args, void* packed, size_t packed_bytes,
                                  vai_stream_t stream);

/* Which kernel vai_linear_launch picks for args (for tests and reports):
 * writes a short name ("slab", "slab_any", "tile_f16_128x128", ...). */
vai_status vai_linear_plan(const vai_linear_args* args, char* name, size_t name_len, uint32_t* split_count);

/* ---------------------------------------------------------------------------
 * Linear over 8-bit weights. No counterpart in the reference. Rows of X are
 * rounded to 8-bit integers in the call, each with a scale of its own, and
 * multiplied with the weight's integers:
 *   x_m = fp32(max_k |I[m,k]| / 127),  a[m,k] = round(I[m,k] / x_m)
 *   A[m,n] = x_m * w_scale[n] * sum_k a[m,k] W[n,k]
 *   O = s * epi(A + bias) + R          (residual_order AFTER)
 *   O = s * epi(A + bias + R)          (residual_order BEFORE)
 * round is to the nearest integer, halves to even, of the exact quotient; the
 * sums are 32-bit integers (exact), the rest fp32, rounded once to o_dtype.
 * I [M,K] fp32 or fp16; W [N] rows of 8-bit integers, each row starting K
 * rounded up to 16 bytes after the one before (what lies between does not
 * count) and the first 16-byte aligned; w_scale [N] fp32. A row of zeros
 * (or below fp32's normal range over 127) gives 0 for A, one that holds a NaN
 * or an infinity NaN. bias, residual, their repeats, epilogue and scalar_scale
 * as in vai_linear_args. K <= 131072.
 * The workspace (vai_linear_i8_workspace_size() bytes, 16-byte aligned; 0 for
 * one or a few short rows) holds the rounded rows of X; calls that overlap in
 * time need one each.
 * ------------------------------------------------------------------------- */
typedef struct {
    void* out;
    const void* in;
    const void* weight;
    const float* w_scale;
    const void* bias;        /* NULL: no bias */
    const void* residual;    /* NULL: no residual */
    void* workspace;
    size_t workspace_bytes;
    uint32_t M, N, K;
    int32_t o_dtype, i_dtype, b_dtype;
    uint32_t epilogue;
    uint32_t residual_order;
    uint32_t bias_repeat;
    uint32_t residual_repeat;
    float scalar_scale;
} vai_linear_i8_args;

vai_status vai_linear_i8_launch(const vai_linear_i8_args* args, vai_stream_t stream);
size_t vai_linear_i8_workspace_size(const vai_linear_i8_args* args);

/* Rounds `rows` rows of K values (fp32 or fp16) as above: out gets rows of K
 * rounded up to 16 bytes (zeros past K, 16-byte aligned), scale one fp32 each.
 * Of a weight [N,K] it makes W and w_scale. K <= 131072. A row with a NaN or
 * an infinity gets scale NaN. */
vai_status vai_quantize_i8_launch(void* out, float* scale, const void* in, int32_t i_dtype,
                                  uint32_t rows, uint32_t K, vai_stream_t stream);

/* GatedMul alone: O[r,j] = epi(I[r,j]) * I[r,H+j], I [rows, 2H].
 * Replaces gated-mul.comp (/root/reference/vai/nodes/gated-mul.h:75-114). */
vai_status vai_gated_mul_launch(void* out, int32_t o_dtype, const void* in, int32_t i_dtype,
                                uint32_t rows, uint32_t H, uint32_t epilogue, vai_stream_t stream);

/* ---------------------------------------------------------------------------
 * Convolution (implicit GEMM): same-padded odd kernel, NCHW.
 *   out[b,co,ho,wo] = epi(scale[co] * sum_{c,kh,kw} W[co,c,kh,kw] X[b,c,ho*s+kh-p,wo*s+kw-p]
 *                         + bias[co] (+R)) (+R),   p = kernel/2, Ho = (Hi-1)/s+1.
 * bias / scale carry w_dtype and may be NULL; residual carries i_dtype.
 * fp16 weights stage both operands as fp16 (fp16 MFMA); fp32 weights stage
 * fp32 (fp32 MFMA). fp16 input needs fp16 weights; fp16 output needs fp16
 * weights (Convolution::validateInputs, /root/reference/vai/nodes/
 * convolution.h:4137-4160). Replaces runK3S1Implicit / the implicit-GEMM
 * plan (/root/reference/vai/nodes/convolution.h:6237-6283, 6616-6644).
 * With fp16 weights the kernel reads them packed per tap in MFMA fragment
 * order (output channels padded to a multiple of 16, input channels to a
 * multiple of 32): pass a buffer that vai_conv2d_pack_weight()
 * filled once as packed_weight (the reference transforms conv weights once,
 * /root/reference/vai/nodes/convolution.h:6224-6235), or leave it NULL and
 * pass a workspace of vai_conv2d_workspace_size() bytes in which every call
 * packs them first.
 * ------------------------------------------------------------------------- */
typedef struct {
    void* out;
    const void* in;
    const void* weight;
    const void* bias;
    const void* scale;
    const void* residual;
    uint32_t batch, ci, hi, wi, co, kernel, stride;
    int32_t o_dtype, i_dtype, w_dtype;
    uint32_t epilogue;
    uint32_t residual_order;
    void* workspace;
    size_t workspace_bytes;
    const void* packed_weight;   /* NULL, or vai_conv2d_pack_weight()'s output */
} vai_conv2d_args;

vai_status vai_conv2d_launch(const vai_conv2d_args* args, vai_stream_t stream);
size_t vai_conv2d_workspace_size(const vai_conv2d_args* args);
/* Size of, and the one-time fill of, the packed weight for args (0 / no-op
 * when args take the fp32 path, which reads the weight as given). */
size_t vai_conv2d_packed_weight_size(const vai_conv2d_args* args);
vai_status vai_conv2d_pack_weight(const vai_conv2d_args* args, void* packed, size_t packed_bytes,
                                  vai_stream_t stream);

/* The reference's MAX_CAUSAL_BLOCKS (/root/reference/vai/shaders/common/
 * spec_constants.h:35). */
#define VAI_MAX_CAUSAL_BLOCKS 32

/* ---------------------------------------------------------------------------
 * Attention scores: S[b,h,i,j] = scale * sum_d Q[b,h,i,d] K[b,h/g,j,d],
 * g = Hq/Hkv, fp32 accumulation, S fp32. causal != 0 hides key j from query i
 * when j > i + (Tkv - Tq) (queries align with the keys' end); span > 0 also
 * hides j < i + Tkv - Tq + 1 - span. Hidden entries are -inf.
 * A block mask (mask_blocks > 0, causal must then be 0) replaces the causal
 * flag with the reference's list of blocks, each causal or fully visible
 * (writeCausalMask, /root/reference/vai/nodes/attention.h:40-55): bit
 * (mask_blocks - 1 - k) of mask_bits marks block k causal, mask_block_end
 * holds the ends (query rows, increasing) of every block but the last, which
 * ends at Tq. A query in a causal block sees keys up to itself, one in a full
 * block sees keys up to its block's end (common/causal_mask.h:25-38): a
 * prefix-LM mask is {2 blocks, bits 0b01, end {prefix}}.
 * Q [batch,Hq,Tq,D], K [batch,Hkv,Tkv,D], same dtype (f16 or f32).
 * The Q.K^T stage of the reference's attention kernels
 * (/root/reference/vai/shaders/attention.comp:155-182,
 *  attention-fa.comp:581-591, common/causal_mask.h:25-42).
 * ------------------------------------------------------------------------- */
typedef struct {
    float* scores;
    const void* q;
    const void* k;
    uint32_t batch, hq, hkv, tq, tkv, head_dim;
    int32_t dtype;
    float scale;
    uint32_t causal;
    uint32_t span;
    uint32_t mask_blocks;                                  /* 0: the causal flag alone */
    uint32_t mask_bits;
    uint32_t mask_block_end[VAI_MAX_CAUSAL_BLOCKS - 1];
} vai_attn_scores_args;

vai_status vai_attn_scores_launch(const vai_attn_scores_args* args, vai_stream_t stream);

/* ---------------------------------------------------------------------------
 * Attention: O[b,i,h,:] = sum_j softmax_j(scale * Q[b,h,i,:].K[b,h/g,j,:] +
 * mask) V[b,h/g,j,:], g = Hq/Hkv -- the reference's Attention node, with or
 * without its KV cache (/root/reference/vai/nodes/attention.h:77-140,
 * 216-245, 979-1304; shaders/attention-fa.comp, attention.comp,
 * attention-fa-reduce.comp).
 *   Q [batch,Hq,Tq,D] in q_dtype, K / V [batch,Hkv,Tkv,D] in kv_dtype (f32 or
 *   f16 each, as typeI / typeKV, attention.h:86-88); O token-major
 *   [batch,Tq,Hq,D] in o_dtype (attention-fa.comp:8,96 and attention.h:
 *   1220-1223), so that [batch,Tq,Hq*D] is a reshape.
 *   Queries and keys align at their ends (query i sits at key i + Tkv - Tq).
 *   The mask is vai_attn_scores_launch's: causal = 0 and mask_blocks = 0 is
 *   no mask at all, the reference's default when setCausalMask was never
 *   called (attention.h:129). A query with no visible key gives zeros.
 *   Any head dim 1..2048. D % 8 == 0 with 16 <= D <= 256 (the reference's
 *   flash-attention gate, attention.h:916-945) and 16-byte aligned operands
 *   take the MFMA flash kernel: fp32 softmax statistics and accumulation,
 *   Q.K^T and P.V on fp16 operands (fp32 Q is rounded to fp16 as the
 *   reference's f16-staged tiles do, fp32 K / V are rounded into workspace
 *   copies first, P enters P.V as fp16). Every other head dim takes a plain
 *   fp32 kernel (the reference's naive attention.comp role).
 *   Long key ranges may be split over workgroups and merged; fp32 K / V and
 *   the split need vai_attention_workspace_size() bytes of workspace.
 * ------------------------------------------------------------------------- */
typedef struct {
    void* out;
    const void* q;
    const void* k;
    const void* v;
    int32_t o_dtype;
    int32_t q_dtype;              /* VAI_DTYPE_F32 or VAI_DTYPE_F16 */
    int32_t kv_dtype;             /* VAI_DTYPE_F32 or VAI_DTYPE_F16, K and V alike */
    uint32_t batch, hq, hkv, tq, tkv, head_dim;
    float scale;                  /* 0: 1/sqrt(head_dim), as attention.h:1254 */
    uint32_t causal;
    uint32_t span;
    void* workspace;              /* vai_attention_workspace_size() bytes, or NULL when that is 0 */
    size_t workspace_bytes;
    uint32_t mask_blocks;                                  /* as vai_attn_scores_args */
    uint32_t mask_bits;
    uint32_t mask_block_end[VAI_MAX_CAUSAL_BLOCKS - 1];
    /* The KV cache (kvCacheSize / kvCacheDtype / kvCacheRing and the counter,
     * attention.h:108-140, 216-245, 1003-1023): cache_size = 0 turns it off.
     * With a cache (batch 1), k_cache / v_cache hold [Hkv, cache_size, D] in
     * cache_dtype, and cache_count points at a device-readable uint32: the
     * positions the cache held before this call, read by the kernels when
     * they run (the reference's kvCacheCount, which the model rewrites before
     * each forward, so a recorded graph follows it). The call appends its Tkv
     * new K / V rows at positions count .. count + Tkv - 1 (row p, or
     * p % cache_size for a ring, whose size must be a multiple of 64), then
     * attends positions [0, count + Tkv): query i sits at position count +
     * max(i + Tkv - Tq, 0) and sees up to count + (its mask end among the
     * new keys), attention-fa.comp:137-146,470-478. K / V may be NULL with
     * Tkv = 0: the call attends the cache alone. The caller keeps count + Tkv
     * <= cache_size without a ring, and advances the count itself.
     * cache_dtype VAI_DTYPE_Q4 keeps the cache in 4 bits (head_dim <= 256; no
     * counterpart in the reference): planes of vai_attention_cache_bytes()
     * bytes, 16-byte aligned, in a layout of the library's own. A row is
     * rounded to fp16 and cut into groups of 32 values (the last may be
     * shorter); a group keeps m = its minimum, s = fp16((max - m) / 15) and
     * codes n = round((x - m) / s) of 0 .. 15, and stands for s n + m (s the
     * fp16 number below where 15 s + m would leave fp16's range). Every
     * key and value is attended as stored, the call's own among them: what the
     * cache holds does not depend on how a sequence was cut into calls. Calls of
     * up to 128 query rows of a KV head (hq / hkv * tq; 256 with cache_size >=
     * 4096, and hq * tq <= 65535) attend the codes themselves, where only V is
     * rounded to fp16: an fp32 result is off by 2e-4 of its norm. Calls of more
     * rows go over copies of the cache whose K and V are rounded to fp16, with a
     * probability as one fp16 number, as an fp16 cache is attended: 4e-4, more
     * where channels of K stand out; the workspace holds two such planes of the
     * cache's size. Head dims that are no multiple of 8 go over fp32 copies, where
     * nothing is rounded. A group
     * with a value that is not finite in fp16 is stored as NaN; a query that
     * sees a row with such a group in K or V is NaN, one it is hidden from is
     * not touched by it. Positions past the count may hold anything. A 4-bit
     * ring is attended as far as it holds: span counts as at most cache_size -
     * Tkv + 1 (0 as that), and Tkv <= cache_size. */
    void* k_cache;
    void* v_cache;
    const uint32_t* cache_count;
    uint32_t cache_size;
    int32_t cache_dtype;          /* VAI_DTYPE_F32, VAI_DTYPE_F16 or VAI_DTYPE_Q4 */
    uint32_t cache_ring;
} vai_attention_args;

vai_status vai_attention_launch(const vai_attention_args* args, vai_stream_t stream);
/* Bytes of workspace a launch needs: nonzero when fp32 K / V take the flash
 * kernel (their fp16 copies; those of a 4-bit cache where a call takes them),
 * or when the query tiles alone do not fill the GPU and long key ranges are split over workgroups (partial results merged by
 * a second pass, the split-K of attention-fa-reduce.comp). */
size_t vai_attention_workspace_size(const vai_attention_args* args);

/* Bytes of one cache plane (k_cache and v_cache each): hkv * cache_size *
 * head_dim values in an fp32 or fp16 cache; a 4-bit one keeps rows of 64, 128
 * or 256 values (the next that holds head_dim) at 5 bits a value, positions
 * rounded up to 32. 0: no such cache. */
size_t vai_attention_cache_bytes(uint32_t hkv, uint32_t cache_size, uint32_t head_dim, int32_t cache_dtype);

/* Rows of a cache as the values they stand for: rows first_row .. first_row +
 * rows - 1 (past the plane's end they go on at row 0) of every head, as
 * [hkv, rows, head_dim] in o_dtype (fp32 or fp16). For a ring, row = position
 * % cache_size. */
typedef struct {
    void* k_out;
    void* v_out;
    const void* k_cache;
    const void* v_cache;
    int32_t o_dtype;
    int32_t cache_dtype;          /* VAI_DTYPE_F32, VAI_DTYPE_F16 or VAI_DTYPE_Q4 */
    uint32_t hkv, cache_size, head_dim;
    uint32_t first_row, rows;
} vai_attention_cache_read_args;

vai_status vai_attention_cache_read(const vai_attention_cache_read_args* args, vai_stream_t stream);

/* ---------------------------------------------------------------------------
 * From the fused query / key / value projection to the planes attention reads:
 * the RMS norm of each query and key head, the position rotation, and token-
 * major rows to head-major planes. No counterpart in the reference's hot path.
 *   qkv [batch,tokens] rows of row_stride elements (0: (hq + 2 hkv) head_dim),
 *   hq query heads, then hkv key heads, then hkv value heads, in i_dtype;
 *   q_out [batch,hq,tokens,head_dim], k_out and v_out [batch,hkv,tokens,
 *   head_dim] in o_dtype, disjoint from qkv. v_out NULL: values stay.
 * norm = 1: y = x / sqrt(mean x^2 + eps) * (w + weight_offset) over each head,
 * w = q_weight / k_weight [head_dim] in w_dtype; NULL: the factor is 1. norm =
 * 0: y = x. Values are only moved.
 * Rotation of the first rot_dim values (even; 0: head_dim) of a head at
 * position p: pair i, (a, e) = (y[i], y[i + rot_dim/2]) (HALVES) or (y[2i],
 * y[2i+1]) (NEIGHBOURS), becomes (a cos - e sin, e cos + a sin) of the angle
 * p * f_i, f_i = inv_freq[i] (fp32, device, rot_dim/2 of them; scaled bases) or,
 * NULL, theta^(-2i/rot_dim). Angles are taken in 64 bits, so far positions keep
 * theirs; the rest is fp32, rounded once to o_dtype.
 * p = positions[batch,tokens] (device uint32), or when NULL *count + token
 * (count: a device uint32 read when the kernel runs, the KV cache's counter;
 * NULL: 0). head_dim <= 2048.
 * ------------------------------------------------------------------------- */
enum { VAI_ROPE_NONE = 0, VAI_ROPE_HALVES = 1, VAI_ROPE_NEIGHBOURS = 2 };

typedef struct {
    void* q_out;
    void* k_out;
    void* v_out;
    const void* qkv;
    const void* q_weight;
    const void* k_weight;
    const uint32_t* positions;
    const uint32_t* count;
    const float* inv_freq;
    uint32_t batch, tokens, hq, hkv, head_dim;
    uint32_t row_stride;
    int32_t i_dtype, o_dtype, w_dtype;
    uint32_t norm;
    float eps, weight_offset;
    uint32_t rope;
    uint32_t rot_dim;
    float theta;
} vai_qk_norm_rope_args;

vai_status vai_qk_norm_rope_launch(const vai_qk_norm_rope_args* args, vai_stream_t stream);

/* ---------------------------------------------------------------------------
 * Many sequences in one forward, over a KV cache in pages. No counterpart in the
 * reference, whose cache holds one sequence.
 *
 * A batch is ragged: the new tokens of sequence s are rows seq_start[s] ..
 * seq_start[s + 1] - 1 of the token-major arrays (increasing; a sequence may
 * bring none). Rows before seq_start[0] or from seq_start[sequences] on are no
 * sequence's: what they hold is not read, and what outputs hold there stays.
 * Before the call sequence s held counts[s] positions; its new token t is at
 * position counts[s] + t.
 * Position p of sequence s lies in page page_table[s][p / page_size], slot p %
 * page_size. A page holds [hkv, page_size, head_dim] values; pages start
 * page_stride elements apart (0: packed; more lets K and V share an allocation).
 * Any page_size; whole 16s (and head dims of whole 8s, 16-byte aligned fp16
 * pages) take the fast kernels. Sequences may share pages that none of them
 * appends to. An entry that is no page (>= num_pages; unused entries hold what
 * they like), and positions past max_pages * page_size, hold nothing: rows
 * appended there are dropped, queries do not see them.
 * seq_start, counts and page_table are device uint32 arrays, read when the
 * kernels run: a recorded graph follows them. Neither call writes them.
 * sequences <= 4096, max_pages * page_size <= 2^30.
 * ------------------------------------------------------------------------- */
typedef struct {
    void* k_pages;
    void* v_pages;
    const uint32_t* page_table;   /* [sequences, max_pages] */
    const uint32_t* seq_start;    /* [sequences + 1] */
    const uint32_t* counts;       /* [sequences] */
    uint64_t page_stride;         /* elements from one page to the next; 0: hkv * page_size * head_dim */
    uint32_t sequences, num_pages, page_size, max_pages;
    int32_t page_dtype;           /* VAI_DTYPE_F32 or VAI_DTYPE_F16, K and V alike */
} vai_kv_pages;

/* From the fused query / key / value projection to the pages: the RMS norm of
 * each query and key head and the position rotation as in vai_qk_norm_rope_args
 * (norm, eps, weights, weight_offset, rope, rot_dim, theta, inv_freq), at the
 * tokens' positions; keys and values go to their pages, queries to q_out.
 *   qkv [tokens] rows of row_stride elements (0: (hq + 2 hkv) head_dim): hq query
 *   heads, then hkv key heads, then hkv value heads, in i_dtype; q_out [tokens,
 *   hq, head_dim] in o_dtype, disjoint from qkv, or NULL: queries stay.
 *   head_dim <= 2048. fp32 until each value's one rounding.
 * Two tokens of a call that land in one slot (a page twice in the table) leave
 * one of the two there. */
typedef struct {
    void* q_out;
    const void* qkv;
    const void* q_weight;
    const void* k_weight;
    const float* inv_freq;
    vai_kv_pages pages;
    uint32_t tokens, hq, hkv, head_dim;
    uint32_t row_stride;
    int32_t i_dtype, o_dtype, w_dtype;
    uint32_t norm;
    float eps, weight_offset;
    uint32_t rope;
    uint32_t rot_dim;
    float theta;
} vai_paged_append_args;

vai_status vai_paged_append_launch(const vai_paged_append_args* args, vai_stream_t stream);

/* Attention of a ragged batch over the pages, its own rows appended before:
 *   O[i,h,:] = sum_j softmax_j(scale * Q[i,h,:].K[j,h/g,:]) V[j,h/g,:], g = hq/hkv,
 * over positions 0 .. counts[s] + n_s - 1 of row i's sequence. causal hides the
 * positions after the query's own; span > 0 those up to its own - span. A query
 * that sees none (or only scores of -infinity) gives zeros.
 *   q [tokens] rows of q_stride elements (0: hq * head_dim) of hq heads in
 *   q_dtype; out [tokens, hq, head_dim] in o_dtype, disjoint from q. head_dim <=
 *   256.
 *   max_new: no sequence brings more tokens (0: tokens). It only chooses kernels
 *   and their workspace: sequences that bring more are attended too.
 *   Statistics and sums are fp32. Over fp16 pages an fp32 q and the probabilities
 *   enter the matrix cores as two fp16 numbers each. fp32 pages, head dims of no
 *   whole 8s and pages of no whole 16s are attended in fp32 throughout.
 *   A table so long that sequences * hkv * max_pages * page_size comes near 2^37, or
 *   tokens * hq * max_pages * page_size near 2^41 (2^45 for prompts on the fast
 *   kernels), is refused: VAI_ERR_UNSUPPORTED.
 *   What hidden positions hold does not matter. A value of V that is not finite
 *   makes its column so for the queries that see it; their other columns may be
 *   NaN too.
 * Calls that overlap in time need a workspace each (vai_paged_attention_
 * workspace_size() bytes, 16-byte aligned). The result does not depend on what
 * it held. */
typedef struct {
    void* out;
    const void* q;
    void* workspace;
    size_t workspace_bytes;
    vai_kv_pages pages;
    uint32_t tokens, max_new, hq, hkv, head_dim;
    uint32_t q_stride;
    int32_t o_dtype, q_dtype;
    float scale;                  /* 0: 1/sqrt(head_dim) */
    uint32_t causal;
    uint32_t span;
} vai_paged_attention_args;

vai_status vai_paged_attention_launch(const vai_paged_attention_args* args, vai_stream_t stream);
size_t vai_paged_attention_workspace_size(const vai_paged_attention_args* args);

/* ---------------------------------------------------------------------------
 * Drafted tokens against the target model's probabilities (speculative
 * sampling). No counterpart in the reference. Sequence s feeds rows seq_start[s]
 * .. seq_start[s + 1] - 1: its pending token, then its drafts; row r's logits
 * are those of the token after row r. For r from the sequence's first row on, with
 * x = tokens[r + 1], p_r = softmax(target[r] / T), q_r = softmax(draft[r] / T), or
 * 1 at x alone where draft is NULL:
 *   x is kept if uniform[r] * q_r(x) < p_r(x); the first that is not ends the
 *   sequence, and its place takes the lowest j with
 *     sum_{i <= j} w_i > uniform[last row] * sum_i w_i,  w = max(p_r - q_r, 0)
 *   (w = p_r if that is 0 everywhere); where all are kept, the token after the
 *   last row is drawn so with w = p of the last row.
 * T = temperature[s] (NULL: 1). T = 0, or any that is not above 0: p and q are 1 at
 * the lowest index of the largest logit. Everything is computed in 64 bits. Logits
 * of -infinity have no probability. A row that is needed and holds a NaN or
 * +infinity, or nothing above -infinity, ends its sequence with the token
 * VAI_NO_TOKEN.
 *   target, draft: [rows] rows of target_stride / draft_stride elements (0:
 *   vocab); draft's row of a sequence's last token is not read. tokens [rows]
 *   uint32, uniform [rows] fp32 in [0, 1); a token >= vocab has no probability.
 *   out_tokens [rows], another array than tokens: row seq_start[s] + i the token at
 *   place i, VAI_NO_TOKEN past the last; accepted [sequences]: drafts kept. new_counts (may be NULL, or
 *   counts itself): counts[s] + accepted + 1, the positions of the cache that
 *   hold. A sequence without rows: accepted 0, its count unchanged. The arrays are
 *   read when the kernels run. sequences <= 4096, rows and vocab < 2^24, and rows
 *   times the 4096s of vocab, rounded up, < 2^24.
 * The workspace (16-byte aligned) as for vai_paged_attention_launch.
 * ------------------------------------------------------------------------- */
#define VAI_NO_TOKEN 0xffffffffu

typedef struct {
    uint32_t* out_tokens;
    uint32_t* accepted;
    uint32_t* new_counts;
    const void* target;
    const void* draft;            /* NULL: drafts without probabilities of their own */
    const uint32_t* tokens;
    const float* uniform;
    const float* temperature;
    const uint32_t* seq_start;    /* [sequences + 1], as in vai_kv_pages */
    const uint32_t* counts;       /* [sequences]; needed with new_counts */
    void* workspace;
    size_t workspace_bytes;
    uint32_t sequences, rows, vocab;
    uint32_t target_stride, draft_stride;
    int32_t target_dtype, draft_dtype;
} vai_verify_drafts_args;

vai_status vai_verify_drafts_launch(const vai_verify_drafts_args* args, vai_stream_t stream);
size_t vai_verify_drafts_workspace_size(const vai_verify_drafts_args* args);

/* ---------------------------------------------------------------------------
 * Device memory and streams: what the host side (vai::Tensor's pooled
 * buffers, the reference's eva::Buffer role) and the tests use.
 * ------------------------------------------------------------------------- */
vai_status vai_device_count(int* count);
vai_status vai_set_device(int device);
vai_status vai_malloc(void** ptr, size_t bytes);
vai_status vai_free(void* ptr);
vai_status vai_memcpy_h2d(void* dst, const void* src, size_t bytes, vai_stream_t stream);
vai_status vai_memcpy_d2h(void* dst, const void* src, size_t bytes, vai_stream_t stream);
vai_status vai_memcpy_d2d(void* dst, const void* src, size_t bytes, vai_stream_t stream);
vai_status vai_memset(void* dst, int value, size_t bytes, vai_stream_t stream);
vai_status vai_stream_create(vai_stream_t* stream);
vai_status vai_stream_destroy(vai_stream_t stream);
vai_status vai_stream_sync(vai_stream_t stream);
vai_status vai_device_sync(void);
const char* vai_status_string(vai_status status);

/* Timing: launches fn-equivalent work is the caller's; these wrap hipEvents
 * recorded on the stream the kernels run on. */
typedef struct ihipEvent_t* vai_event_t;
vai_status vai_event_create(vai_event_t* ev);
vai_status vai_event_destroy(vai_event_t ev);
vai_status vai_event_record(vai_event_t ev, vai_stream_t stream);
vai_status vai_event_sync(vai_event_t ev);
vai_status vai_event_elapsed_ms(float* ms, vai_event_t start, vai_event_t stop);

/* Record once, replay: the launches a stream sees between begin and end are
 * captured into a HIP graph and replayed by vai_graph_launch. This is the
 * gfx950 form of NeuralNet's command buffer that is recorded once and
 * resubmitted while shapes stay the same (/root/reference/vai/engine/
 * neural-net.h:377-449). The stream must not be the null stream. */
typedef struct vai_graph_s* vai_graph_t;
vai_status vai_graph_begin_capture(vai_stream_t stream);
vai_status vai_graph_end_capture(vai_stream_t stream, vai_graph_t* graph);
vai_status vai_graph_launch(vai_graph_t graph, vai_stream_t stream);
vai_status vai_graph_destroy(vai_graph_t graph);

#ifdef __cplusplus
}
#endif
#endif /* VAI_AMD_H */
