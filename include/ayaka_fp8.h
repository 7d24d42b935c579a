/*
 * ayaka_fp8.h -- C ABI of the MI355X (gfx950) FP8 linear library `libayaka_fp8.so`.
 *
 * One entry point per `torch.ops.ayaka.*` operator of the reference's FP8 linear
 * path. Every pointer is a raw device pointer (HIP memory on the current device),
 * every size an int64, every element type a value of `ayk_dtype`, and every call is
 * enqueued on the given stream without host synchronisation. No entry point
 * allocates device memory: the split-K GEMVs take a caller-provided workspace whose
 * size is returned by the matching `*_workspace_bytes` query.
 *
 * Return value: AYK_OK (0), or a nonzero `ayk_status` with a message retrievable by
 * `ayk_last_error()` (thread-local, valid until the next failing call on the thread).
 *
 * Layout conventions (all row-major, innermost stride 1):
 *   activations a / x : [M, K], row stride lda/ldx elements
 *   weights w / b     : [N, K] e4m3 bytes, row stride ldw/ldb bytes
 *   outputs out       : [M, N], row stride ldo elements
 */
#ifndef AYAKA_FP8_H
#define AYAKA_FP8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Opaque stream handle: a hipStream_t (0 = the legacy default stream). */
typedef void* ayk_stream_t;

typedef enum ayk_dtype {
  AYK_F32 = 0,
  AYK_F16 = 1,
  AYK_BF16 = 2,
  AYK_E4M3 = 3, /* OCP float8 e4m3fn */
  AYK_U8 = 4,   /* raw bytes; as a scale: UE8M0 exponent codes */
  AYK_E5M2 = 5  /* OCP float8 e5m2 (KV caches) */
} ayk_dtype;

typedef enum ayk_status {
  AYK_OK = 0,
  AYK_EINVAL = 1,     /* bad argument: shape, stride, dtype or alignment */
  AYK_EARCH = 2,      /* the current device is not gfx950 */
  AYK_ELAUNCH = 3,    /* the HIP launch failed */
  AYK_EWORKSPACE = 4  /* workspace missing or too small */
} ayk_status;

/* Message of the last failing call on this thread ("" if none). */
const char* ayk_last_error(void);

/* Which kernels (and K split) the last GEMM, attention, rotation, 4-bit cache or MoE launch on this thread
 * ran, e.g. "skinny fn=2 fm=2 ks=1 g=2 ch=4 split=1", "pair tail=4" or "moe_small groups=2 runs=16": a diagnostic string,
 * not a stable format. No counterpart in the reference (its Triton launches pick
 * configurations inside Triton's autotuner); tests and profilers read it to assert
 * that a shape reaches the kernel it targets. */
const char* ayk_last_plan(void);

/* Library ABI version (major * 100 + minor). */
int ayk_abi_version(void);

/* 1 if `device` is a gfx950 GPU this library has code for, else 0. */
int ayk_device_supported(int device);

/* ---------------------------------------------------------------- quantizers
 * All quantizers write OCP e4m3fn with round-to-nearest-even after clamping the
 * fp32 quotient to [-448, 448]. `x_dtype` is AYK_F32, AYK_F16 or AYK_BF16.     */

/* Replaces ayaka::per_token_quant_fp8
 * (python/ayaka/kernel/triton/quant/fp8_quant.py:452; oracle reference/quant.py:59-66).
 * scale[m] = max(max|x[m,:]|, 1e-10) / 448 ; q = e4m3(clamp(x / scale[m])). */
int ayk_per_token_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t k,
                            int64_t ldx, void* q, int64_t ldq, float* scale,
                            ayk_stream_t stream);

/* Replaces ayaka::per_token_group_quant_fp8 (fp8_quant.py:297; oracle quant.py:19-29).
 * One fp32 scale per (row, group) stored [rows, k/group] row-major.
 * group: positive power of two dividing k. */
int ayk_per_token_group_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t k,
                                  int64_t ldx, int64_t group, void* q, int64_t ldq,
                                  float* scale, ayk_stream_t stream);

/* per_token_group_quant_fp8 with the scale table's layout given by strides: the scale of
 * (row m, group g) is stored at scale[m * scale_row_stride + g * scale_group_stride],
 * which must describe [rows, k/group] (group stride 1) or [k/group, rows] (row stride 1).
 * No counterpart in the reference, whose quantizer writes row-major scales only: the
 * column-major table is the layout the block-128 GEMM reads fastest at prefill sizes
 * (fp8_blockwise_mm's sa_col_major), written directly instead of transposed afterwards. */
int ayk_per_token_group_quant_fp8_strided(const void* x, int x_dtype, int64_t rows, int64_t k,
                                          int64_t ldx, int64_t group, void* q, int64_t ldq,
                                          float* scale, int64_t scale_row_stride, int64_t scale_group_stride,
                                          ayk_stream_t stream);

/* Replaces ayaka::per_token_group_quant_mxfp8 (fp8_quant.py:374; oracle quant.py:40-56).
 * code[m, g] = 0 for an all-zero group, else clamp(ceil(log2(amax/448)), -126, 127) + 127.
 * group: positive, divides k. */
int ayk_per_token_group_quant_mxfp8(const void* x, int x_dtype, int64_t rows, int64_t k,
                                    int64_t ldx, int64_t group, void* q, int64_t ldq,
                                    uint8_t* code, ayk_stream_t stream);

/* Replaces ayaka::static_quant_fp8 (fp8_quant.py:517; oracle quant.py:69-79).
 * q[i] = e4m3(clamp(x[i] / scale[0])) over n contiguous elements; the scale is read
 * on the device (`scale_dtype` F32/F16/BF16). */
int ayk_static_quant_fp8(const void* x, int x_dtype, int64_t n, const void* scale,
                         int scale_dtype, void* q, ayk_stream_t stream);

/* ------------------------------------------------------------------ GEMMs
 * Output dtype `out_dtype` is AYK_F32, AYK_F16 or AYK_BF16; `bias` may be NULL.
 * fp32 accumulation everywhere; one rounding to the output dtype.             */

/* Replaces ayaka::fp8_scaled_mm (gemm/fp8_gemm.py:246; oracle reference/gemm.py:17-37).
 * out = (a @ b^T) * scale_a * scale_b + bias, with b the [N, K] weight.
 * scale_a: scalar (sa_per_row = 0) or [M]; scale_b: scalar (sb_per_col = 0) or [N].
 * Requires K % 16 == 0, lda/ldb multiples of 16 and 16-byte aligned a/b. */
int ayk_fp8_scaled_mm(const void* a, int64_t lda, const void* b, int64_t ldb,
                      int64_t M, int64_t N, int64_t K,
                      const void* scale_a, int sa_dtype, int sa_per_row,
                      const void* scale_b, int sb_dtype, int sb_per_col,
                      const void* bias, int bias_dtype,
                      void* out, int out_dtype, int64_t ldo,
                      void* workspace, size_t workspace_bytes, ayk_stream_t stream);
/* Bytes of split-K partials ayk_fp8_scaled_mm may need for this shape (0: none). A
 * launch short of one full round of tiles splits K; a launch whose last round of
 * 256 x 256 tiles is at most a third full splits that round's tiles over K; a decode
 * batch (M <= 64) on a narrow projection splits K across workgroups, as the medium tiles
 * do at any M. Each piece writes its fp32 partial and a fixed-order sum adds the bias and
 * rounds once. The size is the largest any of these needs for the shape. With a smaller
 * workspace or none, the launch takes a slower kernel that needs none. */
size_t ayk_fp8_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* fp8_rowwise_linear (gemm/fp8_linear.py:168) for 2 to 8 activation rows in one launch:
 * per-token quantization of x (bf16 / fp16 / fp32, row stride ldx in elements) with the
 * arithmetic of ayk_per_token_quant_fp8, then out = (q @ w^T) * s_token * scale_b + bias,
 * the same result bit for bit as the two launches. No counterpart in the reference,
 * which launches the quantizer and the GEMM separately. Requires 2 <= M <= 8,
 * N * K <= 2^24, K % 16 == 0, M * K <= 64 KiB, 16-byte aligned rows of x and w.
 * scale_b: fp32 scalar (sb_per_col = 0) or [N]. */
int ayk_fp8_rowwise_linear_small(const void* x, int x_dtype, int64_t ldx, int64_t M,
                                 const void* w, int64_t ldw, int64_t N, int64_t K,
                                 const float* scale_b, int sb_per_col, const void* bias,
                                 int bias_dtype, void* out, int out_dtype, int64_t ldo,
                                 ayk_stream_t stream);

/* Replaces ayaka::int8_scaled_mm (gemm/int8_gemm.py:134; oracle reference/gemm.py:192-211).
 * out = float(a @ b^T, int32 accumulation) * scale_a[m] * scale_b[n] + bias, with a the
 * [M, K] int8 activation and b the [N, K] int8 weight; scale_a [M] and scale_b [N] fp32.
 * Requires K % 16 == 0, lda/ldb multiples of 16 and 16-byte aligned a/b. */
int ayk_int8_scaled_mm(const void* a, int64_t lda, const void* b, int64_t ldb,
                       int64_t M, int64_t N, int64_t K,
                       const float* scale_a, const float* scale_b,
                       const void* bias, int bias_dtype,
                       void* out, int out_dtype, int64_t ldo,
                       void* workspace, size_t workspace_bytes, ayk_stream_t stream);
/* Always 0: the INT8 GEMM never splits K (its int32 sums stay exact). */
size_t ayk_int8_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* Replaces ayaka::fp8_blockwise_mm (gemm/fp8_gemm.py:370; oracle reference/gemm.py:40-70).
 * out = sum_kb (a[:, kb] @ b[:, kb]^T) * scale_a[m, kb] * scale_b[n / 128, kb] + bias.
 * scale_a: [M, ceil(K/128)] (or [ceil(K/128), M] when sa_col_major), scale_b:
 * [ceil(N/128), ceil(K/128)], both contiguous. Same alignment rules as above. */
int ayk_fp8_blockwise_mm(const void* a, int64_t lda, const void* b, int64_t ldb,
                         int64_t M, int64_t N, int64_t K,
                         const void* scale_a, int sa_dtype, int sa_col_major,
                         const void* scale_b, int sb_dtype,
                         const void* bias, int bias_dtype,
                         void* out, int out_dtype, int64_t ldo,
                         void* workspace, size_t workspace_bytes, ayk_stream_t stream);
/* Bytes of split-K partials ayk_fp8_blockwise_mm may need for this shape (0: none). A
 * launch with fewer tiles than fill the machine (or, for M <= 64, fewer row groups)
 * splits K and sums fp32 partials in a fixed order before the single rounding. A smaller
 * workspace is treated as by ayk_fp8_scaled_mm. */
size_t ayk_fp8_blockwise_mm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* Replaces fp8_blockwise_scaled_grouped_mm (kernel/triton/moe/moe_grouped_gemm.py:599,
 * kernel :472-585): the MoE grouped block-128 GEMM. Expert e computes rows
 * [expert_offsets[e], + problem_sizes[e][0]) of out:
 *   out[m, n] = sum_kb scales_a[m, kb] * scales_b[e][n / 128][kb] * (a[m, kb] . b[e][n, kb])
 * with a [m_total, k] e4m3, b memory [E][n][k] e4m3, scales_a [m_total, k/128] fp32,
 * scales_a_t nullptr or the same table transposed, [k/128, m_total] (no counterpart in
 * the reference: experts over the whole k read it, at one cache line per 32 rows),
 * scales_b [E][n/128][k/128] fp32, out [m_total, n] bf16/fp16 (row stride n); rows of no
 * expert are not written. problem_sizes [E, 3] int32 (M_e, N_e, K_e) and expert_offsets
 * [E] int32 are read on the device (clamped to the operands). n % 128 == 0,
 * k % 128 == 0, 16-byte aligned a/b/out. */
int ayk_fp8_grouped_blockwise_mm(const void* a, const void* b, const float* scales_a, const float* scales_a_t,
                                 const float* scales_b,
                                 const int32_t* problem_sizes, const int32_t* expert_offsets, int64_t num_experts,
                                 int64_t m_total, int64_t n, int64_t k, void* out, int out_dtype,
                                 ayk_stream_t stream);
/* The same launch, which also fills the reference's per-expert pointer tables and scale
 * descriptors (get_group_gemm_starts, moe_grouped_gemm.py:61-135): int64 addresses
 * [num_experts] each, int32 descriptors [num_experts][>= 5] at row strides ld_sfa / ld_sfb;
 * `transpose` for the swapped operand roles. a_ptrs NULL: no tables. */
int ayk_fp8_grouped_blockwise_mm_tables(const void* a, const void* b, const float* scales_a, const float* scales_a_t,
                                        const float* scales_b, const int32_t* problem_sizes, const int32_t* expert_offsets,
                                        int64_t num_experts, int64_t m_total, int64_t n, int64_t k, void* out, int out_dtype,
                                        int64_t* a_ptrs, int64_t* b_ptrs, int64_t* out_ptrs, int64_t* a_scales_ptrs,
                                        int64_t* b_scales_ptrs, int32_t* layout_sfa, int64_t ld_sfa, int32_t* layout_sfb,
                                        int64_t ld_sfb, int transpose, ayk_stream_t stream);

/* No counterpart in the reference: a mixture-of-experts layer for few tokens (at most 64) with
 * e4m3 experts under 128 x 128 block scales:
 *   out[t] = sum_j weights[t, j] * down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = ids[t, j]
 * gate_up is [experts, 2 * inner, hidden] (gate rows, then up rows) with scales [experts, 2 * inner /
 * 128, hidden / 128], down is [experts, hidden, inner] with [experts, hidden / 128, inner / 128], all
 * contiguous, hidden and inner multiples of 128. x is [tokens, hidden] F16/BF16 and out its dtype,
 * not quantized: products are of the 16-bit activations, sums fp32. Entries of ids outside
 * [0, experts) count nothing; one that a token names twice counts with both weights. weights and ids
 * are [tokens, topk] contiguous. The workspace is needed, 16-byte aligned. */
int ayk_fp8_block_moe_small(const void* x, int x_dtype, int64_t ldx, int64_t tokens, const void* gate_up,
                            const float* gate_up_scale, const void* down, const float* down_scale, int64_t experts,
                            int64_t hidden, int64_t inner, const float* weights, const int32_t* ids, int64_t topk,
                            void* out, int64_t ldo, void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_fp8_block_moe_small_scratch_bytes(int64_t tokens, int64_t topk, int64_t experts, int64_t hidden,
                                             int64_t inner);

/* Replaces ayaka::mxfp8_scaled_mm (gemm/fp8_mxfp8_gemm.py:163; oracle reference/gemm.py:73-92).
 * out = sum_g (a[:, g] @ w[:, g]^T) * 2^(a_scale[m,g]-127) * 2^(w_scale[n,g]-127) + bias
 * over 32-wide K groups g; UE8M0 code 0 decodes to 0 and 0xFF to NaN.
 * K % 32 == 0; a_scale [M, K/32] (row stride ld_as), w_scale [N, K/32] (ld_ws). */
int ayk_mxfp8_scaled_mm(const void* a, int64_t lda, const uint8_t* a_scale, int64_t ld_as,
                        const void* w, int64_t ldw, const uint8_t* w_scale, int64_t ld_ws,
                        int64_t M, int64_t N, int64_t K,
                        const void* bias, int bias_dtype,
                        void* out, int out_dtype, int64_t ldo,
                        void* workspace, size_t workspace_bytes, ayk_stream_t stream);
/* Bytes of split-K partials ayk_mxfp8_scaled_mm may need for this shape (0: none);
 * the same rule as ayk_fp8_scaled_mm_workspace_bytes. */
size_t ayk_mxfp8_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* Replaces ayaka::fp8_weight_only_gemv (gemm/fp8_gemv.py:323; oracle reference/gemm.py:129-157).
 * out[n] = sum_k x[k] * w[n, k] * scale[(n / by) * scale_row_stride + k / bx]
 * x: [K] F16/BF16; scale_dtype: AYK_U8 (UE8M0), AYK_F32 or AYK_BF16; out dtype == x dtype.
 * The workspace holds split-K partials (see ayk_fp8_weight_only_gemv_workspace_bytes). */
int ayk_fp8_weight_only_gemv(const void* x, int x_dtype, const void* w, int64_t ldw,
                             int64_t N, int64_t K, const void* scale, int scale_dtype,
                             int64_t scale_row_stride, int64_t block_size_y,
                             int64_t block_size_x, void* out,
                             void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_fp8_weight_only_gemv_workspace_bytes(int64_t N, int64_t K);

/* No counterpart in the reference. ayk_fp8_weight_only_gemv without a workspace
 * argument, for callers that cannot allocate device memory (code under HIP graph
 * capture, serving loops, harnesses that forbid hipMalloc): the split-K partials live
 * in a static per-device array of ayk_fp8_weight_only_gemv_static_max_bytes() bytes
 * (64 KiB, enough for every shape; a shape needing more is rejected with
 * AYK_EWORKSPACE). Allocates nothing. All calls on one GPU share that array, so calls
 * that overlap on one GPU (different streams, or host threads) race. */
int ayk_fp8_weight_only_gemv_static(const void* x, int x_dtype, const void* w, int64_t ldw,
                                    int64_t N, int64_t K, const void* scale, int scale_dtype,
                                    int64_t scale_row_stride, int64_t block_size_y,
                                    int64_t block_size_x, void* out, ayk_stream_t stream);
size_t ayk_fp8_weight_only_gemv_static_max_bytes(void);

/* Replaces ayaka::fp8_weight_only_gemm (gemm/fp8_w8a16_gemm.py:144; oracle
 * reference/gemm.py:95-126). The [M, K] form of ayk_fp8_weight_only_gemv; out dtype ==
 * x dtype. Each dequantized weight w * scale is rounded to the activation dtype before
 * the product, as the reference does. Launches of any M may use a K split whose partials
 * live in the workspace; ayk_fp8_weight_only_gemm_workspace_bytes(M, N, K, block_size_x)
 * gives its size (0: none needed). With a smaller workspace or none, the launch takes a
 * slower kernel that needs none (AYK_EWORKSPACE where block_size_x is no multiple of 64,
 * which leaves no such kernel for a decode batch that would split). */
int ayk_fp8_weight_only_gemm(const void* x, int x_dtype, int64_t ldx, int64_t M,
                             const void* w, int64_t ldw, int64_t N, int64_t K,
                             const void* scale, int scale_dtype, int64_t scale_row_stride,
                             int64_t block_size_y, int64_t block_size_x,
                             void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                             ayk_stream_t stream);
size_t ayk_fp8_weight_only_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K,
                                                int64_t block_size_x);

/* Replaces ayaka::fp8_blockwise_gemv (gemm/fp8_gemv.py:433; oracle reference/gemm.py:160-189).
 * out[n] = sum_kb (a[kb] . b[n, kb]) * scale_a[kb] * scale_b[n / 128, kb] + bias[n],
 * a: [K] e4m3, scale_a [ceil(K/128)], scale_b [ceil(N/128), ceil(K/128)] contiguous. */
int ayk_fp8_blockwise_gemv(const void* a, const void* b, int64_t ldb, int64_t N, int64_t K,
                           const void* scale_a, int sa_dtype,
                           const void* scale_b, int sb_dtype,
                           const void* bias, int bias_dtype,
                           void* out, int out_dtype,
                           void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_fp8_blockwise_gemv_workspace_bytes(int64_t N, int64_t K);

/* ------------------------------------------------------------------ KV cache
 * Paged caches are [pages, page_size, heads, head_dim], flattened to `num_slots` rows of
 * `width` = heads * head_dim elements; a slot is page * page_size + offset. */

/* Replaces ayaka::cache_write_kv (kernel/triton/cache/cache_ops.py:160; oracle
 * _write_kv_reference :97 with _write_reference :40) and, with `value` == NULL,
 * ayaka::cache_scatter (cache_ops.py:65). Row t of key (and value), `src_row_stride`
 * elements apart, is written to slot slots[t] of key_cache (value_cache). An fp8 cache
 * (AYK_E4M3 / AYK_E5M2) stores round-to-nearest-even(clamp(x * inverse, +-max)); a float
 * cache stores x cast to its dtype. Negative slots are skipped; slots >= num_slots are
 * skipped too (the caller validates them, as the reference requires). */
int ayk_kv_cache_write(const void* key, const void* value, int src_dtype, int64_t num_tokens,
                       int64_t width, int64_t src_row_stride, void* key_cache, void* value_cache,
                       int cache_dtype, int64_t num_slots, const int64_t* slots,
                       float k_inverse, float v_inverse, ayk_stream_t stream);

/* Replaces ayaka::cache_gather (cache_ops.py:230; oracle _gather_reference :206).
 * dest[i] = cache[slots[i]] (repeats allowed), dequantized as float(value) * scale when
 * `dequantize`, else copied / cast to `dest_dtype`. A slot outside [0, num_slots) gives
 * a zero row. */
int ayk_kv_cache_gather(const void* cache, int cache_dtype, int64_t num_slots, int64_t width,
                        const int64_t* slots, int64_t n, void* dest, int dest_dtype, float scale,
                        int dequantize, ayk_stream_t stream);

/* No counterpart in the reference: position rotation of a step's queries and keys with the append
 * to the cache of ayk_kv_cache_write. Rows of q are [tokens, heads, dim] and of k and v [tokens,
 * kv_heads, dim], with the given strides in elements and the elements of a head side by side.
 * cos_sin is [table_rows, rotary_dim] contiguous: the cosines of a position's rotary_dim / 2 angles,
 * then the sines. (x, y) -> (x cos - y sin, y cos + x sin), each operation rounded to fp32, for the
 * pairs (d, d + rotary_dim / 2), or (2d, 2d + 1) when interleaved; dims from rotary_dim on pass
 * through; rotary_dim 0: no rotation (positions and cos_sin unused). q_out, and k_out unless NULL, get
 * the rotated rows in the query's dtype and may be q and k themselves. The caches take the rotated
 * fp32 keys, and the values, as ayk_kv_cache_write does; cache_dtype: fp8 or the keys' dtype. A token
 * whose slot is outside [0, num_slots) is not written; one whose position is outside the table
 * neither, and its rows of q_out and k_out are zeros. No slot may come twice. heads may be 0. */
int ayk_rope_kv_write(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, int64_t k_row_stride,
                      int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, int dtype,
                      int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, const int64_t* positions,
                      const float* cos_sin, int64_t table_rows, int64_t rotary_dim, int interleaved, void* q_out,
                      int64_t qo_row_stride, int64_t qo_head_stride, void* k_out, int64_t ko_row_stride,
                      int64_t ko_head_stride, void* key_cache, void* value_cache, int cache_dtype, int64_t num_slots,
                      const int64_t* slots, float k_inverse, float v_inverse, ayk_stream_t stream);
/* The same into a 4-bit cache. A plane is codes [num_pages, kv_heads, page_size, dim / 2] (OCP
 * e2m1, the even dim in the low half of a byte) and scales [num_pages, kv_heads, page_size, dim / 32]
 * (UE8M0: 2^(code - 127) from code 0 on, where the mxfp8 products have a factor of 0; 0xFF NaN), both contiguous. A group of 32 dims takes the least scale
 * under which no magnitude exceeds 6, codes are rounded to nearest even; zeros have scale code 0, a
 * group with an infinity or NaN has 0xFF. dim % 32 == 0; slot = page * page_size + offset. */
int ayk_rope_kv_write_mxfp4(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, int64_t k_row_stride,
                            int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, int dtype,
                            int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, const int64_t* positions,
                            const float* cos_sin, int64_t table_rows, int64_t rotary_dim, int interleaved, void* q_out,
                            int64_t qo_row_stride, int64_t qo_head_stride, void* k_out, int64_t ko_row_stride,
                            int64_t ko_head_stride, void* key_codes, void* key_scales, void* value_codes,
                            void* value_scales, int64_t num_pages, int64_t page_size, const int64_t* slots,
                            ayk_stream_t stream);
/* dest[i] = the values of slot slots[i] of one 4-bit plane, [n, kv_heads, dim] in fp32, fp16 or bf16.
 * A slot outside the plane gives zeros. fp32 and bf16 hold every value exactly; fp16 rounds, and what is held
 * as 65536 or more (of fp16 rows the magnitudes from 57344 on) comes back infinite. */
int ayk_kv_gather_mxfp4(const void* codes, const void* scales, int64_t num_pages, int64_t page_size, int64_t kv_heads,
                        int64_t dim, const int64_t* slots, int64_t n, void* dest, int dest_dtype, ayk_stream_t stream);

/* ------------------------------------------------------------------ norm
 * No counterpart in the reference's FP8 path: h = x + residual (x without one), rounded to
 * x's dtype into residual_out; y = h * weight / sqrt(mean(h^2) + eps) in fp32 from the
 * unrounded h; then the quantizers' rules. residual and residual_out come together and
 * must not overlap x or each other; residual_out and q are contiguous [rows, k].
 *   group == 0: scale[m] = max(amax(y[m]), 1e-10) / 448                  (fp32)
 *   group > 0:  one scale per (row, group), fp32 (scale_dtype AYK_F32) or UE8M0 codes
 *               (AYK_U8), at scale[m * scale_row_stride + g * scale_group_stride], laid
 *               out [rows, k/group] or [k/group, rows] as in the strided quantizer. */
int ayk_rms_norm_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t ldx,
                           const void* residual, int64_t ldr, const void* weight, int weight_dtype,
                           float eps, int64_t group, int scale_dtype, void* q, void* scale,
                           int64_t scale_row_stride, int64_t scale_group_stride,
                           void* residual_out, ayk_stream_t stream);

/* ------------------------------------------------------------------ attention
 * No counterpart in the reference's FP8 path. Query head h reads kv head h / (heads /
 * kv_heads). Softmax statistics and sums are fp32; the weights p are rounded once to 16
 * bits for the product with V. A query that sees nothing gives 0. With window > 0 a query
 * at position p sees the positions j with p - window < j <= p and j < sinks (j <= p). */

/* One new token per sequence over the paged cache of ayk_kv_cache_write: the query of row b
 * is at position seq_lens[b] - 1 and sees positions below seq_lens[b], position j at page
 * block_tables[b * table_stride + j / page_size], offset j % page_size. The caches are
 * [num_pages, page_size, kv_heads, dim] contiguous, of the query's 16-bit dtype or fp8 with
 * one scale per plane. A length past table_width * page_size is cut there, and positions of
 * a page outside [0, num_pages) count as hidden: neither is read. out: [batch, heads, dim]
 * contiguous, the query's dtype. The launch is chosen from table_width, as lengths are read on the
 * device only. A workspace smaller than the query's answer, or none, leaves the work of each
 * sequence unsplit. */
int ayk_paged_decode_attention(const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                               const void* key_cache, const void* value_cache, int cache_dtype,
                               int64_t num_pages, int64_t page_size, const int32_t* block_tables,
                               int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                               int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, float scale,
                               float k_scale, float v_scale, int64_t window, int64_t sinks, void* out,
                               void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_paged_decode_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim);
/* The same for calls whose longest possible sequence is known, table_width * page_size positions:
 * 0 where every sequence stays whole. */
size_t ayk_paged_decode_attention_split_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int cache_dtype,
                                              int64_t most, int64_t window, int64_t sinks);

/* The same over the 4-bit cache of ayk_rope_kv_write_mxfp4. page_size % 8 == 0, dim % 32 == 0, all four
 * planes 16-byte aligned. The products are of the decoded values, exact but for the weights, which
 * are rounded to 16 significant bits. _split_bytes: the workspace of calls whose longest possible
 * sequence is `most` = table_width * page_size positions (0: none needed). */
int ayk_paged_decode_attention_mxfp4(const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                                     const void* key_codes, const void* key_scales, const void* value_codes,
                                     const void* value_scales, int64_t num_pages, int64_t page_size,
                                     const int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                     const int32_t* seq_lens, int64_t batch, int64_t heads, int64_t kv_heads,
                                     int64_t dim, float scale, int64_t window, int64_t sinks, void* out,
                                     void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_paged_decode_attention_mxfp4_split_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                                        int64_t most, int64_t window, int64_t sinks);

/* Packed sequences: sequence b holds query rows [starts_q[b], starts_q[b + 1]) and key rows
 * [starts_k[b], starts_k[b + 1]); its queries are the last positions of its keys (more
 * queries than keys: the first ones see nothing when causal). Rows are [*, heads, dim] with
 * the given strides in elements; out is contiguous [total_q, heads, dim]. Rows of no sequence give 0;
 * bounds outside the packed rows are cut to them. */
int ayk_varlen_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                         int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                         int64_t v_head_stride, int dtype, const int32_t* starts_q, const int32_t* starts_k,
                         int64_t batch, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                         int64_t dim, float scale, int causal, int64_t window, int64_t sinks, void* out,
                         ayk_stream_t stream);
/* The same with a workspace, in which the keys of few rows (a chunk behind a long prompt) are
 * split over the chip and joined; sequences of less than 1024 keys on average are not. One
 * smaller than the query's answer, or none, leaves them whole. */
int ayk_varlen_attention_split(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                               int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                               int64_t v_head_stride, int dtype, const int32_t* starts_q, const int32_t* starts_k,
                               int64_t batch, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                               int64_t dim, float scale, int causal, int64_t window, int64_t sinks, void* out,
                               void* workspace, size_t workspace_bytes, ayk_stream_t stream);
size_t ayk_varlen_attention_split_workspace_bytes(int64_t batch, int64_t total_q, int64_t heads, int64_t dim);

#ifdef __cplusplus
}
#endif

#endif /* AYAKA_FP8_H */
