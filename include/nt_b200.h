/*
 * nt_b200.h -- C ABI of the B200 (sm_100a) kernel library `libnt_b200.so`.
 *
 * One entry point per operator family that NineToothed's arrange-and-apply
 * programs generate.  Every entry point:
 *   - takes raw device pointers, int64 sizes and element strides, a dtype code
 *     and the caller's CUDA stream (a `cudaStream_t` passed as `void*`);
 *   - never allocates device memory and never synchronises the stream;
 *   - returns 0 on success, a `cudaError_t` value when a launch fails, or one of
 *     the NT_B200_ERR_* codes below when the arguments are rejected on the host
 *     before anything is launched;
 *   - launches nothing when an output has zero elements (returns 0), the same
 *     empty-launch rule as the reference runtime (src/ninetoothed/compiler/
 *     runtime.py:1411-1422).
 *
 * The shape of this ABI follows the launcher the reference CUDA backend emits
 * (src/ninetoothed/backends/emitters/cuda.py:368-380: `extern "C" int
 * launch_<kernel>(..., cudaStream_t stream)` returning `cudaGetLastError()`),
 * with the per-tensor pointer/shape/stride triples that the reference runtime
 * binds (src/ninetoothed/compiler/runtime.py:1301-1332).  Dtype codes are the
 * values of the reference's `NineToothedDataType` enum
 * (src/ninetoothed/backends/materializers/cpp.py:10-23, 26-58).
 */
#ifndef NT_B200_H
#define NT_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types: the NineToothedDataType values of the reference ABI (0-11),
 * extended with the two 8-bit float types the reference's matmul/addmm tests
 * use (torch.float8_e4m3fn, torch.float8_e5m2), which its C++ ABI enum lacks. */
enum NtB200DataType {
    NT_B200_INT8 = 0,
    NT_B200_INT16 = 1,
    NT_B200_INT32 = 2,
    NT_B200_INT64 = 3,
    NT_B200_UINT8 = 4,
    NT_B200_UINT16 = 5,
    NT_B200_UINT32 = 6,
    NT_B200_UINT64 = 7,
    NT_B200_FLOAT16 = 8,
    NT_B200_BFLOAT16 = 9,
    NT_B200_FLOAT32 = 10,
    NT_B200_FLOAT64 = 11,
    NT_B200_FLOAT8_E4M3FN = 12,
    NT_B200_FLOAT8_E5M2 = 13
};

/* Host-side argument errors (no launch happened).  Values are above the
 * cudaError_t range used by CUDA 12 so the two never collide. */
#define NT_B200_ERR_INVALID_ARGUMENT 10001 /* null pointer, negative size, bad window */
#define NT_B200_ERR_UNSUPPORTED_DTYPE 10002 /* dtype not implemented for this op */
#define NT_B200_ERR_SHAPE_MISMATCH 10003   /* output shape inconsistent with inputs */
#define NT_B200_ERR_NO_DEVICE 10004        /* no sm_100 device current */
#define NT_B200_ERR_DEVICE_TIMEOUT 10005   /* a bounded device-side wait gave up */
#define NT_B200_ERR_WORKSPACE_TOO_LARGE 10006 /* staging exceeds the library's fixed array */
#define NT_B200_ERR_INDEX_OUT_OF_RANGE 10007 /* a kernel met a position, page or offset outside its array */

/* Library identity and diagnostics. */
int nt_b200_version(void);
const char *nt_b200_error_string(int code);

/*
 * Reads and clears the device-side error word of the current device after
 * synchronising `stream`.  Pipelined kernels (GEMM, attention, conv) bound every
 * mbarrier wait; a wait that runs out records NT_B200_ERR_DEVICE_TIMEOUT there
 * and the kernel returns early instead of hanging.  `*status` receives 0 or that
 * code.  No counterpart in the reference (its launchers only report launch
 * errors, src/ninetoothed/compiler/runtime.py:31-35).
 */
int nt_b200_device_status(void *stream, int *status);

/*
 * Row softmax over the last dimension: y = exp(x - max(x)) / sum(exp(x - max(x))),
 * fp32 internal math, result rounded to `dtype`.  Replaces the launcher of
 * `softmax_kernel` (tests/test_softmax.py:10-27 in the reference; one program per
 * row, `BLOCK_SIZE = cols`).  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
int nt_b200_softmax(const void *input, void *output, int64_t rows, int64_t cols,
                    int64_t input_stride_row, int64_t input_stride_col,
                    int64_t output_stride_row, int64_t output_stride_col,
                    int dtype, void *stream);

/*
 * output[i] = lhs[i] + rhs[i] for i < size.  Replaces `add_kernel`
 * (tests/test_add.py:9-24).  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
int nt_b200_add(const void *lhs, const void *rhs, void *output, int64_t size,
                int64_t lhs_stride, int64_t rhs_stride, int64_t output_stride,
                int dtype, void *stream);

/*
 * output[i] = pow(input[i], exponent[i]) (CUDA powf, fp32 math).  Replaces
 * `pow_kernel` (tests/test_pow.py:10-31, `libdevice.pow`).
 * dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
int nt_b200_pow(const void *input, const void *exponent, void *output, int64_t size,
                int64_t input_stride, int64_t exponent_stride,
                int64_t output_stride, int dtype, void *stream);

/*
 * output[i] = rand(seed, i) > p ? input[i] / (1 - p) : 0, where rand is
 * Philox4x32-10 on counter (i, 0, 0, 0) with key (seed lo, seed hi), first word
 * mapped to [0, 1) as Triton's `tl.rand` does.  Replaces `dropout_kernel`
 * (tests/test_dropout.py:12-29).  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
int nt_b200_dropout(const void *input, float p, int64_t seed, void *output,
                    int64_t size, int64_t input_stride, int64_t output_stride,
                    int dtype, void *stream);

/*
 * 2-D max pooling over NCHW tensors: output[n,c,p,q] = max over the window rows
 * p*stride_h - pad_h + [0, window_h) and columns q*stride_w - pad_w + [0,
 * window_w) of input, skipping positions outside the input (the reference's
 * `other=-inf` fill).  `out_h`/`out_w` are the caller's output extents (floor or
 * ceil mode is decided by the caller, as in tests/test_max_pool2d.py:39-61).
 * Bit-exact.  Strides are element strides of the 4-D tensors.
 * dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
int nt_b200_max_pool2d(const void *input, void *output, int64_t n, int64_t c,
                       int64_t h, int64_t w, const int64_t *input_strides,
                       int64_t out_h, int64_t out_w, const int64_t *output_strides,
                       int64_t window_h, int64_t window_w, int64_t stride_h,
                       int64_t stride_w, int64_t pad_h, int64_t pad_w, int dtype,
                       void *stream);

/*
 * output[M,N] = cast_out(cast_f16(sum_k lhs[m,k] * rhs[k,n])) with an fp32
 * accumulator: the `matmul` application (tests/test_matmul.py:41-47) rounds the
 * accumulator to float16 before the store converts it to the output dtype.
 * in_dtype: FLOAT16, BFLOAT16, FLOAT8_E4M3FN or FLOAT8_E5M2 (both operands;
 * 8-bit operands run on tcgen05 kind::f8f6f4) or FLOAT32 (exact fp32 on CUDA
 * cores); out_dtype: FLOAT16, BFLOAT16, FLOAT32.  Strides are element strides (row, col) of each 2-D operand.
 */
int nt_b200_matmul(const void *lhs, const void *rhs, void *output, int64_t m,
                   int64_t n, int64_t k, int64_t lhs_stride_row,
                   int64_t lhs_stride_col, int64_t rhs_stride_row,
                   int64_t rhs_stride_col, int64_t output_stride_row,
                   int64_t output_stride_col, int in_dtype, int out_dtype,
                   void *stream);

/*
 * output = beta * input + alpha * cast_f16(mat1 @ mat2), stored in out_dtype:
 * the `addmm` application (tests/test_addmm.py:13-38), whose inlined matmul
 * rounds the fp32 accumulator to float16.  The epilogue follows Triton's typing
 * of a scalar argument against a tensor: beta * input in in_dtype, alpha * the
 * float16 product in float16, their sum in float16 when in_dtype is FLOAT16
 * (fp32 otherwise).  `input` has the output's [M,N] shape and in_dtype.
 */
int nt_b200_addmm(const void *input, const void *mat1, const void *mat2, float beta,
                  float alpha, void *output, int64_t m, int64_t n, int64_t k,
                  int64_t input_stride_row, int64_t input_stride_col,
                  int64_t mat1_stride_row, int64_t mat1_stride_col,
                  int64_t mat2_stride_row, int64_t mat2_stride_col,
                  int64_t output_stride_row, int64_t output_stride_col,
                  int in_dtype, int out_dtype, void *stream);

/*
 * Flash attention with the reference application's numerics
 * (tests/test_attention.py:44-70): q' = round(q * round(log2 e)) in the input
 * dtype, s = q' k^T in fp32 (softmax scale 1; callers pre-scale q), keys beyond
 * seq_kv masked, optional causal mask (query index >= key index), base-2 online
 * softmax with fp32 running max/sum, p rounded to the input dtype before p @ v,
 * o = acc / l.  Tensors are [batch, heads, seq, head_dim]; strides are 4-entry
 * element-stride arrays.  dtype: FLOAT16 or BFLOAT16 (q, k, v and o; tcgen05) or
 * FLOAT32 (CUDA cores).
 */
int nt_b200_attention(const void *q, const void *k, const void *v, int is_causal,
                      void *o, int64_t batch, int64_t heads, int64_t seq_q,
                      int64_t seq_kv, int64_t head_dim, const int64_t *q_strides,
                      const int64_t *k_strides, const int64_t *v_strides,
                      const int64_t *o_strides, int dtype, void *stream);

/*
 * conv2d as an implicit GEMM (tests/test_conv2d.py:14-49 arrangement with the
 * matmul application): output[n,k,p,q] = cast_out(cast_f16(sum over (c,r,s) of
 * input[n,c,p+r-pad_h,q+s-pad_w] * filter[k,c,r,s])), zero outside the input,
 * stride 1, fp32 accumulation.  NCHW input/output, KCRS filter; strides are
 * 4-entry element-stride arrays.  dtype: FLOAT16 or BFLOAT16 (all three tensors).
 *
 * `workspace` is caller-owned device memory of at least
 * nt_b200_conv2d_workspace_size(...) bytes, 256-byte aligned; the tensor-core
 * path stages the input as NHWC and the filter as KRSC there.  With a smaller
 * (or null) workspace the call takes the CUDA-core path instead.
 */
int nt_b200_conv2d(const void *input, const void *filter, void *output, int64_t n,
                   int64_t c, int64_t h, int64_t w, int64_t k, int64_t r, int64_t s,
                   int64_t pad_h, int64_t pad_w, const int64_t *input_strides,
                   const int64_t *filter_strides, const int64_t *output_strides,
                   void *workspace, int64_t workspace_bytes, int dtype, void *stream);

/*
 * conv2d followed by max_pool2d with a 3x3 window, stride 2, padding 1 (floor
 * mode): output[n, k, i, j] = max_pool2d(conv2d(input, filter, padding))[n, k,
 * i, j], bit-identical to the two programs run one after the other
 * (nt_b200_conv2d, then nt_b200_max_pool2d), output [n, k, P2, Q2] with
 * P2 = (P - 1) / 2 + 1, Q2 = (Q - 1) / 2 + 1 for the conv extents P, Q.  The
 * conv result goes to the workspace.  pool_in_conv_kernel = 0 pools it with
 * the max_pool2d kernel after the conv kernel (the faster order on B200);
 * pool_in_conv_kernel = 1 pools inside the tensor-core conv kernel where the
 * shape allows (extra pool warps per CTA read each pool row back from L2 once
 * the warp that completes its last input rows hands it over) and falls back to
 * the two kernels elsewhere.  `workspace` (256-byte aligned) must hold
 * nt_b200_conv2d_max_pool2d_workspace_size(...) bytes (conv staging + the conv
 * result + counters).  No single program of the reference does this; it
 * composes its conv2d and max_pool2d programs (tests/test_conv2d.py,
 * tests/test_max_pool2d.py).
 */
int nt_b200_conv2d_max_pool2d(const void *input, const void *filter, void *output,
                              int64_t n, int64_t c, int64_t h, int64_t w, int64_t k,
                              int64_t r, int64_t s, int64_t pad_h, int64_t pad_w,
                              const int64_t *input_strides, const int64_t *filter_strides,
                              const int64_t *output_strides, void *workspace,
                              int64_t workspace_bytes, int pool_in_conv_kernel, int dtype,
                              void *stream);
int64_t nt_b200_conv2d_max_pool2d_workspace_size(int64_t n, int64_t c, int64_t h, int64_t w,
                                                 int64_t k, int64_t r, int64_t s,
                                                 int64_t pad_h, int64_t pad_w, int dtype);

/*
 * Workspace bytes the tensor-core conv2d path needs for this problem (0 when
 * the path does not apply: 32-bit dtype or channels not a multiple of 8): the
 * input as NHWC with pad_w zero columns on each side of every row, then the
 * filter as KRSC.  No counterpart in the reference (its conv2d program stages
 * nothing).
 */
int64_t nt_b200_conv2d_workspace_size(int64_t n, int64_t c, int64_t h, int64_t w,
                                      int64_t k, int64_t r, int64_t s, int64_t pad_h,
                                      int64_t pad_w, int dtype);

/*
 * conv2d exactly as nt_b200_conv2d, for callers that cannot provide device
 * memory at call time: a C host program without a device allocator, a loop
 * that must not call cudaMalloc (it synchronises the device and stalls other
 * streams), or an application whose memory budget is fixed at start-up.  The
 * NHWC/KRSC staging goes to a 64 MiB array inside the library (held on every
 * GPU that loads the library until the process exits); the call allocates
 * nothing.  Problems needing more staging than 64 MiB return
 * NT_B200_ERR_WORKSPACE_TOO_LARGE without launching.  All calls on a device
 * share the array, so calls whose kernels overlap on the GPU race; calls on
 * one stream are safe.  The first call on a device looks the array's address
 * up with that device current; make it before any stream capture.
 * No counterpart in the reference.
 */
int nt_b200_conv2d_no_alloc(const void *input, const void *filter, void *output,
                            int64_t n, int64_t c, int64_t h, int64_t w, int64_t k,
                            int64_t r, int64_t s, int64_t pad_h, int64_t pad_w,
                            const int64_t *input_strides,
                            const int64_t *filter_strides,
                            const int64_t *output_strides, int dtype, void *stream);

/*
 * clone (tests/test_clone.py:10-47, all four applications): output[i, j] =
 * input[i, j] for a rows x cols matrix with any element strides; a bit copy
 * of any dtype code 0-13.
 */
int nt_b200_clone(const void *input, void *output, int64_t rows, int64_t cols,
                  int64_t input_stride_row, int64_t input_stride_col,
                  int64_t output_stride_row, int64_t output_stride_col, int dtype,
                  void *stream);

/*
 * to_padded_tensor (tests/test_jagged.py:12-49): a jagged 3-D tensor with one
 * ragged dimension -- packed `values` holding element (b, r, d) at
 * (offsets[b] + r) * values_stride_ragged + d * values_stride_inner, device
 * `offsets` [batch + 1] (int64), `inner` elements along the dense dimension --
 * to a dense `output` whose element (b, r, d) sits at output_strides[0] * b +
 * output_strides[1] * r + output_strides[2] * d for r < max_len; positions
 * r >= len_b hold `padding` converted to the dtype (codes 0-11).  Ragged
 * dimension 1: the strides of values [total, D] in order; ragged dimension 2:
 * values [D, total] with its strides swapped.
 */
int nt_b200_jagged_to_padded(const void *values, const int64_t *offsets, int64_t batch,
                             int64_t inner, int64_t values_stride_ragged,
                             int64_t values_stride_inner, double padding, void *output,
                             int64_t max_len, const int64_t *output_strides, int dtype,
                             void *stream);

/*
 * Copy with expand into a jagged tensor (tests/test_jagged.py:104-143): every
 * element (b, r, d) of the jagged tensor (layout as above) becomes
 * src[b * src_stride_batch + d * src_stride_inner], the dense source being
 * broadcast along the ragged dimension.  batch <= 65535.
 */
int nt_b200_jagged_expand(void *values, const int64_t *offsets, int64_t batch, int64_t inner,
                          int64_t values_stride_ragged, int64_t values_stride_inner,
                          const void *src, int64_t src_stride_batch, int64_t src_stride_inner,
                          int dtype, void *stream);

/*
 * Serving operators: rotary positions, a paged cache of 8-bit keys and values,
 * attention over it, and causal attention over packed prompts.  They have no
 * counterpart among the reference's programs.  Each takes its arguments in one
 * struct of 8-byte fields (sizes, strides and codes are int64; strides count
 * elements).  Index arrays (positions, offsets, lengths, block tables) live on
 * the device, all of one call in one dtype, INT32 or INT64 (`index_dtype`).
 * The kernels check every index they read: one that leaves its array records
 * NT_B200_ERR_INDEX_OUT_OF_RANGE in the device error word
 * (nt_b200_device_status) and is not followed; offsets out of order record it
 * too, and leave out some or all tokens of the call.
 */

/*
 * Rotary positions of `input` [tokens, heads, head_dim]: the pairs (a, b) among
 * the first `rotary_dim` elements of each head become (a cos - b sin, b cos +
 * a sin), the rest is copied.  Half layout: a = x[i], b = x[i + rotary_dim/2];
 * interleaved: a = x[2i], b = x[2i+1].  cos, sin: fp32 [table_rows,
 * rotary_dim/2], unit column stride; token t uses row positions[t].  `adjoint`
 * applies the transposed map (sin -> -sin): the gradient of the rotation.
 * Products and sums are rounded to fp32 one by one and the result once to
 * `dtype`.  `output` may be `input`.  A token whose position is outside the
 * table gets NaN in its rotated part.  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
typedef struct NtB200RotaryArgs {
    const void *input;
    const float *cos, *sin;
    const void *positions;
    void *output;
    int64_t tokens, heads, head_dim, rotary_dim, table_rows;
    int64_t input_strides[3], output_strides[3]; /* token, head, element */
    int64_t cos_stride, sin_stride, positions_stride;
    int64_t interleaved, adjoint, dtype, index_dtype;
} NtB200RotaryArgs;
int nt_b200_rotary(const NtB200RotaryArgs *args, void *stream);

/*
 * A paged cache: `pages` pages of `page` tokens each (a multiple of 16, at most
 * 4096), codes of `code_dtype` (FLOAT8_E4M3FN or INT8) in key and value [pages,
 * kv_heads, page, head_dim] with unit element stride, head_dim a multiple of 16, every
 * other stride and both bases multiples of 16; one fp32 scale for each page and
 * head.  A stored element stands for code * scale.
 */
typedef struct NtB200PagedCache {
    void *key, *value;
    float *key_scale, *value_scale;
    int64_t pages, kv_heads, page, head_dim, code_dtype;
    int64_t key_strides[3], value_strides[3];             /* page, head, token */
    int64_t key_scale_strides[2], value_scale_strides[2]; /* page, head */
} NtB200PagedCache;

/*
 * Appends packed new tokens to a paged cache and rotates queries on the way.
 * Sequence s (of `batch`) brings the tokens offsets[s] .. offsets[s+1] - 1 of
 * key and value [tokens, kv_heads, head_dim] and already has past[s] tokens;
 * its token past[s] + i goes to page block_table[s, (past[s] + i) / page], slot
 * (past[s] + i) % page.  With tables (cos not null) keys are rotated as by
 * nt_b200_rotary at those positions before they are stored, and, where given,
 * `query` [tokens, heads, head_dim] is rotated into `query_out` and the rotated
 * key stored in `key_out` in `dtype`.  A query needs tables unless rotary_dim is 0.
 * Tokens that belong to no sequence are written in neither, nor keys that an index
 * out of range keeps from the cache.
 *
 * Scales.  With amax the largest finite magnitude among a page's new elements
 * of a head: E4M3 codes: s = the least power of two, 2^-126 or more, with
 * amax <= 448 s; INT8: s = max(amax * fp32(1 / 127), 2^-126).  A page whose first slots
 * already hold tokens keeps max(its scale, s); where that grows, the held codes
 * are rounded again by old / new (exact for E4M3 down to its subnormals).  code
 * = round(x * (1 / s)) to nearest even, saturated; NaN becomes E4M3's NaN, INT8
 * 0.  A page belongs to one sequence of the call: pages that several sequences
 * share must be full.  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
typedef struct NtB200PagedAppendArgs {
    NtB200PagedCache cache;
    const void *key, *value, *query; /* query may be null */
    const float *cos, *sin;          /* null: no rotation */
    const void *offsets, *past, *block_table;
    void *query_out, *key_out; /* key_out may be null */
    int64_t tokens, batch, heads, rotary_dim, table_rows, table_columns;
    int64_t key_strides[3], value_strides[3], query_strides[3], query_out_strides[3], key_out_strides[3];
    int64_t cos_stride, sin_stride, offsets_stride, past_stride, block_table_strides[2];
    int64_t interleaved, dtype, index_dtype;
} NtB200PagedAppendArgs;
int nt_b200_paged_append(const NtB200PagedAppendArgs *args, void *stream);

/*
 * Attention of each sequence's last `queries` tokens over a paged cache that
 * holds them already: query i of `query` [batch, queries, heads, head_dim] sees
 * the first lengths[b] - queries + 1 + i tokens of sequence b; query head h
 * reads key/value head h / (heads / kv_heads).  Nobody sees the tokens of a page
 * outside the pool.  With s = scale * (q . k) over the tokens seen, output = softmax(s) v and, where `lse` is not null, lse [batch,
 * queries, heads] = ln sum exp(s) (fp32); a query that sees nothing gets 0 and
 * -inf.  Scores, softmax and sums are fp32; the scales must not be negative.
 * FLOAT16 and BFLOAT16 queries of head_dim up to 128 run on tensor cores
 * (probabilities rounded to fp16 there), FLOAT32 ones and head_dim up to 256 on
 * CUDA cores.  `scale` is a double.  `workspace`: 16-byte aligned device memory
 * of nt_b200_paged_attention_workspace_size() bytes (the current device's), for
 * this call alone.
 */
typedef struct NtB200PagedAttentionArgs {
    NtB200PagedCache cache;
    const void *query, *lengths, *block_table;
    void *output;
    float *lse;
    void *workspace;
    int64_t workspace_bytes, batch, queries, heads, table_columns;
    int64_t query_strides[4], output_strides[4], lse_strides[3]; /* batch, query, head, element */
    int64_t lengths_stride, block_table_strides[2];
    int64_t dtype, index_dtype;
    double scale;
} NtB200PagedAttentionArgs;
int nt_b200_paged_attention(const NtB200PagedAttentionArgs *args, void *stream);
int64_t nt_b200_paged_attention_workspace_size(void);

/*
 * Attention over whole prompts packed one after another: sequence b has the
 * queries query_offsets[b] .. query_offsets[b+1] - 1 of `query` [query_tokens,
 * heads, head_dim] and the keys key_offsets[b] .. key_offsets[b+1] - 1 of `key`
 * and `value` [key_tokens, kv_heads, head_dim]; query head h reads key/value
 * head h / (heads / kv_heads).  The last query stands at the last key: with
 * `is_causal`, query i of nq sees the first nk - nq + 1 + i of nk keys.  With s
 * = scale * (q . k), output = softmax(s) v and, where `lse` is not null, lse
 * [query_tokens, heads] = ln sum exp(s) (fp32); a query that sees nothing gets 0
 * and -inf.  Scores, softmax and sums are fp32.  FLOAT16 and BFLOAT16 run on
 * tcgen05 tensor cores (probabilities rounded to the input type there) for
 * head_dim up to 128, unit element strides, other strides and bases on the
 * 16-byte grid and a positive scale; the rest, FLOAT32 and head_dim up to 256,
 * on CUDA cores.  Tokens that belong to no sequence are not written, and none
 * are on tensor cores where any offsets are out of order or leave the tensors.
 * `workspace`: 32-byte aligned device memory of
 * nt_b200_prompt_attention_workspace_size(...) bytes, for this call alone.
 */
typedef struct NtB200PromptAttentionArgs {
    const void *query, *key, *value, *query_offsets, *key_offsets;
    void *output;
    float *lse;
    void *workspace;
    int64_t workspace_bytes, query_tokens, key_tokens, batch, heads, kv_heads, head_dim;
    int64_t query_strides[3], key_strides[3], value_strides[3], output_strides[3]; /* token, head, element */
    int64_t lse_strides[2], query_offsets_stride, key_offsets_stride;
    int64_t is_causal, dtype, index_dtype;
    double scale;
} NtB200PromptAttentionArgs;
int nt_b200_prompt_attention(const NtB200PromptAttentionArgs *args, void *stream);
int64_t nt_b200_prompt_attention_workspace_size(int64_t query_tokens, int64_t batch, int64_t heads, int64_t kv_heads);

/*
 * Causal attention of the next pieces of prompts, packed one after another, over a
 * paged cache that holds them already: sequence b has the queries offsets[b] ..
 * offsets[b+1] - 1 of `query` [tokens, heads, head_dim], the last of its lengths[b]
 * cached tokens; query i of n sees the first lengths[b] - n + 1 + i of them.  Query
 * head h reads key/value head h / (heads / kv_heads); nobody sees the tokens of a page
 * outside the pool.  With s = scale * (q . k) over the tokens seen, output = softmax(s)
 * v and, where `lse` is not null, lse [tokens, heads] = ln sum exp(s) (fp32); a query
 * that sees nothing gets 0 and -inf.  Scores, softmax and sums are fp32; the cache's
 * scales must not be negative, and a value scale that is not finite makes output and, on
 * tensor cores, lse of who sees it NaN.  FLOAT16 and BFLOAT16 queries run on tcgen05 tensor cores
 * (probabilities rounded to fp16 there) for head_dim up to 128, up to 128 query heads to
 * a key/value head and a positive scale; the rest, FLOAT32 and head_dim up to 256, on
 * CUDA cores.  Tokens that belong to no sequence are not written, nor those of a sequence
 * whose offsets are out of order or leave the tensors (recorded as
 * NT_B200_ERR_INDEX_OUT_OF_RANGE; on CUDA cores, which search the offsets, tokens of other
 * sequences may then be left out too).  `workspace`: 16-byte aligned
 * device memory of nt_b200_chunk_attention_workspace_size() bytes (the current
 * device's), for this call alone.
 */
typedef struct NtB200ChunkAttentionArgs {
    NtB200PagedCache cache;
    const void *query, *offsets, *lengths, *block_table;
    void *output;
    float *lse;
    void *workspace;
    int64_t workspace_bytes, tokens, batch, heads, table_columns;
    int64_t query_strides[3], output_strides[3], lse_strides[2]; /* token, head, element */
    int64_t offsets_stride, lengths_stride, block_table_strides[2];
    int64_t dtype, index_dtype;
    double scale;
} NtB200ChunkAttentionArgs;
int nt_b200_chunk_attention(const NtB200ChunkAttentionArgs *args, void *stream);
int64_t nt_b200_chunk_attention_workspace_size(void);

/*
 * Root-mean-square norm of the rows of `input` [rows, width], after the addition
 * of `residual` where it is not null: t = input + residual, rounded to `dtype` and
 * stored in `total` (which may be `residual` or `input`), or t = input; y = (t * r)
 * * weight with r = 1 / sqrt(mean(t^2) + eps).  The mean and its root are taken in
 * 64 bits and r is rounded to fp32, as is each product.  weight: [width], of
 * weight_dtype, `dtype` or FLOAT32.  output_dtype = dtype: output = round(y), and it
 * may be `input`.  output_dtype FLOAT8_E4M3FN or INT8: codes round(y * (1 / s)) with
 * one fp32 scale s in `scale` [rows, ceil(width / group)] for each `group` elements
 * of a row (the last group may be shorter), by the rules of a paged cache's pages
 * (nt_b200_paged_append).  `group`: the width or more, or a multiple of 16; width at
 * most 131072.  dtype: FLOAT16, BFLOAT16, FLOAT32.
 */
typedef struct NtB200RmsNormArgs {
    const void *input, *residual, *weight; /* residual may be null */
    void *output, *total;                  /* total: with a residual */
    float *scale;                          /* with codes */
    int64_t rows, width, group;
    int64_t input_strides[2], residual_strides[2], weight_stride, output_strides[2], total_strides[2],
        scale_strides[2]; /* row, element */
    int64_t dtype, weight_dtype, output_dtype;
    double eps;
} NtB200RmsNormArgs;
int nt_b200_rms_norm(const NtB200RmsNormArgs *args, void *stream);

/*
 * output[m, n] = input_scale[m] * sum_k input[m, k] (q[n, k] - z[n, k / group])
 * scales[n, k / group] for input [rows, inner] and 4-bit weights q, two a byte of
 * `codes` [outer, inner / 2], the even k in the low half.  z = 8 where `zeros` is
 * null, else zeros (uint8) [outer, inner / group], 0 to 63 (larger ones are recorded as
 * NT_B200_ERR_INDEX_OUT_OF_RANGE, and what they give is not specified); scales
 * [outer, inner / group] of scales_dtype; input_scale (fp32, [rows]) may be null.
 * `group` is a multiple of 32 and divides inner.  Products and sums are fp32, the
 * result is rounded once to output_dtype.  dtype: FLOAT16, BFLOAT16, FLOAT32,
 * FLOAT8_E4M3FN or INT8; scales and output: FLOAT16, BFLOAT16, FLOAT32.  Tensor
 * cores take all but FLOAT32 inputs where element strides are 1, rows of input and
 * codes (and both bases) on the 16-byte grid and the bases of scales and zeros on
 * the 4-byte one, for up to 65535 * 32 rows; the rest runs on CUDA cores, for up to
 * 65535 * 8.
 */
typedef struct NtB200Int4MatmulArgs {
    const void *input, *codes, *scales, *zeros; /* zeros may be null */
    const float *input_scale;                   /* or null */
    void *output;
    int64_t rows, inner, outer, group;
    int64_t input_strides[2], codes_strides[2], scales_strides[2], zeros_strides[2], input_scale_stride,
        output_strides[2];
    int64_t dtype, scales_dtype, output_dtype;
} NtB200Int4MatmulArgs;
int nt_b200_int4_matmul(const NtB200Int4MatmulArgs *args, void *stream);

/*
 * Failure-detection self-test (no counterpart in the reference): launches one
 * thread that waits on an mbarrier nothing ever arrives on, through the same
 * bounded wait the pipelined kernels use, with a limit of `limit_ns`
 * (1 us .. 1 s).  The wait gives up, records NT_B200_ERR_DEVICE_TIMEOUT in the
 * device error word and the kernel exits; nt_b200_device_status then reports
 * it.  The context stays usable.
 */
int nt_b200_wait_timeout_selftest(int64_t limit_ns, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NT_B200_H */
