/*
 * s4d_decoder.h -- C ABI of the decoder's dense operators on B200 (sm_100a), the layers that
 * stand around the DeformableFeatureAggregation path of s4d_dfa.h:
 *
 *   s4d_attention_forward / _backward   attention over shared or own heads with scores capped by a
 *                                       tanh, a bias by distance, a document mask and a valid length
 *                                       per batch entry, for one query or many.
 *   s4d_norm_forward / _backward        LayerNorm rows of any width up to 16384 in f32, bf16 or
 *                                       f16, with the gradients of the input, weight and bias.
 *
 * Conventions are those of s4d_dfa.h: device pointers, no allocation, stream-ordered and
 * asynchronous, host-checked arguments, a status code per call and the text of the last failure on
 * the calling thread in s4d_decoder_last_error().  Launches go to the current CUDA device, which
 * has to be the pointers' and the stream's.
 */
#ifndef S4D_DECODER_H_
#define S4D_DECODER_H_

#include "s4d_dfa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of this header: S4D_DTYPE_F32, S4D_DTYPE_BF16 and */
enum { S4D_DTYPE_F16 = 2 };

S4D_API int s4d_decoder_abi_version(void);
S4D_API const char* s4d_decoder_last_error(void);

/* Failure detection of the attention's kernels: a wait on one of their own barriers that takes longer than this
 * many nanoseconds gives up.  The block then sets S4D_FLAG_WAIT_TIMEOUT in the call's error_flag, waits for the
 * copies and products that it has under way and leaves NaNs in its rows of the results (a backward pass also in
 * the rows of dk and dv that those rows reach).  Applies to launches from the calling host thread; default
 * 2,000,000,000 (2 s), never expected to run out.  For tests: with 0 the kernels' copies stop half way, so that
 * waits do run out.  Returns the previous limit. */
S4D_API uint64_t s4d_decoder_set_wait_limit_ns(uint64_t limit_ns);

/* LayerNorm over rows of `width` elements (nn.LayerNorm, biased variance):
 *   y[r, :] = (x[r, :] - mean[r]) * rstd[r] * weight + bias,  rstd = 1 / sqrt(var + eps)
 *   x, y        [rows, width] of `dtype`, unit column stride, row strides x_ld / y_ld (elements;
 *               x_ld may be 0 for one broadcast row, y_ld >= width)
 *   weight/bias [width] of `param_dtype` (S4D_DTYPE_F32 or `dtype`), or NULL
 *   mean, rstd  [rows] f32, written for the backward pass; both or neither may be NULL
 * 1 <= width <= 16384.  Statistics and arithmetic are f32, rounded once into y.  y may be x (the same rows
 * at the same places); otherwise no result overlaps an argument. */
S4D_API int s4d_norm_forward(const void* x, int64_t x_ld, int dtype, const void* weight, const void* bias,
                             int param_dtype, void* y, int64_t y_ld, float* mean, float* rstd, int64_t rows,
                             int64_t width, float eps, void* stream);

/* Gradients of s4d_norm_forward: dx [rows, width] of `dtype` (NULL: not wanted), dweight and dbias
 * [width] of `param_dtype` (each NULL when not wanted) from dy, x and the saved mean and rstd.
 * dweight and dbias are sums over all rows, held in f32 and added in an order that depends on the
 * sizes alone, so that equal calls give equal bits.  rows = 0 writes zeros to them.
 * workspace: s4d_norm_backward_workspace_bytes(rows, width) bytes, 16-byte aligned, read and
 * written by this call only while it runs (may be NULL when that is 0 or neither dweight nor dbias is
 * wanted).  No result overlaps an argument. */
S4D_API size_t s4d_norm_backward_workspace_bytes(int64_t rows, int64_t width);
S4D_API int s4d_norm_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype,
                              const void* weight, int param_dtype, const float* mean, const float* rstd, void* dx,
                              int64_t dx_ld, void* dweight, void* dbias, int64_t rows, int64_t width,
                              void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention.  For batch entry b, head h (shared head g = h / (heads / kv_heads)), query i, key j:
 *   x = scale q_i.k_j;  z = softcap tanh(x / softcap), or x when softcap is 0;
 *   s = z - slope_{b,i,h} |q_pos_i - k_pos_j|   (Euclidean, pos_dim 1 or 2 coordinates);
 *   key j is seen when j < k_len[b] and q_segment_i == k_segment_j >= 0;
 *   out_i = sum_j softmax_j(s) v_j over the seen keys, 0 for a query that sees none;
 *   lse_i = log sum_j exp(s), -inf for such a query.
 * What q, k, v and the positions hold at pairs that are not seen never reaches out: an infinity or
 * a NaN there changes nothing.  An infinity in a value that is seen is one in out, unless its weight
 * underflows in `dtype` (then it may be a NaN).  Distances of two coordinates are roots of an f32 sum of squares, so
 * differences of positions stay below 2^63.  No result overlaps an argument.
 *
 *   dtype         S4D_DTYPE_BF16 or S4D_DTYPE_F16, of q, k, v and out
 *   q             [batch, queries, heads, dim], k and v [batch, keys, kv_heads, dim]: unit stride along
 *                 dim, the other strides (elements: batch, row, head) positive multiples of 8, 16-byte
 *                 aligned; the stride of an axis of one entry is not used
 *   dim           a multiple of 8, 8 to 128; heads a multiple of kv_heads
 *   out           [batch, queries, heads, dim] contiguous, 16-byte aligned
 *   lse           [batch, heads, queries] f32, or NULL
 *   slopes        f32 with strides (elements: batch, query, head; 0 allowed), when pos_dim > 0
 *   q_pos, k_pos  [batch, queries | keys, pos_dim] f32 contiguous, when pos_dim > 0
 *   q_segment, k_segment  [batch, queries | keys] int32 contiguous, both or neither NULL
 *   k_len         [batch] int32 or NULL (all keys); values outside 0 .. keys are clamped
 *   workspace     s4d_attention_forward_workspace_bytes(args) bytes, 16-byte aligned, used by this call
 *                 only while it runs (0 bytes: may be NULL)
 *   error_flag    int32 or NULL: S4D_FLAG_WAIT_TIMEOUT (see s4d_decoder_set_wait_limit_ns)
 *   softcap       0 (none), or up to 1024: a capped score is off by a few 2^-23 softcap
 * P is rounded to `dtype` for its product with v; sums and softmax statistics are f32.  Equal calls
 * give equal bits.  batch and the axes may be 0; rows of one shared head (queries * heads /
 * kv_heads) and keys must stay below 2^31.
 */
typedef struct s4d_attention_args {
  int64_t batch, queries, keys, heads, kv_heads, dim, pos_dim;
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  void* out;
  float* lse;
  const float* slopes;
  int64_t slope_stride[3];
  const float *q_pos, *k_pos;
  const int32_t *q_segment, *k_segment, *k_len;
  void* workspace;
  size_t workspace_bytes;
  int32_t* error_flag;
  float scale, softcap;
  int32_t dtype;
  int32_t dslopes_per_row; /* backward only, from here on */
  const void* dout;
  int64_t dout_stride[3];
  void *dq, *dk, *dv;
  float* dslopes;
} s4d_attention_args;

S4D_API size_t s4d_attention_forward_workspace_bytes(const s4d_attention_args* args);
S4D_API int s4d_attention_forward(const s4d_attention_args* args, void* stream);

/* Gradients of s4d_attention_forward for bf16, from the same arguments, its out and lse, and dout.
 *   dout     [batch, queries, heads, dim], strides as q's
 *   dq       [batch, queries, heads, dim] contiguous; dk, dv [batch, keys, kv_heads, dim] contiguous, or
 *            both NULL when not wanted; all 16-byte aligned
 *   dslopes  f32, or NULL: [batch, queries, heads] when dslopes_per_row, else [heads], the sum over all
 *            rows (0 without a row or a batch entry).  Positions have no gradient.
 *   workspace  s4d_attention_backward_workspace_bytes(args) bytes, 16-byte aligned
 * No atomics: equal calls give equal bits.  Pairs that are not seen take no part, whatever q, k, v,
 * dout and the positions hold there; gradients of rows that see nothing or are seen by nothing are 0.
 * At most 524288 queries and keys. */
S4D_API size_t s4d_attention_backward_workspace_bytes(const s4d_attention_args* args);
S4D_API int s4d_attention_backward(const s4d_attention_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* S4D_DECODER_H_ */
