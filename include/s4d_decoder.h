/*
 * s4d_decoder.h -- C ABI of the decoder's dense operators on B200 (sm_100a), the layers that
 * stand around the DeformableFeatureAggregation path of s4d_dfa.h:
 *
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

/* LayerNorm over rows of `width` elements (nn.LayerNorm, biased variance):
 *   y[r, :] = (x[r, :] - mean[r]) * rstd[r] * weight + bias,  rstd = 1 / sqrt(var + eps)
 *   x, y        [rows, width] of `dtype`, unit column stride, row strides x_ld / y_ld (elements;
 *               x_ld may be 0 for one broadcast row, y_ld >= width)
 *   weight/bias [width] of `param_dtype` (S4D_DTYPE_F32 or `dtype`), or NULL
 *   mean, rstd  [rows] f32, written for the backward pass; both or neither may be NULL
 * 1 <= width <= 16384.  Statistics and arithmetic are f32, rounded once into y. */
S4D_API int s4d_norm_forward(const void* x, int64_t x_ld, int dtype, const void* weight, const void* bias,
                             int param_dtype, void* y, int64_t y_ld, float* mean, float* rstd, int64_t rows,
                             int64_t width, float eps, void* stream);

/* Gradients of s4d_norm_forward: dx [rows, width] of `dtype` (NULL: not wanted), dweight and dbias
 * [width] of `param_dtype` (each NULL when not wanted) from dy, x and the saved mean and rstd.
 * dweight and dbias are sums over all rows, held in f32 and added in an order that depends on the
 * sizes alone, so that equal calls give equal bits.  rows = 0 writes zeros to them.
 * workspace: s4d_norm_backward_workspace_bytes(rows, width) bytes, 16-byte aligned, read and
 * written by this call only while it runs (may be NULL when neither dweight nor dbias is wanted). */
S4D_API size_t s4d_norm_backward_workspace_bytes(int64_t rows, int64_t width);
S4D_API int s4d_norm_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype,
                              const void* weight, int param_dtype, const float* mean, const float* rstd, void* dx,
                              int64_t dx_ld, void* dweight, void* dbias, int64_t rows, int64_t width,
                              void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* S4D_DECODER_H_ */
