/* iblnerf_layers.h — C ABI of the trainable-layer operators: dense layers trained from 8-bit checkpoints of their activations, and table rows by index with the table's
 * gradient by sorted tokens.  They carry what torch autograd does in a training step of the reference for networks outside the fused kernels' shape
 * (nerf_models/ibl_nerf.py:154-208, train.py:479-481); the 8-bit checkpoints and the per-view codes have no counterpart there.
 *
 * Conventions: as iblnerf.h — 0 or a negative iblnerf_status, no exceptions, "d_" pointers are device pointers borrowed for the call, all work is enqueued on `stream` and
 * nothing synchronises — with these differences:
 *   - no ctx: a call keeps nothing.  Scratch memory is the caller's (the *_workspace functions say how much; it may be reused by the next call on the same stream, and a
 *     captured graph needs one of its own).  Calls from several threads, on several streams and devices are independent; the stream must belong to the current device, and
 *     the tensors must lie on it.
 *   - iblnerf_layers_last_error() has the message of the calling thread's last failure.
 *   - `dtype` is the type T of every tensor of the call but indices, codes and scale bytes; sums are held in fp32 and rounded once.  Row strides ("ld_") are in elements,
 *     at least the row's length and at most 2^24; pointers need the alignment of their element type (codes: 8 bytes, workspace: 16 bytes).
 *   - inputs and outputs of a call may not overlap.
 *   - results depend on the inputs alone: the same call gives the same bits. */
#ifndef IBLNERF_LAYERS_H
#define IBLNERF_LAYERS_H

#include "iblnerf.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { IBLNERF_FLOAT32 = 0, IBLNERF_BFLOAT16 = 1, IBLNERF_FLOAT16 = 2 } iblnerf_dtype;

const char* iblnerf_layers_last_error(void);

/* Checkpoint of an activation x [n, k]: d_codes [n, 32 kb] bytes, d_scales [n, kb] bytes, kb = ceil(k / 32).  Per row and block of 32 columns value = code * 2^(scale - 127):
 * signed codes (two's complement) in [-127, 127], unsigned ones (is_signed = 0; negative entries become 0) in [0, 255]; the exponent is the smallest >= -126 that holds the
 * block's largest entry, codes are rounded to nearest (ties to even), a positive entry of an unsigned checkpoint keeps at least code 1.  Columns beyond k are coded 0.  A block
 * with an infinity or NaN has scale 255 and codes 1: its values are NaN.  A finite entry stays finite: what rounds up to one step beyond its type (2^128, or 65536 from float16) is
 * read as 255 * 2^120, or as 65504 where float16 is read. */
int iblnerf_checkpoint(void* stream, int dtype, const void* d_x, int64_t ld_x, int64_t n, int k, int is_signed, uint8_t* d_codes, uint8_t* d_scales);
int iblnerf_checkpoint_values(void* stream, const uint8_t* d_codes, const uint8_t* d_scales, int64_t n, int k, int is_signed, int dtype, void* d_out, int64_t ld_out);

/* y [n, o] = x [n, k] w^T + bias (w [o, k] as nn.Linear holds it; bias [o] or NULL), negative values to 0 if relu; with d_codes / d_scales (both or neither) also y's
 * checkpoint, unsigned if relu, else signed.  float32 products are taken in six bfloat16 products of the operands' three-part splits, exact for magnitudes
 * from 2^-110 on (about fp32's own accuracy; smaller operands are off by up to 2^-134, half of bfloat16's smallest step; one that is infinite or beyond 3.39e38 gives NaN). */
size_t iblnerf_dense_forward_workspace(int dtype, int64_t n, int k, int o);
int iblnerf_dense_forward(void* stream, int dtype, const void* d_x, int64_t ld_x, int64_t n, int k, const void* d_w, int64_t ld_w, int o, const void* d_bias, int relu,
                          void* d_y, int64_t ld_y, uint8_t* d_codes, uint8_t* d_scales, void* d_workspace, size_t workspace_bytes);

/* The backward of that layer from the checkpoint of its input (d_x_codes / d_x_scales, x_is_signed) and, under a ReLU, of its output (d_y_codes; NULL: no ReLU):
 *   dZ = dY where the output's code is not 0 (elsewhere 0, whatever dY holds there);  dX [n, k] = dZ w;  dW [o, k] = dZ^T X;  db [o] = sum over the rows of dZ
 * (float32 by the forward's products: an entry of dZ or w that is infinite or beyond 3.39e38 gives NaN in dX and dW, and in db, which adds up the same parts.)
 * d_dx may be NULL, d_dw and d_db may be NULL together, d_db alone may be.  d_dw and d_db are contiguous and written, not accumulated, in grad_dtype: dtype itself, or
 * IBLNERF_FLOAT32 for parameters that are kept in float32 beside 16-bit activations.  For float16 a checkpoint of float16
 * activations is read exactly (65536 as 65504); values of another origin are rounded to float16. */
size_t iblnerf_dense_backward_workspace(int dtype, int64_t n, int k, int o);
int iblnerf_dense_backward(void* stream, int dtype, const void* d_dy, int64_t ld_dy, int64_t n, int k, int o, const uint8_t* d_x_codes, const uint8_t* d_x_scales, int x_is_signed,
                           const uint8_t* d_y_codes, const void* d_w, int64_t ld_w, void* d_dx, int64_t ld_dx, int grad_dtype, void* d_dw, void* d_db, void* d_workspace,
                           size_t workspace_bytes);

/* out [n rows_per_index, d] = scale * table[index[row / rows_per_index]]; index int32 (index_bits 32) or int64 (64).  A negative index gives a row of zeros, one beyond the
 * table's v rows a row of NaN (the indices are not read on the host). */
int iblnerf_lookup(void* stream, int dtype, const void* d_table, int64_t ld_table, int64_t v, int d, const void* d_index, int index_bits, int64_t n, int64_t rows_per_index, float scale,
                   void* d_out, int64_t ld_out);

/* d table [v, d] (contiguous; written) = scale * the sum of d_dout over each token's rows; rows whose index lies outside the table count nowhere. */
size_t iblnerf_lookup_backward_workspace(int64_t n, int64_t rows_per_index, int64_t v, int d);
int iblnerf_lookup_backward(void* stream, int dtype, const void* d_dout, int64_t ld_dout, const void* d_index, int index_bits, int64_t n, int64_t rows_per_index, int64_t v, int d,
                            float scale, void* d_dtable, void* d_workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif

#endif
