/*
 * maxsim_amd_encoder.h -- C ABI of the operators at the two ends of a training
 * step: token ids looked up in an embedding table with the table's gradient,
 * the norm of all gradients, clipping, and the AdamW step on clipped gradients.
 * None has a counterpart in the reference, whose training example leaves them
 * to torch (README.md:160-205).
 *
 * The conventions are those of maxsim_amd.h: raw device pointers, int64 sizes
 * and strides (in elements), nothing allocated, asynchronous on `stream`, a
 * status code and maxsim_amd_last_error().  Rows and tensors may start at any
 * multiple of the element size, workspaces at any multiple of 16 bytes.
 */
#ifndef MAXSIM_AMD_ENCODER_H_
#define MAXSIM_AMD_ENCODER_H_

#include "maxsim_amd_training.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Token embeddings ---------------------------------------------------- */

/* y [sequences, length, dim] = scale * weight[ids], the product rounded once.
 * weight: `vocab` rows of `dim` elements, `weight_stride` apart, in dtype or
 * float32; vocab at most 2^31 - 1 and dim at most MAXSIM_AMD_MAX_DIM.  ids
 * [sequences, length] and lengths [sequences] (or NULL: every token is real)
 * are int32, or int64 where ids64 / lengths64.  Tokens at or past a sequence's
 * length (below 0 counts as 0) become 0 and their ids are not read; a token
 * whose id is outside [0, vocab) becomes NaN.
 * rows [sequences * length] (or NULL): for the backward, each token's row of
 * the table, -1 where it has none: padding, an id outside, or padding_idx
 * (negative: none).  They need sequences * length < 2^31. */
int maxsim_amd_embed_forward(maxsim_dtype weight_dtype, maxsim_dtype dtype, const void* weight,
                             int64_t vocab, int64_t dim, int64_t weight_stride, const void* ids,
                             int ids64, int64_t sequences, int64_t length, const void* lengths,
                             int lengths64, float scale, int64_t padding_idx, void* y,
                             int32_t* rows, void* stream);

/* Bytes of workspace of the backward. */
size_t maxsim_amd_embed_backward_workspace_size(maxsim_dtype dtype, int64_t tokens, int64_t vocab,
                                                int64_t dim);

/* dweight [vocab, dim] (in weight_dtype: dtype or float32): row v is scale
 * times the sum of the rows of dy [tokens, dim], `dy_stride` apart, whose
 * entry in `rows` is v, and 0 where there is none.  Entries outside
 * [0, vocab) belong to no row.  Sums are fp32, in an order that `rows` and the
 * sizes alone decide, rounded once.  No tokens: dweight becomes 0. */
int maxsim_amd_embed_backward(maxsim_dtype weight_dtype, maxsim_dtype dtype, const void* dy,
                              int64_t dy_stride, const int32_t* rows, int64_t tokens,
                              int64_t vocab, int64_t dim, float scale, void* dweight,
                              void* workspace, size_t workspace_bytes, void* stream);

/* ---- The norm of all gradients ------------------------------------------- */

typedef struct {
  void* grad; /* [numel] of dtype */
  int64_t numel;
  maxsim_dtype dtype;
} maxsim_grad_tensor;

/* Bytes of workspace of the norm and of clipping (partial sums). */
size_t maxsim_amd_grad_norm_workspace_size(const maxsim_grad_tensor* tensors, int64_t count);

/* norm = the root of the sum of all squares of `count` tensors (host array,
 * read before the call returns), summed in 64 bits: gradients of any finite
 * size have one, in an order that the sizes alone decide.
 * factor (or NULL) = min(1, max_norm / (norm + eps)), 1 where norm + eps is 0,
 * NaN for a NaN norm. */
int maxsim_amd_grad_norm(const maxsim_grad_tensor* tensors, int64_t count, double max_norm,
                         double eps, float* norm, float* factor, void* workspace,
                         size_t workspace_bytes, void* stream);

/* The same, and every element times the factor, rounded once, in place; nothing
 * is moved where the factor is 1.  No two tensors overlap. */
int maxsim_amd_clip_grads(const maxsim_grad_tensor* tensors, int64_t count, double max_norm,
                          double eps, float* norm, float* factor, void* workspace,
                          size_t workspace_bytes, void* stream);

/* ---- AdamW on scaled gradients ------------------------------------------- */

/* maxsim_amd_adamw_step with every gradient multiplied by *grad_scale (on the
 * device, read when the kernels run; NULL: 1) on its way in.  The gradients
 * stay as they are. */
int maxsim_amd_adamw_step_scaled(maxsim_dtype param_dtype, maxsim_dtype grad_dtype, int state_bits,
                                 const maxsim_adamw_tensor* tensors, int64_t count,
                                 const float* grad_scale, double lr, const float* lr_on_device,
                                 double beta1, double beta2, double eps, double weight_decay,
                                 int64_t step, const int64_t* step_on_device, uint64_t seed,
                                 void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MAXSIM_AMD_ENCODER_H_ */
