/*
 * maxsim_amd_training.h -- C ABI of the operators around the scoring kernels:
 * layer norm of an encoder's hidden states, token embeddings of unit length
 * (padded or packed) and the AdamW step.  None has a counterpart in the
 * reference, whose training example leaves them to torch (README.md:160-205).
 *
 * The conventions are those of maxsim_amd.h: raw device pointers, int64 sizes
 * and strides (in elements), nothing allocated, asynchronous on `stream`, a
 * status code and maxsim_amd_last_error().  Rows may start at any multiple of
 * the element size.  All sums and statistics are fp32; 16-bit results are
 * rounded once, to nearest even.
 */
#ifndef MAXSIM_AMD_TRAINING_H_
#define MAXSIM_AMD_TRAINING_H_

#include "maxsim_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Layer norm ---------------------------------------------------------- */

/* y [rows, dim] = (x - mean) * rstd * weight + bias over the last axis, with
 * rstd = 1 / sqrt(variance + eps) (the variance over dim, not dim - 1).
 * x: rows of `dim` elements, `row_stride` apart (0 repeats one row).  weight
 * and bias [dim] in weight_dtype (dtype or float32), either may be NULL (1 and
 * 0).  mean, rstd [rows]: what the backward needs, both or NULL.
 * dim <= MAXSIM_AMD_MAX_DIM. */
int maxsim_amd_layer_norm_forward(maxsim_dtype dtype, maxsim_dtype weight_dtype, const void* x,
                                  int64_t rows, int64_t dim, int64_t row_stride,
                                  const void* weight, const void* bias, float eps, void* y,
                                  float* mean, float* rstd, void* stream);

/* Bytes of workspace that the gradients of the weights need (partial sums). */
size_t maxsim_amd_layer_norm_backward_workspace_size(maxsim_dtype dtype, int64_t rows,
                                                     int64_t dim);

/* dx [rows, dim], dweight and dbias [dim] (in weight_dtype; each may be NULL,
 * not wanted) from dy, x and the forward's mean and rstd.  weight may be NULL
 * as in the forward.  The workspace is needed for dweight or dbias only.
 * Every sum is added in an order that the sizes alone decide. */
int maxsim_amd_layer_norm_backward(maxsim_dtype dtype, maxsim_dtype weight_dtype, const void* dy,
                                   int64_t dy_stride, const void* x, int64_t x_stride,
                                   const float* mean, const float* rstd, const void* weight,
                                   int64_t rows, int64_t dim, void* dx, void* dweight,
                                   void* dbias, void* workspace, size_t workspace_bytes,
                                   void* stream);

/* ---- Unit rows ----------------------------------------------------------- */

/* y = x / max(|x|, eps) for each row of x [sequences, length, dim] (sequences
 * x_seq_stride and rows x_row_stride apart), rows of any finite length; eps at
 * least 2^-126; `length` below 2^31 (more rows: as many sequences of one).
 * lengths NULL: every row.  lengths [sequences], int32 (lengths64 0) or int64
 * (1): rows at or past a sequence's
 * length (below 0 counts as 0) are not read.  offsets NULL: y is
 * [sequences, length, dim] and those rows are 0.  offsets [sequences]: y is
 * [packed_rows, dim], row t of sequence s at offsets[s] + t, and they have no
 * row; nothing is written outside y. */
int maxsim_amd_unit_rows_forward(maxsim_dtype dtype, const void* x, int64_t sequences,
                                 int64_t length, int64_t dim, int64_t x_seq_stride,
                                 int64_t x_row_stride, const void* lengths, int lengths64,
                                 const int32_t* offsets, int64_t packed_rows, float eps, void* y,
                                 void* stream);

/* dx [sequences, length, dim] from dy (shaped as y; the strides are those of a
 * padded dy) and x.  Rows that the lengths leave out get 0, and neither x nor
 * dy is read there. */
int maxsim_amd_unit_rows_backward(maxsim_dtype dtype, const void* dy, int64_t dy_seq_stride,
                                  int64_t dy_row_stride, const void* x, int64_t sequences,
                                  int64_t length, int64_t dim, int64_t x_seq_stride,
                                  int64_t x_row_stride, const void* lengths, int lengths64,
                                  const int32_t* offsets, int64_t packed_rows, float eps, void* dx,
                                  void* stream);

/* clamped[s] = lengths[s] in [0, max_len]; offsets[0] = 0 and
 * offsets[s + 1] = offsets[s] + clamped[s], for `sequences` lengths (int32, or
 * int64 where lengths64).  total, if not NULL, is a zeroed word of pinned host
 * memory that gets 2 * offsets[sequences] + 1, for a host that waits for the
 * size alone. */
int maxsim_amd_length_offsets(const void* lengths, int lengths64, int64_t sequences,
                              int64_t max_len, int32_t* clamped, int32_t* offsets,
                              uint64_t* total, void* stream);

/* ---- AdamW --------------------------------------------------------------- */

/* Elements that share the scales of their 8-bit states. */
#define MAXSIM_AMD_STATE_BLOCK 256

typedef struct {
  void* param;       /* [numel] of param_dtype, updated */
  const void* grad;  /* [numel] of grad_dtype */
  void* exp_avg;     /* [numel] fp32, or 8-bit codes, updated */
  void* exp_avg_sq;  /* the same */
  uint8_t* scales;   /* 8-bit states: [ceil(numel / 256)][2], updated; else NULL */
  float* master;     /* fp32 [numel] copy of a 16-bit parameter that the step is
                        taken on, param being its rounding; or NULL */
  int64_t numel;
  uint64_t position; /* of element 0 among the elements of a step, for the random
                        bits of 8-bit states: a multiple of 256 */
} maxsim_adamw_tensor;

/* One AdamW step with decoupled weight decay over `count` tensors (host array,
 * read before the call returns; nothing that one of them updates overlaps
 * another's):
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
 *   p = p (1 - lr weight_decay)
 *       - lr / (1 - beta1^step) m / (sqrt(v) / sqrt(1 - beta2^step) + eps).
 * param_dtype: fp32, fp16 or bf16; grad_dtype: the same or fp32; state_bits 32
 * or 8.  lr_on_device and step_on_device, where not NULL, are read when the
 * kernels run in place of lr and step (a captured graph's next replays see new
 * values).  8-bit states start as zeros, scales among them; they are rounded
 * up or down at random by (seed, step, position). */
int maxsim_amd_adamw_step(maxsim_dtype param_dtype, maxsim_dtype grad_dtype, int state_bits,
                          const maxsim_adamw_tensor* tensors, int64_t count, double lr,
                          const float* lr_on_device, double beta1, double beta2, double eps,
                          double weight_decay, int64_t step, const int64_t* step_on_device,
                          uint64_t seed, void* stream);

/* The values that 8-bit states stand for, in bf16 (exact). */
int maxsim_amd_adamw_state_values(const uint8_t* exp_avg, const uint8_t* exp_avg_sq,
                                  const uint8_t* scales, int64_t numel, void* values,
                                  void* values_sq, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MAXSIM_AMD_TRAINING_H_ */
