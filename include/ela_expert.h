/*
 * ela_expert.h -- C ABI of the expert-layer operators that follow a token-to-
 * expert assignment (libela_auction.so, built from
 * efficient-linear-assignment_b200/csrc/ela_expert.cu and ela_expert_linear.cu).
 *
 * Conventions as in ela_auction.h: plain pointers and sizes, device pointers on
 * the current CUDA device, work enqueued on `stream` and not waited for, status
 * codes ELA_*, element types ELA_DTYPE_*.  Matrices are row-major with unit
 * stride inside a row; `ld*` is the distance between rows in elements.  Pointers lie on
 * whole elements, workspaces on 16 bytes (ELA_ERR_ARGUMENT otherwise).
 *
 * Notation: T tokens, k choices per token, slots s = t*k + j; a slot's bucket is
 * its expert, or E when the expert is outside [0, E) (the solver's -1: no
 * expert).  R = T*k rows sorted by bucket, stable in s.  Row r of the sorted
 * order belongs to expert e when offsets[e] <= r < offsets[e+1]; rows at or past
 * offsets[E] belong to no expert.  Offsets and positions are read with bounds
 * checks: values out of range never lead out of a buffer.
 */
#ifndef ELA_EXPERT_H
#define ELA_EXPERT_H

#include <stddef.h>
#include <stdint.h>

#include "ela_auction.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activation in the product's epilogue.  GELU is the erf form. */
enum { ELA_ACT_NONE = 0, ELA_ACT_RELU = 1, ELA_ACT_GELU = 2, ELA_ACT_SILU = 3 };

/* Largest number of experts. */
#define ELA_EXPERT_MAX 4096

/* Bytes of device workspace ela_expert_plan needs (0 is a valid answer). */
size_t ela_expert_plan_workspace_bytes(int64_t slots, int64_t num_experts);

/*
 * Stable sort of the slots by expert.
 *   expert      device int32 or int64 (id_bytes 4 or 8), contiguous [slots]
 *   offsets     device int32[E+1]; offsets[e] = number of slots in buckets < e
 *   position    device int32[slots]; the sorted row of each slot
 *   source      device int32[slots]; the slot of each sorted row
 * Slots without an expert take the last rows.  1 <= E <= ELA_EXPERT_MAX,
 * slots < 2^31.
 */
int ela_expert_plan(const void* expert, int id_bytes, int64_t slots, int64_t num_experts, int32_t* offsets,
                    int32_t* position, int32_t* source, void* workspace, size_t workspace_bytes, void* stream);

/*
 * rows[position[t*k+j]] = x[t] where the position is below offsets[E], else 0.
 * x (T,H) with row distance ldx, rows (T*k,H) contiguous; fp32, fp16 or bf16.
 */
int ela_expert_dispatch(const void* x, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldx,
                        const int32_t* position, const int32_t* offsets, int64_t num_experts, void* rows,
                        void* stream);

/*
 * out[t] = sum over j with position below offsets[E] of w[t*k+j] * y[position[t*k+j]],
 * summed in fp32 in the order of j and rounded once.  weights: float or `dtype`
 * (weights_dtype), contiguous [T*k], or NULL for 1.  y (T*k,H) with row distance
 * ldy, out (T,H) contiguous.
 */
int ela_expert_combine(const void* y, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldy,
                       const int32_t* position, const int32_t* offsets, int64_t num_experts, const void* weights,
                       int weights_dtype, void* out, void* stream);

/*
 * Gradient of the above: dy[position[t*k+j]] = w[t*k+j] * dout[t] (0 for rows of
 * no expert) and dweights[t*k+j] = <dout[t], y[position[t*k+j]]> (0 where the slot
 * has no expert).  dy or dweights may be NULL.  dout (T,H) with row distance lddo;
 * dy contiguous; dweights in weights_dtype.  y is only read for dweights.
 */
int ela_expert_combine_grad(const void* dout, const void* y, int dtype, int64_t T, int64_t k, int64_t H,
                            int64_t lddo, int64_t ldy, const int32_t* position, const int32_t* offsets,
                            int64_t num_experts, const void* weights, int weights_dtype, void* dy, void* dweights,
                            void* stream);

/* Which pass of the linear operator (for the workspace query). */
enum { ELA_LINEAR_FORWARD = 0, ELA_LINEAR_GRAD_INPUT = 1, ELA_LINEAR_GRAD_WEIGHT = 2, ELA_LINEAR_GRAD_ACT = 3 };

/*
 * Bytes of device workspace a pass of the linear operator needs at these sizes.
 * `aligned`: every matrix that the pass reads starts on a 16-byte boundary and has
 * rows (and expert matrices) a multiple of 16 bytes apart.
 */
size_t ela_expert_linear_workspace_bytes(int pass, int64_t R, int64_t E, int64_t K, int64_t N, int aligned);

/*
 * y[r] = act(W_e x[r] + b_e) + residual[r] for the rows r of each expert e;
 * y[r] = residual[r] (0 without one) for rows of no expert.
 *   x (R,K) ldx; weight (E,N,K): expert distance stride_e, row distance ldw;
 *   bias (E,N) contiguous or NULL; residual (R,N) ldr or NULL; offsets int32[E+1],
 *   or NULL when E == 1 (every row is expert 0's);
 *   y (R,N) contiguous; z (R,N) contiguous or NULL: receives W_e x + b_e, what the
 *   gradient of the activation needs (rows of no expert unwritten): float for
 *   ELA_ACT_GELU and ELA_ACT_SILU; otherwise rounded to dtype, for ELA_ACT_RELU with
 *   the sign of the sum (sums within rounding of 0 are formed again).
 * dtype: fp16 or bf16; products are summed in fp32 and y is rounded once.
 */
int ela_expert_linear(const void* x, const void* weight, const void* bias, const void* residual,
                      const int32_t* offsets, int dtype, int64_t R, int64_t E, int64_t K, int64_t N, int64_t ldx,
                      int64_t stride_e, int64_t ldw, int64_t ldr, int activation, void* y, void* z, void* workspace,
                      size_t workspace_bytes, void* stream);

/*
 * dz = dy * act'(z), and dbias[e] = sum of dz over the expert's rows (fp32 sums in a
 * fixed order).  dy, z, dz (R,N) contiguous, z as ela_expert_linear writes it.  dz NULL when only dbias is wanted;
 * dbias (E,N) or NULL; z NULL for ELA_ACT_NONE.  Rows of no expert: dz unwritten.
 */
int ela_expert_linear_grad_act(const void* dy, const void* z, const int32_t* offsets, int dtype, int64_t R,
                               int64_t E, int64_t N, int activation, void* dz, void* dbias, void* workspace,
                               size_t workspace_bytes, void* stream);

/* dx[r] = dz[r] W_e for the rows of each expert, 0 for rows of no expert.  dz (R,N), dx (R,K) contiguous. */
int ela_expert_linear_grad_input(const void* dz, const void* weight, const int32_t* offsets, int dtype, int64_t R,
                                 int64_t E, int64_t K, int64_t N, int64_t stride_e, int64_t ldw, void* dx,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* dweight[e] = sum over the expert's rows of dz[r] x[r]^T; dz (R,N) contiguous, x (R,K) ldx, dweight (E,N,K) contiguous. */
int ela_expert_linear_grad_weight(const void* dz, const void* x, const int32_t* offsets, int dtype, int64_t R,
                                  int64_t E, int64_t K, int64_t N, int64_t ldx, void* dweight, void* workspace,
                                  size_t workspace_bytes, void* stream);

/*
 * Error of the linear kernels on the current device since the last call: ELA_OK, or
 * ELA_ERR_TIMEOUT when a device-side wait ran out (the results of that call are
 * incomplete).  Waits for the device and clears the error.
 */
int ela_expert_status(int* status);

#ifdef __cplusplus
}
#endif

#endif /* ELA_EXPERT_H */
