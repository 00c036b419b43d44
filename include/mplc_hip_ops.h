/*
 * mplc_hip_ops.h - operators on lockstep batches of models (part of the mplc_hip.h C ABI): a dense layer of any size
 * with its epilogue and its gradients, and the orthogonalised (Muon) update of weight matrices.
 *
 * A batch holds n_models models.  Every tensor is addressed as base + model * <t>_stride + row * <t>_ld + column, in
 * elements, with unit stride along a row: a matrix may be a view into the models' parameter rows (model stride =
 * MPLC_CNN_STRIDE, ld = its columns).  Any alignment of the element type is accepted.
 *
 * Conventions are those of mplc_hip.h: device pointers, caller-owned buffers and workspace, work enqueued on `stream`,
 * nothing synchronises, MPLC_E_ARG / MPLC_E_WORKSPACE / MPLC_E_SHAPE before anything is enqueued.  All launches are
 * plain kernels (no memset, copy or allocation), so a call can be captured into a graph; calls that may run at the same
 * time, or captured graphs that may, need workspaces of their own.  Results do not depend on timing: no atomics.
 */
#ifndef MPLC_HIP_OPS_H
#define MPLC_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MPLC_DTYPE_F32 0
#define MPLC_DTYPE_BF16 1
#define MPLC_DTYPE_F16 2

#define MPLC_ACT_NONE 0
#define MPLC_ACT_RELU 1
#define MPLC_ACT_GELU 2 /* z (1 + erf(z / sqrt 2)) / 2; relative error before the rounding to dtype below 2^-19 (16-bit
                         * types 2^-16) in the negative tail too, down to results of 2^-120                             */
#define MPLC_ACT_SILU 3 /* z / (1 + exp(-z)) */

/* ------------------------------------------------------------------------------------------------
 * Dense layer, batched over models:
 *   z[g] = x[g] w[g] + bias[g],   y[g] = act(z[g]) + residual[g],   rows r < counts[g]
 * x [rows][in], w [in][out] (the framework's kernel layout), bias [out], residual / y / z [rows][out].  x, w, bias,
 * residual, y and the gradients have the type `dtype`; sums are fp32 and each result is rounded to dtype once.  z is
 * kept in fp32 for the backward pass (a 16-bit z would add its rounding to every gradient).
 * x_shared != 0: all models read the one x [rows][in] (x_stride is ignored).
 * counts (NULL = every row): rows of each model's batch; values outside [0, rows] are clamped.  Rows at or behind a
 * model's count are neither read nor written.
 * Backward, from dy and z (z is read only for an activation):
 *   dz = dy act'(z),  dx = dz w^T (x_shared: summed over the models),  dw = x^T dz,  db = sum over the rows of dz
 * A model adds nothing to the rows of a shared x's dx behind its count, whatever its weights hold; a row that no model
 * reaches gets 0.  act'(0) = 0 for relu.  The gradient of the residual is dy.  Each of dx, dw, db may be NULL (not wanted).  A model
 * whose count is 0 gets dw = db = 0.  Where an activation is differentiated, dz enters the two products rounded to
 * dtype; db is summed before that rounding.
 * ---------------------------------------------------------------------------------------------- */
typedef struct {
  int32_t n_models, rows, in, out;
  int32_t dtype, activation, x_shared, pad0;
  const int32_t* counts;  /* [n_models] or NULL                      */
  const void* x;
  int64_t x_stride, x_ld;
  const void* w;
  int64_t w_stride, w_ld;
  const void* bias;  /* NULL = none (forward)                          */
  int64_t bias_stride;
  const void* residual;  /* NULL = none (forward)                      */
  int64_t residual_stride, residual_ld;
  void* y; /* forward output                                         */
  int64_t y_stride, y_ld;
  float* z; /* forward: written unless NULL; backward: read if activation != NONE */
  int64_t z_stride, z_ld;
  const void* dy; /* backward                                          */
  int64_t dy_stride, dy_ld;
  void* dx;
  int64_t dx_stride, dx_ld;
  void* dw;
  int64_t dw_stride, dw_ld;
  void* db;
  int64_t db_stride;
  void* workspace; /* 16-byte aligned                                  */
  size_t workspace_bytes;
} mplc_dense_t;

/* Bytes of workspace the call needs (0 possible); only sizes, dtype, activation, x_shared and which of dx / dw / db are
 * wanted are read. */
size_t mplc_dense_forward_workspace_bytes(const mplc_dense_t* t);
size_t mplc_dense_backward_workspace_bytes(const mplc_dense_t* t);
int mplc_dense_forward(const mplc_dense_t* t, void* stream);
int mplc_dense_backward(const mplc_dense_t* t, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Orthogonalised update.  For each model's matrix U [rows][cols]:
 *   X_0 = U / |U|_F,   X_{t+1} = a X_t + b (X_t X_t^T) X_t + c (X_t X_t^T)^2 X_t,   O(U) = X_steps
 * which acts on the singular values alone: s -> a s + b s^3 + c s^5.  O(0) = 0; a matrix that holds an infinity or a NaN
 * gives NaN throughout, and leaves the other models' results alone.  O does not depend on the scale of U.
 * Requirements: 1 <= steps <= 16, and the singular values must stay in [0, 2]: the largest |a s + b s^3 + c s^5| over the
 * range reached so far, from [0, 1], may not exceed 2 at any step (MPLC_E_ARG otherwise).
 *   mplc_orthogonalize:  out = O(g), in dtype.
 *   mplc_muon_step:      m = beta m + g;  u = nesterov ? g + beta m : m;  w = (1 - lr * weight_decay) w - lr * scale * O(u)
 *                        with fp32 m and w, updated in place; g in dtype.
 * ---------------------------------------------------------------------------------------------- */
typedef struct {
  int32_t n_models, rows, cols, dtype;
  int32_t steps, nesterov;
  int32_t invariant;  /* != 0: a model's result does not depend on n_models (sums are split as for 16 models) */
  float a, b, c;
  float lr, beta, weight_decay, scale;
  const void* g;
  int64_t g_stride, g_ld;
  void* out; /* mplc_orthogonalize                                     */
  int64_t out_stride, out_ld;
  float* m; /* mplc_muon_step                                         */
  int64_t m_stride, m_ld;
  float* w;
  int64_t w_stride, w_ld;
  void* workspace; /* 16-byte aligned                                  */
  size_t workspace_bytes;
} mplc_muon_t;

/* Bytes of workspace of either call; only sizes, dtype, steps and invariant are read. */
size_t mplc_muon_workspace_bytes(const mplc_muon_t* t);
int mplc_orthogonalize(const mplc_muon_t* t, void* stream);
int mplc_muon_step(const mplc_muon_t* t, void* stream);

/* Layout query (checked when the host binds): sizeof(mplc_dense_t) for 0, sizeof(mplc_muon_t) for 1, else -1. */
int64_t mplc_ops_layout(int what);

#ifdef __cplusplus
}
#endif

#endif /* MPLC_HIP_OPS_H */
