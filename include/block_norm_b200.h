/*
 * block_norm_b200.h -- C ABI of the norms around a block in libema_ssd_b200.so (sm_100a).
 *
 * After a block, with its gate z (silu(z) = z sigmoid(z)), per group of `group_size` channels:
 *   norm_before_gate != 0:  y = x rstd(x) w silu(z)
 *   norm_before_gate == 0:  t = x silu(z),  y = t rstd(t) w
 * Before the next block, on the residual stream:
 *   h = residual + scale x  (rounded to the residual's type),  y = h rstd(h) w
 * with rstd(t) = (mean(t^2) + eps)^-1/2 over the group (the row), in fp32.
 *
 * Tensors are (rows, dim) with channel stride 1 and a row stride in elements; x, z, y, dy, dx, dz share
 * one element type, the residual stream (residual, h, dh, d_residual) has its own: the same or fp32.
 * The weight is (dim,) contiguous in any of the three types, its gradient fp32.  Launchers are
 * asynchronous on the given stream, allocate nothing and return an EMA_* code (ema_ssd_b200.h) with the
 * text in ema_last_error(); zero rows are a valid no-op (a backward then writes a zero weight gradient).
 */
#ifndef BLOCK_NORM_B200_H_
#define BLOCK_NORM_B200_H_

#include "ema_ssd_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct GatedNormArgs {
  int64_t rows, dim, group_size;
  int32_t dtype;                /* EMA_DTYPE_*: x, z, y, dy, dx, dz */
  int32_t weight_dtype;
  int32_t norm_before_gate;
  float eps;
  const void* x;  int64_t x_stride;
  const void* z;  int64_t z_stride;
  const void* weight;
  void* y;        int64_t y_stride;   /* forward only */
  /* backward */
  const void* dy; int64_t dy_stride;
  void* dx;       int64_t dx_stride;
  void* dz;       int64_t dz_stride;
  float* dweight;               /* (dim,) fp32, written (not accumulated), in a fixed order of sums */
  void* workspace;              /* block_norm_workspace_bytes(); contents need not be initialised */
  size_t workspace_bytes;
} GatedNormArgs;

typedef struct ResidualNormArgs {
  int64_t rows, dim;
  int32_t dtype;                /* x, y, dy, dx */
  int32_t residual_dtype;       /* residual, h, dh, d_residual: dtype or EMA_DTYPE_F32 */
  int32_t weight_dtype;
  float eps, scale;
  int32_t reserved;
  const void* x;        int64_t x_stride;
  const void* residual; int64_t residual_stride;  /* NULL: h = scale x */
  const void* weight;
  void* y;              int64_t y_stride;   /* forward only */
  void* h;              int64_t h_stride;   /* forward: written; backward: read */
  /* backward */
  const void* dy; int64_t dy_stride;
  const void* dh; int64_t dh_stride;        /* NULL: zero */
  void* dx;       int64_t dx_stride;
  void* d_residual; int64_t d_residual_stride;  /* NULL: not wanted */
  float* dweight;
  void* workspace;
  size_t workspace_bytes;
} ResidualNormArgs;

/* Scratch of a backward over (rows, dim) in groups of group_size (dim for the residual norm). */
EMA_API size_t block_norm_workspace_bytes(int64_t rows, int64_t dim, int64_t group_size);
EMA_API int gated_norm_fwd_launch(const GatedNormArgs* args, void* stream);
EMA_API int gated_norm_bwd_launch(const GatedNormArgs* args, void* stream);
EMA_API int residual_norm_fwd_launch(const ResidualNormArgs* args, void* stream);
EMA_API int residual_norm_bwd_launch(const ResidualNormArgs* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BLOCK_NORM_B200_H_ */
