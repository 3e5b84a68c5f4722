// C interface of the norms around a block (libbshmem_fused.so).
//
// Row by row over H values, sums and statistics in fp32:
//   z = h * rsqrt(mean(h^2) + eps) * (post + weight_offset)       z = h where `post` is null
//   r = residual_scale * residual + branch_scale * gate * z       r = residual_scale * residual where `h` is null
//   y = r * rsqrt(mean(r^2) + eps) * (pre + weight_offset)        not computed where `y` is null
// y is computed from r before its rounding to the residual's type.
// Backward takes dr and dy (either may be null: zero) and writes the gradients whose pointers are given.  It needs the
// statistics that forward left in `stat`, and computes r again from h and residual.
// No entry allocates; gradients that are sums over rows are added in a fixed order (the same bits every time).
#pragma once
#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BSHMEM_NORM_MAX_H 16384

enum { BSHMEM_NORM_BF16 = 0, BSHMEM_NORM_F16 = 1, BSHMEM_NORM_F32 = 2 };
enum { BSHMEM_NORM_GATE_NONE = 0, BSHMEM_NORM_GATE_CHANNEL = 1 /*[H]*/, BSHMEM_NORM_GATE_TOKEN = 2 /*[T]*/, BSHMEM_NORM_GATE_FULL = 3 /*[T][H]*/ };
enum { BSHMEM_NORM_OK = 0, BSHMEM_NORM_ERR_ARGS = 1, BSHMEM_NORM_ERR_SHAPE = 2, BSHMEM_NORM_ERR_DRIVER = 3 };

typedef struct {
  int T, H;
  int type;       /* of h, y and their gradients */
  int res_type;   /* of residual, r and their gradients: `type` or F32 */
  int wt_type;    /* of post, pre, gate and their gradients: `type` or F32 */
  int gate_mode;
  int64_t h_stride, res_stride, gate_stride, dr_stride, dy_stride; /* elements between rows; outputs are dense */
  float residual_scale, branch_scale, eps, weight_offset;
  const void *h, *residual, *post, *pre, *gate;
  void *r, *y;    /* forward */
  float* stat;    /* [2][T]: the two reciprocal root mean squares; forward writes it unless null, backward reads it */
  /* backward */
  const void *dr, *dy;
  void *dh, *dresidual, *dpost, *dpre, *dgate;
  int* error_flag;  /* device int; set to 1 if a copy inside a kernel did not arrive in time */
  float* partials;  /* bshmem_block_norms_partials(T, H) floats, 16-byte aligned, needed for dpost, dpre and the channel gate's gradient */
} bshmem_norm_args_t;

int bshmem_block_norms(const bshmem_norm_args_t* args, cudaStream_t stream);
int bshmem_block_norms_backward(const bshmem_norm_args_t* args, cudaStream_t stream);
size_t bshmem_block_norms_partials(int T, int H);

#ifdef __cplusplus
}
#endif
