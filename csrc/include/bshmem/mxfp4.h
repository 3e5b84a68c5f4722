// C interface of microscaled 4-bit floating point (libbshmem_fused.so): quantisation, reading back, and the product.
//
// A matrix [R][K] (K a multiple of 32, below 2^26) is held as
//   data    [R][K/2] bytes: two E2M1 values each, the lower K in the low four bits
//   scales  E8M0, one byte per 32 values along K, in blocks of 512 bytes that hold 128 rows by 4 scales the way the tensor
//           core's scale operand wants them: row r, scale s of a block at (r % 32) * 16 + (r / 32) * 4 + s; block (rb, kb) of
//           rows 128 rb.. and K 128 kb.. at (rb * KB + kb) * 512, with KB even.  Bytes of rows and K past the end are 0.
// Quantisation (the OCP microscaling format): scale 2^(floor(log2 amax) - 2), at least 2^-127; elements x / scale rounded to the
// nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to even), saturating at 6.  A block with an infinity or a NaN gets the scale NaN.
#pragma once
#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { BSHMEM_MX_BF16 = 0, BSHMEM_MX_F16 = 1, BSHMEM_MX_F32 = 2 };
enum { BSHMEM_MX_OK = 0, BSHMEM_MX_ERR_ARGS = 1, BSHMEM_MX_ERR_SHAPE = 2, BSHMEM_MX_ERR_ALIGNMENT = 3, BSHMEM_MX_ERR_DRIVER = 4 };

/* Bytes of the scales of a matrix. */
size_t bshmem_mxfp4_scale_bytes(int64_t R, int64_t K);
/* x: [R][K] of `type`, `stride` elements between rows. */
int bshmem_mxfp4_quantize(const void* x, int type, int64_t R, int64_t K, int64_t stride, void* data, void* scales, cudaStream_t stream);
/* out: dense [R][K] of `type`. */
int bshmem_mxfp4_dequantize(const void* data, const void* scales, int64_t R, int64_t K, int type, void* out, cudaStream_t stream);

typedef struct {
  const void *x, *x_scales;  /* [M][K] */
  const void *w, *w_scales;  /* [N][K] */
  void* out;                 /* bf16 [M][N]: x w^T, accumulated in fp32 */
  int64_t M, N, K;
  uint32_t wait_limit_ms;    /* bound of the waits inside the kernel (0: 10 s) */
  int* error_flag;           /* device int; set to 1 if a wait ran out */
  /* Optional: x before quantisation, [M][K] of raw_type with raw_stride elements between rows.  It is quantised into x and x_scales
   * (which are then room for it) by a kernel of its own ahead of the product. */
  const void* raw_x;
  int raw_type;
  int64_t raw_stride;
} bshmem_mxfp4_gemm_args_t;

/* data pointers 16-byte aligned.  The sum over K is divided by a rule on M, N and K: a row's last bits may differ with the number of rows. */
int bshmem_mxfp4_gemm(const bshmem_mxfp4_gemm_args_t* args, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
