// C interface of the expert router and its balance loss (libbshmem_fused.so).
//
// route: the K experts of every token and their weights, from logits [T][E].
//   choice   the K largest logits, or the K largest of score + bias where `bias` is given (computed in 64 bits, so that the
//            order does not depend on roundings of the exponential); ties go to the lowest expert.  A logit (or score + bias)
//            that is -inf or NaN is never chosen; places left over get expert -1 and weight 0.  The softmax of the biased choice is
//            taken over the logits that are numbers, and those of +inf share it evenly.
//   weight   the score of the chosen expert (softmax over all experts, or sigmoid), divided by the sum over the chosen ones
//            where `renormalize` is set, times `scale`; NaN for a softmax with a NaN or +inf among the token's logits
// balance: loss = E * sum_e f_e P_e over the n valid tokens, f_e = counts_e / (n K), P_e = mean over them of the softmax of the
//   logits (or of the sigmoids divided by their sum)
// A token whose `valid` byte is 0 gets experts -1 and weights 0, counts nowhere and has a gradient of 0.
// No entry allocates.  Sums over tokens are taken in a fixed order.
#pragma once
#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BSHMEM_ROUTE_MAX_EXPERTS 1024
#define BSHMEM_ROUTE_MAX_TOPK 16

enum { BSHMEM_ROUTE_BF16 = 0, BSHMEM_ROUTE_F16 = 1, BSHMEM_ROUTE_F32 = 2 };
enum { BSHMEM_ROUTE_SOFTMAX = 0, BSHMEM_ROUTE_SIGMOID = 1 };
enum { BSHMEM_ROUTE_OK = 0, BSHMEM_ROUTE_ERR_ARGS = 1, BSHMEM_ROUTE_ERR_SHAPE = 2, BSHMEM_ROUTE_ERR_DRIVER = 3 };

typedef struct {
  int T, E, K, type, score, renormalize;
  int64_t stride;           /* elements between rows of the logits; dlogits is dense */
  float scale;
  const void* logits;
  const float* bias;        /* [E] or null */
  const uint8_t* valid;     /* [T] or null */
  int32_t* idx;             /* [T][K]: written by route, read by the other entries */
  float* weight;            /* [T][K] */
  /* route, backward */
  const float* dweight;     /* [T][K] */
  void* dlogits;            /* [T][E] of the logits' type */
  /* balance */
  float* loss;              /* [1] */
  int32_t* counts;          /* [E] */
  float* coef;              /* [E]: dloss / dp_te less its mean over e; written by balance unless null, read by its backward */
  void* workspace;          /* bshmem_balance_workspace(T, E) bytes */
  const float* dloss;       /* [1], device */
} bshmem_route_args_t;

int bshmem_route(const bshmem_route_args_t* args, cudaStream_t stream);
int bshmem_route_backward(const bshmem_route_args_t* args, cudaStream_t stream);
int bshmem_balance(const bshmem_route_args_t* args, cudaStream_t stream);
int bshmem_balance_backward(const bshmem_route_args_t* args, cudaStream_t stream);
size_t bshmem_balance_workspace(int T, int E);

#ifdef __cplusplus
}
#endif
