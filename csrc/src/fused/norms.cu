// Norms before and after a block, fused with the block's gate and the scaled residual: the C entry points.
#include "../../include/bshmem/norms.h"

namespace bshmem {
namespace norms {

int run_bf16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);
int run_f16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);
int run_f32(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);

static int check(const bshmem_norm_args_t* a) {
  if (!a || a->T < 0 || a->H < 1 || a->H > BSHMEM_NORM_MAX_H) return BSHMEM_NORM_ERR_SHAPE;
  if (a->type < 0 || a->type > 2 || (a->res_type != a->type && a->res_type != BSHMEM_NORM_F32) || (a->wt_type != a->type && a->wt_type != BSHMEM_NORM_F32)) return BSHMEM_NORM_ERR_ARGS;
  if (a->gate_mode < 0 || a->gate_mode > 3 || (a->gate_mode && (!a->gate || !a->h)) || !a->residual || (a->post && !a->h)) return BSHMEM_NORM_ERR_ARGS;
  if ((a->y || a->dy) && !a->pre) return BSHMEM_NORM_ERR_ARGS;
  return BSHMEM_NORM_OK;
}

static int run(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) {
  return a->type == BSHMEM_NORM_BF16 ? run_bf16(a, backward, stream) : a->type == BSHMEM_NORM_F16 ? run_f16(a, backward, stream) : run_f32(a, backward, stream);
}

}  // namespace norms
}  // namespace bshmem

using namespace bshmem::norms;

// Two sums per column and CTA: at most eight CTAs of 64 threads an SM, and no more than there are rows.
extern "C" size_t bshmem_block_norms_partials(int T, int H) {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return T > 0 && H > 0 ? (size_t)(T < sms * 8 ? T : sms * 8) * 2 * H : 0;
}

extern "C" int bshmem_block_norms(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  if ((!a->r && !a->y) || !a->error_flag) return BSHMEM_NORM_ERR_ARGS;
  return run(a, false, stream);
}

extern "C" int bshmem_block_norms_backward(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  const bool sums = a->dpost || a->dpre || (a->dgate && a->gate_mode == BSHMEM_NORM_GATE_CHANNEL);
  if ((!a->dr && !a->dy) || (a->dpre && !a->dy) || (a->dpost && !a->post) || ((a->dh || a->dgate) && !a->h) || (a->dgate && !a->gate_mode)) return BSHMEM_NORM_ERR_ARGS;
  if ((sums && (!a->partials || ((uintptr_t)a->partials & 15))) || ((a->post || a->dy) && !a->stat) || !a->error_flag) return BSHMEM_NORM_ERR_ARGS;
  bshmem_norm_args_t args = *a;
  if (!sums) args.partials = nullptr;
  return run(&args, true, stream);
}
