// Norms around a block: rows of __nv_bfloat16.
#include "norms.cuh"

int bshmem::norms::run_bf16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) { return run<__nv_bfloat16>(a, backward, stream); }
