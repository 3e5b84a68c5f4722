// Norms around a block: rows of __half.
#include "norms.cuh"

int bshmem::norms::run_f16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) { return run<__half>(a, backward, stream); }
