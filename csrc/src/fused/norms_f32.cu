// Norms around a block: rows of float.
#include "norms.cuh"

int bshmem::norms::run_f32(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) { return run<float>(a, backward, stream); }
