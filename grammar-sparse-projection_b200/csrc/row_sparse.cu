// Row-sparse projection with fp16, bf16 and fp32 operands (kernels and their
// description in row_sparse.cuh).
#include "row_sparse.cuh"

namespace gsp {

cudaError_t launch_row_sparse(const RowSparseParams& p, int dtype, cudaStream_t stream) {
  const bool sample = p.sample_index != nullptr;
  if (dtype == 2) {
    if (sample) return cudaErrorNotSupported;  // the sampler takes half-precision inputs only
    return launch_row_sparse_typed<float, false>(p, stream);
  }
  if (dtype == 1) return sample ? launch_row_sparse_typed<__nv_bfloat16, true>(p, stream) : launch_row_sparse_typed<__nv_bfloat16, false>(p, stream);
  return sample ? launch_row_sparse_typed<__half, true>(p, stream) : launch_row_sparse_typed<__half, false>(p, stream);
}

}  // namespace gsp
