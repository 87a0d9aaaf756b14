// Block and dense projection with fp16 and bf16 operands (kernels and their
// description in block_gemm.cuh).
#include "block_gemm.cuh"

namespace gsp {

cudaError_t launch_block_gemm(const BlockGemmParams& p, int dtype, cudaStream_t stream) {
  if (dtype == 1) return launch_block_gemm_typed<__nv_bfloat16>(p, stream);
  return launch_block_gemm_typed<__half>(p, stream);
}

}  // namespace gsp
