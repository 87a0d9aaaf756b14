// Block and dense projection with int8 operands and scales per token and per
// vocabulary row (kernels and their description in block_gemm.cuh).
#include "block_gemm.cuh"

namespace gsp {

// out_dtype: 0 fp16, 1 bf16, 2 fp32 logits.
cudaError_t launch_block_gemm_int8(const BlockGemmParams& p, int out_dtype, cudaStream_t stream) {
  if (out_dtype == 2) return launch_block_gemm_typed<Int8Rows<float>>(p, stream);
  if (out_dtype == 1) return launch_block_gemm_typed<Int8Rows<__nv_bfloat16>>(p, stream);
  return launch_block_gemm_typed<Int8Rows<__half>>(p, stream);
}

}  // namespace gsp
