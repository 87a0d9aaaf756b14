// Parameters and pieces shared by the fp8 head's kernels.
#pragma once

#include "fp8_quantize.cuh"
#include "gsp_common.cuh"
#include "gsp_internal.h"

namespace gsp {

struct Fp8Params {
  // hidden states: e4m3 values with scales per 128 columns, or rows still to be quantised
  const void* raw;  // raw_dtype GSP_DTYPE_*, or nullptr
  int64_t raw_stride;
  int raw_dtype;
  const uint8_t* hidden;  // (raw: the buffer for the values, written by the prologue)
  int64_t hidden_stride;
  const float* hidden_scales;  // [batch, blocks], the caller's (raw: nullptr)
  int64_t hidden_scales_stride;
  const uint8_t* weight;
  int64_t weight_stride;
  const float* weight_scales;  // [ceil(vocab / 128), blocks]
  int64_t weight_scales_stride;
  const uint32_t* mask;  // nullptr: every token legal
  int64_t mask_stride;
  int batch;
  int vocab;
  int hidden_dim;
  int nw;      // ceil(vocab / 32)
  int blocks;  // ceil(hidden_dim / 128)
  int64_t vocab_offset;
  void* logits;
  int64_t logits_stride;
  float* top_value;
  int64_t* top_index;
  int64_t* top_key;
  // scratch of this call (contents undefined on entry)
  unsigned long long* keys;  // [batch] running top-1 keys, zeroed by the prologue
  unsigned int* tickets;     // [batch] (tensor-core kernel: the first only), zeroed by the prologue
  float* scales;             // [batch, scales_stride]: the hidden states' scales
  int scales_stride;         // blocks rounded up to 4: rows of whole 16-byte vectors
  int32_t* groups;           // active 32-row vocabulary groups, kListGroups slots a builder block
  int32_t* group_counts;     // per builder block
  uint32_t* group_bits;      // the active groups as bits
  int* device_error;
  bool dense;
};

constexpr int kListGroups = 128;  // mask words of a builder block

// out_dtype: 0 fp16, 1 bf16, 2 fp32 logits.
cudaError_t launch_fp8_row_sparse(const Fp8Params& p, int out_dtype, cudaStream_t stream);
cudaError_t launch_fp8_tensor(const Fp8Params& p, int out_dtype, cudaStream_t stream);

}  // namespace gsp
