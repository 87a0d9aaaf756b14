// Rows to e4m3 with a scale per 128 columns, and weights to e4m3 with a scale per
// 128 x 128 block (sm_100a), for the fp8 head (rules in fp8_quantize.cuh).
//
// One pass over memory, bound by its bytes (2 or 4 read, 1 written per element).
// Rows: 16 or 32 lanes hold a block (64 x 2,048 bf16 3 us, 16,384 x 8,192 128 us, 3.1 TB/s:
// one vector a thread under way). Weights: a CTA holds a block in the rows' own type, eight
// units a thread (248,320 x 2,048 fp16 355 us, 4.3 TB/s; held as fp32 766).
#include <algorithm>

#include "../../include/gsp_b200.h"
#include "fp8_quantize.cuh"
#include "gsp_internal.h"

namespace gsp {
namespace {

constexpr int kThreads = 256;

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    quantize_rows_fp8_kernel(const typename DTypeTraits<T>::Bits* __restrict__ src, int64_t src_stride, int64_t rows,
                             int cols, uint8_t* values, int64_t values_stride, float* scales, int64_t scales_stride) {
  using U = Units<T, kVec>;
  constexpr int kE = U::kElems;
  const int n = U::count(cols), width = (n + 31) & ~31;  // (whole warps within a row)
  const int64_t total = rows * width, step = (int64_t)gridDim.x * kThreads;
  for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < total; at += step) {
    // (the 64-bit division is some 100 instructions)
    const int64_t row = total <= 0xffffffffll ? (int64_t)((uint32_t)at / (uint32_t)width) : at / width;
    const int i = (int)(at - row * width);
    float f[kE];
    uint32_t top = 0u;
    if (i < n) {
      U::load(src + row * src_stride, i, cols, f);
      top = U::magnitude(f);
    }
    const BlockScale s = block_scale(lanes_max<U::kLanes>(top));
    if (i >= n) continue;
    uint32_t w[kE / 4];
#pragma unroll
    for (int k = 0; k < kE / 4; ++k) w[k] = to_e4m3(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3], s);
    U::store_bytes(values + row * values_stride, i, cols, w);
    if (i % U::kLanes == 0) scales[row * scales_stride + i / U::kLanes] = s.scale;
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    quantize_weight_fp8_kernel(const typename DTypeTraits<T>::Bits* __restrict__ src, int64_t src_stride, int rows,
                               int cols, uint8_t* values, int64_t values_stride, float* scales, int64_t scales_stride,
                               int col_blocks) {
  using U = Units<T, kVec>;
  constexpr int kE = U::kElems;
  constexpr int kRowsAtOnce = kThreads / U::kLanes, kSteps = kBlock / kRowsAtOnce;
  __shared__ uint32_t s_top[kThreads / 32];
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  const int lane_unit = threadIdx.x % U::kLanes, first = threadIdx.x / U::kLanes;
  const int i = cb * U::kLanes + lane_unit, n = U::count(cols);
  uint4 held[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int row = rb * kBlock + k * kRowsAtOnce + first;
    held[k] = row < rows && i < n ? U::load_packed(src + (int64_t)row * src_stride, i, cols) : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t top = 0u;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    float f[kE];
    U::unpack(held[k], f);
    top = max(top, U::magnitude(f));
  }
  top = __reduce_max_sync(FULL_MASK, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int k = 0; k < kThreads / 32; ++k) top = max(top, s_top[k]);
  const BlockScale s = block_scale(top);
  if (threadIdx.x == 0) scales[rb * scales_stride + cb] = s.scale;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int row = rb * kBlock + k * kRowsAtOnce + first;
    if (row >= rows || i >= n) continue;
    float f[kE];
    U::unpack(held[k], f);
    uint32_t w[kE / 4];
#pragma unroll
    for (int q = 0; q < kE / 4; ++q) w[q] = to_e4m3(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3], s);
    U::store_bytes(values + (int64_t)row * values_stride, i, cols, w);
  }
}

template <typename T>
bool vector_rows(const void* src, int64_t src_stride, int64_t rows, int cols, const void* values, int64_t values_stride) {
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  return cols % kPer == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0 &&
         reinterpret_cast<uintptr_t>(values) % kPer == 0 &&
         (rows == 1 || (src_stride * (int64_t)sizeof(T) % 16 == 0 && values_stride % kPer == 0));
}

template <typename T>
cudaError_t launch_rows(const void* src, int64_t src_stride, int64_t rows, int cols, uint8_t* values,
                        int64_t values_stride, float* scales, int64_t scales_stride, cudaStream_t stream) {
  int dev = 0;
  const cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const auto* s = static_cast<const typename DTypeTraits<T>::Bits*>(src);
  const bool vec = vector_rows<T>(src, src_stride, rows, cols, values, values_stride);
  const int64_t units = vec ? cols / DTypeTraits<T>::kPerVec : ((int64_t)cols + kBlock - 1) / kBlock * 32;
  const int64_t blocks = (rows * ((units + 31) / 32 * 32) + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, (int64_t)num_sms(dev) * 64);
  if (vec)
    quantize_rows_fp8_kernel<T, true><<<grid, kThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, scales_stride);
  else
    quantize_rows_fp8_kernel<T, false><<<grid, kThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, scales_stride);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_weight(const void* src, int64_t src_stride, int rows, int cols, uint8_t* values,
                          int64_t values_stride, float* scales, int64_t scales_stride, cudaStream_t stream) {
  const auto* s = static_cast<const typename DTypeTraits<T>::Bits*>(src);
  const int cb = (cols + kBlock - 1) / kBlock;
  const int64_t grid = ((int64_t)rows + kBlock - 1) / kBlock * cb;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (vector_rows<T>(src, src_stride, rows, cols, values, values_stride))
    quantize_weight_fp8_kernel<T, true><<<(unsigned)grid, kThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, scales_stride, cb);
  else
    quantize_weight_fp8_kernel<T, false><<<(unsigned)grid, kThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, scales_stride, cb);
  return cudaGetLastError();
}

int32_t check(const char* fn, const void* src, int64_t src_row_stride, int64_t rows, int32_t cols, int32_t dtype,
              const void* values, int64_t values_row_stride, const void* scales, int64_t scales_row_stride) {
  if (rows < 0 || cols < 1) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: rows must be >= 0 and cols positive", fn);
  if (dtype != GSP_DTYPE_F16 && dtype != GSP_DTYPE_BF16 && dtype != GSP_DTYPE_F32)
    return record_error(GSP_ERR_UNSUPPORTED, "%s: dtype must be GSP_DTYPE_F16, GSP_DTYPE_BF16 or GSP_DTYPE_F32", fn);
  if (rows == 0) return GSP_OK;
  if (rows > INT32_MAX) return record_error(GSP_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", fn);
  if (cols > (1 << 24)) return record_error(GSP_ERR_UNSUPPORTED, "%s: more than 2^24 columns", fn);
  if (!src || !values || !scales)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: src, values and scales are required", fn);
  if (rows > 1 && (src_row_stride < 0 || values_row_stride < cols || scales_row_stride < (cols + kBlock - 1) / kBlock))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: a row stride is negative or shorter than its row", fn);
  return GSP_OK;
}

int32_t status(const char* fn, cudaError_t err) {
  if (err == cudaSuccess) return GSP_OK;
  return record_error(GSP_ERR_CUDA, "%s: %s (%s)", fn, cudaGetErrorName(err), cudaGetErrorString(err));
}

}  // namespace
}  // namespace gsp

using namespace gsp;

extern "C" {

int32_t gsp_quantize_rows_fp8(const void* src, int64_t src_row_stride, int64_t rows, int32_t cols, int32_t dtype,
                              uint8_t* values, int64_t values_row_stride, float* scales, int64_t scales_row_stride,
                              void* stream) {
  const char* fn = "gsp_quantize_rows_fp8";
  const int32_t st = check(fn, src, src_row_stride, rows, cols, dtype, values, values_row_stride, scales, scales_row_stride);
  if (st != GSP_OK || rows == 0) return st;
  auto launch = dtype == 2 ? launch_rows<float> : dtype == 1 ? launch_rows<__nv_bfloat16> : launch_rows<__half>;
  return status(fn, launch(src, src_row_stride, rows, cols, values, values_row_stride, scales, scales_row_stride,
                           static_cast<cudaStream_t>(stream)));
}

int32_t gsp_quantize_weight_fp8(const void* src, int64_t src_row_stride, int64_t rows, int32_t cols, int32_t dtype,
                                uint8_t* values, int64_t values_row_stride, float* scales, int64_t scales_row_stride,
                                void* stream) {
  const char* fn = "gsp_quantize_weight_fp8";
  const int32_t st = check(fn, src, src_row_stride, rows, cols, dtype, values, values_row_stride, scales, scales_row_stride);
  if (st != GSP_OK || rows == 0) return st;
  auto launch = dtype == 2 ? launch_weight<float> : dtype == 1 ? launch_weight<__nv_bfloat16> : launch_weight<__half>;
  return status(fn, launch(src, src_row_stride, (int)rows, cols, values, values_row_stride, scales, scales_row_stride,
                           static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
