// Rows to int8 with one scale each (sm_100a), for the int8 head: the weight's
// rows once, the step's hidden states before each projection.
//
//   scale = max |x| / 127 (fp32 division; or max |x| * fp32(1 / 127), as the
//   caller says), value = x / scale rounded to the nearest integer, ties to even
//   (fp32 division, then rounding), in -127..127.
//
// A row of zeros has scale 0 and values 0. A row that holds an infinity or NaN
// has scale NaN and values 0, so that everything computed from it is NaN.
//
// One pass over memory: a group of 1 to 8 warps holds one row in registers
// (16-byte vectors, up to kHeld per thread, neighbouring lanes holding
// neighbouring vectors), takes the maximum, then writes a vector's 8 (fp32: 4)
// bytes. Rows longer than a group's registers are read
// twice, the second time mostly from L2. Bound: HBM bytes (2 or 4 read, 1
// written per element) for a whole weight, latency for a step's few rows, where
// the group is widened until every SM-resident thread holds little.
#include <algorithm>

#include "gsp_common.cuh"
#include "gsp_internal.h"
#include "int8_quantize.cuh"

namespace gsp {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantWarps = kQuantThreads / 32;
constexpr int kHeld = 8;     // vectors a thread holds

// Maximum over the row's group of `gw` warps (uniform over the CTA).
template <typename T>
__device__ __forceinline__ float group_max(uint32_t running, int gw, float* s_max) {
  const uint32_t bits = __reduce_max_sync(FULL_MASK, __float_as_uint(magnitude<T>(running)));
  if (gw == 1) return __uint_as_float(bits);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) s_max[warp] = __uint_as_float(bits);
  __syncthreads();
  uint32_t m = 0u;
  for (int i = 0; i < gw; ++i) m = max(m, __float_as_uint(s_max[warp / gw * gw + i]));
  return __uint_as_float(m);
}

// kVec: rows and outputs aligned to 16 bytes, rows whole vectors long.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_rows_kernel(const T* __restrict__ src, int64_t src_stride, int64_t rows, int cols, int8_t* values,
                         int64_t values_stride, float* scales, int gw, bool by_product) {
  __shared__ float s_max[kQuantWarps];
  // a staged projection launched behind this kernel may have its CTAs in place
  // already (it waits for this kernel's end before it does anything)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_block = kQuantWarps / gw;
  const int group = threadIdx.x / (32 * gw), t = threadIdx.x - group * 32 * gw, nt = 32 * gw;
  const int64_t row = (int64_t)blockIdx.x * per_block + group;
  const bool live = row < rows;
  const T* x = src + (live ? row : 0) * src_stride;
  int8_t* out = values + (live ? row : 0) * values_stride;
  uint32_t running = 0u;
  if constexpr (kVec) {
    const int n = live ? cols / DTypeTraits<T>::kPerVec : 0;
    const void* base = x;
    uint4 v[kHeld];
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      const int i = t + c * nt;
      v[c] = i < n ? ld_stream_v4(static_cast<const uint4*>(base) + i) : make_uint4(0u, 0u, 0u, 0u);
      running = vector_max<T>(running, v[c]);
    }
    for (int i = t + kHeld * nt; i < n; i += nt)
      running = vector_max<T>(running, ld_stream_v4(static_cast<const uint4*>(base) + i));
    const RowScale r = row_scale(group_max<T>(running, gw, s_max), by_product);
    if (live && t == 0) scales[row] = r.scale;
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      const int i = t + c * nt;
      if (i < n) store_packed<T>(out, i, quantize_vector<T>(v[c], r));
    }
    for (int i = t + kHeld * nt; i < n; i += nt)
      store_packed<T>(out, i, quantize_vector<T>(ld_stream_v4(static_cast<const uint4*>(base) + i), r));
  } else {
    using Bits = typename DTypeTraits<T>::Bits;
    const Bits* xb = reinterpret_cast<const Bits*>(x);
    const int n = live ? cols : 0;
    // (four loads under way while all lanes have four; the second time they come
    // from L1: 248,320 x 1,023 fp16 517 -> 337 us, one row of 8,191 10.7 -> 7.0)
    int i = t;
    for (; i - t + 4 * nt <= n; i += 4 * nt) {
      const uint32_t x0 = __ldg(xb + i), x1 = __ldg(xb + i + nt), x2 = __ldg(xb + i + 2 * nt), x3 = __ldg(xb + i + 3 * nt);
      running = word_max<T>(word_max<T>(word_max<T>(word_max<T>(running, x0), x1), x2), x3);
    }
    for (; i < n; i += nt) running = word_max<T>(running, (uint32_t)__ldg(xb + i));
    const RowScale r = row_scale(group_max<T>(running, gw, s_max), by_product);
    if (live && t == 0) scales[row] = r.scale;
    for (i = t; i - t + 4 * nt <= n; i += 4 * nt) {
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = DTypeTraits<T>::bits_to_float(__ldg(xb + i + k * nt));
#pragma unroll
      for (int k = 0; k < 4; ++k) out[i + k * nt] = quantize_value(f[k], r);
    }
    for (; i < n; i += nt) out[i] = quantize_value(DTypeTraits<T>::bits_to_float(__ldg(xb + i)), r);
  }
}

template <typename T>
cudaError_t launch_typed(const void* src, int64_t src_stride, int64_t rows, int cols, bool by_product, int8_t* values,
                         int64_t values_stride, float* scales, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const bool vec = cols % DTypeTraits<T>::kPerVec == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(values) & 15) == 0 &&
                   (rows == 1 || ((src_stride * (int64_t)sizeof(T)) % 16 == 0 && values_stride % 8 == 0));
  // Warps per row: enough to hold the row in registers; with few rows, more,
  // until the grid fills the SMs or a thread is left with one vector (or one
  // element of the unaligned path).
  const int64_t units = vec ? cols / DTypeTraits<T>::kPerVec : cols;
  int gw = 1;
  while (gw < kQuantWarps && ((vec && units > (int64_t)32 * gw * kHeld) ||
                              (units > 32 * gw && rows * gw < (int64_t)num_sms(dev) * kQuantWarps)))
    gw *= 2;
  const int64_t per_block = kQuantWarps / gw;
  const unsigned grid = (unsigned)((rows + per_block - 1) / per_block);
  const T* s = static_cast<const T*>(src);
  if (vec)
    quantize_rows_kernel<T, true><<<grid, kQuantThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, gw, by_product);
  else
    quantize_rows_kernel<T, false><<<grid, kQuantThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, gw, by_product);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows_int8(const void* src, int64_t src_stride, int64_t rows, int cols, int dtype,
                                      bool by_product, int8_t* values, int64_t values_stride, float* scales,
                                      cudaStream_t stream) {
  auto launch = dtype == 2 ? launch_typed<float> : dtype == 1 ? launch_typed<__nv_bfloat16> : launch_typed<__half>;
  return launch(src, src_stride, rows, cols, by_product, values, values_stride, scales, stream);
}

}  // namespace gsp
