// Rows to int8 with one scale each (sm_100a), for the int8 head: the weight's
// rows once, the step's hidden states before each projection.
//
//   scale = max |x| / 127 (fp32 division), value = x / scale rounded to the
//   nearest integer, ties to even (fp32 division, then rounding), in -127..127.
//
// A row of zeros has scale 0 and values 0. A row that holds an infinity or NaN
// has scale NaN and values 0, so that everything computed from it is NaN.
//
// One pass over memory: a group of 1 to 8 warps holds one row in registers
// (chunks of 16 elements, up to kChunks per thread), takes the maximum, then
// writes 16 bytes per chunk. Rows longer than a group's registers are read
// twice, the second time mostly from L2. Bound: HBM bytes (2 or 4 read, 1
// written per element) for a whole weight, latency for a step's few rows, where
// the group is widened until every SM-resident thread holds little.
//
// The division: a quotient's rounding differs from that of x * (1 / scale) only
// where the product lies within its error (three roundings, 3 * 2^-24
// relative, at most 127.5 * 2^-22 absolute) of a half; only those elements
// divide.
#include <algorithm>

#include "gsp_common.cuh"
#include "gsp_internal.h"

namespace gsp {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantWarps = kQuantThreads / 32;
constexpr int kChunk = 16;   // elements: one 16-byte store
constexpr int kChunks = 4;   // chunks a thread holds

template <typename T>
struct ChunkWords {
  static constexpr int value = kChunk * (int)sizeof(T) / 4;
};

// |x| as ordered fp32 bits: the maximum of the bits is the maximum of the
// magnitudes, infinities and NaN above every finite value.
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t running, uint32_t w) {
  if constexpr (sizeof(T) == 4)
    return max(running, w & 0x7fffffffu);
  else
    return __vmaxu2(running, w & 0x7fff7fffu);  // two 16-bit magnitudes
}

template <typename T>
__device__ __forceinline__ float magnitude(uint32_t running) {
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(running);
  else
    return DTypeTraits<T>::bits_to_float((uint16_t)max(running & 0xffffu, running >> 16));
}

struct RowScale {
  float scale, inverse;
  bool zero;  // nothing but zeros, or not finite: every value is 0
};

__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  const bool finite = amax < INFINITY;  // false for NaN
  r.scale = finite ? __fdiv_rn(amax, 127.f) : __int_as_float(0x7fc00000);
  r.zero = !finite || !(r.scale > 0.f);
  r.inverse = r.zero ? 0.f : __fdiv_rn(1.f, r.scale);
  return r;
}

__device__ __forceinline__ int quantize(float x, const RowScale& r) {
  if (r.zero) return 0;
  const float t = x * r.inverse;
  float q = rintf(t);
  // a denormal scale has an infinite inverse: its quotients divide too
  if (!(fabsf(t - q) < 0.4999f)) q = rintf(__fdiv_rn(x, r.scale));
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

template <typename T>
__device__ __forceinline__ float element(const uint32_t* words, int i) {
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(words[i]);
  else
    return DTypeTraits<T>::bits_to_float((uint16_t)(words[i >> 1] >> (16 * (i & 1))));
}

template <typename T>
__device__ __forceinline__ void load_chunk(const T* src, uint32_t (&w)[ChunkWords<T>::value]) {
  const uint4* p = reinterpret_cast<const uint4*>(src);
#pragma unroll
  for (int v = 0; v < ChunkWords<T>::value / 4; ++v) {
    const uint4 x = ld_stream_v4(p + v);
    w[4 * v] = x.x;
    w[4 * v + 1] = x.y;
    w[4 * v + 2] = x.z;
    w[4 * v + 3] = x.w;
  }
}

template <typename T>
__device__ __forceinline__ uint4 quantize_chunk(const uint32_t (&w)[ChunkWords<T>::value], const RowScale& r) {
  uint32_t out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    out[k] = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[k] |= ((uint32_t)quantize(element<T>(w, 4 * k + j), r) & 0xffu) << (8 * j);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

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

// kVec: rows and outputs aligned to 16 bytes and whole chunks long.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_rows_kernel(const T* __restrict__ src, int64_t src_stride, int64_t rows, int cols, int8_t* values,
                         int64_t values_stride, float* scales, int gw) {
  __shared__ float s_max[kQuantWarps];
  // a projection launched behind this kernel may set itself up already
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_block = kQuantWarps / gw;
  const int group = threadIdx.x / (32 * gw), t = threadIdx.x - group * 32 * gw, nt = 32 * gw;
  const int64_t row = (int64_t)blockIdx.x * per_block + group;
  const bool live = row < rows;
  const T* x = src + (live ? row : 0) * src_stride;
  int8_t* out = values + (live ? row : 0) * values_stride;
  uint32_t running = 0u;
  if constexpr (kVec) {
    const int n = live ? cols / kChunk : 0;
    uint32_t w[kChunks][ChunkWords<T>::value];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int i = t + c * nt;
      if (i < n) {
        load_chunk(x + (int64_t)i * kChunk, w[c]);
#pragma unroll
        for (int k = 0; k < ChunkWords<T>::value; ++k) running = word_max<T>(running, w[c][k]);
      }
    }
    for (int i = t + kChunks * nt; i < n; i += nt) {
      uint32_t y[ChunkWords<T>::value];
      load_chunk(x + (int64_t)i * kChunk, y);
#pragma unroll
      for (int k = 0; k < ChunkWords<T>::value; ++k) running = word_max<T>(running, y[k]);
    }
    const RowScale r = row_scale(group_max<T>(running, gw, s_max));
    if (live && t == 0) scales[row] = r.scale;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int i = t + c * nt;
      if (i < n) reinterpret_cast<uint4*>(out)[i] = quantize_chunk<T>(w[c], r);
    }
    for (int i = t + kChunks * nt; i < n; i += nt) {
      uint32_t y[ChunkWords<T>::value];
      load_chunk(x + (int64_t)i * kChunk, y);
      reinterpret_cast<uint4*>(out)[i] = quantize_chunk<T>(y, r);
    }
  } else {
    using Bits = typename DTypeTraits<T>::Bits;
    const Bits* xb = reinterpret_cast<const Bits*>(x);
    const int n = live ? cols : 0;
    for (int i = t; i < n; i += nt) running = word_max<T>(running, (uint32_t)__ldg(xb + i));
    const RowScale r = row_scale(group_max<T>(running, gw, s_max));
    if (live && t == 0) scales[row] = r.scale;
    for (int i = t; i < n; i += nt) out[i] = (int8_t)quantize(DTypeTraits<T>::bits_to_float(__ldg(xb + i)), r);
  }
}

template <typename T>
cudaError_t launch_typed(const void* src, int64_t src_stride, int64_t rows, int cols, int8_t* values,
                         int64_t values_stride, float* scales, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const bool vec = cols % kChunk == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(values) & 15) == 0 &&
                   (rows == 1 || ((src_stride * (int64_t)sizeof(T)) % 16 == 0 && values_stride % 16 == 0));
  // Warps per row: enough to hold the row in registers; with few rows, more,
  // until the grid fills the SMs or a thread is left with one chunk (or one
  // element of the unaligned path).
  const int64_t units = vec ? cols / kChunk : cols;
  int gw = 1;
  while (gw < kQuantWarps && ((vec && units > (int64_t)32 * gw * kChunks) ||
                              (units > 32 * gw && rows * gw < (int64_t)num_sms(dev) * kQuantWarps)))
    gw *= 2;
  const int64_t per_block = kQuantWarps / gw;
  const unsigned grid = (unsigned)((rows + per_block - 1) / per_block);
  const T* s = static_cast<const T*>(src);
  if (vec)
    quantize_rows_kernel<T, true><<<grid, kQuantThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, gw);
  else
    quantize_rows_kernel<T, false><<<grid, kQuantThreads, 0, stream>>>(s, src_stride, rows, cols, values, values_stride, scales, gw);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows_int8(const void* src, int64_t src_stride, int64_t rows, int cols, int dtype,
                                      int8_t* values, int64_t values_stride, float* scales, cudaStream_t stream) {
  if (dtype == 2) return launch_typed<float>(src, src_stride, rows, cols, values, values_stride, scales, stream);
  if (dtype == 1) return launch_typed<__nv_bfloat16>(src, src_stride, rows, cols, values, values_stride, scales, stream);
  return launch_typed<__half>(src, src_stride, rows, cols, values, values_stride, scales, stream);
}

}  // namespace gsp
