// Root-mean-square norm with the residual's addition, and an output in the input's
// type, in int8 with a scale per row, or in e4m3 with a scale per 128 columns
// (sm_100a): the step before the LM head.
//
//   h = round_T(x + residual)      (what the residual stream holds from here on)
//   y = h * (1 / sqrt(mean(h^2) + eps)) * weight        (fp32)
//   out = round_T(y), or
//   int8:  scale = max |y| / 127 over the row, value = y / scale to the nearest
//          integer, ties to even (gsp_quantize_rows_int8's rule);
//   e4m3:  scale = max |y| / 448 over 128 columns, value = y / scale to the nearest
//          (gsp_quantize_rows_fp8's rule).
//
// The 8-bit outputs are taken from y in fp32: rounding it to T first, as a norm
// followed by a quantiser does, would add half a step of T.
//
// One pass over memory (2 + 2 read, 2 + 1 written per element of a 16-bit row with
// residual and 8-bit output): 1 to 16 warps hold a row's h in registers, and the squares,
// the row's maximum and the blocks' maxima are reduced from there. What of a row is past
// the registers (over 16,384 columns) is read again.
//
// Measured, 16,384 x 8,192 bf16 with residual: rounded output 204 us (5.3 TB/s, 81% of
// measured), e4m3 221 us (4.2 TB/s; floor 146), int8 250 us: with an 8-bit output the
// instructions of the quantisation bound it beside memory. 64 x 2,048: 2.9-3.3 us, a launch.
#include <algorithm>
#include <cmath>

#include "../../include/gsp_b200.h"
#include "fp8_quantize.cuh"
#include "gsp_internal.h"
#include "int8_quantize.cuh"

namespace gsp {
namespace {

enum NormOut { kSame, kInt8, kE4m3 };

struct NormParams {
  const void* x;
  int64_t x_stride;
  const void* residual;  // optional
  int64_t residual_stride;
  const void* weight;  // optional: 1
  int64_t rows;
  int cols;
  float eps;
  void* residual_out;  // with residual
  int64_t residual_out_stride;
  void* out;
  int64_t out_stride;
  float* scales;
  int64_t scales_stride;  // e4m3
  int group_warps;
};

// Sum, or maximum, of a value over the warps of a row's group (every thread of the CTA calls).
template <bool kMax>
__device__ __forceinline__ float over_group(float v, int gw, float* s_part) {
  if constexpr (kMax) v = __uint_as_float(__reduce_max_sync(FULL_MASK, __float_as_uint(v)));  // (v >= 0, or NaN)
  else v = warp_sum(v);
  if (gw == 1) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) s_part[warp] = v;
  __syncthreads();
  float r = 0.f;
  for (int i = 0; i < gw; ++i) {
    const float y = s_part[warp / gw * gw + i];
    if constexpr (kMax) r = __uint_as_float(max(__float_as_uint(r), __float_as_uint(y)));
    else r += y;
  }
  return r;
}

// Four values as four int8 bytes, by the reciprocal where that rounds to the same integers.
__device__ __forceinline__ uint32_t to_int8(float a, float b, float c, float d, const RowScale& s) {
  return ((uint32_t)quantize_value(a, s) & 0xffu) | (((uint32_t)quantize_value(b, s) & 0xffu) << 8) |
         (((uint32_t)quantize_value(c, s) & 0xffu) << 16) | (((uint32_t)quantize_value(d, s) & 0xffu) << 24);
}

// kHeld: units a thread holds, in the row's type. kLong: rows may be longer than that.
template <typename T, bool kVec, int kOut, int kHeld, int kThreads, int kThreadsPerSm, bool kLong>
__global__ void __launch_bounds__(kThreads, kThreadsPerSm / kThreads) rms_norm_kernel(const __grid_constant__ NormParams p) {
  using U = Units<T, kVec>;
  using Bits = typename U::Bits;
  constexpr int kE = U::kElems;
  __shared__ float s_sum[kThreads / 32], s_max[kThreads / 32];
  const int gw = p.group_warps, nt = 32 * gw;
  const int group = threadIdx.x / nt, t = threadIdx.x - group * nt;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / nt) + group;
  const bool live = row < p.rows;
  const int64_t at = live ? row : 0;
  const int cols = p.cols;
  const Bits* x = static_cast<const Bits*>(p.x) + at * p.x_stride;
  const Bits* res = p.residual ? static_cast<const Bits*>(p.residual) + at * p.residual_stride : nullptr;
  Bits* res_out = p.residual ? static_cast<Bits*>(p.residual_out) + at * p.residual_out_stride : nullptr;
  const Bits* weight = static_cast<const Bits*>(p.weight);
  const int n = live ? U::count(cols) : 0;

  // h of a unit: with a residual their rounded sum, which the residual stream takes
  const auto sum_of = [&](int i, const uint4& v) {
    if (!res) return v;
    float a[kE], b[kE];
    U::unpack(v, a);
    U::unpack(U::load_packed(res, i, cols), b);
#pragma unroll
    for (int j = 0; j < kE; ++j) a[j] += b[j];
    const uint4 h = U::pack(a);
    U::store_packed(res_out, i, cols, h);
    return h;
  };
  const auto again = [&](int i, float (&h)[kE]) {  // (this thread's own store, or the input)
    if (!res) {
      U::load(x, i, cols, h);
      return;
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const int c = U::column(i, j);
      h[j] = c < cols ? DTypeTraits<T>::bits_to_float(*(volatile const Bits*)(res_out + c)) : 0.f;
    }
  };
  const auto squares_of = [&](const uint4& v) {
    float f[kE], sum = 0.f;
    U::unpack(v, f);
#pragma unroll
    for (int j = 0; j < kE; ++j) sum = fmaf(f[j], f[j], sum);
    return sum;
  };

  uint4 held[kHeld];
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const int i = t + c * nt;
    held[c] = i < n ? U::load_packed(x, i, cols) : make_uint4(0u, 0u, 0u, 0u);
  }
  float squares = 0.f;
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const int i = t + c * nt;
    if (i < n) held[c] = sum_of(i, held[c]);
    squares += squares_of(held[c]);
  }
  if constexpr (kLong) {
    for (int i = t + kHeld * nt; i < n; i += nt) squares += squares_of(sum_of(i, U::load_packed(x, i, cols)));
  }
  // (each thread's part of the mean: the sum over the row of squares near fp32's largest would pass it)
  const float mean = over_group<false>(__fdiv_rn(squares, (float)cols), gw, s_sum);
  const float by = __frcp_rn(__fsqrt_rn(mean + p.eps));

  const auto normed = [&](int i, float (&v)[kE]) {  // h -> y
    if (weight) {
      float w[kE];
      if constexpr (kVec) U::unpack(__ldg(reinterpret_cast<const uint4*>(weight) + i), w);
      else U::load(weight, i, cols, w);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = v[j] * by * w[j];
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = v[j] * by;
    }
  };
  // every unit of the thread's, as y
  const auto each = [&](auto&& use) {
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      const int i = t + c * nt;
      float v[kE];
      U::unpack(held[c], v);
      if (i < n) normed(i, v);
      use(i, v);
    }
    if constexpr (kLong) {
      for (int i = t + kHeld * nt; i < ((n + 31) & ~31); i += nt) {  // (whole warps)
        float v[kE];
        if (i < n) {
          again(i, v);
          normed(i, v);
        }
        use(i, v);
      }
    }
  };

  if constexpr (kOut == kSame) {
    Bits* out = static_cast<Bits*>(p.out) + at * p.out_stride;
    each([&](int i, const float (&v)[kE]) {
      if (i < n) U::store(out, i, cols, v);
    });
  } else if constexpr (kOut == kInt8) {
    uint8_t* out = static_cast<uint8_t*>(p.out) + at * p.out_stride;
    uint32_t top = 0u;
    each([&](int i, const float (&v)[kE]) {
      if (i < n) top = max(top, U::magnitude(v));
    });
    const RowScale scale = row_scale(over_group<true>(__uint_as_float(top), gw, s_max), false);
    if (live && t == 0) p.scales[row] = scale.scale;
    each([&](int i, const float (&v)[kE]) {
      if (i >= n) return;
      uint32_t w[kE / 4];
#pragma unroll
      for (int k = 0; k < kE / 4; ++k) w[k] = to_int8(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3], scale);
      U::store_bytes(out, i, cols, w);
    });
  } else {
    uint8_t* out = static_cast<uint8_t*>(p.out) + at * p.out_stride;
    float* scales = p.scales + at * p.scales_stride;
    each([&](int i, const float (&v)[kE]) {  // (lanes past the row take part in the blocks' maxima)
      const BlockScale s = block_scale(lanes_max<U::kLanes>(i < n ? U::magnitude(v) : 0u));
      if (i >= n) return;
      uint32_t w[kE / 4];
#pragma unroll
      for (int k = 0; k < kE / 4; ++k) w[k] = to_e4m3(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3], s);
      U::store_bytes(out, i, cols, w);
      if (i % U::kLanes == 0) scales[i / U::kLanes] = s.scale;
    });
  }
}

template <typename T, bool kVec, int kOut>
cudaError_t launch_norm(NormParams p, cudaStream_t stream) {
  int dev = 0;
  const cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  constexpr int kE = Units<T, kVec>::kElems;
  // Warps per row: 8 values a thread, past 4,096 columns 16, past 8,192 32: a row is soon
  // done, and most of the SM's threads are resident. Rows of few warps share a CTA.
  const int64_t units = kVec ? p.cols / kE : ((int64_t)p.cols + kBlock - 1) / kBlock * 32;
  int gw = 1;
  while (gw < 16 && units * kE > (int64_t)32 * gw * 8) gw *= 2;
  p.group_warps = gw;
  const int threads = std::max(256, 32 * gw);
  const int64_t per_cta = threads / 32 / gw, grid = (p.rows + per_cta - 1) / per_cta;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned g = (unsigned)grid;
  const int64_t floats = units * kE, row_threads = 32 * gw;
  const auto run = [&](auto kernel) { kernel<<<g, (unsigned)threads, 0, stream>>>(p); };
  if (threads == 256) run(rms_norm_kernel<T, kVec, kOut, 8 / kE, 256, 1536, false>);
  else if (floats <= row_threads * 8) run(rms_norm_kernel<T, kVec, kOut, 8 / kE, 512, 1536, false>);
  else if (floats <= row_threads * 16) run(rms_norm_kernel<T, kVec, kOut, 16 / kE, 512, 1536, false>);
  else if (floats <= row_threads * 32) run(rms_norm_kernel<T, kVec, kOut, 32 / kE, 512, 1024, false>);
  else run(rms_norm_kernel<T, kVec, kOut, 32 / kE, 512, 1024, true>);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const NormParams& p, int out_kind, cudaStream_t stream) {
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  const auto aligned = [&](const void* q, int64_t stride, int64_t size, int64_t to) {
    return (reinterpret_cast<uintptr_t>(q) % to) == 0 && (p.rows == 1 || stride * size % to == 0);
  };
  const int64_t out_size = out_kind == kSame ? sizeof(T) : 1, out_to = out_kind == kSame ? 16 : kPer;
  const bool vec = p.cols % kPer == 0 && aligned(p.x, p.x_stride, sizeof(T), 16) &&
                   (!p.residual || (aligned(p.residual, p.residual_stride, sizeof(T), 16) &&
                                    aligned(p.residual_out, p.residual_out_stride, sizeof(T), 16))) &&
                   (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0 && aligned(p.out, p.out_stride, out_size, out_to);
  if (out_kind == kInt8) return vec ? launch_norm<T, true, kInt8>(p, stream) : launch_norm<T, false, kInt8>(p, stream);
  if (out_kind == kE4m3) return vec ? launch_norm<T, true, kE4m3>(p, stream) : launch_norm<T, false, kE4m3>(p, stream);
  return vec ? launch_norm<T, true, kSame>(p, stream) : launch_norm<T, false, kSame>(p, stream);
}

}  // namespace
}  // namespace gsp

using namespace gsp;

extern "C" int32_t gsp_rms_norm(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride,
                                const void* weight, int64_t rows, int32_t cols, float eps, int32_t dtype,
                                void* residual_out, int64_t residual_out_row_stride, int32_t out_dtype, void* out,
                                int64_t out_row_stride, float* scales, int64_t scales_row_stride, void* stream) {
  const char* fn = "gsp_rms_norm";
  if (rows < 0 || cols < 1) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: rows must be >= 0 and cols positive", fn);
  if (dtype != GSP_DTYPE_F16 && dtype != GSP_DTYPE_BF16 && dtype != GSP_DTYPE_F32)
    return record_error(GSP_ERR_UNSUPPORTED, "%s: dtype must be GSP_DTYPE_F16, GSP_DTYPE_BF16 or GSP_DTYPE_F32", fn);
  if (out_dtype != dtype && out_dtype != GSP_DTYPE_I8 && out_dtype != GSP_DTYPE_E4M3)
    return record_error(GSP_ERR_UNSUPPORTED, "%s: out_dtype must be dtype, GSP_DTYPE_I8 or GSP_DTYPE_E4M3", fn);
  if (rows > INT32_MAX) return record_error(GSP_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", fn);
  if (cols > (1 << 24)) return record_error(GSP_ERR_UNSUPPORTED, "%s: more than 2^24 columns", fn);
  if (!(eps >= 0.f) || std::isinf(eps))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", fn);
  if (rows == 0) return GSP_OK;
  if (!x || !out) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: x and out are required", fn);
  if ((residual == nullptr) != (residual_out == nullptr))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: residual and residual_out go together", fn);
  const int64_t blocks = ((int64_t)cols + kBlock - 1) / kBlock;
  if (out_dtype != dtype && !scales) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: scales is required", fn);
  if (rows > 1 && (x_row_stride < 0 || residual_row_stride < 0 || out_row_stride < cols ||
                   (residual_out && residual_out_row_stride < cols) ||
                   (out_dtype == GSP_DTYPE_E4M3 && scales_row_stride < blocks)))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: a row stride is negative or shorter than its row", fn);
  NormParams p{};
  p.x = x;
  p.x_stride = rows > 1 ? x_row_stride : 0;
  p.residual = residual;
  p.residual_stride = rows > 1 ? residual_row_stride : 0;
  p.weight = weight;
  p.rows = rows;
  p.cols = cols;
  p.eps = eps;
  p.residual_out = residual_out;
  p.residual_out_stride = rows > 1 ? residual_out_row_stride : 0;
  p.out = out;
  p.out_stride = rows > 1 ? out_row_stride : 0;
  p.scales = scales;
  p.scales_stride = rows > 1 ? scales_row_stride : 0;
  const int kind = out_dtype == dtype ? kSame : out_dtype == GSP_DTYPE_I8 ? kInt8 : kE4m3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == GSP_DTYPE_F32    ? launch_typed<float>(p, kind, s)
                          : dtype == GSP_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(p, kind, s)
                                                    : launch_typed<__half>(p, kind, s);
  if (err == cudaSuccess) return GSP_OK;
  return record_error(GSP_ERR_CUDA, "%s: %s (%s)", fn, cudaGetErrorName(err), cudaGetErrorString(err));
}
