// Device code that turns a row into int8 values and one scale, shared by the
// row quantiser and the row-sparse kernels that quantise their hidden states
// themselves (same bits):
//
//   scale = max |x| / 127 (fp32 division; or max |x| * fp32(1 / 127), as the
//   caller says), value = x / scale rounded to the nearest integer, ties to even
//   (fp32 division, then rounding), in -127..127.
//
// The division: x * (1 / scale) is within 3 * 2^-24 relative of the quotient
// (at most 2.3e-5 absolute), so their roundings to an integer differ only where
// the product lies that near a half; a vector that has such an element divides.
// Rounding by adding 1.5 * 2^23 leaves the integer in the low byte, ready to be
// packed: an element costs about six instructions (with a float-to-integer
// conversion, two clamps and a branch each, a weight of 248,320 x 2,048 fp16
// took 490 us).
#pragma once

#include "gsp_common.cuh"

namespace gsp {
namespace {

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
  bool zero;    // nothing but zeros, or not finite: every value is 0
  bool divide;  // the inverse is not finite (a denormal scale)
};

// by_product: the scale is the product with the rounded reciprocal of 127,
// which torch takes on the GPU for amax / 127.0 (one step off the division's in
// some rows).
__device__ __forceinline__ RowScale row_scale(float amax, bool by_product) {
  constexpr float kInverse127 = 1.f / 127.f;
  RowScale r;
  const bool finite = amax < INFINITY;  // false for NaN
  r.scale = !finite ? __int_as_float(0x7fc00000) : by_product ? __fmul_rn(amax, kInverse127) : __fdiv_rn(amax, 127.f);
  r.zero = !finite || !(r.scale > 0.f);
  r.inverse = r.zero ? 0.f : __fdiv_rn(1.f, r.scale);
  r.divide = !(r.inverse < INFINITY);
  return r;
}

// The definition itself (the scale is positive); a denormal scale may be so
// coarse that its quotients pass 127.
__device__ __forceinline__ int quantize_by_division(float x, float scale) {
  return (int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.f), 127.f);
}

// One value, by the reciprocal where that cannot round to another integer.
__device__ __forceinline__ int8_t quantize_value(float x, const RowScale& r) {
  constexpr float kMagic = 12582912.f;
  const float t = fmaf(x, r.inverse, kMagic);
  if (r.divide || fabsf(fmaf(x, r.inverse, kMagic - t)) > 0.4999f) return (int8_t)quantize_by_division(x, r.scale);
  return r.zero ? (int8_t)0 : (int8_t)(__float_as_uint(t) & 0xffu);
}

template <typename T>
__device__ __forceinline__ float element(const uint32_t* words, int i) {
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(words[i]);
  else
    return DTypeTraits<T>::bits_to_float((uint16_t)(words[i >> 1] >> (16 * (i & 1))));
}

// A vector's values, 8 (fp32: 4) bytes.
template <typename T>
struct Packed {
  static constexpr int kWords = DTypeTraits<T>::kPerVec / 4;
  uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ Packed<T> quantize_vector(const uint4& v, const RowScale& r) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, ties to even
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  Packed<T> out;
  float farthest = 0.f;  // from the integer
#pragma unroll
  for (int k = 0; k < Packed<T>::kWords; ++k) {
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = element<T>(w, 4 * k + j);
      const float t = fmaf(x, r.inverse, kMagic);
      farthest = fmaxf(farthest, fabsf(fmaf(x, r.inverse, kMagic - t)));
      q[j] = __float_as_uint(t);
    }
    out.w[k] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  }
  if (r.divide || farthest > 0.4999f) {
#pragma unroll
    for (int k = 0; k < Packed<T>::kWords; ++k) {
      out.w[k] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out.w[k] |= ((uint32_t)quantize_by_division(element<T>(w, 4 * k + j), r.scale) & 0xffu) << (8 * j);
    }
  }
  if (r.zero) {
#pragma unroll
    for (int k = 0; k < Packed<T>::kWords; ++k) out.w[k] = 0u;
  }
  return out;
}

template <typename T>
__device__ __forceinline__ void store_packed(int8_t* row, int i, const Packed<T>& v) {
  if constexpr (Packed<T>::kWords == 2)
    reinterpret_cast<uint2*>(row)[i] = make_uint2(v.w[0], v.w[1]);
  else
    reinterpret_cast<uint32_t*>(row)[i] = v.w[0];
}

template <typename T>
__device__ __forceinline__ uint32_t vector_max(uint32_t running, const uint4& v) {
  return word_max<T>(word_max<T>(word_max<T>(word_max<T>(running, v.x), v.y), v.z), v.w);
}

}  // namespace
}  // namespace gsp
