// Device code that turns a block of values into e4m3 and one scale, shared by the
// quantisers and the norm that quantises its own output (same bits):
//
//   scale = max |x| / 448 (fp32 division), value = x / scale (fp32 division) to the
//   nearest e4m3, ties to even, at most 448 in magnitude.
//
// A block of zeros, or one whose scale rounds to 0, has values 0; a block that holds
// an infinity or NaN has scale NaN and values 0, so that everything computed from it
// is NaN.
#pragma once

#include <cuda_fp8.h>

#include "gsp_common.cuh"

namespace gsp {
namespace {

constexpr int kBlock = 128;  // columns (and, of a weight, rows) that share a scale

struct BlockScale {
  float scale, below, above;  // the scale's reciprocal, less and more 2^-21 of it
  bool zero, divide;          // divide: the reciprocal is not finite (a denormal scale)
};

// magnitude: the largest |x| as fp32 bits (infinities and NaN above every finite value).
__device__ __forceinline__ BlockScale block_scale(uint32_t magnitude) {
  const float amax = __uint_as_float(magnitude);
  BlockScale s;
  const bool finite = amax < INFINITY;  // false for NaN
  s.scale = finite ? __fdiv_rn(amax, 448.f) : __int_as_float(0x7fc00000);
  s.zero = !finite || !(s.scale > 0.f);
  float inverse;  // (within 2^-23; a denormal scale's is infinite)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s.scale));
  s.below = inverse * (1.f - 0x1p-21f);
  s.above = inverse * (1.f + 0x1p-21f);
  s.divide = !(s.above < INFINITY);
  return s;
}

__device__ __forceinline__ uint32_t e4m3_pair_of(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// Four values as four e4m3 bytes. The quotients lie between the products with the two
// reciprocals (each within 2^-22 of its exact value); where both products round to
// one e4m3, and rounding is monotonic, so do the quotients, and that is nearly always.
// Else they are divided out.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d, const BlockScale& s) {
  if (s.zero) return 0u;
  const uint32_t lo = e4m3_pair_of(a * s.below, b * s.below) | (e4m3_pair_of(c * s.below, d * s.below) << 16);
  const uint32_t hi = e4m3_pair_of(a * s.above, b * s.above) | (e4m3_pair_of(c * s.above, d * s.above) << 16);
  if (lo == hi && !s.divide) return lo;
  return e4m3_pair_of(__fdiv_rn(a, s.scale), __fdiv_rn(b, s.scale)) |
         (e4m3_pair_of(__fdiv_rn(c, s.scale), __fdiv_rn(d, s.scale)) << 16);
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Largest of the values over `lanes` neighbouring lanes (a power of two), in each of them.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (kLanes == 32) {
    return __reduce_max_sync(FULL_MASK, v);
  } else {
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) v = max(v, __shfl_xor_sync(FULL_MASK, v, o));
    return v;
  }
}

// A row's elements as a thread holds them, in units: with whole 16-byte vectors
// (kVec) a unit is one vector, and 16 (fp32: 32) neighbouring lanes hold a block of
// 128; else a unit is four elements 32 apart, and the warp's lanes hold the block.
template <typename T, bool kVec>
struct Units {
  static constexpr int kElems = kVec ? DTypeTraits<T>::kPerVec : 4;
  static constexpr int kLanes = kBlock / kElems;  // that share a block
  using Bits = typename DTypeTraits<T>::Bits;

  static __device__ __forceinline__ int count(int cols) {  // units of a row, whole warps
    return kVec ? cols / kElems : (cols + kBlock - 1) / kBlock * 32;
  }
  static __device__ __forceinline__ int column(int unit, int j) {
    return kVec ? unit * kElems + j : (unit >> 5) * kBlock + (unit & 31) + 32 * j;
  }
  // A unit as it is held: a vector in the row's type, or four fp32 values.
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[kElems]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (!kVec || sizeof(Bits) == 4) {
        f[k] = __uint_as_float(w[k]);
      } else {
        const float2 two = DTypeTraits<T>::pair_to_float2(w[k]);
        f[2 * k] = two.x;
        f[2 * k + 1] = two.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kElems]) {  // rounded to the row's type
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(Bits) == 4) w[k] = __float_as_uint(f[k]);
      else if constexpr (!kVec) w[k] = __float_as_uint(DTypeTraits<T>::bits_to_float(DTypeTraits<T>::round_bits(f[k])));
      else w[k] = (uint32_t)DTypeTraits<T>::round_bits(f[2 * k]) | ((uint32_t)DTypeTraits<T>::round_bits(f[2 * k + 1]) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint4 load_packed(const Bits* row, int unit, int cols) {
    if constexpr (kVec) return ld_stream_v4(reinterpret_cast<const uint4*>(row) + unit);
    float f[kElems];
    load(row, unit, cols, f);
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ void store_packed(Bits* row, int unit, int cols, const uint4& v) {
    if constexpr (kVec) {
      reinterpret_cast<uint4*>(row)[unit] = v;
    } else {
      float f[kElems];
      unpack(v, f);
      store(row, unit, cols, f);
    }
  }
  // (elements past the row are 0)
  static __device__ __forceinline__ void load(const Bits* row, int unit, int cols, float (&f)[kElems]) {
    if constexpr (kVec) {
      unpack(ld_stream_v4(reinterpret_cast<const uint4*>(row) + unit), f);
    } else {
#pragma unroll
      for (int j = 0; j < kElems; ++j) {
        const int at = column(unit, j);
        f[j] = at < cols ? DTypeTraits<T>::bits_to_float(__ldg(row + at)) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(Bits* row, int unit, int cols, const float (&f)[kElems]) {
    if constexpr (kVec) {
      reinterpret_cast<uint4*>(row)[unit] = pack(f);
    } else {
#pragma unroll
      for (int j = 0; j < kElems; ++j) {
        const int at = column(unit, j);
        if (at < cols) row[at] = DTypeTraits<T>::round_bits(f[j]);
      }
    }
  }
  // kElems bytes of an 8-bit row, packed four to a word
  static __device__ __forceinline__ void store_bytes(uint8_t* row, int unit, int cols, const uint32_t (&w)[kElems / 4]) {
    if constexpr (kVec && kElems == 8) {
      reinterpret_cast<uint2*>(row)[unit] = make_uint2(w[0], w[1]);
    } else if constexpr (kVec) {
      reinterpret_cast<uint32_t*>(row)[unit] = w[0];
    } else {
#pragma unroll
      for (int j = 0; j < kElems; ++j) {
        const int at = column(unit, j);
        if (at < cols) row[at] = (uint8_t)(w[0] >> (8 * j));
      }
    }
  }
  static __device__ __forceinline__ uint32_t magnitude(const float (&f)[kElems]) {
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < kElems; ++j) m = max(m, magnitude_bits(f[j]));
    return m;
  }
};

}  // namespace
}  // namespace gsp
