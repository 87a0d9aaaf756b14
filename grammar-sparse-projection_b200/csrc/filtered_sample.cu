// Sampling with temperature, top-k, min-p and top-p from given uniform numbers
// (sm_100a), on the logits the head's routes write or on packed legal rows.
//
// For one row with legal logits x_i (bit set, not NaN, not -inf), in the order
// "falling logit, ties by rising position", and w_i = exp((x_i - max) / T):
//   top-k   keep the first k                                  (k <= 0: all)
//   min-p   keep w_i >= min_p           (min_p <= 0: all; above 1 it counts as 1)
//   top-p   keep the shortest prefix with sum >= top_p * sum  (top_p >= 1: all)
//   draw    the first kept i with w_1 + ... + w_i > u * (sum of the kept)
// Each filter leaves a prefix of that order, so a kept set is a border key and
// a number of ties kept at it, and the draw is one more such border: all four
// are the search for the first position where a running sum (of ones or of
// weights) passes a target.
//
// The weights are 64-bit integers in units of 2^-shift (shift = 62 - the bit
// length of n, at most 50): their sums are exact, so no order of additions and
// no split over threads or CTAs changes a token, and equal calls give equal
// answers bit for bit. The unit is at most 2^-43 for rows up to 2^18 tokens.
//
// Two kernels; long 16-bit rows in batches take the one that counts values (its
// description below). In the other, one cluster of CTAs per row; the row is read from global memory once and held
// in the CTAs' shared memory (-inf where the mask says not legal). A search
// counts or weighs the tokens in 512 bins of shared memory, the CTAs read one
// another's bins over distributed shared memory after one cluster barrier, and
// each picks the bin at which the running sum passes the target.
//   * The first bins are chosen by value, so that few tokens share one:
//     sixteenths of an octave of the weight, or (top-k) 64ths of an octave of
//     the distance to the maximum. They do not depend on the target, so top-p
//     and the draw use the same weighing.
//   * The tokens of the picked bins (for top-p: of the border's bin and of those
//     the draw can fall into) are then listed, key and position, in the first
//     CTA's shared memory; the other CTAs are done and leave, and the rest of the
//     search needs no cluster barrier: the range of keys narrows 512-fold per
//     pass over the list. Where a list does not fit, the search goes on in the
//     whole row, 512-fold per pass all the same.
//   * Rows with few legal tokens (a grammar's) are listed whole at once, and
//     after top-k or min-p the kept tokens are; up to 256 tokens left are put in
//     order by comparing each with all, and one running sum gives both borders.
//
// Bound: for long kept sets one 64-bit exponential per weighed token (11
// double-precision operations, about 35 in all) and one shared-memory atomic;
// for short ones the cluster barriers and the passes between them.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "gsp_async.cuh"
#include "gsp_common.cuh"
#include "gsp_internal.h"

namespace gsp {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBinBits = 9;
constexpr int kBins = 1 << kBinBits;
constexpr int kMaxCluster = 16;
constexpr int kMaxShift = 50;
constexpr int kExpTable = 16;
constexpr int kTiesCap = 512;    // tokens of one value whose positions are set side by side
constexpr int kFew = 256;        // tokens left that are put in order at once
constexpr int kListTotal = 4096; // tokens a cluster lists
static_assert(kBins == kSampleThreads, "one bin per thread");
static_assert(32 * 16 <= kBins, "32 octaves of weights in sixteenths");
static_assert(kMaxCluster <= kSampleWarps, "a warp for each part of the list");
static_assert(2 * kFew <= kSampleThreads, "two threads per token of few");

// 2^(j / 16) and log2(1 + j / 16).
__constant__ double kExp2[kExpTable] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
__constant__ double kLog2[kExpTable] = {
    0.0, 0.0874628412503394, 0.16992500144231237, 0.2479275134435855,
    0.32192809488736235, 0.3923174227787603, 0.45943161863729726, 0.5235619560570128,
    0.5849625007211562, 0.6438561897747247, 0.7004397181410922, 0.7548875021634686,
    0.8073549220576041, 0.8579809951275721, 0.9068905956085185, 0.9541963103868752};

// Order-preserving keys: larger logit, larger key (-0 and +0 alike); 0 for NaN
// and -inf, which are never drawn.
template <typename T>
struct SampleKey {
  static constexpr uint32_t kNegInf = std::is_same<T, __half>::value ? 0x8000u - 0x7C00u : 0x8000u - 0x7F80u;
  static __device__ __forceinline__ uint32_t from_value(float f) {
    uint32_t bits;
    if constexpr (std::is_same<T, __half>::value)
      bits = __half_as_ushort(__float2half_rn(f));
    else
      bits = __float_as_uint(f) >> 16;
    return from_bits(bits);
  }
  static __device__ __forceinline__ uint32_t from_bits(uint32_t bits) {
    const uint32_t o = (bits & 0x8000u) ? 0x8000u - (bits & 0x7fffu) : (bits | 0x8000u);
    return o > kNegInf ? o : 0u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    const uint32_t bits = key >= 0x8000u ? (key & 0x7fffu) : (0x8000u | (0x8000u - key));
    return DTypeTraits<T>::bits_to_float((uint16_t)bits);
  }
  // smallest value of the type that is >= x
  static __device__ __forceinline__ float value_at_least(double x) {
    const float f = __double2float_ru(x);
    if constexpr (std::is_same<T, __half>::value)
      return __half2float(__float2half_ru(f));
    else
      return __bfloat162float(__float2bfloat16_ru(f));
  }
};
template <>
struct SampleKey<float> {
  static constexpr uint32_t kNegInf = 0x007FFFFFu;
  static __device__ __forceinline__ uint32_t from_value(float f) {
    const uint32_t o = ordered_bits(f);
    return o > kNegInf ? o : 0u;
  }
  static __device__ __forceinline__ float value(uint32_t key) { return from_ordered_bits(key); }
  static __device__ __forceinline__ float value_at_least(double x) { return __double2float_ru(x); }
};

struct SampleSmemHeader {
  uint32_t lo[kBins + 32];                 // bins being filled: low and high halves of 64-bit sums (and a
  uint32_t hi[kBins + 32];                 // place for each lane's values that have none)
  unsigned long long tot[kBins];           // this CTA's bins, read by the cluster
  unsigned long long list[kListTotal];     // (key, position in the row), in parts (rank 0's is used)
  unsigned long long scan[kSampleWarps];
  unsigned long long pick[2][4];           // picked bin, sum before it, its own sum; [.][3] of 0: sum of all bins
  unsigned long long word[2][kMaxCluster]; // one value per CTA (all-gather)
  double exp2_table[kExpTable];            // Weigher's
  uint32_t ties_at[kTiesCap];              // positions of the drawn value's tokens
  uint32_t warp[2][kSampleWarps];
  uint32_t list_count[kMaxCluster];        // tokens in each part of the list
  uint32_t listed;                         // tokens this CTA has offered to the list
};

constexpr size_t kHeaderBytes = (sizeof(SampleSmemHeader) + 127) / 128 * 128;

template <typename T>
struct Row {
  const typename DTypeTraits<T>::Bits* x;  // the row's first logit
  const uint32_t* mask;                    // its mask words, or nullptr
  int n;                                   // tokens
};

// Request b's row; *start: its first position in the packed arrays. Positions
// outside those are not read, whatever the offsets say, nor more than 2^30 of them.
template <typename T>
__device__ __forceinline__ Row<T> row_of(const FilteredSampleParams& p, int b, int64_t* start) {
  const auto* x = static_cast<const typename DTypeTraits<T>::Bits*>(p.logits);
  *start = 0;
  if (p.offsets) {
    *start = min(max(p.offsets[b], (int64_t)0), p.capacity);
    const int64_t end = min(max(p.offsets[b + 1], *start), p.capacity);
    return Row<T>{x + *start, nullptr, (int)min(end - *start, (int64_t)1 << 30)};
  }
  return Row<T>{x + (int64_t)b * p.row_stride, p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr, p.vocab};
}

// Value at position i, read from global memory; -inf where not legal or NaN.
template <typename T>
__device__ __forceinline__ float load_value(const Row<T>& r, int64_t i) {
  if (r.mask && !((__ldg(r.mask + (i >> 5)) >> (i & 31)) & 1u)) return -INFINITY;
  const float f = DTypeTraits<T>::bits_to_float(__ldg(r.x + i));
  return f == f ? f : -INFINITY;
}

// ---- comparisons of the values in one 32-bit word (two 16-bit ones, or one) ----
// All ones in the half (word) of a value that is above, or at least, `x`, a
// value of the type. NaN is neither.
template <typename T>
__device__ __forceinline__ uint32_t pair_above(uint32_t w, float x) {
  if constexpr (std::is_same<T, __half>::value)
    return __hgt2_mask(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(x));
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __hgt2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(x));
  else
    return __uint_as_float(w) > x ? 0xffffffffu : 0u;
}
template <typename T>
__device__ __forceinline__ uint32_t pair_at_least(uint32_t w, float x) {
  if constexpr (std::is_same<T, __half>::value)
    return __hge2_mask(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(x));
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(x));
  else
    return __uint_as_float(w) >= x ? 0xffffffffu : 0u;
}
// Counts of such masks add up in both halves of a word, over a vector's words.
template <typename T>
__device__ __forceinline__ uint32_t pair_count(uint32_t mask) {
  return sizeof(typename DTypeTraits<T>::Bits) == 4 ? mask & 1u : mask & 0x00010001u;
}
template <typename T>
__device__ __forceinline__ uint32_t pair_total(uint32_t count) {
  return sizeof(typename DTypeTraits<T>::Bits) == 4 ? count : (count & 0xffffu) + (count >> 16);
}
// Running maximum of pairs; NaN never wins.
template <typename T>
struct PairMax {
  float a = -INFINITY;
  __device__ __forceinline__ void add(uint32_t w) { a = fmaxf(a, __uint_as_float(w)); }
  __device__ __forceinline__ float value() const { return a; }
};
template <>
struct PairMax<__half> {
  __half2 a = __float2half2_rn(-INFINITY);
  __device__ __forceinline__ void add(uint32_t w) { a = __hmax2(a, *reinterpret_cast<const __half2*>(&w)); }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(a), __high2float(a)); }
};
template <>
struct PairMax<__nv_bfloat16> {
  __nv_bfloat162 a = __float2bfloat162_rn(-INFINITY);
  __device__ __forceinline__ void add(uint32_t w) { a = __hmax2(a, *reinterpret_cast<const __nv_bfloat162*>(&w)); }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(a), __high2float(a)); }
};

// One CTA's part of the row: positions [lo, lo + len), as 16-byte vectors
// aligned in global memory (position lo has place `phase` in the first). The
// first `held_vectors` are kept in shared memory by load(), the others are read
// from global memory (mostly L2) in every pass.
template <typename T>
struct Slice {
  using Bits = typename DTypeTraits<T>::Bits;
  static constexpr int kVec = 16 / (int)sizeof(Bits);
  Row<T> row;
  const uint4* base;     // vector 0
  uint4* held;
  int first;             // position of vector 0's first value (up to `phase` before the part)
  int lo, len;
  int vectors, held_vectors;
  int whole0, whole1;    // vectors [whole0, whole1) are the part's own throughout

  __device__ __forceinline__ void set(const Row<T>& r, int lo_, int len_, unsigned char* smem, int room) {
    row = r;
    lo = lo_;
    len = len_;
    held = reinterpret_cast<uint4*>(smem);
    const int phase = (int)((reinterpret_cast<uintptr_t>(row.x + lo) & 15) / sizeof(Bits));
    base = reinterpret_cast<const uint4*>(row.x + lo - phase);
    first = lo - phase;
    vectors = (phase + len + kVec - 1) / kVec;
    whole0 = phase > 0 ? 1 : 0;
    whole1 = (phase + len) / kVec;
    held_vectors = min(vectors, room);
  }

  static __device__ __forceinline__ float unpack(const uint32_t (&w)[4], int j) {
    if constexpr (sizeof(Bits) == 4)
      return __uint_as_float(w[j]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    else
      return DTypeTraits<T>::bits_to_float((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
  }

  // Value at a position of the part.
  __device__ __forceinline__ float at(uint32_t pos) const {
    const int slot = (int)pos - first;
    return slot / kVec < held_vectors ? DTypeTraits<T>::bits_to_float(reinterpret_cast<const Bits*>(held)[slot])
                                      : load_value(row, pos);
  }

  // A vector at the part's ends, of which only some places are its own (by
  // value: nothing of the caller's goes through memory).
  static __device__ __noinline__ uint4 end_vector(Row<T> row, int pos, int begin, int end) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const bool mine = pos + j >= begin && pos + j < end;
      const uint32_t bits = DTypeTraits<T>::round_bits(mine ? load_value(row, pos + j) : -INFINITY);
      if constexpr (sizeof(Bits) == 4) w[j] = bits;
      else w[j >> 1] |= bits << (16 * (j & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }

  // Vector v from global memory (in two steps, so that several can be under
  // way): its words, then -inf where the mask says not legal. NaN stays (every
  // comparison with it is false).
  __device__ __forceinline__ uint4 fetch(int v, uint32_t* legal) const {
    *legal = 0xffffffffu;
    if (v < whole0 || v >= whole1) return end_vector(row, first + v * kVec, lo, lo + len);
    if (row.mask) {
      const int pos = first + v * kVec, w0 = pos >> 5, sh = pos & 31;
      const uint32_t a = __ldg(row.mask + w0);
      const uint32_t b = sh + kVec > 32 ? __ldg(row.mask + w0 + 1) : 0u;
      *legal = __funnelshift_r(a, b, sh);
    }
    return ld_stream_v4(base + v);
  }
  __device__ __forceinline__ void settle(const uint4& q, uint32_t legal, uint32_t (&w)[4]) const {
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    if (row.mask == nullptr) return;
    constexpr uint32_t kIllegal = DTypeTraits<T>::kNegInfBits;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const bool ok = (legal >> j) & 1u;
      if constexpr (sizeof(Bits) == 4)
        w[j] = ok ? w[j] : kIllegal;
      else if (j & 1)
        w[j >> 1] = ok ? w[j >> 1] : (w[j >> 1] & 0xffffu) | (kIllegal << 16);
      else
        w[j >> 1] = ok ? w[j >> 1] : (w[j >> 1] & 0xffff0000u) | kIllegal;
    }
  }

  // The places of vector v that hold a value, as bits.
  __device__ __forceinline__ uint32_t places_of(int v, float x) const {
    uint32_t legal = 0xffffffffu, w[4], m = 0u;
    const uint4 q = v < held_vectors ? held[v] : fetch(v, &legal);
    settle(q, legal, w);
#pragma unroll
    for (int j = 0; j < kVec; ++j) m |= unpack(w, j) == x ? 1u << j : 0u;
    return m;
  }

  // Reads the whole part, keeping the held vectors; returns the thread's
  // largest value and its number of legal tokens. Four loads under way.
  __device__ __forceinline__ float load(uint32_t& legal_count) {
    constexpr int kAhead = 4;
    PairMax<T> most;
    legal_count = 0u;
    for (int v0 = threadIdx.x; v0 < vectors; v0 += kAhead * kSampleThreads) {
      uint4 q[kAhead];
      uint32_t legal[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = v0 + k * kSampleThreads;
        q[k] = make_uint4(0u, 0u, 0u, 0u);
        legal[k] = 0u;
        if (v < vectors) q[k] = fetch(v, &legal[k]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = v0 + k * kSampleThreads;
        if (v >= vectors) break;
        uint32_t w[4];
        settle(q[k], legal[k], w);
        uint32_t c = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          most.add(w[j]);
          c += pair_count<T>(pair_above<T>(w[j], -INFINITY));
        }
        legal_count += pair_total<T>(c);
        if (v < held_vectors) held[v] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return most.value();
  }

  // fn(words, position of the first value) for every vector of the part (-inf
  // or NaN: not legal, or not of the part); the next two are under way meanwhile.
  template <typename Fn>
  __device__ __forceinline__ void each_vector(Fn fn) const {
    uint4 q0 = make_uint4(0u, 0u, 0u, 0u), q1 = q0;
    uint32_t legal0 = 0u, legal1 = 0u;
    const auto get = [&](int v) {
      if (v < held_vectors) {
        q1 = held[v];
        legal1 = 0xffffffffu;
      } else if (v < vectors) {
        q1 = fetch(v, &legal1);
      }
    };
    get(threadIdx.x);
    q0 = q1, legal0 = legal1;
    get(threadIdx.x + kSampleThreads);
    for (int v = threadIdx.x; v < vectors; v += kSampleThreads) {
      uint32_t w[4];
      settle(q0, legal0, w);
      q0 = q1, legal0 = legal1;
      get(v + 2 * kSampleThreads);
      fn(w, (uint32_t)(first + v * kVec));
    }
  }
  // fn(value) one by one
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    each_vector([&](const uint32_t (&w)[4], uint32_t pos) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) fn(unpack(w, j), pos + j);
    });
  }
  // fn(four values) for all of them
  template <typename Fn>
  __device__ __forceinline__ void each_four(Fn fn) const {
    each_vector([&](const uint32_t (&w)[4], uint32_t) {
#pragma unroll
      for (int h = 0; h < kVec / 4; ++h) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = unpack(w, 4 * h + j);
        fn(f);
      }
    });
  }
  // fn(value, position) for the values in [from, to] or [from2, to2], which are
  // few; returns how many are above `to`. (Pairs are compared at once; a mask
  // per vector, then its set bits.)
  template <typename Fn>
  __device__ __forceinline__ uint32_t each_between(float from, float to, float from2, float to2, Fn fn) const {
    uint32_t above = 0u;
    each_vector([&](const uint32_t (&w)[4], uint32_t pos) {
      uint32_t in[4], c = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t over = pair_above<T>(w[j], to);
        c += pair_count<T>(over);
        in[j] = (pair_at_least<T>(w[j], from) & ~over) | (pair_at_least<T>(w[j], from2) & ~pair_above<T>(w[j], to2));
      }
      above += pair_total<T>(c);
      if ((in[0] | in[1] | in[2] | in[3]) == 0u) return;
      uint32_t m = 0u;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (sizeof(Bits) == 4) m |= in[j] & (1u << j);
        else m |= ((in[j >> 1] >> (16 * (j & 1))) & 1u) << j;
      }
      while (m) {
        const uint32_t i = pos + (uint32_t)(__ffs(m) - 1);
        m &= m - 1u;
        fn(at(i), i);
      }
    });
    return above;
  }
};

// The listed tokens: one part per CTA of the cluster (or, listed whole, a
// single part), each with a share of the warps.
template <typename T>
struct List {
  const SampleSmemHeader* s;
  int room;        // tokens a part can hold
  uint32_t share;  // this thread's part, its first token there and its step (a byte, two 12-bit fields)
  __device__ __forceinline__ List(const SampleSmemHeader* s_, int parts) : s(s_), room(kListTotal / parts) {
    const uint32_t warp = threadIdx.x >> 5, part = warp % parts;
    const uint32_t step = (kSampleWarps - part + parts - 1u) / parts * 32u;
    share = part | (warp / parts * 32u + (threadIdx.x & 31u)) << 8 | step << 20;
  }
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    const int part = (int)(share & 0xffu), step = (int)(share >> 20), n = (int)s->list_count[part];
    const unsigned long long* e = s->list + part * room;
    for (int i = (int)(share >> 8 & 0xfffu); i < n; i += step) {
      const unsigned long long x = e[i];
      fn(SampleKey<T>::value((uint32_t)(x >> 32)), (uint32_t)x);
    }
  }
};

// A finite value of type T as a double by integer operations (the conversion
// unit is slower); zero and subnormals become some value below 2^-126, which
// moves no weight. 16-bit types end in the high word.
template <typename T>
__device__ __forceinline__ double widen(float f) {
  const uint32_t u = __float_as_uint(f);
  return __hiloint2double((int)((((uint32_t)((int)u >> 3)) & 0x8fffffffu) + (896u << 20)),
                          sizeof(typename DTypeTraits<T>::Bits) == 2 ? 0 : (int)(u << 29));
}

// Weight of a value in units of 2^-shift: with y = shift + log2 w, the nearest
// multiple of 1/16 is q / 16, and 2^y = 2^(q / 16) * 2^(y - q / 16): a table
// entry with its exponent, and the Taylor polynomial of 2^r = exp(r ln 2) to
// degree 5 on |r| <= 1/32 (the next term is below 1.5e-13 and nearly the same
// for all). Sixteen entries take each of the 32 banks once: whatever entries a
// warp's lanes want, there is no bank conflict (with 256 entries and degree 3
// the loads met 5 to a bank, and shared memory was what bound the pass).
template <typename T>
struct Weigher {
  int shift;
  double vmax, per_octave, octave;  // the largest value; log2(e) / T and its inverse
  const double* table;              // 2^(j / 16), j << 16 taken off the high word

  // The weight of a value of at least cut(), as a double before its rounding.
  __device__ __forceinline__ double unrounded(float v) const {
    constexpr double kMagic = 422212465065984.0;  // 1.5 * 2^48: its last place is 1/16
    const double y = fma(widen<T>(v) - vmax, per_octave, (double)shift);
    const double t = y + kMagic;
    const double r = y - (t - kMagic);
    const int q = __double2loint(t);
    double p = fma(r, 1.3333558146428443e-03, 9.6181291076284772e-03);  // ln2^5 / 120, ln2^4 / 24
    p = fma(p, r, 5.5504108664821580e-02);                              // ln2^3 / 6
    p = fma(p, r, 2.4022650695910072e-01);                              // ln2^2 / 2
    p = fma(p, r, 6.9314718055994531e-01);                              // ln2
    const double e = table[q & (kExpTable - 1)];
    const double m = __hiloint2double(__double2hiint(e) + (q << 16), __double2loint(e));
    return fma(p * r, m, m);
  }
  static __device__ __forceinline__ unsigned long long round(double w) {
    // adding 2^52 rounds to an integer, held in the low mantissa bits
    const double rounded = w + 4503599627370496.0;
    return ((unsigned long long)(uint32_t)(__double2hiint(rounded) - 0x43300000) << 32) |
           (uint32_t)__double2loint(rounded);
  }
  // Weighing bin: sixteenths of the weight's octaves, read off its exponent and
  // leading mantissa bits; all below 2^-32 of the maximum share the last.
  __device__ __forceinline__ int bin(double w) const {
    return min(((1023 + shift) << 4) - (__double2hiint(w) >> 16), kBins - 1);
  }
  // Values below this weigh nothing (they would round to 0).
  __device__ __forceinline__ double cut() const { return vmax - (double)(shift + 1) * octave; }
  __device__ __forceinline__ unsigned long long operator()(float v) const { return round(unrounded(v)); }
  // Values that the bins first..last may hold: [*lo, *hi], wider by 2^-20 octave
  // on both sides (rounding moves a border by far less).
  __device__ __forceinline__ void bin_values(int first, int last, double* lo, double* hi) const {
    const auto border = [&](int k) {  // log2 of the least weight of bin k, below the maximum
      // (in doubles: with an integer shift here, nvcc 12.9 lost the shift where
      // first == last)
      const double e = -0.0625 * k, whole = floor(e);
      return whole + kLog2[(int)((e - whole) * 16.0)];
    };
    *hi = vmax + (border(first - 1) + 9.5367431640625e-07) * octave;
    *lo = last == kBins - 1 ? cut() : vmax + (border(last) - 9.5367431640625e-07) * octave;
  }
};

// x in [0, 1) as a multiple of 2^-64 (exact unless x < 2^-40).
__device__ __forceinline__ unsigned long long fraction64(float x) {
  return (unsigned long long)((double)x * 18446744073709551616.0);
}

// The shortest prefix with sum >= x * total is the first whose sum passes
// ceil(x * total) - 1; at least one token (x <= 0).
__device__ __forceinline__ unsigned long long prefix_target(float x, unsigned long long total) {
  const unsigned long long frac = x > 0.f ? fraction64(x) : 0ull;
  if (frac == 0ull) return 0ull;
  return __umul64hi(frac, total) - (frac * total == 0ull ? 1ull : 0ull);
}

// State of the cluster's cooperation; every decision is taken from sums that
// all CTAs hold, so that all of them take the same steps and barriers.
struct Team {
  SampleSmemHeader* s;  // (this CTA's)
  cg::cluster_group cluster;
  int rank, size;
  int room;  // tokens in a CTA's part of the list
  int buf;  // which half of `word` the next all-gather uses

  // All-gather of one value per CTA (the same in all its threads): the returned
  // array holds rank r's at index r until the all-gather after the next.
  __device__ __forceinline__ const unsigned long long* gather(unsigned long long v) {
    unsigned long long* mine = s->word[buf];
    if ((int)threadIdx.x < size) cluster.map_shared_rank(mine, threadIdx.x)[rank] = v;
    cluster.sync();
    buf ^= 1;
    return mine;
  }
};

__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(FULL_MASK, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

// Block-wide sum (in every thread).
__device__ __forceinline__ uint32_t block_sum(uint32_t a, SampleSmemHeader* s) {
  a = __reduce_add_sync(FULL_MASK, a);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s->warp[0][threadIdx.x >> 5] = a;
  __syncthreads();
  return __reduce_add_sync(FULL_MASK, (threadIdx.x & 31) < kSampleWarps ? s->warp[0][threadIdx.x & 15] : 0u);
}

// Sum of a count over the cluster.
__device__ __forceinline__ unsigned long long cluster_sum(Team& team, uint32_t count) {
  const unsigned long long* all = team.gather(block_sum(count, team.s));
  unsigned long long sum = 0ull;
  for (int r = 0; r < team.size; ++r) sum += all[r];
  return sum;
}

// ---- bins ----------------------------------------------------------------------
__device__ __forceinline__ void clear_bins(SampleSmemHeader* s) {
  s->lo[threadIdx.x] = 0u;
  s->hi[threadIdx.x] = 0u;
  __syncthreads();
}

// 64-bit sum in two 32-bit words: the old low word tells the carry.
__device__ __forceinline__ void add_to_bin(SampleSmemHeader* s, uint32_t bin, unsigned long long m) {
  const uint32_t m_lo = (uint32_t)m;
  uint32_t m_hi = (uint32_t)(m >> 32);
  const uint32_t old = atomicAdd(&s->lo[bin], m_lo);
  m_hi += (old + m_lo < old) ? 1u : 0u;
  if (m_hi) atomicAdd(&s->hi[bin], m_hi);
}

// Four at a time: the additions of the low words are under way together before
// the first carry is waited for. Bins from kBins on take anything.
__device__ __forceinline__ void add_to_bins(SampleSmemHeader* s, const uint32_t (&bin)[4],
                                            const unsigned long long (&m)[4]) {
  uint32_t old[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) old[k] = atomicAdd(&s->lo[bin[k]], (uint32_t)m[k]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t hi = (uint32_t)(m[k] >> 32) + (old[k] + (uint32_t)m[k] < old[k] ? 1u : 0u);
    if (hi) atomicAdd(&s->hi[bin[k]], hi);
  }
}

// Sum of a thread's bin and the running sum before it.
struct BinSums {
  unsigned long long before, own;
  // If the bin is where the running sum passes the target, publishes it in
  // s->pick[slot] (read after the next barrier).
  __device__ __forceinline__ void pick(SampleSmemHeader* s, int slot, unsigned long long target) const {
    if (before <= target && target < before + own) {
      s->pick[slot][0] = threadIdx.x;
      s->pick[slot][1] = before;
      s->pick[slot][2] = own;
    }
  }
};

// The block's inclusive running sum, and the sum of all.
__device__ __forceinline__ unsigned long long block_scan_u64(unsigned long long v, SampleSmemHeader* s,
                                                             unsigned long long* total) {
  const int tid = threadIdx.x;
  const unsigned long long incl = warp_scan_u64(v);
  if ((tid & 31) == 31) s->scan[tid >> 5] = incl;
  __syncthreads();
  // every warp scans the warps' totals
  const unsigned long long w = warp_scan_u64((tid & 31) < kSampleWarps ? s->scan[tid & (kSampleWarps - 1)] : 0ull);
  const unsigned long long before_warp = __shfl_sync(FULL_MASK, w, max((tid >> 5) - 1, 0));
  *total = __shfl_sync(FULL_MASK, w, 31);
  return incl + (tid >= 32 ? before_warp : 0ull);
}

// Closes a filling pass: the bins' sums over the cluster, or (local) this
// CTA's; *total: the sum of all bins.
__device__ __forceinline__ BinSums sum_bins(Team& team, bool local, unsigned long long* total) {
  SampleSmemHeader* s = team.s;
  const int tid = threadIdx.x;
  __syncthreads();
  BinSums v;
  v.own = s->lo[tid] + ((unsigned long long)s->hi[tid] << 32);
  if (!local) {
    s->tot[tid] = v.own;
    team.cluster.sync();
    v.own = 0ull;
    for (int r0 = 0; r0 < team.size; r0 += 8) {  // independent loads, eight in flight
      unsigned long long x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = r0 + k < team.size ? team.cluster.map_shared_rank(s->tot, r0 + k)[tid] : 0ull;
#pragma unroll
      for (int k = 0; k < 8; ++k) v.own += x[k];
    }
  }
  v.before = block_scan_u64(v.own, s, total) - v.own;
  return v;
}

// Where a running sum passes a target: the key, the sums above and at it.
struct Found {
  uint32_t key;
  unsigned long long above, own;
};

// Goes on with a search inside keys [klo, khi] of `tokens` (those that
// take(value, &measure) accepts): the first key, from khi down, at which the
// running sum of the measure passes `target`, which it does (the caller knows
// the sum). local: every CTA holds all the tokens.
template <typename T, typename Tokens, typename Take>
__device__ __forceinline__ Found search(Team& team, bool local, const Tokens& tokens, uint32_t klo, uint32_t khi,
                                        Take take, unsigned long long target) {
  SampleSmemHeader* s = team.s;
  Found f{khi, 0ull, 0ull};
  for (int slot = 0;; slot ^= 1) {
    const int width = 32 - __clz(khi - klo);  // bits of the range (0: a single key)
    const int sh = width > kBinBits ? width - kBinBits : 0;
    clear_bins(s);
    tokens.each([&](float v, uint32_t) {
      const uint32_t key = SampleKey<T>::from_value(v);
      unsigned long long m;
      if (key >= klo && key <= khi && take(v, &m)) add_to_bin(s, (khi - key) >> sh, m);
    });
    unsigned long long total;
    sum_bins(team, local, &total).pick(s, slot, target);
    if (local) __syncthreads();
    else team.cluster.sync();  // (and the CTAs have read one another's bins)
    const uint32_t bin = (uint32_t)s->pick[slot][0] & (kBins - 1);
    f.above += s->pick[slot][1];
    f.own = s->pick[slot][2];
    target -= s->pick[slot][1];
    khi -= bin << sh;
    f.key = khi;
    if (sh == 0) {
      __syncthreads();  // the pick has been read
      return f;
    }
    const uint32_t span = (1u << sh) - 1u;
    klo = khi - klo > span ? khi - span : klo;
  }
}

// ---- listing ---------------------------------------------------------------------
__device__ __forceinline__ void open_list(Team& team) {
  __syncthreads();
  if (threadIdx.x == 0) team.s->listed = 0u;
  __syncthreads();
}

// Writes an entry of the first CTA's list.
__device__ __forceinline__ void put_in_list(const Team& team, uint32_t i, uint32_t key, uint32_t at) {
  team.cluster.map_shared_rank(team.s->list, 0)[i] = ((unsigned long long)key << 32) | at;
}

// Offers a token to the CTA's part of the list.
__device__ __forceinline__ void list_token(const Team& team, uint32_t key, uint32_t at) {
  const uint32_t i = atomicAdd(&team.s->listed, 1u);
  if (i < (uint32_t)team.room) put_in_list(team, (uint32_t)(team.rank * team.room) + i, key, at);
}

// After a listing pass: whether every CTA's part fits (then the first CTA has
// them all and goes on alone), and the cluster's sum of `count`. A list that
// does not fit is not read, so the next may be written at once.
__device__ __forceinline__ bool close_list(Team& team, uint32_t count, unsigned long long* sum) {
  SampleSmemHeader* s = team.s;
  const uint32_t part = (uint32_t)team.room;
  count = block_sum(count, s);
  const uint32_t mine = min(s->listed, part + 1u);
  const unsigned long long* all = team.gather(((unsigned long long)mine << 32) | count);
  unsigned long long total = 0ull;
  bool fits = true;
  for (int r = 0; r < team.size; ++r) {
    total += (uint32_t)all[r];
    fits &= (uint32_t)(all[r] >> 32) <= part;
  }
  if (threadIdx.x < kMaxCluster)
    s->list_count[threadIdx.x] = (int)threadIdx.x < team.size ? (uint32_t)(all[threadIdx.x] >> 32) : 0u;
  __syncthreads();
  *sum = total;
  return fits;
}

// Puts up to kFew of the first CTA's listed tokens, those that take(value) says,
// in order. gather_few: how many it says (beyond kFew, they are not kept).
template <typename T, typename Take>
__device__ __forceinline__ int gather_few(SampleSmemHeader* s, const List<T>& list, Take take) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) s->listed = 0u;
  s->lo[tid] = 0u;
  __syncthreads();
  list.each([&](float v, uint32_t at) {
    if (!take(v)) return;
    const uint32_t i = atomicAdd(&s->listed, 1u);
    if (i < (uint32_t)kFew) s->tot[i] = ((unsigned long long)SampleKey<T>::from_value(v) << 32) | (uint32_t)~at;
  });
  __syncthreads();
  return (int)s->listed;
}
// The gathered token of rank threadIdx.x as (key, ~position), 0 past the last.
// Each is compared with all others, by two threads with half of them each.
__device__ __forceinline__ unsigned long long order_few(SampleSmemHeader* s, int count) {
  const int tid = threadIdx.x;
  const int i = tid & (kFew - 1), half = (count + 1) / 2;
  const unsigned long long mine = i < count ? s->tot[i] : 0ull;
  if (i < count) {
    uint32_t before = 0u;
    const int k0 = tid < kFew ? 0 : half, k1 = tid < kFew ? half : count;
#pragma unroll 8
    for (int k = k0; k < k1; ++k) before += s->tot[k] > mine ? 1u : 0u;
    if (before) atomicAdd(&s->lo[i], before);
  }
  __syncthreads();
  if (tid < count) s->tot[kFew + s->lo[tid]] = mine;
  __syncthreads();
  return tid < count ? s->tot[kFew + tid] : 0ull;
}

// Tokens in the list.
__device__ __forceinline__ uint32_t listed_tokens(const SampleSmemHeader* s) {
  const uint32_t lane = threadIdx.x & 31u;
  return __reduce_add_sync(FULL_MASK, lane < (uint32_t)kMaxCluster ? s->list_count[lane] : 0u);
}

// Bin of the top-k search: 64ths of an octave of the distance to the maximum,
// from 1/4 to 64; nearer and farther tokens share the first and last.
constexpr uint32_t kDistanceShift = 17, kDistanceBase = 0x3e800000u >> kDistanceShift;
__device__ __forceinline__ uint32_t distance_bin(float vmax, float v) {
  return min((__float_as_uint(vmax - v + 0.25f) >> kDistanceShift) - kDistanceBase, (uint32_t)kBins - 1u);
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) filtered_sample_kernel(const FilteredSampleParams p) {
  using K = SampleKey<T>;
  using Bits = typename DTypeTraits<T>::Bits;
  extern __shared__ __align__(128) unsigned char smem[];
  SampleSmemHeader* s = reinterpret_cast<SampleSmemHeader*>(smem);
  Team team{s, cg::this_cluster(), 0, 0, 0, 0};
  team.rank = (int)team.cluster.block_rank();
  team.size = (int)team.cluster.num_blocks();
  team.room = kListTotal / team.size;
  const int b = blockIdx.x / team.size, tid = threadIdx.x;

  // ---- the row and its settings ---------------------------------------------
  int64_t start;
  const Row<T> row = row_of<T>(p, b, &start);
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const int64_t top_k = p.top_ks ? p.top_ks[b] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[b] : p.min_p;
  const float u = p.uniforms[b];
  // every CTA of the cluster runs before its shared memory is written to
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  Slice<T> slice;
  const int n = row.n;
  const int64_t part = (((int64_t)n + team.size - 1) / team.size + 31) / 32 * 32;
  const int lo = (int)min(part * team.rank, (int64_t)n);
  slice.set(row, lo, (int)min(part, (int64_t)(n - lo)), smem + kHeaderBytes, p.held_vectors);

  // ---- the row into shared memory, largest value, number of legal tokens ----------
  uint32_t legal = 0u;
  float vmax = slice.load(legal);
  if (tid < kExpTable) {
    const double e = kExp2[tid];
    s->exp2_table[tid] = __hiloint2double(__double2hiint(e) - (tid << 16), __double2loint(e));
  }
  if (tid == 0) s->listed = 0u;
  {
    const uint32_t key = __reduce_max_sync(FULL_MASK, K::from_value(vmax));
    legal = __reduce_add_sync(FULL_MASK, legal);
    if ((tid & 31) == 0) {
      s->warp[0][tid >> 5] = key;
      s->warp[1][tid >> 5] = legal;
    }
  }
  __syncthreads();
  uint32_t kmax = __reduce_max_sync(FULL_MASK, s->warp[0][tid & (kSampleWarps - 1)]);
  legal = __reduce_add_sync(FULL_MASK, (tid & 31) < kSampleWarps ? s->warp[1][tid & (kSampleWarps - 1)] : 0u);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  unsigned long long kept = 0ull;  // tokens left so far
  uint32_t list_base = 0u;         // legal tokens of the CTAs before this one
  {
    const unsigned long long* all = team.gather(((unsigned long long)legal << 32) | kmax);
    for (int r = 0; r < team.size; ++r) {
      const unsigned long long x = all[r];
      kmax = max(kmax, (uint32_t)x);
      kept += x >> 32;
      if (r < team.rank) list_base += (uint32_t)(x >> 32);
    }
  }
  const bool valid = temperature >= 0.f && temperature < INFINITY && top_p == top_p && min_p == min_p && u >= 0.f &&
                     u < 1.f;
  if (!valid || kmax == 0u) {  // not to be drawn, or nothing is legal
    if (team.rank == 0 && tid == 0) {
      p.token_ids[b] = valid ? 0 : -1;
      if (p.logprobs) p.logprobs[b] = valid ? -INFINITY : __int_as_float(0x7fc00000);
      if (p.kept) p.kept[b] = 0;
    }
    return;
  }
  vmax = K::value(kmax);
  const float vmin = K::value(K::kNegInf + 1u);  // the lowest legal value
  const bool infinite = !(vmax < INFINITY);
  List<T> list{s, team.size};

  float draw_value = vmax;
  unsigned long long ordinal = 0ull;  // among the tokens of draw_value, by rising position
  float logprob = 0.f;
  bool solo = false;  // the list holds all that is still needed: this CTA goes on alone
  // the answer: the token at a position
  const auto put = [&](int64_t at) {
    p.token_ids[b] = p.ids ? p.ids[start + at] : p.vocab_offset + at;
    if (p.logprobs) p.logprobs[b] = logprob;
    if (p.kept) p.kept[b] = (int32_t)kept;
  };
  if (temperature > 0.f && !infinite) {
    Weigher<T> weigh;
    weigh.shift = min(kMaxShift, 62 - (64 - __clzll((unsigned long long)n)));
    weigh.vmax = widen<T>(vmax);
    weigh.per_octave = 1.4426950408889634 / (double)temperature;
    weigh.octave = 0.6931471805599453 * (double)temperature;
    weigh.table = s->exp2_table;
    // ---- the kept set: values above `border`, and `ties` tokens at it --------------
    float border = vmin;
    unsigned long long ties = ~0ull, excess = 0ull;  // excess: tokens at the border beyond `ties`
    bool in_list = false;                            // the list holds every kept token
    const auto logprob_of = [&](const Weigher<T>& weigh, float v, unsigned long long sum) {
      return (float)(((double)v - (double)vmax) / (double)temperature -
                     log((double)sum / (double)(1ull << weigh.shift)));
    };
    const auto one = [](float, unsigned long long* m) {
      *m = 1ull;
      return true;
    };
    if (kept <= kListTotal) {
      // few legal tokens: all of them, each CTA's behind the others'
      slice.each_between(vmin, vmax, vmin, vmax, [&](float v, uint32_t at) {
        put_in_list(team, list_base + atomicAdd(&s->listed, 1u), K::from_value(v), at);
      });
      if (tid < kMaxCluster) s->list_count[tid] = tid == 0 ? (uint32_t)kept : 0u;
      list = List<T>(s, 1);
      __syncthreads();
      team.cluster.sync();
      if (team.rank != 0) return;
      in_list = solo = true;
    }
    if (top_k > 0 && (unsigned long long)top_k < kept) {
      const unsigned long long target = (unsigned long long)top_k - 1ull;
      uint32_t klo = 1u;
      if (in_list) {  // the lowest listed key bounds the range
        uint32_t low = kmax;
        list.each([&](float v, uint32_t) { low = min(low, K::from_value(v)); });
        low = __reduce_min_sync(FULL_MASK, low);
        if ((tid & 31) == 0) s->warp[0][tid >> 5] = low;
        __syncthreads();
        klo = __reduce_min_sync(FULL_MASK, s->warp[0][tid & (kSampleWarps - 1)]);
      } else {
        clear_bins(s);
        slice.each([&](float v, uint32_t) {
          if (v > -INFINITY) atomicAdd(&s->lo[distance_bin(vmax, v)], 1u);
        });
        unsigned long long total;
        sum_bins(team, false, &total).pick(s, 0, target);
        __syncthreads();
        // every token down to the picked bin: its lower border, a little wider
        const int j = (int)s->pick[0][0] & (kBins - 1);
        float low = vmin;
        if (j < kBins - 1) {
          const float edge = __uint_as_float((uint32_t)(j + 1 + kDistanceBase) << kDistanceShift) - 0.25f;
          low = fmaxf(vmin, K::value_at_least((double)vmax - (double)edge * 1.00001 - 1e-6 * fabs((double)vmax)));
        }
        open_list(team);
        slice.each_between(low, vmax, low, vmax,
                           [&](float v, uint32_t at) { list_token(team, K::from_value(v), at); });
        unsigned long long unused;
        in_list = solo = close_list(team, 0u, &unused);
        if (solo && team.rank != 0) return;
        if (in_list) klo = K::from_value(low);
      }
      const Found f = in_list ? search<T>(team, true, list, klo, kmax, one, target)
                              : search<T>(team, false, slice, klo, kmax, one, target);
      border = K::value(f.key);
      ties = (unsigned long long)top_k - f.above;
      excess = f.own - ties;
      kept = (unsigned long long)top_k;
    }
    if (min_p > 0.f) {
      const float low =
          min_p >= 1.f ? vmax : fminf(vmax, K::value_at_least((double)vmax + (double)temperature * log((double)min_p)));
      if (low > border) {
        border = low;
        ties = ~0ull;
        excess = 0ull;
        uint32_t count = 0u;
        if (in_list) {
          list.each([&](float v, uint32_t) { count += v >= border ? 1u : 0u; });
          kept = block_sum(count, s);
        } else {
          open_list(team);
          slice.each_between(border, vmax, border, vmax, [&](float v, uint32_t at) {
            ++count;
            list_token(team, K::from_value(v), at);
          });
          in_list = solo = close_list(team, count, &kept);
          if (solo && team.rank != 0) return;
        }
      }
    }
    const float lowest = fmaxf(border, fminf(vmax, K::value_at_least(weigh.cut())));
    // ---- few are left (a top-k, a grammar's tokens): all in order, then running sums --
    if (in_list && kept + excess <= kFew) {
      const int left = gather_few<T>(s, list, [&](float v) { return v >= border; });  // kept + excess
      const unsigned long long token = order_few(s, left);
      const float v = K::value((uint32_t)(token >> 32));
      const unsigned long long w = (unsigned long long)tid < kept && v >= lowest ? weigh(v) : 0ull;
      unsigned long long sum;
      const unsigned long long upto = block_scan_u64(w, s, &sum);
      if (top_p < 1.f) {  // the last kept: the first whose running sum passes the target
        const unsigned long long target = prefix_target(top_p, sum);
        if (upto - w <= target && target < upto) {
          s->pick[0][0] = (unsigned long long)tid + 1ull;
          s->pick[0][1] = upto;
        }
        __syncthreads();
        kept = s->pick[0][0];
        sum = s->pick[0][1];
      }
      const unsigned long long target = __umul64hi(fraction64(u), sum);
      if (upto - w <= target && target < upto) {
        logprob = logprob_of(weigh, v, sum);
        put((uint32_t)~(uint32_t)token);
      }
      return;
    }
    // ---- weigh what is left, by bins ---------------------------------------------
    clear_bins(s);
    const auto into_bin = [&](float v, uint32_t) {
      const double w = weigh.unrounded(v);
      if (v >= lowest) add_to_bin(s, (uint32_t)weigh.bin(w), weigh.round(w));
    };
    if (in_list) {
      list.each(into_bin);
    } else {
      slice.each_four([&](const float (&f)[4]) {
        uint32_t bin[4];
        unsigned long long m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const double w = weigh.unrounded(f[k]);
          m[k] = weigh.round(w);
          bin[k] = f[k] >= lowest ? (uint32_t)weigh.bin(w) : (uint32_t)kBins + (tid & 31);
        }
        add_to_bins(s, bin, m);
      });
    }
    unsigned long long sum;
    const BinSums bins = sum_bins(team, in_list, &sum);
    if (excess && border >= lowest) sum -= excess * weigh(border);
    // Values of a bin, as [*from, *to], a little wider than it.
    const auto bin_values = [&](int first, int last, float* from, float* to) {
      double lo, hi;
      weigh.bin_values(first, last, &lo, &hi);
      *from = fmaxf(lowest, K::value_at_least(lo));
      *to = fmaxf(*from, fminf(vmax, K::value_at_least(hi)));
    };
    // The search for `target` inside bin j (its sum before the bin, its values).
    const auto within = [&](int j, float from, float to, unsigned long long before, unsigned long long target) {
      const auto in_bin = [&](float v, unsigned long long* m) {
        const double w = weigh.unrounded(v);
        *m = weigh.round(w);
        return weigh.bin(w) == j;
      };
      const uint32_t klo = K::from_value(from), khi = K::from_value(to);
      Found f = solo ? search<T>(team, true, list, klo, khi, in_bin, target - before)
                     : search<T>(team, false, slice, klo, khi, in_bin, target - before);
      f.above += before;
      return f;
    };
    const unsigned long long p_target = top_p < 1.f ? prefix_target(top_p, sum) : 0ull;
    int p_bin = 0;
    unsigned long long p_before = 0ull, most = sum;  // most: the kept weight, at most
    float p_from = 0.f, p_to = 0.f;
    if (top_p < 1.f) {
      bins.pick(s, 0, p_target);
      __syncthreads();
      p_bin = (int)s->pick[0][0];
      p_before = s->pick[0][1];
      most = min(sum, p_before + s->pick[0][2]);
      bin_values(p_bin, p_bin, &p_from, &p_to);
      __syncthreads();  // the pick has been read
    }
    unsigned long long n_above = 0ull;  // tokens above p_to (list of bins)
    // the bins that the draw can fall into, the sums before the first and of all
    bins.pick(s, 0, __umul64hi(fraction64(u), top_p < 1.f ? p_before + 1ull : sum));
    bins.pick(s, 1, __umul64hi(fraction64(u), most));
    __syncthreads();
    if (!in_list) {
      // list the border's bin and the draw's
      float from, to;
      bin_values((int)s->pick[0][0], (int)s->pick[1][0], &from, &to);
      if (!(top_p < 1.f)) p_from = from, p_to = to;
      open_list(team);
      const uint32_t above = slice.each_between(
          p_from, p_to, from, to, [&](float v, uint32_t at) { list_token(team, K::from_value(v), at); });
      solo = close_list(team, above, &n_above);
      if (solo && team.rank != 0) return;
    }
    // ---- few tokens in those bins: in order, and their running sums ------------------
    // (a list of bins holds little else; of a list of all tokens they are a small part)
    if (solo && (in_list || listed_tokens(s) <= (uint32_t)kFew)) {
      const int j0 = (int)s->pick[0][0], j1 = (int)s->pick[1][0];
      const float top = in_list ? vmax : p_to;
      uint32_t others = 0u;  // tokens of bins before the border's that are not gathered (less those counted in n_above)
      const int count = gather_few<T>(s, list, [&](float v) {
        if (!(v >= lowest)) return false;
        const int j = weigh.bin(weigh.unrounded(v));
        const bool take = (j >= j0 && j <= j1) || (top_p < 1.f && j == p_bin);
        if (top_p < 1.f && j < p_bin) others += (v <= top ? 1u : 0u) - (take ? 1u : 0u);
        return take;
      });
      if (count <= kFew) {
        others = block_sum(others, s);
        const unsigned long long token = order_few(s, count);
        const float v = K::value((uint32_t)(token >> 32));
        const double unrounded = weigh.unrounded(v);
        const int j = weigh.bin(unrounded);
        const unsigned long long w = tid < count ? weigh.round(unrounded) : 0ull;
        const unsigned long long j_before = s->pick[0][1], j_sum = s->pick[1][1] + s->pick[1][2] - j_before;
        unsigned long long all;  // (its barrier: the picks have been read)
        unsigned long long upto = block_scan_u64(w, s, &all);
        upto = j <= j1 ? j_before + upto : p_before + (upto - j_sum);  // (the draw's bins come first)
        if (top_p < 1.f) {
          if (j == p_bin && upto - w <= p_target && p_target < upto) {
            s->pick[0][0] = (unsigned long long)(tid + 1);
            s->pick[0][1] = upto;
          }
          __syncthreads();
          kept = n_above + (unsigned long long)(int32_t)others + s->pick[0][0];
          sum = s->pick[0][1];
        }
        const unsigned long long target = __umul64hi(fraction64(u), sum);
        if (j <= j1 && upto - w <= target && target < upto) {
          logprob = logprob_of(weigh, v, sum);
          put((uint32_t)~(uint32_t)token);
        }
        return;
      }
    }
    if (top_p < 1.f) {
      const Found f = within(p_bin, p_from, p_to, p_before, p_target);
      const float value = K::value(f.key);
      const unsigned long long w = weigh(value);
      ties = (p_target - f.above) / w + 1ull;
      sum = f.above + ties * w;
      // how many that keeps (of a list of bins: those above the border's bin have been counted)
      uint32_t count = 0u;
      if (solo) {
        const float top = in_list ? vmax : p_to;
        list.each([&](float v, uint32_t) { count += v > value && v <= top ? 1u : 0u; });
        kept = ties + block_sum(count, s) + n_above;
      } else {
        slice.each([&](float v, uint32_t) { count += v > value ? 1u : 0u; });
        kept = ties + cluster_sum(team, count);
      }
    }
    // ---- the draw ------------------------------------------------------------------
    const unsigned long long target = __umul64hi(fraction64(u), sum);
    bins.pick(s, 0, target);
    __syncthreads();
    const int j = (int)s->pick[0][0];
    const unsigned long long before = s->pick[0][1];
    __syncthreads();  // the pick has been read
    float from, to;
    bin_values(j, j, &from, &to);
    const Found f = within(j, from, to, before, target);
    draw_value = K::value(f.key);
    ordinal = (target - f.above) / weigh(draw_value);
    logprob = logprob_of(weigh, draw_value, sum);
  } else if (temperature > 0.f) {
    // a maximum of +inf: its tokens weigh 1 each, every other nothing
    uint32_t at_max = 0u;
    slice.each([&](float v, uint32_t) { at_max += v == vmax ? 1u : 0u; });
    unsigned long long m = cluster_sum(team, at_max);
    if (top_k > 0) kept = min(kept, (unsigned long long)top_k);
    m = min(m, kept);
    if (min_p > 0.f) kept = m;
    if (top_p < 1.f) kept = m = prefix_target(top_p, m) + 1ull;
    ordinal = __umul64hi(fraction64(u), m);
    logprob = (float)-log((double)m);
  } else {
    kept = 1ull;
  }

  // ---- the drawn token: the ordinal-th of draw_value, by rising position ----------------
  if (solo) {
    // the positions of draw_value's tokens; each counts those before it
    uint32_t* ties_at = s->ties_at;
    __syncthreads();
    if (tid == 0) s->listed = 0u;
    __syncthreads();
    list.each([&](float v, uint32_t at) {
      if (v != draw_value) return;
      const uint32_t i = atomicAdd(&s->listed, 1u);
      if (i < kTiesCap) ties_at[i] = at;
    });
    __syncthreads();
    const uint32_t m = s->listed;
    if (m > kTiesCap) {  // very many ties: each counts those before it in the list itself
      list.each([&](float v, uint32_t at) {
        if (v != draw_value) return;
        uint32_t lower = 0u;
        for (int r = 0; r < kMaxCluster; ++r)  // (parts that there are not have count 0)
          for (uint32_t k = 0; k < s->list_count[r]; ++k) {
            const unsigned long long e = s->list[(uint32_t)(r * list.room) + k];
            lower += ((uint32_t)(e >> 32) == K::from_value(draw_value) && (uint32_t)e < at) ? 1u : 0u;
          }
        if (lower == ordinal) put(at);
      });
      return;
    }
    for (uint32_t i = tid; i < m; i += kSampleThreads) {
      const uint32_t at = ties_at[i];
      uint32_t lower = 0u;
#pragma unroll 4
      for (uint32_t k = 0; k < m; ++k) lower += ties_at[k] < at ? 1u : 0u;
      if (lower == ordinal) put(at);
    }
    return;
  }
  uint32_t here = 0u;
  slice.each([&](float v, uint32_t) { here += v == draw_value ? 1u : 0u; });
  here = block_sum(here, s);
  const unsigned long long* all = team.gather(here);
  for (int r = 0; r < team.rank; ++r) ordinal -= all[r];  // wraps for CTAs behind the owner
  if (ordinal >= here) return;
  // a vector per thread at a time, in order
  constexpr int kVec = Slice<T>::kVec;
  for (int v0 = 0; v0 < slice.vectors; v0 += kSampleThreads) {
    const uint32_t hits = v0 + tid < slice.vectors ? slice.places_of(v0 + tid, draw_value) : 0u;
    uint32_t incl = __popc(hits);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(FULL_MASK, incl, o);
      if ((tid & 31) >= o) incl += t;
    }
    __syncthreads();
    if ((tid & 31) == 31) s->warp[0][tid >> 5] = incl;
    __syncthreads();
    const uint32_t of_warp = (tid & 31) < kSampleWarps ? s->warp[0][tid & (kSampleWarps - 1)] : 0u;
    const uint32_t in_block = __reduce_add_sync(FULL_MASK, of_warp);
    if (ordinal >= in_block) {
      ordinal -= in_block;
      continue;
    }
    const uint32_t last = incl + __reduce_add_sync(FULL_MASK, (tid & 31) < (tid >> 5) ? of_warp : 0u);
    const uint32_t before = last - __popc(hits);
    if (before <= ordinal && ordinal < last) {
      uint32_t m = hits;
      for (uint32_t i = before; i < (uint32_t)ordinal; ++i) m &= m - 1u;
      put(slice.first + (v0 + tid) * kVec + (__ffs(m) - 1));
    }
    return;
  }
}

// ===========================================================================
// rows of 16-bit logits, one CTA per row: every value is counted
// ===========================================================================
// A row of fp16 or bf16 logits has few distinct values (some thousand), so one
// shared-memory addition per token, whatever its weight, is all that the row's
// pass costs: count[m] holds, for the magnitude m (the value's bits without the
// sign), how many tokens have it (low half) and how many of those are negative
// (high half). The exponentials are then taken once per distinct value, and
// every search (top-k, top-p, the draw) is one over the counts. The row is read
// a second time, from L2, to find the drawn value's positions.
//
// A magnitude of more than 65,535 tokens overflows its half; the sum of the
// counts then differs from the number of tokens (every overflow makes it
// smaller), and the counts of a chunk are taken from the row each time they are
// needed, in 32 bits (several passes: right, but slow).
//
// Order: chunks of 1024 magnitudes, positive ones from the largest magnitude
// down, then negative ones up; within a chunk thread t has the t-th value.
constexpr int kCountThreads = 1024;
constexpr int kCountWarps = kCountThreads / 32;
constexpr int kMagnitudes = 1 << 15;
constexpr int kChunks = 2 * kMagnitudes / kCountThreads;
static_assert(kChunks == 64 && kCountWarps == 32, "a warp scans the chunks and the warps");

struct CountSmem {
  uint32_t count[kMagnitudes];
  uint32_t lo[kChunks], hi[kChunks];  // weights of the chunks, in 64 bits
  uint32_t tokens[kChunks];           // tokens of the chunks
  unsigned long long scan[kCountWarps];
  unsigned long long pick[4];
  double exp2_table[kExpTable];
  uint32_t warp[2][kCountWarps];
};

// Magnitude and sign of chunk o's place t.
struct Place {
  uint32_t m;
  bool negative;
};
__device__ __forceinline__ Place place_of(int o, int t) {
  return o < kChunks / 2 ? Place{(uint32_t)((kChunks / 2 - 1 - o) * kCountThreads + (kCountThreads - 1 - t)), false}
                         : Place{(uint32_t)((o - kChunks / 2) * kCountThreads + t), true};
}
__device__ __forceinline__ int chunk_of(uint32_t m, bool negative) {
  const int j = (int)(m / kCountThreads);
  return negative ? kChunks / 2 + j : kChunks / 2 - 1 - j;
}

template <typename T>
struct Counted {
  static constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  CountSmem* s;
  const Slice<T>* row;
  bool overflow;

  // fn(16-bit pattern) for every token that the mask allows and whose pattern is
  // not -inf (NaN included)
  template <typename Fn>
  __device__ __forceinline__ void each_pattern(Fn fn) const {
    constexpr int kAhead = 4;
    for (int v0 = threadIdx.x; v0 < row->vectors; v0 += kAhead * kCountThreads) {
      uint4 q[kAhead];
      uint32_t legal[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = v0 + k * kCountThreads;
        q[k] = make_uint4(0u, 0u, 0u, 0u);
        legal[k] = 0u;
        if (v < row->vectors) q[k] = row->fetch(v, &legal[k]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (v0 + k * kCountThreads >= row->vectors) break;
        const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu;
          if (b != (0x8000u | kInf) && (legal[k] & (1u << j))) fn(b);
        }
      }
    }
  }

  // Fills the counts; returns the thread's number of tokens counted.
  __device__ __forceinline__ uint32_t count_all() const {
    uint32_t counted = 0u;
    each_pattern([&](uint32_t b) {
      ++counted;
      atomicAdd(&s->count[b & 0x7fffu], ((b & 0x8000u) << 1) | 1u);
    });
    return counted;
  }

  // Before chunk o's counts are asked for (all threads): after an overflow they
  // are counted from the row.
  __device__ __forceinline__ void prepare(int o) const {
    if (!overflow) return;
    __syncthreads();
    s->count[threadIdx.x] = 0u;
    __syncthreads();
    each_pattern([&](uint32_t b) {
      const uint32_t m = b & 0x7fffu;
      const bool negative = (b & 0x8000u) != 0u && m != 0u;
      if (m > kInf || (negative && m == kInf) || chunk_of(m, negative) != o) return;
      atomicAdd(&s->count[negative ? m % kCountThreads : kCountThreads - 1u - m % kCountThreads], 1u);
    });
    __syncthreads();
  }
  // Tokens of chunk o's place threadIdx.x.
  __device__ __forceinline__ uint32_t tokens(int o) const {
    if (overflow) return s->count[threadIdx.x];
    const Place at = place_of(o, threadIdx.x);
    if (at.m > kInf) return 0u;
    const uint32_t c = s->count[at.m];
    if (at.m == 0u) return at.negative ? 0u : c & 0xffffu;  // -0 is 0
    return at.negative ? c >> 16 : (c & 0xffffu) - (c >> 16);
  }
  static __device__ __forceinline__ float value(int o, int t) {
    const Place at = place_of(o, t);
    return DTypeTraits<T>::bits_to_float((uint16_t)(at.m | (at.negative ? 0x8000u : 0u)));
  }
};

__device__ __forceinline__ uint32_t count_block_sum(uint32_t a, CountSmem* s) {
  a = __reduce_add_sync(FULL_MASK, a);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s->warp[0][threadIdx.x >> 5] = a;
  __syncthreads();
  return __reduce_add_sync(FULL_MASK, s->warp[0][threadIdx.x & 31]);
}

// The chunk (of two per lane: a, b) at which the running sum passes the target:
// its number, and the sum before it. All warps compute the same.
__device__ __forceinline__ int pick_chunk(unsigned long long a, unsigned long long b, unsigned long long target,
                                          unsigned long long* before) {
  const unsigned long long incl = warp_scan_u64(a + b), excl = incl - (a + b);
  const bool here = excl <= target && target < incl, second = target >= excl + a;
  const unsigned m = __ballot_sync(FULL_MASK, here);
  const int lane = m ? __ffs(m) - 1 : 31;
  *before = __shfl_sync(FULL_MASK, second ? excl + a : excl, lane);
  return __shfl_sync(FULL_MASK, 2 * (int)(threadIdx.x & 31) + (second ? 1 : 0), lane);
}

// The place at which the running sum over the block's `own` passes the target
// (which it does); pick: {place, sum before it, its own}.
__device__ __forceinline__ void pick_place(CountSmem* s, unsigned long long own, unsigned long long target) {
  const int tid = threadIdx.x;
  const unsigned long long incl_w = warp_scan_u64(own);
  __syncthreads();  // the last pick has been read
  if ((tid & 31) == 31) s->scan[tid >> 5] = incl_w;
  __syncthreads();
  const unsigned long long w = warp_scan_u64(s->scan[tid & 31]);
  const unsigned long long warp_before = __shfl_sync(FULL_MASK, w, max((tid >> 5) - 1, 0));
  const unsigned long long incl = incl_w + (tid >= 32 ? warp_before : 0ull), excl = incl - own;
  if (excl <= target && target < incl) {
    s->pick[0] = tid;
    s->pick[1] = excl;
    s->pick[2] = own;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kCountThreads, 1) counted_sample_kernel(const FilteredSampleParams p) {
  using K = SampleKey<T>;
  using Bits = typename DTypeTraits<T>::Bits;
  extern __shared__ __align__(128) unsigned char smem[];
  CountSmem* s = reinterpret_cast<CountSmem*>(smem);
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;

  // ---- the row and its settings ---------------------------------------------
  int64_t start;
  const Row<T> row = row_of<T>(p, b, &start);
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const int64_t top_k = p.top_ks ? p.top_ks[b] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[b] : p.min_p;
  const float u = p.uniforms[b];
  const int n = row.n;
  Slice<T> slice;
  slice.set(row, 0, n, nullptr, 0);

  // ---- count ------------------------------------------------------------------
#pragma unroll
  for (int i = 0; i < kMagnitudes / 4 / kCountThreads; ++i)
    reinterpret_cast<uint4*>(s->count)[i * kCountThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
  if (tid < kChunks) s->lo[tid] = s->hi[tid] = s->tokens[tid] = 0u;
  if (tid < kExpTable) {
    const double e = kExp2[tid];
    s->exp2_table[tid] = __hiloint2double(__double2hiint(e) - (tid << 16), __double2loint(e));
  }
  __syncthreads();
  Counted<T> c{s, &slice, false};
  const uint32_t counted = count_block_sum(c.count_all(), s);
  // tokens of each chunk; all magnitudes' low halves must add up to what was counted
  uint32_t low = 0u, top = 0u;  // top: the largest key met
  for (int j = 0; j < kMagnitudes / kCountThreads; ++j) {
    const uint32_t m = (uint32_t)(j * kCountThreads + tid), x = s->count[m];
    low += x & 0xffffu;
    if (__ballot_sync(FULL_MASK, x != 0u) == 0u) continue;
    const uint32_t negative = m == 0u || m >= Counted<T>::kInf ? 0u : x >> 16;
    const uint32_t positive = m > Counted<T>::kInf ? 0u : (x & 0xffffu) - (m == 0u ? 0u : x >> 16);
    top = max(top, positive ? 0x8000u + m : negative ? 0x8000u - m : 0u);
    const uint32_t a = __reduce_add_sync(FULL_MASK, positive), d = __reduce_add_sync(FULL_MASK, negative);
    if (lane == 0 && a) atomicAdd(&s->tokens[chunk_of(m, false)], a);
    if (lane == 0 && d) atomicAdd(&s->tokens[chunk_of(m, true)], d);
  }
  top = __reduce_max_sync(FULL_MASK, top);
  if (lane == 0) s->warp[1][tid >> 5] = top;
  c.overflow = count_block_sum(low, s) != counted;
  if (c.overflow) {
    __syncthreads();
    if (tid < kChunks) s->tokens[tid] = 0u;
    __syncthreads();
    c.each_pattern([&](uint32_t x) {
      const uint32_t m = x & 0x7fffu;
      const bool negative = (x & 0x8000u) != 0u && m != 0u;
      if (m <= Counted<T>::kInf && !(negative && m == Counted<T>::kInf))
        atomicAdd(&s->tokens[chunk_of(m, negative)], 1u);
    });
    __syncthreads();
  }
  // two chunks per lane, in every warp
  const uint32_t t0 = s->tokens[2 * lane], t1 = s->tokens[2 * lane + 1];
  unsigned long long kept = __reduce_add_sync(FULL_MASK, t0 + t1);  // tokens left so far
  const unsigned long long filled =
      (unsigned long long)__ballot_sync(FULL_MASK, t0 != 0u) | ((unsigned long long)__ballot_sync(FULL_MASK, t1 != 0u) << 32);
  const auto is_filled = [&](int o) { return ((filled >> ((o & 1) * 32 + (o >> 1))) & 1ull) != 0ull; };
  const bool valid = temperature >= 0.f && temperature < INFINITY && top_p == top_p && min_p == min_p && u >= 0.f &&
                     u < 1.f;
  if (!valid || kept == 0ull) {  // not to be drawn, or nothing is legal
    if (tid == 0) {
      p.token_ids[b] = valid ? 0 : -1;
      if (p.logprobs) p.logprobs[b] = valid ? -INFINITY : __int_as_float(0x7fc00000);
      if (p.kept) p.kept[b] = 0;
    }
    return;
  }

  // The value at which the running number of tokens passes a target.
  struct Border {
    float value;
    unsigned long long above, own;  // tokens above it, and of it
  };
  const auto by_tokens = [&](unsigned long long target) {
    unsigned long long before;
    const int o = pick_chunk(t0, t1, target, &before);
    c.prepare(o);
    pick_place(s, c.tokens(o), target - before);
    return Border{Counted<T>::value(o, (int)s->pick[0]), before + s->pick[1], s->pick[2]};
  };
  const float vmax = c.overflow ? by_tokens(0ull).value : K::value(__reduce_max_sync(FULL_MASK, s->warp[1][lane]));
  const bool infinite = !(vmax < INFINITY);
  float draw_value = vmax;
  unsigned long long ordinal = 0ull;  // among the tokens of draw_value, by rising position
  float logprob = 0.f;
  if (temperature > 0.f && !infinite) {
    Weigher<T> weigh;
    weigh.shift = min(kMaxShift, 62 - (64 - __clzll((unsigned long long)n)));
    weigh.vmax = widen<T>(vmax);
    weigh.per_octave = 1.4426950408889634 / (double)temperature;
    weigh.octave = 0.6931471805599453 * (double)temperature;
    weigh.table = s->exp2_table;
    // ---- the kept set: values above `border`, and `ties` tokens at it ----------------
    float border = -INFINITY;
    unsigned long long ties = ~0ull, excess = 0ull;
    if (top_k > 0 && (unsigned long long)top_k < kept) {
      const Border f = by_tokens((unsigned long long)top_k - 1ull);
      border = f.value;
      ties = (unsigned long long)top_k - f.above;
      excess = f.own - ties;
      kept = (unsigned long long)top_k;
    }
    const float lowest_weighed = fminf(vmax, K::value_at_least(weigh.cut()));
    bool below = false;  // min-p moved the border
    if (min_p > 0.f) {
      const float low_value =
          min_p >= 1.f ? vmax : fminf(vmax, K::value_at_least((double)vmax + (double)temperature * log((double)min_p)));
      if (low_value > border) {
        border = low_value;
        ties = ~0ull;
        excess = 0ull;
        below = true;
      }
    }
    // ---- weigh the chunks' values -------------------------------------------------------
    const float lowest = fmaxf(border, lowest_weighed);
    const auto weight_here = [&](int o) {
      const uint32_t x = c.tokens(o);
      const float v = Counted<T>::value(o, tid);
      return x != 0u && v >= lowest ? (unsigned long long)x * weigh(v) : 0ull;
    };
    uint32_t n_kept = 0u;
    const auto add_chunk = [&](int o, uint32_t x, float v, unsigned long long w) {
      if (below) n_kept += v >= border ? x : 0u;
      // (w < 2^62: three parts whose sums over the warp fit 32 bits)
      const unsigned long long sum_w =
          (unsigned long long)__reduce_add_sync(FULL_MASK, (uint32_t)w & 0x7ffffffu) +
          ((unsigned long long)__reduce_add_sync(FULL_MASK, (uint32_t)(w >> 27) & 0x7ffffffu) << 27) +
          ((unsigned long long)__reduce_add_sync(FULL_MASK, (uint32_t)(w >> 54)) << 54);
      if (lane == 31 && sum_w) {
        const uint32_t old = atomicAdd(&s->lo[o], (uint32_t)sum_w);
        const uint32_t hi = (uint32_t)(sum_w >> 32) + (old + (uint32_t)sum_w < old ? 1u : 0u);
        if (hi) atomicAdd(&s->hi[o], hi);
      }
    };
    if (c.overflow) {
      for (int o = 0; o < kChunks; ++o) {
        if (!is_filled(o)) continue;
        c.prepare(o);
        const uint32_t x = c.tokens(o);
        const float v = Counted<T>::value(o, tid);
        add_chunk(o, x, v, x != 0u && v >= lowest ? (unsigned long long)x * weigh(v) : 0ull);
      }
    } else {
      // every warp by itself, over the chunks in which its places have tokens;
      // two at a time, so that their chains of arithmetic run side by side
      uint32_t busy_lo = 0u, busy_hi = 0u;  // those chunks, a bit each
      for (int o = 0; o < kChunks; ++o) {
        if (!is_filled(o)) continue;
        if (__ballot_sync(FULL_MASK, c.tokens(o) != 0u) == 0u) continue;
        if (o < 32) busy_lo |= 1u << o;
        else busy_hi |= 1u << (o - 32);
      }
      unsigned long long busy = ((unsigned long long)busy_hi << 32) | busy_lo;
      while (busy) {
        const int o0 = __ffsll((long long)busy) - 1;
        busy &= busy - 1ull;
        const int o1 = busy ? __ffsll((long long)busy) - 1 : o0;
        const bool two = busy != 0ull;
        busy &= busy - 1ull;  // (0 stays 0)
        const uint32_t x0 = c.tokens(o0), x1 = c.tokens(o1);
        const float v0 = Counted<T>::value(o0, tid), v1 = Counted<T>::value(o1, tid);
        const unsigned long long e0 = weigh(v0), e1 = weigh(v1);
        add_chunk(o0, x0, v0, x0 != 0u && v0 >= lowest ? (unsigned long long)x0 * e0 : 0ull);
        if (two) add_chunk(o1, x1, v1, x1 != 0u && v1 >= lowest ? (unsigned long long)x1 * e1 : 0ull);
      }
    }
    if (below) kept = count_block_sum(n_kept, s);
    __syncthreads();
    const unsigned long long w0 = s->lo[2 * lane] + ((unsigned long long)s->hi[2 * lane] << 32);
    const unsigned long long w1 = s->lo[2 * lane + 1] + ((unsigned long long)s->hi[2 * lane + 1] << 32);
    unsigned long long sum = __shfl_sync(FULL_MASK, warp_scan_u64(w0 + w1), 31);
    if (excess && border >= lowest) sum -= excess * weigh(border);
    // The value at which the running weight passes a target, its chunk and place.
    const auto by_weight = [&](unsigned long long target, int* o, int* place) {
      unsigned long long before;
      *o = pick_chunk(w0, w1, target, &before);
      c.prepare(*o);
      pick_place(s, weight_here(*o), target - before);
      *place = (int)s->pick[0];
      return Border{Counted<T>::value(*o, *place), before + s->pick[1], s->pick[2]};
    };
    if (top_p < 1.f) {
      const unsigned long long target = prefix_target(top_p, sum);
      int o, place;
      const Border f = by_weight(target, &o, &place);
      const unsigned long long w = weigh(f.value);
      ties = (target - f.above) / w + 1ull;
      sum = f.above + ties * w;
      // the tokens above it: of the chunks before, and of its chunk's places before
      const uint32_t upto = (2 * lane < o ? t0 : 0u) + (2 * lane + 1 < o ? t1 : 0u);
      kept = ties + __reduce_add_sync(FULL_MASK, upto) + count_block_sum(tid < place ? c.tokens(o) : 0u, s);
    }
    // ---- the draw ------------------------------------------------------------------------
    const unsigned long long target = __umul64hi(fraction64(u), sum);
    int o, place;
    const Border f = by_weight(target, &o, &place);
    draw_value = f.value;
    ordinal = (target - f.above) / weigh(draw_value);
    logprob = (float)(((double)draw_value - (double)vmax) / (double)temperature -
                      log((double)sum / (double)(1ull << weigh.shift)));
  } else if (temperature > 0.f) {
    // a maximum of +inf: its tokens weigh 1 each, every other nothing
    unsigned long long m = by_tokens(0ull).own;
    if (top_k > 0) kept = min(kept, (unsigned long long)top_k);
    m = min(m, kept);
    if (min_p > 0.f) kept = m;
    if (top_p < 1.f) kept = m = prefix_target(top_p, m) + 1ull;
    ordinal = __umul64hi(fraction64(u), m);
    logprob = (float)-log((double)m);
  } else {
    kept = 1ull;
  }

  // ---- the drawn token: the ordinal-th of draw_value, by rising position ----------------
  // The row is gone over in quarters, until the one that holds it; in a quarter
  // each warp has a run of vectors, and the warp whose run holds it goes over
  // that again in order.
  constexpr int kVec = Slice<T>::kVec;
  // the vector's places that hold the value, as bits
  const auto hits = [&](const uint4& q, uint32_t legal) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t same = pair_at_least<T>(w[j], draw_value) & ~pair_above<T>(w[j], draw_value);
      m |= ((same & 1u) | ((same >> 15) & 2u)) << (2 * j);
    }
    return m & legal;
  };
  const int quarter = max((slice.vectors + 3) / 4, 8 * kCountThreads / kVec);
  uint32_t passed = 0u;  // its tokens in the quarters before
  for (int q_lo = 0; q_lo < slice.vectors; q_lo += quarter) {
    const int q_hi = min(q_lo + quarter, slice.vectors), run = (q_hi - q_lo + kCountWarps - 1) / kCountWarps;
    const int v_lo = min(q_lo + (tid >> 5) * run, q_hi), v_hi = min(v_lo + run, q_hi);
    uint32_t here = 0u;
    for (int v0 = v_lo + lane; v0 < v_hi; v0 += 8 * 32) {
      uint4 q[8];
      uint32_t legal[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        legal[k] = 0u;
        q[k] = make_uint4(0u, 0u, 0u, 0u);
        if (v0 + 32 * k < v_hi) q[k] = slice.fetch(v0 + 32 * k, &legal[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (v0 + 32 * k < v_hi) here += __popc(hits(q[k], legal[k]));
    }
    here = __reduce_add_sync(FULL_MASK, here);
    __syncthreads();
    if (lane == 0) s->warp[0][tid >> 5] = here;
    __syncthreads();
    const uint32_t mine = s->warp[0][lane];
    const uint32_t incl_runs = (uint32_t)warp_scan_u64(mine), total = __shfl_sync(FULL_MASK, incl_runs, 31);
    if (ordinal >= (unsigned long long)passed + total) {
      passed += total;
      continue;
    }
    // hits before this warp's run
    const uint32_t before = passed + __shfl_sync(FULL_MASK, incl_runs - mine, tid >> 5);
    if (ordinal < before || ordinal >= (unsigned long long)before + here) return;
    uint32_t left = (uint32_t)ordinal - before;
    for (int v0 = v_lo; v0 < v_hi; v0 += 32) {
      const int v = v0 + lane;
      uint32_t legal, m = 0u;
      if (v < v_hi) {
        const uint4 q = slice.fetch(v, &legal);
        m = hits(q, legal);
      }
      const uint32_t k = __popc(m), incl = (uint32_t)warp_scan_u64(k), found = __shfl_sync(FULL_MASK, incl, 31);
      if (left >= found) {
        left -= found;
        continue;
      }
      if (incl - k <= left && left < incl) {
        for (uint32_t i = incl - k; i < left; ++i) m &= m - 1u;
        const int64_t at = slice.first + v * kVec + (__ffs(m) - 1);
        p.token_ids[b] = p.ids ? p.ids[start + at] : p.vocab_offset + at;
        if (p.logprobs) p.logprobs[b] = logprob;
        if (p.kept) p.kept[b] = (int32_t)kept;
      }
      return;
    }
    return;
  }
}

template <typename T>
cudaError_t launch_counted(const FilteredSampleParams& p, int batch, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  auto k = counted_sample_kernel<T>;
  if ((err = raise_smem_limit(reinterpret_cast<const void*>(k), sizeof(CountSmem), dev)) != cudaSuccess) return err;
  k<<<batch, kCountThreads, sizeof(CountSmem), stream>>>(p);
  return cudaGetLastError();
}

// ---- launch: one cluster per row ------------------------------------------------
constexpr size_t kSmemFull = 227 * 1024, kSmemHalf = kSmemFull / 2 - 1024;  // a CTA alone on its SM, or two

// How many clusters of `size` CTAs with that shared memory the device holds at a
// time: a cluster lies within one GPC, and what a GPC has left over is lost (of
// 148 SMs, 45 clusters of 3 CTAs alone on their SMs, 93 of half the shared memory).
template <typename T>
int resident_clusters(int dev, int size, bool full) {
  static std::atomic<int> known[32][kMaxCluster + 1][2];  // plus one; 0: not asked yet
  const bool keep = dev < 32;
  if (keep) {
    const int n = known[dev][size][full].load(std::memory_order_relaxed);
    if (n > 0) return n - 1;
  }
  auto k = filtered_sample_kernel<T>;
  const size_t smem = full ? kSmemFull : kSmemHalf;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (raise_smem_limit(reinterpret_cast<const void*>(k), smem, dev) != cudaSuccess ||
      (size > 8 && cudaFuncSetAttribute(reinterpret_cast<const void*>(k),
                                        cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
      cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess) {
    cudaGetLastError();  // (then that size is not taken)
    n = 0;
  }
  if (keep) known[dev][size][full].store(n + 1, std::memory_order_relaxed);
  return n;
}

// CTAs per row, and whether each has its SM's shared memory to itself. Every
// row's cluster has to be resident at once (a second wave doubles the time); of
// those sizes, the one that is done first by this count, in tokens: those of a
// CTA (1.75 times as many where two share an SM), and for every CTA of the
// cluster what the barriers cost, about 1,000 tokens' time, more past 8 CTAs.
// Measured, no filter / top-k 50, us (normal logits): 48 x 262,144 fp32 in
// clusters of 6 (a second wave) 80 / 47, of 5 65 / 35, of 4 75 / 39, of 3 on
// half the shared memory 96 / 49; 40 x 50,257 bf16 of 7 26 / 22, of 3 21 / 14;
// 16 x 262,144 fp32 of 16 45 / 31, of 6 38 / 22; 8 x 151,936 bf16 of 16 21 / 19,
// of 8 24 / 14; 4 x 262,144 fp32 of 16 24 / 17, of 8 29 / 19.
struct LaunchShape {
  int size;
  bool full;
};
template <typename T>
LaunchShape launch_shape(int dev, int batch, int64_t max_len) {
  const int sms = num_sms(dev);
  LaunchShape best{1, false};
  if (batch > sms) return best;
  int64_t best_cost = INT64_MAX;
  for (int size = 1; size <= kMaxCluster; size = size < 8 ? size + 1 : 2 * size) {
    const int64_t ctas = (int64_t)batch * size, part = (max_len + size - 1) / size;
    const int64_t barriers = 1000 * size + (size > 8 ? 4000 : 0);
    for (const bool full : {true, false}) {
      const int64_t cost = (full ? part : part + part * 3 / 4) + barriers;
      if (ctas > (full ? 1 : 2) * (int64_t)sms || cost >= best_cost ||
          resident_clusters<T>(dev, size, full) < batch)
        continue;
      best_cost = cost;
      best = LaunchShape{size, full};
    }
  }
  return best;
}

template <typename T>
cudaError_t launch_typed(FilteredSampleParams p, int batch, int64_t max_len, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const LaunchShape shape = launch_shape<T>(dev, batch, max_len);
  const int size = shape.size;
  // what shared memory does not hold is read again from L2
  const size_t room = (shape.full ? kSmemFull : kSmemHalf) - kHeaderBytes;
  const int64_t part = ((max_len + size - 1) / size + 31) / 32 * 32;
  const int64_t part_vectors = (part * (int64_t)sizeof(typename DTypeTraits<T>::Bits) + 15) / 16 + 1;
  p.held_vectors = (int)std::min<int64_t>((int64_t)(room / 16), part_vectors);
  const size_t smem = kHeaderBytes + (size_t)p.held_vectors * 16;
  auto k = filtered_sample_kernel<T>;
  if ((err = raise_smem_limit(reinterpret_cast<const void*>(k), smem, dev)) != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * size));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, p);
}

// Whether rows of 16-bit logits are better counted, one CTA per row, than
// weighed by a cluster each. Counting costs a row some 18 us (fp16, which has
// more distinct values: 36) and 1 us per 8,000 tokens, a row per SM at a time;
// clusters some 13 us and 1 us per 312,500 tokens of the batch. A top-k or min-p
// known to leave few tokens spares a cluster the weighing, and is left to it.
// Measured, counted / clusters, no filter and top-k 50, us (normal logits): 128 x
// 248,320 bf16 49 / 117 and 50 / 48, fp16 69 / 114 and 67 / 49; 64 x 151,936 bf16
// 37 / 46 and 38 / 23, fp16 56 / 44 and 54 / 23; 64 x 65,536 bf16 27 / 27 and
// 28 / 16; 256 x 32,768 bf16 43 / 37; 32 x 248,320 fp16 69 / 39. Greedy, 64 x
// 151,936 bf16 28 / 15, 128 x 248,320 fp16 42 / 40. Settings per request are not
// known here and count as no filter.
bool counting_pays(const FilteredSampleParams& p, int dtype, int batch, int64_t max_len, int sms) {
  const bool few = (p.top_ks == nullptr && p.top_k > 0 && p.top_k <= 1000) ||
                   (p.min_ps == nullptr && p.min_p >= 0.02f) || (p.temperatures == nullptr && p.temperature == 0.f);
  if (few) return false;
  const int64_t waves = (batch + sms - 1) / sms;
  const double counted = (double)waves * ((dtype == 1 ? 18.0 : 36.0) + (double)max_len / 8000.0);
  const double clusters = 13.0 + (double)batch * (double)max_len / 312500.0;
  return counted < clusters;
}

}  // namespace

cudaError_t launch_filtered_sample(const FilteredSampleParams& p, int dtype, int batch, int64_t max_len,
                                   cudaStream_t stream) {
  if (dtype == 2) return launch_typed<float>(p, batch, max_len, stream);
  int dev = 0;
  const cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (counting_pays(p, dtype, batch, max_len, num_sms(dev)))
    return dtype == 1 ? launch_counted<__nv_bfloat16>(p, batch, stream) : launch_counted<__half>(p, batch, stream);
  if (dtype == 1) return launch_typed<__nv_bfloat16>(p, batch, max_len, stream);
  return launch_typed<__half>(p, batch, max_len, stream);
}

}  // namespace gsp
