// Sampling with temperature, top-k, min-p and top-p from given uniform numbers
// (sm_100a), on the logits the head's routes write or on packed legal rows.
//
// For one row with legal logits x_i (bit set, not NaN, not -inf), in the order
// "falling logit, ties by rising position", and w_i = exp((x_i - max) / T):
//   top-k   keep the first k                                  (k <= 0: all)
//   min-p   keep w_i >= min_p                                 (min_p <= 0: all)
//   top-p   keep the shortest prefix with sum >= top_p * sum  (top_p >= 1: all)
//   draw    the first kept i with w_1 + ... + w_i > u * (sum of the kept)
// Each filter leaves a prefix of that order, so a kept set is a border key and
// a number of ties kept at it, and the draw is one more such border: all four
// are the search for the first position where a running sum (of ones or of
// weights) passes a target.
//
// The weights are 64-bit integers in units of 2^-shift (shift = 62 -
// ceil(log2 n), at most 52): their sums are exact, so no order of additions
// and no split over threads or CTAs changes a token, and equal calls give equal
// answers bit for bit. The unit is below 2^-44 for rows up to 2^18 tokens.
//
// One cluster of CTAs per row; the row is read from global memory once and held
// in the CTAs' shared memory (-inf where not legal). A search counts or weighs
// the tokens in 1024 bins of shared memory, the CTAs read one another's bins
// over distributed shared memory after one cluster barrier, and each picks the
// bin at which the running sum passes the target.
//   * The first bins are chosen by value, so that few tokens share one:
//     sixteenths of an octave of the weight, or (top-k) 128ths of an octave of
//     the distance to the maximum. They do not depend on the target, so top-p
//     and the draw use the same weighing.
//   * The picked bin's tokens are then listed (key and position, every CTA
//     writing its own to all), and the rest of the search is each CTA's own,
//     without cluster barriers: the range of keys narrows 1024-fold per pass. A
//     list that does not fit leaves the search in the whole row.
//   * After top-k or min-p the kept tokens themselves are listed if they fit,
//     and only they are weighed.
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
constexpr int kBinBits = 10;
constexpr int kBins = 1 << kBinBits;
constexpr int kMaxCluster = 16;
constexpr int kMaxShift = 50;
constexpr int kExpBits = 8;
constexpr int kExpTable = 1 << kExpBits;
constexpr int kOctaveBits = 4;   // weighing bins per octave: 2^kOctaveBits
constexpr int kListTotal = 2048; // tokens a cluster lists, an equal part for each CTA
static_assert(kBins == 2 * kSampleThreads, "two bins per thread");
static_assert(((kMaxShift + 1) << kOctaveBits) < kBins, "every weight has a bin");

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
  uint32_t lo[kBins];                      // bins being filled: low and high halves of 64-bit sums
  uint32_t hi[kBins];
  ulonglong2 tot[kBins / 2];               // this CTA's bins, read by the cluster
  unsigned long long list[kListTotal];     // (key, position in the row); part r holds rank r's tokens
  unsigned long long scan[kSampleWarps];
  unsigned long long pick[4];              // picked bin, sum before it, its own sum, sum of all bins
  unsigned long long word[2][kMaxCluster]; // one value per CTA (all-gather)
  double exp2_table[kExpTable];            // 2^(j / kExpTable)
  uint32_t warp[2][kSampleWarps];
  uint32_t list_count[kMaxCluster];        // tokens in each part of the list
  uint32_t listed;                         // tokens this CTA has offered to the list
};

constexpr size_t kHeaderBytes = (sizeof(SampleSmemHeader) + 127) / 128 * 128;

template <typename T>
struct Row {
  const typename DTypeTraits<T>::Bits* x;  // the row's first logit
  const uint32_t* mask;                    // its mask words, or nullptr
  int64_t n;                               // tokens
};

// Value at position i, read from global memory; -inf where not legal or NaN.
template <typename T>
__device__ __forceinline__ float load_value(const Row<T>& r, int64_t i) {
  if (r.mask && !((__ldg(r.mask + (i >> 5)) >> (i & 31)) & 1u)) return -INFINITY;
  const float f = DTypeTraits<T>::bits_to_float(__ldg(r.x + i));
  return f == f ? f : -INFINITY;
}

// One CTA's part of the row: positions [lo, lo + len), the first `resident`
// of them in shared memory at index `phase` on (so that 16-byte loads of the
// row and stores to shared memory are both aligned), the rest read from global
// memory in every pass.
template <typename T>
struct Slice {
  using Bits = typename DTypeTraits<T>::Bits;
  static constexpr int kVec = 16 / (int)sizeof(Bits);
  Row<T> row;
  Bits* held;
  int64_t lo, len;
  int phase, resident;

  __device__ __forceinline__ int vectors() const { return (phase + resident + kVec - 1) / kVec; }

  static __device__ __forceinline__ float unpack(const uint32_t (&w)[4], int j) {
    if constexpr (sizeof(Bits) == 4)
      return __uint_as_float(w[j]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    else
      return DTypeTraits<T>::bits_to_float((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
  }

  // Fills the resident part; returns the thread's largest value and its number
  // of legal tokens over the whole part.
  __device__ __forceinline__ float load(uint32_t& legal_count) {
    float top = -INFINITY;
    legal_count = 0u;
    const int nv = vectors();
#pragma unroll 2
    for (int v = threadIdx.x; v < nv; v += kSampleThreads) {
      const int64_t i0 = lo + (int64_t)v * kVec - phase;
      float f[kVec];
      if (v * kVec >= phase && v * kVec + kVec <= phase + resident) {
        const uint4 q = ld_stream_v4(row.x + i0);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        uint32_t legal = 0xffffffffu;
        if (row.mask) {
          const int64_t w0 = i0 >> 5;
          const int s = (int)(i0 & 31);
          const uint32_t a = __ldg(row.mask + w0);
          const uint32_t b = s + kVec > 32 ? __ldg(row.mask + w0 + 1) : 0u;
          legal = __funnelshift_r(a, b, s);
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          f[j] = unpack(w, j);
          if (!((legal >> j) & 1u) || f[j] != f[j]) f[j] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int at = v * kVec + j;
          f[j] = (at >= phase && at < phase + resident) ? load_value(row, i0 + j) : -INFINITY;
        }
      }
      uint32_t out[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        top = fmaxf(top, f[j]);
        legal_count += f[j] > -INFINITY ? 1u : 0u;
        if constexpr (sizeof(Bits) == 4)
          out[j] = __float_as_uint(f[j]);
        else
          out[j >> 1] |= (uint32_t)DTypeTraits<T>::round_bits(f[j]) << (16 * (j & 1));
      }
      reinterpret_cast<uint4*>(held)[v] = make_uint4(out[0], out[1], out[2], out[3]);
    }
    for (int64_t i = resident + threadIdx.x; i < len; i += kSampleThreads) {
      const float f = load_value(row, lo + i);
      top = fmaxf(top, f);
      legal_count += f > -INFINITY ? 1u : 0u;
    }
    return top;
  }

  // fn(value, position in the row) for every position of the CTA's part (-inf: not legal)
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    const int nv = vectors();
    for (int v = threadIdx.x; v < nv; v += kSampleThreads) {
      const uint4 q = reinterpret_cast<const uint4*>(held)[v];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < kVec; ++j) fn(unpack(w, j), (uint32_t)(lo - phase + v * kVec + j));
    }
    for (int64_t i = resident + threadIdx.x; i < len; i += kSampleThreads)
      fn(load_value(row, lo + i), (uint32_t)(lo + i));
  }
};

// The cluster's listed tokens, all of them in every CTA.
template <typename T>
struct List {
  const SampleSmemHeader* s;
  int part_bits;  // log2 of the entries in one CTA's part
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
#pragma unroll
    for (int i = threadIdx.x; i < kListTotal; i += kSampleThreads) {
      if ((uint32_t)(i & ((1 << part_bits) - 1)) >= s->list_count[i >> part_bits]) continue;
      const unsigned long long e = s->list[i];
      fn(SampleKey<T>::value((uint32_t)(e >> 32)), (uint32_t)e);
    }
  }
};

// A finite float as a double by integer operations (the conversion unit is
// slower); zero and subnormals become some value below 2^-126, which moves no
// weight.
__device__ __forceinline__ double widen(float f) {
  const uint32_t u = __float_as_uint(f);
  return __hiloint2double((int)((((uint32_t)((int)u >> 3)) & 0x8fffffffu) + (896u << 20)), (int)(u << 29));
}

// Weight of a value in units of 2^-shift: with y = shift + log2 w, the nearest
// multiple of 1/256 is q / 256, and 2^y = 2^(q / 256) * 2^(y - q / 256): a table
// entry, an exponent, and the Taylor polynomial of 2^r = exp(r ln 2) to degree
// 3 on |r| <= 1/512 (the next term is below 1.4e-13 and nearly the same for all).
struct Weigher {
  int shift;
  double vmax, per_octave;  // the largest value; log2(e) / T
  const double* table;

  __device__ __forceinline__ double log_weight(float v, int* q, double* r) const {
    constexpr double kMagic = 26388279066624.0;  // 1.5 * 2^44: its last place is 1/256
    const double y = fma(widen(v) - vmax, per_octave, (double)shift);
    const double t = y + kMagic;
    *q = __double2loint(t);
    *r = y - (t - kMagic);
    return y;
  }
  // Weighing bin: 2^kOctaveBits per octave below the maximum (only for y >= -1).
  __device__ __forceinline__ int bin(int q) const { return (shift * kExpTable - q) >> (kExpBits - kOctaveBits); }
  __device__ __forceinline__ int bin_of(float v) const {
    int q;
    double r;
    return log_weight(v, &q, &r) >= -1.0 ? bin(q) : kBins;
  }
  __device__ __forceinline__ unsigned long long weigh(float v, int* q) const {
    double r;
    const double y = log_weight(v, q, &r);
    if (!(y >= -1.0)) return 0ull;  // rounds to nothing
    double p = fma(r, 5.5504108664821580e-02, 2.4022650695910072e-01);  // ln2^3 / 6, ln2^2 / 2
    p = fma(p, r, 6.9314718055994531e-01);                             // ln2
    const double m = table[*q & (kExpTable - 1)];
    p = fma(p * r, m, m);
    const double w =
        __hiloint2double(__double2hiint(p) + ((*q & ~(kExpTable - 1)) << (20 - kExpBits)), __double2loint(p));
    // adding 2^52 rounds to an integer, held in the low mantissa bits
    const double rounded = w + 4503599627370496.0;
    return ((unsigned long long)(uint32_t)(__double2hiint(rounded) - 0x43300000) << 32) |
           (uint32_t)__double2loint(rounded);
  }
  __device__ __forceinline__ unsigned long long operator()(float v) const {
    int q;
    return weigh(v, &q);
  }
  // Values that bin j may hold: [lo, hi], 0.02 of a multiple of 1/256 wider than
  // the bin on both sides (rounding moves a border by less).
  __device__ __forceinline__ void bin_range(int j, double* lo, double* hi) const {
    constexpr double kWidth = kExpTable >> kOctaveBits;
    *hi = vmax + (-kWidth * j + 0.52) / kExpTable / per_octave;
    *lo = vmax + (-kWidth * (j + 1) + 0.48) / kExpTable / per_octave;
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
  int rank, size, size_bits;
  int buf;          // which half of `word` the next all-gather uses
  bool list_in_use; // a list may still be read by other CTAs

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
  // lo and hi together are one array of 2 * kBins words
  reinterpret_cast<uint4*>(s->lo)[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
}
static_assert(2 * kBins == 4 * kSampleThreads, "one 16-byte store per thread clears the bins");

// 64-bit sum in two 32-bit words: the old low word tells the carry.
__device__ __forceinline__ void add_to_bin(SampleSmemHeader* s, uint32_t bin, unsigned long long m) {
  const uint32_t m_lo = (uint32_t)m;
  uint32_t m_hi = (uint32_t)(m >> 32);
  const uint32_t old = atomicAdd(&s->lo[bin], m_lo);
  m_hi += (old + m_lo < old) ? 1u : 0u;
  if (m_hi) atomicAdd(&s->hi[bin], m_hi);
}

// Sums of a thread's two bins and the running sum before them.
struct BinSums {
  unsigned long long before, a, b;
  // Whether one of the two is where the running sum passes the target; if so
  // publishes it.
  __device__ __forceinline__ void pick(SampleSmemHeader* s, unsigned long long target) const {
    if (before <= target && target < before + a + b) {
      const bool second = target >= before + a;
      s->pick[0] = 2 * threadIdx.x + (second ? 1 : 0);
      s->pick[1] = second ? before + a : before;
      s->pick[2] = second ? b : a;
    }
    __syncthreads();
  }
};

// Closes a filling pass: the bins' sums over the cluster, or (local) this
// CTA's. s->pick[3] holds the sum of all bins after the next barrier.
__device__ __forceinline__ BinSums sum_bins(Team& team, bool local) {
  SampleSmemHeader* s = team.s;
  const int tid = threadIdx.x;
  __syncthreads();
  const uint2 lo = reinterpret_cast<const uint2*>(s->lo)[tid], hi = reinterpret_cast<const uint2*>(s->hi)[tid];
  BinSums v;
  v.a = lo.x + ((unsigned long long)hi.x << 32);
  v.b = lo.y + ((unsigned long long)hi.y << 32);
  if (!local && team.size > 1) {
    s->tot[tid] = make_ulonglong2(v.a, v.b);
    team.cluster.sync();
    v.a = v.b = 0ull;
    for (int r0 = 0; r0 < team.size; r0 += 4) {  // independent loads, four in flight
      ulonglong2 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[k] = r0 + k < team.size ? team.cluster.map_shared_rank(s->tot, r0 + k)[tid] : make_ulonglong2(0ull, 0ull);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v.a += x[k].x;
        v.b += x[k].y;
      }
    }
  }
  const unsigned long long incl = warp_scan_u64(v.a + v.b);
  if ((tid & 31) == 31) s->scan[tid >> 5] = incl;
  __syncthreads();
  v.before = incl - (v.a + v.b);
  unsigned long long total = 0ull;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    const unsigned long long x = s->scan[w];
    if (w < (tid >> 5)) v.before += x;
    total += x;
  }
  if (tid == 0) s->pick[3] = total;
  return v;
}

// Where a running sum passes a target: the key, the sums above and at it.
struct Found {
  uint32_t key;
  unsigned long long above, own;
};

// Goes on with a search inside keys [klo, khi] of `tokens` (those that `member`
// accepts): the first key, from khi down, at which the running sum of
// measure(value) passes `target`, which it does (the caller knows the sum).
// local: every CTA holds all the tokens.
template <typename T, typename Tokens, typename Measure, typename Member>
__device__ __forceinline__ Found search(Team& team, bool local, const Tokens& tokens, uint32_t klo, uint32_t khi,
                                        Measure measure, Member member, unsigned long long target) {
  SampleSmemHeader* s = team.s;
  Found f{khi, 0ull, 0ull};
  for (;;) {
    const int width = 32 - __clz(khi - klo);  // bits of the range (0: a single key)
    const int sh = width > kBinBits ? width - kBinBits : 0;
    clear_bins(s);
    tokens.each([&](float v, uint32_t) {
      const uint32_t key = SampleKey<T>::from_value(v);
      if (key >= klo && key <= khi && member(v)) add_to_bin(s, (khi - key) >> sh, measure(v));
    });
    const BinSums sums = sum_bins(team, local);
    sums.pick(s, target);
    const uint32_t bin = (uint32_t)s->pick[0] & (kBins - 1);
    f.above += s->pick[1];
    f.own = s->pick[2];
    target -= s->pick[1];
    khi -= bin << sh;
    f.key = khi;
    if (!local) team.cluster.sync();  // the CTAs have read one another's bins
    else __syncthreads();             // the pick has been read
    if (sh == 0) return f;
    const uint32_t span = (1u << sh) - 1u;
    klo = khi - klo > span ? khi - span : klo;
  }
}

// ---- listing ---------------------------------------------------------------------
__device__ __forceinline__ void open_list(Team& team) {
  if (team.list_in_use) team.cluster.sync();  // nobody reads the last list any more
  team.list_in_use = true;
  __syncthreads();
  if (threadIdx.x == 0) team.s->listed = 0u;
  __syncthreads();
}

// Offers a token to the list: every CTA of the cluster gets it.
__device__ __forceinline__ void list_token(const Team& team, uint32_t key, uint32_t at) {
  const uint32_t i = atomicAdd(&team.s->listed, 1u);
  const uint32_t part = kListTotal >> team.size_bits;
  if (i >= part) return;
  const unsigned long long e = ((unsigned long long)key << 32) | at;
  for (int r = 0; r < team.size; ++r) team.cluster.map_shared_rank(team.s->list, r)[team.rank * part + i] = e;
}

// After a listing pass: whether every CTA's part fits, and the cluster's sum of `count`.
__device__ __forceinline__ bool close_list(Team& team, uint32_t count, unsigned long long* sum) {
  SampleSmemHeader* s = team.s;
  const uint32_t part = kListTotal >> team.size_bits;
  count = block_sum(count, s);
  const uint32_t mine = min(s->listed, part + 1u);
  const unsigned long long* all = team.gather(((unsigned long long)mine << 32) | count);
  unsigned long long total = 0ull;
  bool fits = true;
  for (int r = 0; r < team.size; ++r) {
    total += (uint32_t)all[r];
    fits &= (uint32_t)(all[r] >> 32) <= part;
  }
  if ((int)threadIdx.x < team.size) s->list_count[threadIdx.x] = (uint32_t)(all[threadIdx.x] >> 32);
  __syncthreads();
  *sum = total;
  return fits;
}

// Bin of the top-k search: 128ths of an octave of the distance to the maximum,
// from 1/4 to 64; nearer and farther tokens share the first and last.
constexpr uint32_t kDistanceBase = 0x3e800000u >> 16;
__device__ __forceinline__ uint32_t distance_bin(float vmax, float v) {
  return min((__float_as_uint(vmax - v + 0.25f) >> 16) - kDistanceBase, (uint32_t)kBins - 1u);
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) filtered_sample_kernel(const FilteredSampleParams p) {
  using K = SampleKey<T>;
  using Bits = typename DTypeTraits<T>::Bits;
  extern __shared__ __align__(128) unsigned char smem[];
  SampleSmemHeader* s = reinterpret_cast<SampleSmemHeader*>(smem);
  Team team{s, cg::this_cluster(), 0, 0, 0, 0, false};
  team.rank = (int)team.cluster.block_rank();
  team.size = (int)team.cluster.num_blocks();
  team.size_bits = 31 - __clz(team.size);
  const int b = blockIdx.x / team.size, tid = threadIdx.x;
  const bool leader = team.rank == 0 && tid == 0;

  // ---- the row and its settings ---------------------------------------------
  Slice<T> slice;
  int64_t start = 0;
  if (p.offsets) {
    // positions outside the packed arrays are not read, whatever the offsets say
    start = min(max(p.offsets[b], (int64_t)0), p.capacity);
    const int64_t end = min(max(p.offsets[b + 1], start), p.capacity);
    slice.row = Row<T>{static_cast<const Bits*>(p.logits) + start, nullptr, end - start};
  } else {
    slice.row = Row<T>{static_cast<const Bits*>(p.logits) + (int64_t)b * p.row_stride,
                       p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr, p.vocab};
  }
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const int64_t top_k = p.top_ks ? p.top_ks[b] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[b] : p.min_p;
  const float u = p.uniforms[b];
  const bool valid = temperature >= 0.f && temperature < INFINITY && top_p == top_p && min_p == min_p && u >= 0.f &&
                     u < 1.f;
  if (!valid) {
    if (leader) {
      p.token_ids[b] = -1;
      if (p.logprobs) p.logprobs[b] = __int_as_float(0x7fc00000);
      if (p.kept) p.kept[b] = 0;
    }
    return;  // the whole cluster returns
  }
  // every CTA of the cluster runs before its shared memory is written to
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const int64_t n = slice.row.n;
  const int64_t part = ((n + team.size - 1) / team.size + 31) / 32 * 32;
  slice.lo = min(part * team.rank, n);
  slice.len = min(part, n - slice.lo);
  slice.held = reinterpret_cast<Bits*>(smem + kHeaderBytes);
  slice.phase = (int)((reinterpret_cast<uintptr_t>(slice.row.x + slice.lo) & 15) / sizeof(Bits));
  slice.resident = (int)min(slice.len, (int64_t)p.resident);

  // ---- the row into shared memory, largest value, number of legal tokens ----------
  uint32_t legal = 0u;
  float vmax = slice.load(legal);
  if (tid < kExpTable) s->exp2_table[tid] = exp2((double)tid / kExpTable);
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
  {
    const unsigned long long* all = team.gather(((unsigned long long)legal << 32) | kmax);
    for (int r = 0; r < team.size; ++r) {
      kmax = max(kmax, (uint32_t)all[r]);
      kept += all[r] >> 32;
    }
  }
  if (kmax == 0u) {  // nothing is legal
    if (leader) {
      p.token_ids[b] = 0;
      if (p.logprobs) p.logprobs[b] = -INFINITY;
      if (p.kept) p.kept[b] = 0;
    }
    return;
  }
  vmax = K::value(kmax);
  const bool infinite = !(vmax < INFINITY);
  const List<T> list{s, 31 - __clz(kListTotal) - team.size_bits};

  float draw_value = vmax;
  unsigned long long ordinal = 0ull;  // among the tokens of draw_value, by rising position
  float logprob = 0.f;
  bool listed = false;  // the list holds every token of draw_value
  if (temperature > 0.f && !infinite) {
    Weigher weigh;
    weigh.shift = min(kMaxShift, 62 - (64 - __clzll((unsigned long long)n)));
    weigh.vmax = widen(vmax);
    weigh.per_octave = 1.4426950408889634 / (double)temperature;
    weigh.table = s->exp2_table;
    // ---- the kept set: values above `border`, and `ties` tokens at it --------------
    float border = -INFINITY;             // (none: every legal token)
    unsigned long long ties = ~0ull, excess = 0ull;  // excess: tokens at the border beyond `ties`
    bool in_list = false;                 // the list holds every token >= border
    const auto all_of = [](float) { return true; };
    if (top_k > 0 && (unsigned long long)top_k < kept) {
      const auto one = [](float) { return 1ull; };
      clear_bins(s);
      slice.each([&](float v, uint32_t) {
        if (v > -INFINITY) atomicAdd(&s->lo[distance_bin(vmax, v)], 1u);
      });
      const unsigned long long target = (unsigned long long)top_k - 1ull;
      sum_bins(team, false).pick(s, target);
      // every token down to the picked bin: its lower border, a little wider
      const int j = (int)s->pick[0] & (kBins - 1);
      float low = -INFINITY;
      if (j < kBins - 1) {
        const float edge = __uint_as_float((uint32_t)(j + 1 + kDistanceBase) << 16) - 0.25f;
        low = K::value_at_least((double)vmax - (double)edge * 1.00001 - 1e-6 * fabs((double)vmax));
      }
      open_list(team);
      slice.each([&](float v, uint32_t at) {
        if (v >= low && v > -INFINITY) list_token(team, K::from_value(v), at);
      });
      unsigned long long unused;
      in_list = close_list(team, 0u, &unused);
      const uint32_t klo = max(K::from_value(low), 1u);
      const Found f = in_list ? search<T>(team, true, list, klo, kmax, one, all_of, target)
                              : search<T>(team, false, slice, 1u, kmax, one, all_of, target);
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
          slice.each([&](float v, uint32_t at) {
            if (v >= border && v > -INFINITY) {
              ++count;
              list_token(team, K::from_value(v), at);
            }
          });
          in_list = close_list(team, count, &kept);
        }
      }
    }
    // ---- weigh what is left, by bins ---------------------------------------------
    clear_bins(s);
    const auto into_bin = [&](float v, uint32_t) {
      if (!(v >= border)) return;
      int q;
      const unsigned long long w = weigh.weigh(v, &q);
      if (w) add_to_bin(s, (uint32_t)weigh.bin(q), w);
    };
    if (in_list) list.each(into_bin);
    else slice.each(into_bin);
    const BinSums bins = sum_bins(team, in_list);
    __syncthreads();
    unsigned long long sum = s->pick[3];
    if (excess) sum -= excess * weigh(border);
    // The bin at which the running sum passes `target`, and the search inside
    // it; *n_above: tokens in the bins above it (where the list holds the bin alone).
    const auto find = [&](unsigned long long target, unsigned long long* n_above) {
      bins.pick(s, target);
      const int j = (int)s->pick[0];
      const unsigned long long before = s->pick[1];
      double lo, hi;
      weigh.bin_range(j, &lo, &hi);
      const float flo = fmaxf(border, K::value_at_least(lo)), fhi = fminf(vmax, K::value_at_least(hi));
      const uint32_t khi = K::from_value(fhi), klo = min(max(K::from_value(flo), 1u), khi);
      const auto in_bin = [&](float v) { return weigh.bin_of(v) == j; };
      Found f;
      if (in_list) {
        listed = true;
        __syncthreads();  // the pick has been read
        f = search<T>(team, true, list, klo, khi, weigh, in_bin, target - before);
      } else {
        open_list(team);
        uint32_t count = 0u;
        slice.each([&](float v, uint32_t at) {
          if (v > fhi) {
            ++count;
          } else if (v >= flo && v > -INFINITY) {
            const int mine = weigh.bin_of(v);
            if (mine == j) list_token(team, K::from_value(v), at);
            else count += mine < j ? 1u : 0u;
          }
        });
        listed = close_list(team, count, n_above);
        f = listed ? search<T>(team, true, list, klo, khi, weigh, all_of, target - before)
                   : search<T>(team, false, slice, klo, khi, weigh, in_bin, target - before);
      }
      f.above += before;
      return f;
    };
    if (top_p < 1.f) {
      const unsigned long long target = prefix_target(top_p, sum);
      unsigned long long n_above = 0ull;
      const Found f = find(target, &n_above);
      const float value = K::value(f.key);
      const unsigned long long w = weigh(value);
      ties = (target - f.above) / w + 1ull;
      sum = f.above + ties * w;
      // how many that keeps: those above the bin, and above the value within it
      uint32_t count = 0u;
      const auto above_value = [&](float v, uint32_t) { count += v > value ? 1u : 0u; };
      if (listed) {
        list.each(above_value);
        kept = ties + block_sum(count, s) + (in_list ? 0ull : n_above);
      } else {
        slice.each(above_value);
        kept = ties + cluster_sum(team, count);
      }
    }
    // ---- the draw ------------------------------------------------------------------
    const unsigned long long target = __umul64hi(fraction64(u), sum);
    unsigned long long unused;
    const Found f = find(target, &unused);
    draw_value = K::value(f.key);
    ordinal = (target - f.above) / weigh(draw_value);
    logprob = (float)(((double)draw_value - (double)vmax) / (double)temperature -
                      log((double)sum / (double)(1ull << weigh.shift)));
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
  const auto put = [&](int64_t at) {
    p.token_ids[b] = p.ids ? p.ids[start + at] : p.vocab_offset + at;
    if (p.logprobs) p.logprobs[b] = logprob;
    if (p.kept) p.kept[b] = (int32_t)kept;
  };
  if (listed) {  // every CTA holds all of them: the first one answers
    if (team.rank != 0) return;
    // the positions of draw_value's tokens, into the bins' space; each counts those before it
    uint32_t* ties_at = s->lo;
    static_assert(kListTotal <= 2 * kBins, "the listed positions fit the bins' space");
    __syncthreads();
    if (tid == 0) s->listed = 0u;
    __syncthreads();
    list.each([&](float v, uint32_t at) {
      if (v == draw_value) ties_at[atomicAdd(&s->listed, 1u)] = at;
    });
    __syncthreads();
    const uint32_t m = s->listed;
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
  // blocks of kSampleThreads positions in order
  for (int64_t i0 = 0; i0 < slice.len; i0 += kSampleThreads) {
    const int64_t i = i0 + tid;
    float v = -INFINITY;
    if (i < slice.resident) v = DTypeTraits<T>::bits_to_float(slice.held[slice.phase + i]);
    else if (i < slice.len) v = load_value(slice.row, slice.lo + i);
    const bool hit = v == draw_value;
    const unsigned hits = __ballot_sync(FULL_MASK, hit);
    __syncthreads();
    if ((tid & 31) == 0) s->warp[0][tid >> 5] = __popc(hits);
    __syncthreads();
    unsigned long long before = 0ull, in_block = 0ull;
    for (int w = 0; w < kSampleWarps; ++w) {
      if (w < (tid >> 5)) before += s->warp[0][w];
      in_block += s->warp[0][w];
    }
    before += __popc(hits & ((1u << (tid & 31)) - 1u));
    if (hit && before == ordinal) put(slice.lo + i);
    if (ordinal < in_block) break;
    ordinal -= in_block;
  }
}

// Launch: one cluster per row.
template <typename T>
cudaError_t launch_typed(FilteredSampleParams p, int batch, int64_t max_len, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  using Key = typename DTypeTraits<T>::Bits;
  constexpr size_t kSmemMax = 227 * 1024;
  // CTAs per row: one for short rows; for long ones enough that a CTA's part
  // leaves room for a second CTA on the SM (their barriers overlap), and more
  // while the batch leaves SMs idle.
  const size_t room = (kSmemMax - kHeaderBytes - 64) / sizeof(Key) / 32 * 32;
  constexpr size_t kShare = (kSmemMax / 2 - 1024 - kHeaderBytes - 64) / sizeof(Key);
  int size = 1;
  while (size < kMaxCluster &&
         ((int64_t)(size < 8 ? kShare : room) * size < max_len ||
          (max_len > (int64_t)4096 * size && (int64_t)batch * size * 2 <= 2 * num_sms(dev))))
    size *= 2;
  const int64_t part = ((max_len + size - 1) / size + 31) / 32 * 32;
  p.resident = (int)std::min<int64_t>((int64_t)room, std::max<int64_t>(part, 32));
  const size_t smem = kHeaderBytes + ((size_t)p.resident + 16) * sizeof(Key);
  auto k = filtered_sample_kernel<T>;
  if ((err = raise_smem_limit(reinterpret_cast<const void*>(k), smem, dev)) != cudaSuccess) return err;
  static std::atomic<uint64_t> wide_ok[2];  // devices on which clusters of 16 have been allowed
  if (size > 8 && dev < 128 && !((wide_ok[dev >> 6].load() >> (dev & 63)) & 1u)) {
    if ((err = cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeNonPortableClusterSizeAllowed,
                                    1)) != cudaSuccess)
      return err;
    wide_ok[dev >> 6].fetch_or(1ull << (dev & 63));
  }
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

}  // namespace

cudaError_t launch_filtered_sample(const FilteredSampleParams& p, int dtype, int batch, int64_t max_len,
                                   cudaStream_t stream) {
  if (dtype == 2) return launch_typed<float>(p, batch, max_len, stream);
  if (dtype == 1) return launch_typed<__nv_bfloat16>(p, batch, max_len, stream);
  return launch_typed<__half>(p, batch, max_len, stream);
}

}  // namespace gsp
