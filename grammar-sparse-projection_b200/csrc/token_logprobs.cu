// Log probabilities of given tokens, entropy, logsumexp and the top alternatives
// of logits rows, and their gradient (sm_100a).
//
// With x the legal logits of a row (bit set, not NaN, not -inf), T its
// temperature, z = x / T, m = max x:
//
//   S = sum exp((x - m) / T),  A = sum exp((x - m) / T) (x - m) / T
//   logprob_t = (x_t - m) / T - ln S       (-inf for a token that is not legal)
//   entropy   = ln S - A / S               (0 for a row without a legal token)
//   logsumexp = m / T + ln S
//   top n     = the n legal tokens that come first by falling x, ties by rising id
//
//   dL/dx_j = (p_j (gL - sum_k g_k - gH (ln p_j + entropy)) + sum_k g_k [j = t_k]) / T
//
// Forward: one pass over the row, which is bound by its bytes. A row belongs to
// one CTA, or to a cluster of CTAs whose shares are merged over distributed
// shared memory when there are few rows. A thread keeps its own running (m, S, A)
// in powers of two (d = (x - m) log2(e) / T, clamped at -200 so that an excluded
// value adds exactly nothing) and compares a vector's maximum, two packed
// instructions per four elements, with both m and the n-th alternative so far:
// the two rare cases (a new maximum, a candidate) share that one test. All
// threads start from the maximum of the CTA's first batch of vectors, and the
// alternatives from the n-th largest of its lanes' maxima in 64 groups, so hardly any
// vector takes the slow path after it. Candidates gather in a list that is ranked by
// counting each time the row read has doubled; a list that overflows (rows in rising
// order, equal values) is made again with a barrier for every vector: time, not results.
//
// Measured (device): 1,999 x 151,936 bf16, four tokens a row, 132-135 us (4.5 TB/s, 70% of
// measured; issue slots 65% busy, the exponentials' pipe 54%, the rest waits for loads);
// 128 x 248,320 bf16 with masks and five alternatives 42 us (floor 10.5: issue slots 44%
// busy; what waits, waits for loads and, a third as often, at the rankings' barriers; 40 of
// 148 SMs have half the work of the others); one row of 248,320 with 20 alternatives 14 us,
// 7 of them the alternatives' rankings and barriers.
//
// Sums run in fp32: a thread adds a row's terms over 512 (CTAs of 256 threads) or over 1,024
// times the row's CTAs in each of two sums, 300 at 151,936 tokens and 131,072 at 2^30, then
// a tree.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "../../include/gsp_b200.h"
#include "gsp_common.cuh"
#include "gsp_internal.h"
#include "gsp_pairs.cuh"

namespace cg = cooperative_groups;

namespace gsp {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kGroups = 64;      // groups of lanes whose maxima place the first border
constexpr int kParts = 8;        // lanes that count for one key
constexpr int kUnroll = 4;       // 16-byte vectors a thread has under way
constexpr int kMaxTop = 64;      // alternatives
constexpr int kListSize = 1024;  // candidates held at a time
constexpr int kMaxClusterSize = 8;
constexpr int kMaxTokens = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNothing = -200.f;  // exponent whose power of two is 0 in fp32
constexpr float kFurthest = -1e30f;  // no exponent of a half is below it

struct LogprobParams {
  const void* logits;
  int64_t row_stride;
  const uint32_t* mask;
  int64_t mask_stride;
  int vocab;               // row length (packed rows: ignored)
  const int64_t* offsets;  // packed rows: [batch + 1], else nullptr
  const int64_t* ids;      // packed rows: token id of each position, rising in a row
  int64_t capacity;        // packed rows: positions that exist
  float temperature;
  const float* temperatures;
  const int64_t* token_ids;  // [batch, tokens]
  int tokens;
  int top_n;
  float* logprobs;      // [batch, tokens]
  float* entropy;       // [batch] (optional)
  float* logsumexp;     // [batch] (optional)
  int64_t* top_ids;     // [batch, top_n]
  float* top_logprobs;  // [batch, top_n]
  float4* stats;        // [batch]: m, S, entropy, 1 / T (optional)
};

// One row as 16-byte vectors from an aligned base: vector i holds elements
// i * kPerVec - phase and on; those before 0 and from len on are not the row's.
struct Row {
  const uint4* base;
  int phase;
  int64_t len;
  const uint32_t* mask;
  int64_t first;  // position of element 0 in the packed arrays
  int last;       // vector that holds the last element
};

template <typename T>
__device__ __forceinline__ void set_row(Row& r, const void* logits, int64_t start, int64_t len) {
  using Bits = typename DTypeTraits<T>::Bits;
  const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<const Bits*>(logits) + start);
  r.base = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
  r.phase = (int)((at & 15) / sizeof(Bits));
  r.len = len;
  r.first = start;
  r.last = len > 0 ? (int)((len + r.phase + DTypeTraits<T>::kPerVec - 1) / DTypeTraits<T>::kPerVec) - 1 : -1;
}

// Which of vector i's elements belong to the row and are legal. Rows that start on a
// vector read the vector's own bits alone.
template <typename T, bool kMask>
__device__ __forceinline__ uint32_t legal_bits(const Row& r, int i) {
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  uint32_t bits = (1u << kPer) - 1u;
  if constexpr (kMask) {
    if (r.phase == 0) {
      const uint32_t byte = __ldg(reinterpret_cast<const uint8_t*>(r.mask) + (kPer == 8 ? i : i >> 1));
      bits &= kPer == 8 ? byte : byte >> (4 * (i & 1));
    } else {
      const int e0 = i * kPer - r.phase, w = e0 >> 5, shift = e0 & 31, nw = (int)((r.len + 31) >> 5);
      const uint32_t lo = w >= 0 ? __ldg(r.mask + w) : 0u;
      const uint32_t hi = shift + kPer > 32 && w + 1 < nw ? __ldg(r.mask + w + 1) : 0u;
      bits &= __funnelshift_r(lo, hi, shift);
    }
  }
  if (i == r.last || i == 0) {  // (the row's edges)
    const int e0 = i * kPer - r.phase, left = (int)r.len - e0;
    if (e0 < 0) bits &= ~((1u << -e0) - 1u);
    if (left < kPer) bits &= (1u << left) - 1u;
  }
  return bits;
}

// -inf in the elements whose bit is not set.
template <typename T>
__device__ __forceinline__ void exclude(uint4& v, uint32_t bits) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(typename DTypeTraits<T>::Bits) == 2) {
    // bits 2k and 2k + 1 to the tops of a word's halves, whose signs spread over them
    const uint32_t z = bits | (bits << 15), ninf = DTypeTraits<T>::kNegInfBits * 0x00010001u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t keep = spread_half_signs(z << (15 - 2 * k));
      w[k] = (w[k] & keep) | (ninf & ~keep);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = ((bits >> k) & 1u) ? w[k] : 0xff800000u;
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
}

// Largest element; NaN counts as absent.
template <typename T>
__device__ __forceinline__ float vector_top(const uint4& v) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmaxf(fmaxf(__uint_as_float(v.x), -INFINITY), __uint_as_float(v.y)),
                 fmaxf(fmaxf(__uint_as_float(v.z), -INFINITY), __uint_as_float(v.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(&v);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    uint32_t w;
    w = *reinterpret_cast<const uint32_t*>(&m);
    const float2 f = DTypeTraits<T>::pair_to_float2(w);
    return fmaxf(fmaxf(f.x, -INFINITY), f.y);
  }
}

template <typename T>
__device__ __forceinline__ float2 element_pair(const uint4& v, int k) {  // elements 2k, 2k + 1
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (std::is_same<T, float>::value) return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
  else return DTypeTraits<T>::pair_to_float2(w[k]);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The exponents d = (x - m) c of a vector's elements, in pairs, none below kNothing
// (-inf, NaN and what is far below: nothing). Halves are held back at `floor` before they
// are widened: a value of the type at or below m + kNothing / c, two in each word. Where m
// is large the next such value may lie far below that (at the largest bf16 one step is
// 1.3e36), so far that its exponent would pass fp32 and 0 times it be NaN: then, too, the
// exponents are held back in fp32.
template <typename T>
struct Exponents {
  unsigned long long neg, by;
  uint32_t floor;
  bool deep;  // the type has no such value (a maximum near its lowest), or one too far: held back in fp32
  float lowest;  // no exponent is below it
  __device__ __forceinline__ void set(float m, float c) {
    neg = pack2(-m, -m);
    by = pack2(c, c);
    // (a maximum so large that the difference is lost in it: the number below it, whose
    // weight is nothing as well)
    float low = m + kNothing / c;
    if (!(low < m)) low = m > 0.f ? __uint_as_float(__float_as_uint(m) - 1u) : __uint_as_float(__float_as_uint(m) + 1u);
    floor = 0u;
    deep = true;
    lowest = kNothing;
    if constexpr (!std::is_same<T, float>::value) {
      float held;  // the floor's value (-inf where the type has none)
      if constexpr (std::is_same<T, __half>::value) {
        const __half h = __float2half_rd(low);
        floor = (uint32_t)__half_as_ushort(h) * 0x00010001u;
        held = __half2float(h);
      } else {
        const __nv_bfloat16 h = __float2bfloat16_rd(low);
        floor = (uint32_t)__bfloat16_as_ushort(h) * 0x00010001u;
        held = __bfloat162float(h);
      }
      const float d = (held - m) * c;
      deep = !(d >= kFurthest);
      if (!deep) lowest = d;
    }
  }
  template <bool kDeep>
  __device__ __forceinline__ unsigned long long at(const uint4& v, int k) const {  // of elements 2k, 2k + 1
    if constexpr (kDeep) {
      const float2 x = element_pair<T>(v, k);
      const float2 d = unpack2(mul2(add2(pack2(x.x, x.y), neg), by));
      return pack2(fmaxf(d.x, kNothing), fmaxf(d.y, kNothing));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const T2 held = __hmax2(*reinterpret_cast<const T2*>(&w[k]), *reinterpret_cast<const T2*>(&floor));
      const float2 x = DTypeTraits<T>::pair_to_float2(*reinterpret_cast<const uint32_t*>(&held));
      return mul2(add2(pack2(x.x, x.y), neg), by);
    }
  }
};

// A thread's running maximum and sums relative to it, in two lanes each.
template <typename T>
struct Running {
  float m;
  unsigned long long s, a;
  Exponents<T> d;
  __device__ __forceinline__ void start(float top, float c) {
    m = top;
    s = a = 0ull;
    d.set(m, c);
  }
  // Moves the reference from m up to `to`: s 2^delta, a -> 2^delta (a + delta s).
  __device__ __forceinline__ void raise(float to, float c) {
    const float delta = fmaxf((m - to) * c, kNothing);
    const float f = exp2_approx(delta);
    a = mul2(pack2(f, f), fma2(pack2(delta, delta), s, a));
    s = mul2(pack2(f, f), s);
    m = to;
    d.set(m, c);
  }
  template <bool kDeep>
  __device__ __forceinline__ void add(const uint4& v) {
#pragma unroll
    for (int k = 0; k < DTypeTraits<T>::kPerVec / 2; ++k) {
      const unsigned long long dd = d.template at<kDeep>(v, k);
      const float2 one = unpack2(dd);
      const unsigned long long e = pack2(exp2_approx(one.x), exp2_approx(one.y));
      s = add2(s, e);
      a = fma2(e, dd, a);
    }
  }
};

struct Sums {
  float m, s, a;
};
__device__ __forceinline__ Sums merge(Sums x, Sums y, float c) {
  const float m = fmaxf(x.m, y.m);
  const float dx = fmaxf((x.m - m) * c, kNothing), dy = fmaxf((y.m - m) * c, kNothing);
  const float fx = exp2_approx(dx), fy = exp2_approx(dy);
  return Sums{m, fx * x.s + fy * y.s, fx * fmaf(dx, x.s, x.a) + fy * fmaf(dy, y.s, y.a)};
}

struct Shared {
  Sums part[kMaxThreads / 32];
  Sums total[kMaxClusterSize];  // every CTA's, written by them
  unsigned int ninf, all_ninf[kMaxClusterSize];
  float group_top[kGroups];
  unsigned int count;
  int listed, overflow;
  unsigned long long border;
  alignas(16) unsigned long long list[kListSize];
  unsigned long long best[kMaxTop];
  // CTA 0's: the lists of all (n keys each in falling order, 0: none), written by them
  alignas(16) unsigned long long all[kMaxClusterSize * kMaxTop];
};

// Sum over the kParts neighbouring lanes of a key.
__device__ __forceinline__ int over_parts(int v) {
#pragma unroll
  for (int o = 1; o < kParts; o <<= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// The n largest of the list's keys, in falling order, at its front: a key's place is the
// number of larger ones, which kParts lanes count. Called by the whole CTA between
// barriers of its own; afterwards s.border is the n-th.
template <int kThreads>
__device__ __forceinline__ void rank_list(Shared& s, int n) {
  __syncthreads();
  const int count = min((int)s.count, kListSize), part = threadIdx.x % kParts;
  for (int t0 = 0; t0 < count; t0 += kThreads / kParts) {
    const int t = t0 + threadIdx.x / kParts;
    const unsigned long long key = t < count ? s.list[t] : ~0ull;
    int rank = 0;
    for (int j = part; j < count; j += kParts) rank += s.list[j] > key;
    rank = over_parts(rank);
    if (part == 0 && t < count && rank < n) s.best[rank] = key;
  }
  __syncthreads();
  const int kept = min(count, n);
  if ((int)threadIdx.x < kept) s.list[threadIdx.x] = s.best[threadIdx.x];
  if (threadIdx.x == 0) {
    s.count = (unsigned)kept;
    s.listed = kept;
    if (count >= n) s.border = s.best[n - 1];
  }
  __syncthreads();
}

__device__ __forceinline__ float border_value(unsigned long long border) {
  return border == 0ull ? -INFINITY : from_ordered_bits((uint32_t)(border >> 32));
}

// Of vector v's elements, those past the border.
template <typename T>
__device__ __forceinline__ uint32_t candidates(const uint4& v, float least) {
  uint32_t found = 0u;
#pragma unroll
  for (int k = 0; k < DTypeTraits<T>::kPerVec / 2; ++k) {
    const float2 x = element_pair<T>(v, k);
    if (x.x >= least && x.x > -INFINITY) found |= 1u << (2 * k);
    if (x.y >= least && x.y > -INFINITY) found |= 2u << (2 * k);
  }
  return found;
}

// Lists vector v's waiting elements past the border; those that find no room stay waiting.
template <typename T>
__device__ __forceinline__ uint32_t list_candidates(Shared& s, const uint4& v, uint32_t waiting, int e0,
                                                    unsigned long long border) {
#pragma unroll
  for (int j = 0; j < DTypeTraits<T>::kPerVec; ++j) {
    if (!((waiting >> j) & 1u)) continue;
    const float2 x = element_pair<T>(v, j / 2);
    const unsigned long long key = top1_key(j & 1 ? x.y : x.x, (uint64_t)(e0 + j));
    if (key > border) {
      const unsigned at = atomicAdd(&s.count, 1u);
      if (at >= (unsigned)kListSize) continue;
      s.list[at] = key;
    }
    waiting &= ~(1u << j);
  }
  return waiting;
}

// The n largest keys of the vectors lo .. hi - 1 when the list has not held the
// candidates (rows in rising order, or of equal values): a vector a thread and time, what
// finds no room tried again against the border of what is listed.
template <typename T, bool kMask, int kThreads>
__device__ __noinline__ void list_again(Shared& s, const Row& r, int lo, int hi, int n) {
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  if (threadIdx.x == 0) {
    s.count = 0u;
    if (s.border != 0ull) s.border -= 1ull;  // (the key on the border is to be found again)
  }
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    uint32_t waiting = 0u;
    unsigned long long border = s.border;
    if (i < hi) {
      v = ld_stream_v4(r.base + i);
      exclude<T>(v, legal_bits<T, kMask>(r, i));
      waiting = candidates<T>(v, border_value(border));
    }
    for (;;) {
      if (waiting) waiting = list_candidates<T>(s, v, waiting, i * kPer - r.phase, border);
      if (!__syncthreads_or(waiting != 0u)) break;
      rank_list<kThreads>(s, n);
      border = s.border;
    }
  }
}

__device__ __forceinline__ bool valid_temperature(float t) { return t > 0.f && t < INFINITY; }

// (x - m) / T - ln S; infinite maxima share the weight among themselves.
__device__ __forceinline__ float logprob_of(float x, float m, float t, float log_s) {
  if (!(x > -INFINITY)) return -INFINITY;  // (NaN too)
  if (x == m) return -log_s;
  if (m - x == INFINITY) return 2.f * __fdiv_rn(0.5f * x - 0.5f * m, t) - log_s;  // (the lowest value beside the largest)
  return __fdiv_rn(x - m, t) - log_s;
}

template <typename T, bool kMask, bool kTop, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) token_logprobs_kernel(const LogprobParams p) {
  using Bits = typename DTypeTraits<T>::Bits;
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  constexpr uint32_t kAll = (1u << kPer) - 1u;
  constexpr int kGroupLanes = kThreads / kGroups;
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  // (nothing is written to a CTA's shared memory before it runs)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  Row r;
  if (p.offsets) {
    int64_t lo = p.offsets[b], hi = p.offsets[b + 1];
    lo = lo < 0 ? 0 : lo > p.capacity ? p.capacity : lo;
    hi = hi > p.capacity ? p.capacity : hi;
    set_row<T>(r, p.logits, lo, hi > lo ? min(hi - lo, (int64_t)1 << 30) : 0);  // (vectors are counted in 32 bits)
  } else {
    set_row<T>(r, p.logits, b * p.row_stride, p.vocab);
  }
  r.mask = kMask ? p.mask + b * p.mask_stride : nullptr;
  const float t = p.temperatures ? p.temperatures[b] : p.temperature;
  const bool valid = valid_temperature(t);
  const float c = fminf(kLog2e / t, 3e38f);
  const int nv = valid ? r.last + 1 : 0;
  const int lo = (int)((int64_t)nv * rank / size), hi = (int)((int64_t)nv * (rank + 1) / size);
  const int n = p.top_n;

  if (tid == 0) {
    s.count = 0u;
    s.listed = s.overflow = 0;
    s.border = 0ull;
    s.ninf = 0u;
  }

  uint4 v[kUnroll];
  uint32_t bits[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = lo + u * kThreads + tid;
    bits[u] = i < hi ? legal_bits<T, kMask>(r, i) : 0u;
    v[u] = i < hi ? ld_stream_v4(r.base + i) : make_uint4(0u, 0u, 0u, 0u);
  }

  // the CTA's first batch: everyone's first maximum, and the first border
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    exclude<T>(v[u], bits[u]);
    bits[u] = kAll;
    top = fmaxf(top, vector_top<T>(v[u]));
  }
#pragma unroll
  for (int o = 1; o < kGroupLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
  if (lane % kGroupLanes == 0) s.group_top[tid / kGroupLanes] = top;
  __syncthreads();
  {
    float m = fmaxf(s.group_top[lane], s.group_top[lane + 32]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
    top = m;
    if constexpr (kTop) {  // the n-th largest of the 64: at least n elements are no smaller
#pragma unroll
      for (int g0 = 0; g0 < kGroups; g0 += kThreads / kParts) {
        const int g = g0 + tid / kParts;
        const float x = s.group_top[g];
        int above = 0;
#pragma unroll
        for (int j = tid % kParts; j < kGroups; j += kParts) {
          const float y = s.group_top[j];
          above += y > x || (y == x && j < g);
        }
        above = over_parts(above);
        if (above == n - 1 && tid % kParts == 0 && x > -INFINITY) s.border = (unsigned long long)ordered_bits(x) << 32;
      }
    }
  }
  unsigned long long border = 0ull;
  float least = INFINITY;
  if constexpr (kTop) {
    __syncthreads();
    border = s.border;
    least = border_value(border);
  }
  Running<T> run;
  run.start(top, c);

  for (int i0 = lo, batch = 0; i0 < hi; i0 += kUnroll * kThreads, ++batch) {
    float most = -INFINITY;  // of the batch's vectors
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (kMask || bits[u] != kAll) exclude<T>(v[u], bits[u]);
      most = fmaxf(most, vector_top<T>(v[u]));
    }
    if (most >= (kTop ? fminf(least, run.m) : run.m)) {  // rarely
      if (most > run.m) run.raise(most, c);
      if (kTop && most >= least) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const uint32_t found = candidates<T>(v[u], least);
          if (found && list_candidates<T>(s, v[u], found, (i0 + u * kThreads + tid) * kPer - r.phase, border)) s.overflow = 1;
        }
      }
    }
    const bool some = most > -INFINITY;
    if (some && (std::is_same<T, float>::value || run.d.deep)) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) run.template add<true>(v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int after = i0 + (kUnroll + u) * kThreads + tid;
      if constexpr (!std::is_same<T, float>::value) {
        if (some && !run.d.deep) run.template add<false>(v[u]);
      }
      bits[u] = after < hi ? legal_bits<T, kMask>(r, after) : 0u;
      if (after < hi) v[u] = ld_stream_v4(r.base + after);
    }
    // After 1, 2, 4, ... batches the list is ranked and the border with it: each doubling
    // of what has been read brings about n candidates more.
    if (kTop && (batch & (batch + 1)) == 0 && i0 + kUnroll * kThreads < hi) {
      rank_list<kThreads>(s, n);
      border = s.border;
      least = border_value(border);
    }
  }
  if constexpr (kTop) {
    __syncthreads();
    if (s.overflow) list_again<T, kMask, kThreads>(s, r, lo, hi, n);
  }

  // this CTA's sums
  const float2 run_s = unpack2(run.s), run_a = unpack2(run.a);
  Sums mine = merge(Sums{run.m, run_s.x, run_a.x}, Sums{run.m, run_s.y, run_a.y}, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    mine = merge(mine, Sums{__shfl_xor_sync(FULL_MASK, mine.m, o), __shfl_xor_sync(FULL_MASK, mine.s, o),
                            __shfl_xor_sync(FULL_MASK, mine.a, o)}, c);
  if (lane == 0) s.part[warp] = mine;
  if constexpr (kTop) rank_list<kThreads>(s, n);
  else __syncthreads();
  if (warp == 0) {
    mine = s.part[lane & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1)
      mine = merge(mine, Sums{__shfl_xor_sync(FULL_MASK, mine.m, o), __shfl_xor_sync(FULL_MASK, mine.s, o),
                              __shfl_xor_sync(FULL_MASK, mine.a, o)}, c);
    if (lane == 0) s.part[0] = mine;
  }
  __syncthreads();
  // to the other CTAs' shared memory (all of them run: the barrier at the start): what a
  // CTA would have to fetch took it 15 us for 16 lists of 20
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (size > 1) {
    if (tid < size) cluster.map_shared_rank(s.total, tid)[rank] = s.part[0];
    if (kTop && tid < n) cluster.map_shared_rank(s.all, 0)[rank * n + tid] = tid < s.listed ? s.list[tid] : 0ull;
    cluster.sync();
  } else {
    if (tid == 0) s.total[0] = s.part[0];
    if (kTop && tid < n) s.all[tid] = tid < s.listed ? s.list[tid] : 0ull;
    __syncthreads();
  }
  // the cluster's, the same in every thread (merged in rank order)
  Sums sum = s.total[0];
  for (int q = 1; q < size; ++q) sum = merge(sum, s.total[q], c);
  if (sum.m == INFINITY) {  // infinite logits share the weight: S counts them
    unsigned int found = 0u;
    for (int i = lo + tid; i < hi; i += kThreads) {
      uint4 x = ld_stream_v4(r.base + i);
      exclude<T>(x, legal_bits<T, kMask>(r, i));
#pragma unroll
      for (int k = 0; k < kPer / 2; ++k) {
        const float2 f = element_pair<T>(x, k);
        found += (f.x == INFINITY) + (f.y == INFINITY);
      }
    }
    if (found) atomicAdd(&s.ninf, found);
    __syncthreads();
    if (tid == 0) cluster.map_shared_rank(s.all_ninf, 0)[rank] = s.ninf;
    if (size > 1) cluster.sync();
    else __syncthreads();
    unsigned int all = 0u;
    for (int q = 0; q < size; ++q) all += s.all_ninf[q];  // (CTA 0's are all there)
    sum.s = (float)all;
    sum.a = 0.f;
  }

  if (rank == 0) {
    const bool some = sum.m > -INFINITY;
    const float nan = __int_as_float(0x7fc00000);
    const float log_s = !valid ? nan : some ? logf(sum.s) : 0.f;
    const float rounded = log_s - kLn2 * (sum.a / sum.s);
    const float entropy = !valid ? nan : some && !(rounded < 0.f) ? rounded : 0.f;
    if (tid == 0) {
      if (p.entropy) p.entropy[b] = entropy;
      if (p.logsumexp) p.logsumexp[b] = !valid ? nan : some ? __fdiv_rn(sum.m, t) + log_s : -INFINITY;
      if (p.stats) p.stats[b] = make_float4(sum.m, sum.s, entropy, valid ? fminf(__fdiv_rn(1.f, t), 3e38f) : nan);
    }
    for (int k = tid; k < p.tokens; k += kThreads) {
      const int64_t id = p.token_ids[b * p.tokens + k];
      int64_t at = id;
      if (p.offsets && id >= 0) {  // its place among the row's rising ids
        int64_t a = 0, z = r.len;
        while (a < z) {
          const int64_t mid = (a + z) >> 1;
          if (p.ids[r.first + mid] < id) a = mid + 1;
          else z = mid;
        }
        at = a < r.len && p.ids[r.first + a] == id ? a : r.len;
      }
      float lp = -INFINITY;
      if (id >= 0 && at < r.len && (!kMask || ((__ldg(r.mask + (at >> 5)) >> (at & 31)) & 1u)))
        lp = logprob_of(DTypeTraits<T>::bits_to_float(__ldg(static_cast<const Bits*>(p.logits) + r.first + at)), sum.m, t,
                        log_s);
      p.logprobs[b * p.tokens + k] = !valid ? nan : id < 0 ? 0.f : lp;
    }
    if constexpr (kTop) {
      // a key's place is the number of larger ones, counted in the other lists one by one
      for (int i0 = 0; i0 < size * n; i0 += kThreads / kParts) {
        const int i = i0 + tid / kParts, q = i / n;
        const unsigned long long key = i < size * n ? s.all[i] : 0ull;
        int place = 0;
        if (key != 0ull) {
          for (int o = tid % kParts; o < size; o += kParts) {
            if (o == q) continue;
            const unsigned long long* other = s.all + o * n;
            int a = 0, z = n;
            while (a < z) {  // larger keys come first, and none (0) last
              const int mid = (a + z) >> 1;
              if (other[mid] > key) a = mid + 1;
              else z = mid;
            }
            place += a;
          }
        }
        place = over_parts(place) + i - q * n;
        if (key == 0ull || place >= n || tid % kParts != 0) continue;
        const int64_t at_row = key_index(key);
        p.top_ids[b * n + place] = p.offsets ? p.ids[r.first + at_row] : at_row;
        p.top_logprobs[b * n + place] = logprob_of(key_value(key), sum.m, t, log_s);
      }
      int listed = 0;
      for (int i = lane; i < size * n; i += 32) listed += s.all[i] != 0ull;
      listed = warp_sum(listed);
      for (int i = min(listed, n) + tid; i < n; i += kThreads) {
        p.top_ids[b * n + i] = -1;
        p.top_logprobs[b * n + i] = valid ? -INFINITY : nan;
      }
    }
  }
}

template <typename T, bool kMask, bool kTop, int kThreads>
cudaError_t launch_forward(const LogprobParams& p, int batch, int size, cudaStream_t stream) {
  auto k = token_logprobs_kernel<T, kMask, kTop, kThreads>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)batch * (unsigned)size);
  cfg.blockDim = dim3(kThreads);
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

template <typename T, bool kMask, bool kTop>
cudaError_t launch_shaped(const LogprobParams& p, int batch, int64_t max_len, cudaStream_t stream) {
  int dev = 0;
  const cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const int sms = num_sms(dev);
  // Many rows: a CTA of 256 threads each, four on an SM, so that one's start and end pass
  // while the others read (1,999 x 151,936 bf16: 132 us, two of 512 threads 151).
  if (batch >= 4 * sms) return launch_forward<T, kMask, kTop, 256>(p, batch, 1, stream);
  // Few: CTAs of 512 threads, as many for a row as keep half a batch of vectors each while
  // the device holds them all, two on an SM; and no more than 8, past which the cluster's
  // barriers cost what the shorter shares gain (one row of 248,320, 20 alternatives: 8 and
  // 16 alike, 4 take a fifth longer).
  const int64_t half = (int64_t)kMaxThreads * kUnroll * DTypeTraits<T>::kPerVec / 2;
  int size = 1;
  while (size < kMaxClusterSize && (int64_t)batch * size * 2 <= 2 * (int64_t)sms && max_len > half * size) size *= 2;
  return launch_forward<T, kMask, kTop, 512>(p, batch, size, stream);
}

template <typename T>
cudaError_t launch_typed(const LogprobParams& p, int batch, int64_t max_len, cudaStream_t stream) {
  if (p.mask) return p.top_n ? launch_shaped<T, true, true>(p, batch, max_len, stream)
                             : launch_shaped<T, true, false>(p, batch, max_len, stream);
  return p.top_n ? launch_shaped<T, false, true>(p, batch, max_len, stream)
                 : launch_shaped<T, false, false>(p, batch, max_len, stream);
}

// ---- gradient -------------------------------------------------------------------
// Reads the logits once more and writes the gradient once (with the forward pass 2,048 x
// 151,936 bf16 538 us, floor 295); a CTA takes a batch of
// vectors of one row. A given token's own term is added by a second store of the
// CTA that holds its element, after a barrier: the element is computed again from
// its logit, with every term that names it, and rounded once.
struct LogprobGradParams {
  const void* logits;
  int64_t row_stride;
  const uint32_t* mask;
  int64_t mask_stride;
  int vocab;
  const int64_t* token_ids;
  int tokens;
  const float4* stats;
  const float* grad_logprobs;   // [batch, tokens] (optional)
  const float* grad_entropy;    // [batch] (optional)
  const float* grad_logsumexp;  // [batch] (optional)
  void* grad;
  int64_t grad_stride;
  int slices;
};

constexpr int kGradThreads = 256;

// y = p (base - gH ln p) / T: with d = (x - m) log2(e) / T, p = 2^d / S and
// ln p = d ln 2 - ln S, so y = 2^d (first + slope d) with the factors folded in.
struct RowGrad {
  float m, c, first, slope, inv_t;
  bool inf;  // infinite logits share the weight; the others have none
  __device__ __forceinline__ float at(float x) const {
    float d = inf ? (x == m ? 0.f : -INFINITY) : (x - m) * c;
    d = fmaxf(d, kNothing);  // (NaN, -inf: p = 0)
    const float e = exp2_approx(d);
    return e > 0.f ? e * fmaf(slope, d, first) : 0.f;  // (the factor may be infinite)
  }
};

template <typename T, bool kMask>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(const LogprobGradParams p) {
  using Bits = typename DTypeTraits<T>::Bits;
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  __shared__ float s_sum;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - b * p.slices);
  Row r;
  set_row<T>(r, p.logits, b * p.row_stride, p.vocab);
  r.mask = kMask ? p.mask + b * p.mask_stride : nullptr;
  const int nv = r.last + 1, i0 = slice * kGradThreads * kUnroll, hi = min(nv, i0 + kGradThreads * kUnroll);
  uint4 v[kUnroll];
  uint32_t bits[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = i0 + u * kGradThreads + tid;
    bits[u] = i < hi ? legal_bits<T, kMask>(r, i) : 0u;
    v[u] = i < hi ? ld_stream_v4(r.base + i) : make_uint4(0u, 0u, 0u, 0u);
  }
  const float4 st = p.stats[b];
  const int64_t* ids = p.token_ids + b * p.tokens;
  const float* g = p.grad_logprobs ? p.grad_logprobs + b * p.tokens : nullptr;
  if (tid < 32) {
    float sum = 0.f;
    if (g)
      for (int k = tid; k < p.tokens; k += 32) sum += ids[k] >= 0 ? g[k] : 0.f;
    sum = warp_sum(sum);
    if (tid == 0) s_sum = sum;
  }
  __syncthreads();
  RowGrad row;
  row.m = st.x;
  row.inv_t = st.w;
  row.c = fminf(kLog2e * st.w, 3e38f);
  const float gh = p.grad_entropy ? p.grad_entropy[b] : 0.f, share = __fdiv_rn(1.f, st.y) * st.w;
  row.first = ((p.grad_logsumexp ? p.grad_logsumexp[b] : 0.f) - s_sum + gh * (logf(st.y) - st.z)) * share;
  row.slope = -gh * kLn2 * share;
  row.inf = st.x == INFINITY;
  const bool none = !(st.x > -INFINITY);
  const float nothing = st.w != st.w ? st.w : 0.f;  // (a temperature that is not valid: NaN, as the row reports)
  Exponents<T> exponents;
  exponents.set(st.x, row.c);
  constexpr bool kDeep = std::is_same<T, float>::value;
  // (else element by element: where a factor passes fp32, 0 times it would be NaN)
  const bool plain = !none && !row.inf && (kDeep || !exponents.deep) &&
                     fabsf(row.first) + fabsf(row.slope * exponents.lowest) < INFINITY;
  const unsigned long long first2 = pack2(row.first, row.first), slope2 = pack2(row.slope, row.slope);

  Bits* out = static_cast<Bits*>(p.grad) + b * p.grad_stride;
  // (element 0 of the gradient's row lies as far into a 16-byte vector as the logits')
  const bool same_phase = (reinterpret_cast<uintptr_t>(out - r.phase) & 15) == 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = i0 + u * kGradThreads + tid;
    if (i >= hi) continue;
    uint4 x = v[u];
    if (kMask || bits[u] != (1u << kPer) - 1u) exclude<T>(x, bits[u]);
    float y[kPer];
    if (plain) {
#pragma unroll
      for (int k = 0; k < kPer / 2; ++k) {
        const unsigned long long d = exponents.template at<kDeep>(x, k);
        const float2 one = unpack2(d);
        const float2 two = unpack2(mul2(pack2(exp2_approx(one.x), exp2_approx(one.y)), fma2(slope2, d, first2)));
        y[2 * k] = two.x;
        y[2 * k + 1] = two.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPer / 2; ++k) {
        const float2 f = element_pair<T>(x, k);
        y[2 * k] = !(f.x > -INFINITY) ? 0.f : none ? nothing : row.at(f.x);
        y[2 * k + 1] = !(f.y > -INFINITY) ? 0.f : none ? nothing : row.at(f.y);
      }
    }
    const int e0 = i * kPer - r.phase;
    if (same_phase && e0 >= 0 && e0 + kPer <= r.len) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(y[2 * k], y[2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * k], y[2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          w[k] = __float_as_uint(y[k]);
        }
      }
      *reinterpret_cast<uint4*>(out + e0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (e0 + j >= 0 && e0 + j < r.len) out[e0 + j] = DTypeTraits<T>::round_bits(y[j]);
    }
  }
  if (!g || none) return;
  __syncthreads();  // the stores above come before those below
  const int64_t first = (int64_t)i0 * kPer - r.phase, last = (int64_t)hi * kPer - r.phase;
  for (int k = tid; k < p.tokens; k += kGradThreads) {
    const int64_t id = ids[k];
    if (id < 0 || id < first || id >= last || id >= r.len) continue;
    if (kMask && !((__ldg(r.mask + (id >> 5)) >> (id & 31)) & 1u)) continue;
    const float x = DTypeTraits<T>::bits_to_float(__ldg(static_cast<const Bits*>(p.logits) + r.first + id));
    if (!(x > -INFINITY)) continue;
    bool earlier = false;
    for (int j = 0; j < k && !earlier; ++j) earlier = ids[j] == id;
    if (earlier) continue;
    float own = 0.f;
    for (int j = k; j < p.tokens; ++j)
      if (ids[j] == id) own += g[j];
    out[id] = DTypeTraits<T>::round_bits(fmaf(own, st.w, row.at(x)));
  }
}

template <typename T>
cudaError_t launch_grad(LogprobGradParams p, int batch, cudaStream_t stream) {
  // (one vector more than the length needs, for rows that start inside one)
  const int64_t per_cta = (int64_t)kGradThreads * kUnroll;
  const int64_t vectors = ((int64_t)p.vocab + DTypeTraits<T>::kPerVec - 1) / DTypeTraits<T>::kPerVec + 1;
  const int64_t slices = (vectors + per_cta - 1) / per_cta, grid = slices * batch;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  p.slices = (int)slices;
  if (p.mask) token_logprobs_grad_kernel<T, true><<<(unsigned)grid, kGradThreads, 0, stream>>>(p);
  else token_logprobs_grad_kernel<T, false><<<(unsigned)grid, kGradThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

int32_t check(const char* fn, int32_t dtype, int32_t batch, const int64_t* token_ids, int32_t tokens) {
  if (dtype != GSP_DTYPE_F16 && dtype != GSP_DTYPE_BF16 && dtype != GSP_DTYPE_F32)
    return record_error(GSP_ERR_UNSUPPORTED, "%s: dtype must be GSP_DTYPE_F16, GSP_DTYPE_BF16 or GSP_DTYPE_F32", fn);
  if (batch < 1 || batch > (1 << 26)) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: batch must be in 1..2^26", fn);
  if (tokens < 0 || tokens > kMaxTokens)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: tokens must be in 0..%d", fn, kMaxTokens);
  if (tokens > 0 && !token_ids) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: token_ids is required", fn);
  return GSP_OK;
}

int32_t check_rows(const char* fn, const void* logits, int64_t row_stride, const int32_t* bitmask,
                   int64_t bitmask_row_stride, int32_t batch, int32_t vocab) {
  if (!logits) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: logits is required", fn);
  if (vocab < 1) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: vocab must be positive", fn);
  if (vocab > (1 << 30)) return record_error(GSP_ERR_UNSUPPORTED, "%s: vocab above 2^30", fn);
  if (row_stride < 0) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: negative logits_row_stride", fn);
  const int64_t nw = ((int64_t)vocab + 31) / 32;
  if (bitmask && (bitmask_row_stride < 0 || (batch > 1 && bitmask_row_stride != 0 && bitmask_row_stride < nw)))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: bitmask_row_stride must be 0 or >= ceil(vocab/32)", fn);
  return GSP_OK;
}

int32_t forward(const char* fn, const LogprobParams& p, int32_t dtype, int32_t batch, int64_t max_len, void* stream) {
  if (!p.temperatures && !(p.temperature > 0.f && p.temperature < INFINITY))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: temperature must be positive and finite", fn);
  if (p.top_n < 0 || p.top_n > kMaxTop)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: top_n must be in 0..%d", fn, kMaxTop);
  if (p.tokens > 0 && !p.logprobs) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: logprobs is required", fn);
  if (p.top_n > 0 && (!p.top_ids || !p.top_logprobs))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: top_ids and top_logprobs are required", fn);
  if (reinterpret_cast<uintptr_t>(p.stats) & 15)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: stats must be 16-byte aligned", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == GSP_DTYPE_F32    ? launch_typed<float>(p, batch, max_len, s)
                          : dtype == GSP_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(p, batch, max_len, s)
                                                    : launch_typed<__half>(p, batch, max_len, s);
  if (err == cudaSuccess) return GSP_OK;
  return record_error(GSP_ERR_CUDA, "%s: %s (%s)", fn, cudaGetErrorName(err), cudaGetErrorString(err));
}

}  // namespace
}  // namespace gsp

using namespace gsp;

extern "C" {

int32_t gsp_token_logprobs(const void* logits, int64_t logits_row_stride, int32_t dtype, const int32_t* bitmask,
                           int64_t bitmask_row_stride, int32_t batch, int32_t vocab, float temperature,
                           const float* temperatures, const int64_t* token_ids, int32_t tokens, int32_t top_n,
                           float* logprobs, float* entropy, float* logsumexp, int64_t* top_ids, float* top_logprobs,
                           float* stats, void* stream) {
  const char* fn = "gsp_token_logprobs";
  int32_t st = check(fn, dtype, batch, token_ids, tokens);
  if (st == GSP_OK) st = check_rows(fn, logits, logits_row_stride, bitmask, bitmask_row_stride, batch, vocab);
  if (st != GSP_OK) return st;
  LogprobParams p{};
  p.logits = logits;
  p.row_stride = batch > 1 ? logits_row_stride : 0;
  p.mask = reinterpret_cast<const uint32_t*>(bitmask);
  p.mask_stride = batch > 1 ? bitmask_row_stride : 0;
  p.vocab = vocab;
  p.temperature = temperature;
  p.temperatures = temperatures;
  p.token_ids = token_ids;
  p.tokens = tokens;
  p.top_n = top_n;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.logsumexp = logsumexp;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.stats = reinterpret_cast<float4*>(stats);
  return forward(fn, p, dtype, batch, vocab, stream);
}

int32_t gsp_token_logprobs_compact(const void* compact_logits, const int64_t* compact_ids,
                                   const int64_t* request_offsets, int64_t capacity, int32_t max_len, int32_t dtype,
                                   int32_t batch, float temperature, const float* temperatures,
                                   const int64_t* token_ids, int32_t tokens, int32_t top_n, float* logprobs,
                                   float* entropy, float* logsumexp, int64_t* top_ids, float* top_logprobs,
                                   void* stream) {
  const char* fn = "gsp_token_logprobs_compact";
  const int32_t st = check(fn, dtype, batch, token_ids, tokens);
  if (st != GSP_OK) return st;
  if (capacity < 0 || max_len < 0)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: capacity and max_len must not be negative", fn);
  if (!request_offsets) return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: request_offsets is required", fn);
  if (capacity > 0 && (!compact_logits || !compact_ids))
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: compact_logits and compact_ids are required", fn);
  LogprobParams p{};
  p.logits = compact_logits;
  p.ids = compact_ids;
  p.offsets = request_offsets;
  p.capacity = capacity;
  p.temperature = temperature;
  p.temperatures = temperatures;
  p.token_ids = token_ids;
  p.tokens = tokens;
  p.top_n = top_n;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.logsumexp = logsumexp;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  return forward(fn, p, dtype, batch, max_len, stream);
}

int32_t gsp_token_logprobs_grad(const void* logits, int64_t logits_row_stride, int32_t dtype, const int32_t* bitmask,
                                int64_t bitmask_row_stride, int32_t batch, int32_t vocab, const int64_t* token_ids,
                                int32_t tokens, const float* stats, const float* grad_logprobs,
                                const float* grad_entropy, const float* grad_logsumexp, void* grad_logits,
                                int64_t grad_row_stride, void* stream) {
  const char* fn = "gsp_token_logprobs_grad";
  int32_t st = check(fn, dtype, batch, token_ids, tokens);
  if (st == GSP_OK) st = check_rows(fn, logits, logits_row_stride, bitmask, bitmask_row_stride, batch, vocab);
  if (st != GSP_OK) return st;
  if (!stats || !grad_logits)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: stats and grad_logits are required", fn);
  if (reinterpret_cast<uintptr_t>(stats) & 15)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: stats must be 16-byte aligned", fn);
  if (batch > 1 && grad_row_stride < vocab)
    return record_error(GSP_ERR_INVALID_ARGUMENT, "%s: grad_row_stride < vocab", fn);
  LogprobGradParams p{};
  p.logits = logits;
  p.row_stride = batch > 1 ? logits_row_stride : 0;
  p.mask = reinterpret_cast<const uint32_t*>(bitmask);
  p.mask_stride = batch > 1 ? bitmask_row_stride : 0;
  p.vocab = vocab;
  p.token_ids = token_ids;
  p.tokens = tokens;
  p.stats = reinterpret_cast<const float4*>(stats);
  p.grad_logprobs = tokens > 0 ? grad_logprobs : nullptr;
  p.grad_entropy = grad_entropy;
  p.grad_logsumexp = grad_logsumexp;
  p.grad = grad_logits;
  p.grad_stride = batch > 1 ? grad_row_stride : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == GSP_DTYPE_F32    ? launch_grad<float>(p, batch, s)
                          : dtype == GSP_DTYPE_BF16 ? launch_grad<__nv_bfloat16>(p, batch, s)
                                                    : launch_grad<__half>(p, batch, s);
  if (err == cudaSuccess) return GSP_OK;
  return record_error(GSP_ERR_CUDA, "%s: %s (%s)", fn, cudaGetErrorName(err), cudaGetErrorString(err));
}

}  // extern "C"
