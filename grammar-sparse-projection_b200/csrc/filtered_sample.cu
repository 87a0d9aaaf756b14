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
// One cluster of CTAs per row, the row's order-preserving keys (16 or 32 bits,
// 0: not legal) held in the CTAs' shared memory; one pass over the logits in
// global memory. A search narrows the range of keys 256-fold per pass: every
// CTA counts (or weighs) its keys in 256 bins of shared memory, the CTAs read
// one another's bins over distributed shared memory after one cluster barrier,
// and each picks the bin that passes the target.
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
constexpr int kBins = 256;
constexpr int kReplicas = 4;  // copies of the bins, by lane: equal keys of a warp meet on fewer addresses
constexpr int kMaxCluster = 16;
constexpr int kMaxShift = 52;

// Order-preserving keys: larger logit, larger key; NaN and -inf (never drawn)
// and illegal entries 0.
template <typename T>
struct SampleKey {
  using Key = uint16_t;
  static constexpr uint32_t kNegInf = std::is_same<T, __half>::value ? 0x8000u - 0x7C00u : 0x8000u - 0x7F80u;
  static constexpr uint32_t kPosInf = std::is_same<T, __half>::value ? 0xFC00u : 0xFF80u;
  static __device__ __forceinline__ uint32_t from_bits(uint32_t bits) {
    const uint32_t o = (bits & 0x8000u) ? 0x8000u - (bits & 0x7fffu) : (bits | 0x8000u);
    return (o > kNegInf && o <= kPosInf) ? o : 0u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    const uint32_t bits = key >= 0x8000u ? (key & 0x7fffu) : (0x8000u | (0x8000u - key));
    return DTypeTraits<T>::bits_to_float((uint16_t)bits);
  }
  // smallest key whose value is >= x
  static __device__ __forceinline__ uint32_t at_least(double x) {
    const float f = __double2float_ru(x);
    uint32_t bits;
    if constexpr (std::is_same<T, __half>::value)
      bits = __half_as_ushort(__float2half_ru(f));
    else
      bits = __bfloat16_as_ushort(__float2bfloat16_ru(f));
    const uint32_t o = (bits & 0x8000u) ? 0x8000u - (bits & 0x7fffu) : (bits | 0x8000u);
    return o <= kNegInf ? 1u : o;
  }
};
template <>
struct SampleKey<float> {
  using Key = uint32_t;
  static constexpr uint32_t kNegInf = 0x007FFFFFu;
  static constexpr uint32_t kPosInf = 0xFF800000u;
  static __device__ __forceinline__ uint32_t from_bits(uint32_t bits) {
    const uint32_t o = ordered_bits(__uint_as_float(bits));
    return (o > kNegInf && o <= kPosInf) ? o : 0u;
  }
  static __device__ __forceinline__ float value(uint32_t key) { return from_ordered_bits(key); }
  static __device__ __forceinline__ uint32_t at_least(double x) {
    const uint32_t o = ordered_bits(__double2float_ru(x));
    return o <= kNegInf ? 1u : o;
  }
};

struct SampleSmemHeader {
  uint32_t lo[kReplicas][kBins];            // bins being filled: low and high halves of 64-bit sums
  uint32_t hi[kReplicas][kBins];
  unsigned long long tot[2][kBins];         // this CTA's bins, read by the cluster (double-buffered)
  unsigned long long side[2][2];            // further values the cluster sums with the bins
  unsigned long long scan[kSampleWarps];
  unsigned long long pick[4];               // picked bin, sum before it, its own sum, sum of all bins
  unsigned long long word[2][kMaxCluster];  // one value per CTA (all-gather)
  uint32_t warp[kSampleWarps];
};

constexpr size_t kHeaderBytes = (sizeof(SampleSmemHeader) + 127) / 128 * 128;

template <typename T>
struct Row {
  const typename DTypeTraits<T>::Bits* x;  // the row's first logit
  const uint32_t* mask;                    // its mask words, or nullptr
  int64_t n;                               // tokens
};

// Key of position i, read from global memory.
template <typename T>
__device__ __forceinline__ uint32_t load_key(const Row<T>& r, int64_t i) {
  if (r.mask && !((__ldg(r.mask + (i >> 5)) >> (i & 31)) & 1u)) return 0u;
  return SampleKey<T>::from_bits(__ldg(r.x + i));
}

// One CTA's part of the row: positions [lo, lo + len), the first `resident`
// of them as keys in shared memory at index `phase` on (so that 16-byte loads
// of the row and stores of the keys are both aligned), the rest read from
// global memory in every pass.
template <typename T>
struct Slice {
  using Key = typename SampleKey<T>::Key;
  static constexpr int kVec = 16 / (int)sizeof(Key);
  Row<T> row;
  Key* keys;
  int64_t lo, len;
  int phase, resident;

  __device__ __forceinline__ int vectors() const { return (phase + resident + kVec - 1) / kVec; }

  __device__ __forceinline__ void load() {
    const int nv = vectors();
    for (int v = threadIdx.x; v < nv; v += kSampleThreads) {
      const int64_t i0 = lo + (int64_t)v * kVec - phase;
      uint32_t k[kVec];
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
          const uint32_t bits = sizeof(Key) == 4 ? w[j % 4] : (w[(j >> 1) % 4] >> (16 * (j & 1))) & 0xffffu;
          k[j] = ((legal >> j) & 1u) ? SampleKey<T>::from_bits(bits) : 0u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int at = v * kVec + j;
          k[j] = (at >= phase && at < phase + resident) ? load_key(row, i0 + j) : 0u;
        }
      }
      uint4 out;
      if constexpr (sizeof(Key) == 4)
        out = make_uint4(k[0], k[1], k[2], k[3]);
      else
        out = make_uint4(k[0] | (k[1] << 16), k[2] | (k[3] << 16), k[4 % kVec] | (k[5 % kVec] << 16),
                         k[6 % kVec] | (k[7 % kVec] << 16));
      reinterpret_cast<uint4*>(keys)[v] = out;
    }
  }

  // fn(key) for every position of the CTA's part (key 0: not legal)
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    const int nv = vectors();
    for (int v = threadIdx.x; v < nv; v += kSampleThreads) {
      const uint4 q = reinterpret_cast<const uint4*>(keys)[v];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < kVec; ++j) fn(sizeof(Key) == 4 ? w[j % 4] : (w[(j >> 1) % 4] >> (16 * (j & 1))) & 0xffffu);
    }
    for (int64_t i = resident + threadIdx.x; i < len; i += kSampleThreads) fn(load_key(row, lo + i));
  }
};

// Weight of a key in units of 2^-shift.
template <typename T>
struct Weigher {
  uint32_t kmax;
  double vmax, inv_t;
  int shift;
  __device__ __forceinline__ double score(uint32_t key) const {
    return key == kmax ? 0.0 : ((double)SampleKey<T>::value(key) - vmax) * inv_t;
  }
  __device__ __forceinline__ unsigned long long operator()(uint32_t key) const {
    if (key == kmax) return 1ull << shift;
    return (unsigned long long)__double2ll_rn(exp(score(key)) * (double)(1ull << shift));
  }
};

// x in [0, 1) as a multiple of 2^-64 (exact unless x < 2^-40).
__device__ __forceinline__ unsigned long long fraction64(float x) {
  return (unsigned long long)((double)x * 18446744073709551616.0);
}

// The shortest prefix with sum >= x * total is the first whose sum passes
// ceil(x * total) - 1; at least one position (x <= 0).
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
  int buf;  // which of the double buffers the next exchange uses

  // All-gather of one value per CTA (the same in all its threads): the returned
  // array holds rank r's at index r until the exchange after the next.
  __device__ __forceinline__ unsigned long long* gather(unsigned long long v) {
    unsigned long long* mine = s->word[buf];
    if (threadIdx.x < size) {
      unsigned long long* theirs = cluster.map_shared_rank(mine, threadIdx.x);
      theirs[rank] = v;
    }
    cluster.sync();
    buf ^= 1;
    return mine;
  }
};

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s_warp) {
  v = __reduce_max_sync(FULL_MASK, v);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = __reduce_max_sync(FULL_MASK, s_warp[threadIdx.x & (kSampleWarps - 1)]);
  __syncthreads();
  return v;
}

__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(FULL_MASK, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += t;
  }
  return v;
}

struct Found {
  uint32_t key;               // border key
  unsigned long long above;   // sum over larger keys
  unsigned long long own;     // sum over the keys equal to it
  unsigned long long total;   // sum over the searched range
  bool any;                   // the running sum passes the target
};

// The first key, from khi down to klo, at which the running sum of measure(key)
// passes target(total of the range).
template <typename T, typename Measure, typename Target>
__device__ __forceinline__ Found search(Team& team, const Slice<T>& slice, uint32_t klo, uint32_t khi, Measure measure,
                                        Target target_of) {
  SampleSmemHeader* s = team.s;
  const int tid = threadIdx.x, rep = tid & (kReplicas - 1);
  Found f{0u, 0ull, 0ull, 0ull, false};
  unsigned long long target = 0ull;
  bool first = true;
  for (;;) {
    const int width = 32 - __clz(khi - klo);  // bits of the range (0: a single key)
    const int sh = width > 8 ? width - 8 : 0;
    for (int i = tid; i < kReplicas * kBins; i += kSampleThreads) {
      s->lo[0][i] = 0u;
      s->hi[0][i] = 0u;
    }
    __syncthreads();
    slice.each([&](uint32_t key) {
      if (key < klo || key > khi || key == 0u) return;
      const uint32_t bin = (khi - key) >> sh;
      const unsigned long long m = measure(key);
      const uint32_t m_lo = (uint32_t)m;
      uint32_t m_hi = (uint32_t)(m >> 32);
      if (m_lo) {
        const uint32_t old = atomicAdd(&s->lo[rep][bin], m_lo);
        m_hi += (old + m_lo < old) ? 1u : 0u;
      }
      if (m_hi) atomicAdd(&s->hi[rep][bin], m_hi);
    });
    __syncthreads();
    if (tid < kBins) {
      unsigned long long t = 0ull;
#pragma unroll
      for (int r = 0; r < kReplicas; ++r) t += s->lo[r][tid] + ((unsigned long long)s->hi[r][tid] << 32);
      s->tot[team.buf][tid] = t;
    }
    team.cluster.sync();
    unsigned long long t = 0ull;
    if (tid < kBins) {
      for (int r = 0; r < team.size; ++r) t += team.cluster.map_shared_rank(s->tot[team.buf], r)[tid];
    }
    team.buf ^= 1;
    // inclusive scan over the bins, largest keys first
    const unsigned long long incl_w = warp_scan_u64(t);
    if ((tid & 31) == 31) s->scan[tid >> 5] = incl_w;
    if (tid < 4) s->pick[tid] = ~0ull;
    __syncthreads();
    unsigned long long before = 0ull, total = 0ull;
    for (int w = 0; w < kBins / 32; ++w) {
      if (w < (tid >> 5)) before += s->scan[w];
      total += s->scan[w];
    }
    if (first) {
      f.total = total;
      target = target_of(total);
      first = false;
    }
    const unsigned long long incl = before + incl_w, excl = incl - t;
    if (tid < kBins && excl <= target && target < incl) {
      s->pick[0] = (unsigned long long)tid;
      s->pick[1] = excl;
      s->pick[2] = t;
    }
    __syncthreads();
    const unsigned long long bin = s->pick[0];
    if (bin == ~0ull) return f;  // the whole range does not pass the target
    f.above += s->pick[1];
    target -= s->pick[1];
    f.own = s->pick[2];
    khi -= (uint32_t)bin << sh;
    if (sh == 0) {
      f.key = khi;
      f.any = true;
      return f;
    }
    const uint32_t span = (1u << sh) - 1u;
    klo = khi - klo > span ? khi - span : klo;
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) filtered_sample_kernel(const FilteredSampleParams p) {
  using K = SampleKey<T>;
  using Bits = typename DTypeTraits<T>::Bits;
  extern __shared__ __align__(128) unsigned char smem[];
  SampleSmemHeader* s = reinterpret_cast<SampleSmemHeader*>(smem);
  Team team{s, cg::this_cluster(), 0, 0, 0};
  team.rank = (int)team.cluster.block_rank();
  team.size = (int)team.cluster.num_blocks();
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
  slice.keys = reinterpret_cast<typename K::Key*>(smem + kHeaderBytes);
  slice.phase = (int)((reinterpret_cast<uintptr_t>(slice.row.x + slice.lo) & 15) / sizeof(Bits));
  slice.resident = (int)min(slice.len, (int64_t)p.resident);

  // ---- keys into shared memory, largest key -----------------------------------
  slice.load();
  __syncthreads();
  uint32_t kmax = 0u;
  slice.each([&](uint32_t key) { kmax = max(kmax, key); });
  kmax = block_max(kmax, s->warp);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  {
    const unsigned long long* all = team.gather(kmax);
    for (int r = 0; r < team.size; ++r) kmax = max(kmax, (uint32_t)all[r]);
  }
  if (kmax == 0u) {  // nothing is legal
    if (leader) {
      p.token_ids[b] = 0;
      if (p.logprobs) p.logprobs[b] = -INFINITY;
      if (p.kept) p.kept[b] = 0;
    }
    return;
  }

  Weigher<T> weigh;
  weigh.kmax = kmax;
  weigh.vmax = (double)K::value(kmax);
  weigh.inv_t = temperature > 0.f ? 1.0 / (double)temperature : 0.0;
  weigh.shift = min(kMaxShift, 62 - (64 - __clzll((unsigned long long)n)));

  uint32_t draw_key = kmax;
  unsigned long long ordinal = 0ull;  // among the positions of draw_key, by rising position
  float logprob = 0.f;
  unsigned long long kept = 1ull;
  if (temperature > 0.f) {
    // ---- the kept set: keys above `border`, and `ties` positions at it --------
    uint32_t border = 1u;
    unsigned long long ties = ~0ull, excess = 0ull;  // excess: positions at the border beyond `ties`
    if (top_k > 0 && top_k < n) {
      const Found f = search(
          team, slice, 1u, kmax, [](uint32_t) { return 1ull; },
          [&](unsigned long long) { return (unsigned long long)top_k - 1ull; });
      if (f.any) {
        border = f.key;
        ties = (unsigned long long)top_k - f.above;
        excess = f.own - ties;
      }
    }
    if (min_p > 0.f) {
      const uint32_t k = min_p >= 1.f ? kmax : K::at_least(weigh.vmax + (double)temperature * log((double)min_p));
      if (k > border) {
        border = min(k, kmax);
        ties = ~0ull;
        excess = 0ull;
      }
    }
    unsigned long long sum = 0ull;
    if (top_p < 1.f) {
      unsigned long long target = 0ull;
      const Found f = search(team, slice, border, kmax, weigh, [&](unsigned long long total) {
        if (excess) total -= excess * weigh(border);
        target = prefix_target(top_p, total);
        return target;
      });
      const unsigned long long w = weigh(f.key);
      border = f.key;
      ties = (target - f.above) / w + 1ull;
      excess = f.own / w - ties;
      sum = f.above + ties * w;
    }
    // ---- the draw ------------------------------------------------------------
    unsigned long long target = 0ull;
    const Found f = search(team, slice, border, kmax, weigh, [&](unsigned long long total) {
      if (sum == 0ull) sum = total - (excess ? excess * weigh(border) : 0ull);
      target = __umul64hi(fraction64(u), sum);
      return target;
    });
    draw_key = f.key;
    ordinal = (target - f.above) / weigh(f.key);
    logprob = (float)(weigh.score(draw_key) - log((double)sum * (1.0 / (double)(1ull << weigh.shift))));
    // ---- how many were kept ------------------------------------------------------
    uint32_t above = 0u, at = 0u;
    slice.each([&](uint32_t key) {
      above += key > border ? 1u : 0u;
      at += key == border ? 1u : 0u;
    });
    above = __reduce_add_sync(FULL_MASK, above);
    at = __reduce_add_sync(FULL_MASK, at);
    if ((tid & 31) == 0) s->scan[tid >> 5] = ((unsigned long long)at << 32) | above;
    __syncthreads();
    unsigned long long mine = 0ull;
    for (int w = 0; w < kSampleWarps; ++w) mine += s->scan[w];
    const unsigned long long* all = team.gather(mine);
    unsigned long long n_above = 0ull, n_at = 0ull;
    for (int r = 0; r < team.size; ++r) {
      n_above += all[r] & 0xffffffffull;
      n_at += all[r] >> 32;
    }
    kept = n_above + min(n_at, ties);
  }

  // ---- the drawn position: the ordinal-th of draw_key, by rising position -------
  uint32_t here = 0u;
  slice.each([&](uint32_t key) { here += key == draw_key ? 1u : 0u; });
  here = __reduce_add_sync(FULL_MASK, here);
  __syncthreads();
  if ((tid & 31) == 0) s->warp[tid >> 5] = here;
  __syncthreads();
  unsigned long long mine = 0ull;
  for (int w = 0; w < kSampleWarps; ++w) mine += s->warp[w];
  const unsigned long long* all = team.gather(mine);
  for (int r = 0; r < team.rank; ++r) ordinal -= all[r];  // wraps for CTAs behind the owner
  if (ordinal < mine) {
    // this CTA owns it: blocks of kSampleThreads positions in order
    for (int64_t i0 = 0; i0 < slice.len; i0 += kSampleThreads) {
      const int64_t i = i0 + tid;
      uint32_t key = 0u;
      if (i < slice.resident) key = slice.keys[slice.phase + i];
      else if (i < slice.len) key = load_key(slice.row, slice.lo + i);
      const bool hit = key == draw_key;
      const unsigned hits = __ballot_sync(FULL_MASK, hit);
      __syncthreads();
      if ((tid & 31) == 0) s->warp[tid >> 5] = __popc(hits);
      __syncthreads();
      unsigned long long before = 0ull, in_block = 0ull;
      for (int w = 0; w < kSampleWarps; ++w) {
        if (w < (tid >> 5)) before += s->warp[w];
        in_block += s->warp[w];
      }
      before += __popc(hits & ((1u << (tid & 31)) - 1u));
      if (hit && before == ordinal) {
        const int64_t at = slice.lo + i;
        p.token_ids[b] = p.ids ? p.ids[start + at] : p.vocab_offset + at;
        if (p.logprobs) p.logprobs[b] = logprob;
        if (p.kept) p.kept[b] = (int32_t)kept;
      }
      if (ordinal < in_block) break;
      ordinal -= in_block;
    }
  }
}

// Launch: one cluster per row.
template <typename T>
cudaError_t launch_typed(FilteredSampleParams p, int batch, int64_t max_len, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  using Key = typename SampleKey<T>::Key;
  constexpr size_t kSmemMax = 227 * 1024;
  // CTAs per row: one for short rows; for long ones as many as the batch leaves
  // SMs for, and no fewer than hold the row in shared memory (up to 16).
  const size_t room = (kSmemMax - kHeaderBytes - 32) / sizeof(Key) / 32 * 32;
  int size = 1;
  while (size < kMaxCluster && ((int64_t)room * size < max_len ||
                                (max_len > (int64_t)2048 * size && (int64_t)batch * size * 2 <= num_sms(dev))))
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
