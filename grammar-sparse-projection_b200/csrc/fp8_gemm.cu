// The fp8 head on the tensor cores (sm_100a): block-sparse and dense routes, and the
// plain product (no mask) over the positions of a prompt.
//
//   y[b, v] = sum_kb hs[b, kb] ws[v / 128, kb] sum_{k in block kb} q[b, k] w[v, k]
//
// One block of 128 columns is one stage of the pipeline: four tcgen05.mma
// (kind::f8f6f4, 32 columns each) give the inner sums in a TMEM accumulator of their
// own, and the epilogue warps add them, times their two scales, to fp32 sums in
// registers. M is the 128 hidden states (TMEM lanes: a thread's scale hs is one
// register and its logits lie side by side in memory), N the vocabulary rows, in
// groups of 32: one mask word, a quarter of a scale block, so that a column group
// shares one scale per stage and an addition costs one packed fp32 operation per two
// products. Rows of the operand tile past the batch hold whatever the stage held;
// their lanes are never read.
//
// Batches up to 128 are bound by the weight's bytes: a CTA's share of the active
// groups is even to one group, in tiles of four (N <= 128, four accumulators).
// Larger batches take tiles of eight groups (N = 256, two accumulators) strided so
// that the CTAs under way share the weight's tiles through L2.
//
//   warp 0      TMA producer: the active groups' 32 rows x 128 bytes each, and the
//               hidden states' rows x 128 bytes, 128-byte swizzle;
//   warp 1      TMEM, and one lane's tcgen05.mma;
//   warps 2-9   epilogue, two per TMEM lane quadrant, alternating groups.
//
// A prologue kernel quantises (or turns round the scales of) the hidden states,
// clears the top-1 keys, and in block mode lists the 32-row groups that hold a legal
// token of some request; the -inf of the other groups is stored by the epilogue warps
// before their first accumulator.
//
// Every wait is bounded; one that runs out sets the device's error word and the
// kernel drains its copies and tensor-core work before it returns.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "fp8_head.cuh"
#include "gsp_async.cuh"
#include "gsp_pairs.cuh"
#include "gsp_tcgen05.cuh"

namespace gsp {
namespace {

constexpr int kChunkRows = 128;  // hidden states of a tile
constexpr int kGroupRows = 32;
constexpr uint32_t kGroupBytes = kGroupRows * kBlock;
constexpr int kEpilogueWarps = 8;
constexpr int kGemmThreads = 32 * (2 + kEpilogueWarps);
constexpr int kMaxStages = 10;
constexpr int kMaxAcc = 4;
constexpr int kMaxBuilders = 256;  // prefix sums that fit the CTA's table: 2^20 tokens; past it they are searched in global memory

struct GemmConfig {
  int chunks;  // of kChunkRows hidden states
  int xrows;   // rows loaded of a chunk
  int stages;
  int builders;
};

// ---- prologue -------------------------------------------------------------------
constexpr int kPrologueThreads = 512;

template <typename T, bool kVec>
__device__ __forceinline__ void quantize_hidden(const Fp8Params& p, int64_t first, int64_t step) {
  using U = Units<T, kVec>;
  constexpr int kE = U::kElems;
  const int n = U::count(p.hidden_dim), width = (n + 31) & ~31;
  const int64_t total = (int64_t)p.batch * width;
  uint8_t* values = const_cast<uint8_t*>(p.hidden);
  for (int64_t at = first; at < total; at += step) {
    const int row = (int)(at / width), i = (int)(at - (int64_t)row * width);
    float f[kE];
    uint32_t top = 0u;
    if (i < n) {
      U::load(static_cast<const typename U::Bits*>(p.raw) + row * p.raw_stride, i, p.hidden_dim, f);
      top = U::magnitude(f);
    }
    const BlockScale s = block_scale(lanes_max<U::kLanes>(top));
    if (i >= n) continue;
    uint32_t w[kE / 4];
#pragma unroll
    for (int k = 0; k < kE / 4; ++k) w[k] = to_e4m3(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3], s);
    U::store_bytes(values + row * p.hidden_stride, i, p.hidden_dim, w);
    if (i % U::kLanes == 0) p.scales_t[(int64_t)(i / U::kLanes) * p.batch + row] = s.scale;
  }
}

// Blocks [0, builders): the active groups of kListGroups mask words each; the others:
// the hidden states.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kPrologueThreads) fp8_prologue_kernel(const __grid_constant__ Fp8Params p, int builders) {
  __shared__ uint32_t s_any[kListGroups];
  const int tid = threadIdx.x;
  // (the projection may take its place and set itself up; it waits for this grid's end)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if ((int)blockIdx.x >= builders) {
    const int64_t first = (int64_t)(blockIdx.x - builders) * kPrologueThreads + tid;
    const int64_t step = (int64_t)(gridDim.x - builders) * kPrologueThreads;
    for (int64_t b = first; b < p.batch; b += step) {
      p.keys[b] = 0ull;
      p.tickets[b] = 0u;
    }
    if (p.raw) {
      quantize_hidden<T, kVec>(p, first, step);
    } else {
      const int64_t total = (int64_t)p.batch * p.blocks;
      for (int64_t at = first; at < total; at += step) {
        const int kb = (int)(at / p.batch);
        const int64_t row = at - (int64_t)kb * p.batch;
        p.scales_t[at] = __ldg(p.hidden_scales + row * p.hidden_scales_stride + kb);
      }
    }
    return;
  }
  const int w0 = blockIdx.x * kListGroups;
  const int at = w0 + tid % kListGroups;
  if (tid < kListGroups) s_any[tid] = 0u;
  __syncthreads();
  uint32_t any = 0u;
  if (at < p.nw) {
#pragma unroll 8
    for (int b = tid / kListGroups; b < p.batch; b += kPrologueThreads / kListGroups)
      any |= __ldg(p.mask + (int64_t)b * p.mask_stride + at);
    any = tail_clip(any, at, p.vocab);
  }
  if (any) atomicOr(&s_any[tid % kListGroups], any);
  __syncthreads();
  __shared__ int s_before[kListGroups / 32];
  unsigned active = 0u;
  if (tid < kListGroups) {
    active = __ballot_sync(FULL_MASK, s_any[tid] != 0u);
    if ((tid & 31) == 0) {
      s_before[tid >> 5] = __popc(active);
      const int word = (w0 + tid) >> 5;
      if (word < (p.nw + 31) / 32) p.group_bits[word] = active;
    }
  }
  __syncthreads();
  if (tid < kListGroups) {
    int pos = __popc(active & ((1u << (tid & 31)) - 1u));
    for (int j = 0; j < (tid >> 5); ++j) pos += s_before[j];
    if (s_any[tid] != 0u) p.groups[w0 + pos] = w0 + tid;
    if (tid == kListGroups - 1) p.group_counts[blockIdx.x] = pos + (s_any[tid] != 0u);
  }
}

// ---- projection -----------------------------------------------------------------
template <int kGroups>
struct GemmLayout {
  static constexpr uint32_t kWBytes = kGroups * kGroupBytes;
  uint32_t x, bars, tmem, misc, prefix, total;
  __host__ __device__ GemmLayout(const GemmConfig& c) {
    x = (uint32_t)c.stages * kWBytes;
    // (the MMA reads 128 rows of a stage's hidden states, loaded or not)
    bars = x + (uint32_t)(c.stages - 1) * (uint32_t)c.xrows * kBlock + kChunkRows * kBlock;
    tmem = bars + 8 * (2 * kMaxStages + 2 * kMaxAcc);
    misc = tmem + 16;
    prefix = misc + 16;
    total = prefix + 4 * (kMaxBuilders + 1);
  }
};

// A tile: `n` groups from compacted position `pos` on, for chunk `chunk`.
struct Tile {
  int chunk, pos, n;
};

// The CTA's i-th tile; false past the last.
template <int kGroups>
__device__ __forceinline__ bool tile_of(int i, int total, int chunks, Tile& t) {
  if (chunks == 1) {
    const int lo = (int)((int64_t)total * blockIdx.x / gridDim.x), hi = (int)((int64_t)total * (blockIdx.x + 1) / gridDim.x);
    t.chunk = 0;
    t.pos = lo + i * kGroups;
    t.n = min(kGroups, hi - t.pos);
    return t.n > 0;
  }
  const int64_t item = (int64_t)blockIdx.x + (int64_t)i * gridDim.x;
  const int64_t tile = item / chunks;
  t.chunk = (int)(item - tile * chunks);
  if (tile * kGroups >= total) return false;
  t.pos = (int)(tile * kGroups);
  t.n = min(kGroups, total - t.pos);
  return true;
}

// Group (mask word) at compacted position `pos`.
__device__ __forceinline__ int group_at(const Fp8Params& p, const int* s_prefix, int builders, int pos) {
  if (p.dense) return pos;
  int lo = 0, hi = builders;  // s_prefix[lo] <= pos < s_prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_prefix[mid] <= pos) lo = mid;
    else hi = mid;
  }
  return p.groups[lo * kListGroups + pos - s_prefix[lo]];
}

// -inf in the groups without a legal token of any request: 32 groups' logits of one
// request a warp at a time.
template <typename Out>
__device__ __forceinline__ void fill_inactive(const Fp8Params& p, int ew, int lane) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  constexpr int kVec = 16 / (int)sizeof(OutBits), kSteps = 1024 / (32 * kVec);
  const OutBits ninf = DTypeTraits<Out>::kNegInfBits;
  const uint32_t x = sizeof(OutBits) == 2 ? (uint32_t)ninf * 0x00010001u : (uint32_t)ninf;
  const uint4 x4 = make_uint4(x, x, x, x);
  const bool vec = (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 && p.logits_stride % kVec == 0;
  const int words = (p.nw + 31) / 32;
  const int64_t units = (int64_t)words * p.batch, step = (int64_t)gridDim.x * kEpilogueWarps;
  for (int64_t u = (int64_t)blockIdx.x * kEpilogueWarps + ew; u < units; u += step) {
    const int b = (int)(u / words), word = (int)(u - (int64_t)b * words);
    const uint32_t active = p.group_bits[word];
    if (active == 0xffffffffu) continue;
    const int v0 = word * 1024;
    OutBits* row = static_cast<OutBits*>(p.logits) + b * p.logits_stride;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int at = (k * 32 + lane) * kVec;
      if ((active >> (at >> 5)) & 1u) continue;
      if (vec && v0 + at + kVec <= p.vocab) {
        *reinterpret_cast<uint4*>(row + v0 + at) = x4;
      } else {
        for (int j = 0; j < kVec && v0 + at + j < p.vocab; ++j) row[v0 + at + j] = ninf;
      }
    }
  }
}

// One group's 32 logits of a request: masked, rounded, stored; the largest as a top-1 key.
template <typename Out>
__device__ __forceinline__ unsigned long long finish_group(const float (&y)[32], uint32_t legal, typename DTypeTraits<Out>::OutBits* out,
                                                           bool vec, int left, int64_t first_id) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  uint32_t best = 0u;  // (ordered bits: a NaN is the largest, as for the other heads)
  int at = -1;
  OutBits bits[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const OutBits r = DTypeTraits<Out>::round_bits(y[j]);
    const bool ok = (legal >> j) & 1u;
    bits[j] = ok ? r : (OutBits)DTypeTraits<Out>::kNegInfBits;
    const uint32_t o = ordered_bits(DTypeTraits<Out>::bits_to_float(r));
    if (ok && o > best) {
      best = o;
      at = j;
    }
  }
  if (out) {
    if (vec && left >= 32) {
      constexpr int kPer = 16 / (int)sizeof(OutBits);
#pragma unroll
      for (int k = 0; k < 32 / kPer; ++k) {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (sizeof(OutBits) == 2) w[q] = (uint32_t)bits[k * 8 + 2 * q] | ((uint32_t)bits[k * 8 + 2 * q + 1] << 16);
          else w[q] = bits[k * 4 + q];
        }
        reinterpret_cast<uint4*>(out)[k] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < left) out[j] = bits[j];
    }
  }
  return at < 0 ? 0ull : top1_key(from_ordered_bits(best), (uint64_t)(first_id + at));
}

template <typename Out, int kGroups>
__global__ void __launch_bounds__(kGemmThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                    const __grid_constant__ Fp8Params p, const GemmConfig c) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  constexpr int kUnits = kGroups / 2;               // groups of an epilogue warp
  constexpr int kAcc = 512 / (kGroupRows * kGroups);  // accumulators: all of TMEM
  constexpr uint32_t kAccCols = kGroupRows * kGroups;
  static_assert(kAcc <= kMaxAcc, "accumulator barriers");
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const GemmLayout<kGroups> L(c);
  unsigned char* s_w = smem;
  unsigned char* s_x = smem + L.x;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* tempty = tfull + kMaxAcc;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L.tmem);
  int* s_misc = reinterpret_cast<int*>(smem + L.misc);  // [0] abort, [1] last CTA, [2] total
  int* s_prefix = reinterpret_cast<int*>(smem + L.prefix);
  volatile int* abort_flag = s_misc;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool want_top = (p.top_value != nullptr) | (p.top_index != nullptr) | (p.top_key != nullptr);
  // quadrants of 32 hidden states that exist (with several chunks, all of them)
  const int quads = c.chunks == 1 ? (p.batch + 31) / 32 : 4;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < c.stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(tfull + a, 1);
      mbar_init(tempty + a, 2 * (uint32_t)quads);
    }
    fence_mbar_init();
    s_misc[0] = 0;
    s_misc[1] = 0;
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the prologue's outputs are there
  if (warp == 2) {
    int carry = 0;
    if (!p.dense) {
      for (int j0 = 0; j0 < c.builders; j0 += 32) {
        const int j = j0 + lane, v = j < c.builders ? p.group_counts[j] : 0;
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(FULL_MASK, incl, o);
          if (lane >= o) incl += x;
        }
        if (j < c.builders) s_prefix[j] = carry + incl - v;
        carry += __shfl_sync(FULL_MASK, incl, 31);
      }
    }
    if (lane == 0) s_misc[2] = p.dense ? p.nw : carry;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *s_tmem;
  const int total = s_misc[2];

  if (warp == 0) {
    if (lane == 0) {
      uint32_t parity = 1, issued = 0;
      int s = 0;
      Tile t;
      for (int i = 0; !*abort_flag && tile_of<kGroups>(i, total, c.chunks, t); ++i) {
        int row[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          row[g] = g < t.n ? group_at(p, s_prefix, c.builders, t.pos + g) * kGroupRows : 0;
        const uint32_t bytes = (uint32_t)t.n * kGroupBytes + (uint32_t)c.xrows * kBlock;
        for (int kb = 0; kb < p.blocks; ++kb) {
          if (!mbar_wait(empty + s, parity, abort_flag)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(full + s, bytes);
          unsigned char* w = s_w + (size_t)s * GemmLayout<kGroups>::kWBytes;
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
            if (g < t.n) tma_load_2d(w + g * kGroupBytes, &tmap_w, kb * kBlock, row[g], full + s);
          tma_load_2d(s_x + (size_t)s * c.xrows * kBlock, &tmap_x, kb * kBlock, t.chunk * kChunkRows, full + s);
          ++issued;
          if (++s == c.stages) {
            s = 0;
            parity ^= 1u;
          }
        }
      }
      if (*abort_flag) {  // every copy issued lands before the CTA ends
        for (uint32_t k = issued > (uint32_t)c.stages ? issued - c.stages : 0; k < issued; ++k)
          mbar_wait(full + (k % (uint32_t)c.stages), (k / (uint32_t)c.stages) & 1u, nullptr);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint64_t x_desc = tc_desc_sw128(s_x), w_desc = tc_desc_sw128(s_w);
      const uint32_t x_step = ((uint32_t)c.xrows * kBlock) >> 4, w_step = GemmLayout<kGroups>::kWBytes >> 4;
      uint32_t parity = 0, last_parity = 0, it = 0;
      int s = 0, last_stage = -1;
      Tile t;
      bool ok = true;
      for (int i = 0; ok && !*abort_flag && tile_of<kGroups>(i, total, c.chunks, t); ++i) {
        const uint32_t idesc = tc_idesc_e4m3((uint32_t)(t.n * kGroupRows));
        for (int kb = 0; kb < p.blocks; ++kb, ++it) {
          const uint32_t acc = it % kAcc, use = it / kAcc;
          if ((use > 0 && !mbar_wait(tempty + acc, (use - 1) & 1u, abort_flag)) || !mbar_wait(full + s, parity, abort_flag)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t xd = x_desc + (uint64_t)((uint32_t)s * x_step), wd = w_desc + (uint64_t)((uint32_t)s * w_step);
          const uint32_t d = tmem_base + acc * kAccCols;
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k) tc_mma_f8(d, xd + 2ull * k, wd + 2ull * k, idesc, k != 0);
          tc_commit(empty + s);
          tc_commit(tfull + acc);
          last_stage = s;
          last_parity = parity;
          if (++s == c.stages) {
            s = 0;
            parity ^= 1u;
          }
        }
      }
      if (last_stage >= 0) mbar_wait(empty + last_stage, last_parity, nullptr);  // all tensor-core work is done
    }
  } else {
    const int ew = warp - 2, q = warp & 3, half = ew >> 2;
    if (!p.dense && p.logits) fill_inactive<Out>(p, ew, lane);
    constexpr int kVec = 16 / (int)sizeof(OutBits);
    const bool vec = (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 && p.logits_stride % kVec == 0;
    unsigned long long best = 0ull;  // of request `best_row`
    int best_row = -1;
    const auto flush = [&]() {
      if (best != 0ull && best > *(volatile unsigned long long*)(p.keys + best_row)) atomicMax(p.keys + best_row, best);
      best = 0ull;
    };
    uint32_t it = 0;
    Tile t;
    bool ok = q < quads;
    for (int i = 0; ok && tile_of<kGroups>(i, total, c.chunks, t); ++i) {
      const int b = t.chunk * kChunkRows + q * 32 + lane;
      const bool mine = b < p.batch;
      int group[kUnits];
      uint32_t legal[kUnits];
      float2 acc[kUnits][16];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int g = 2 * u + half;
        group[u] = g < t.n ? group_at(p, s_prefix, c.builders, t.pos + g) : 0;
        legal[u] = 0u;
        if (g < t.n && mine)
          legal[u] = tail_clip(p.mask ? __ldg(p.mask + (int64_t)b * p.mask_stride + group[u]) : 0xffffffffu, group[u], p.vocab);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[u][j] = make_float2(0.f, 0.f);
      }
      // scales: the request's, four blocks ahead; the groups', a lane each for 32 blocks
      float hs[4], hs_next[4], ws[kUnits];
      const auto load_hs = [&](int kb, float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = mine && kb + j < p.blocks ? p.scales_t[(int64_t)(kb + j) * p.batch + b] : 0.f;
      };
      load_hs(0, hs_next);
      for (int kb0 = 0; ok && kb0 < p.blocks; kb0 += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) hs[j] = hs_next[j];
        load_hs(kb0 + 4, hs_next);
        if ((kb0 & 31) == 0) {
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
            ws[u] = kb0 + lane < p.blocks ? __ldg(p.weight_scales + (int64_t)(group[u] >> 2) * p.weight_scales_stride + kb0 + lane) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!ok || kb0 + j >= p.blocks) break;
          const uint32_t a = it % kAcc;
          if (!mbar_wait(tfull + a, (it / kAcc) & 1u, abort_flag)) {
            if (lane == 0) *abort_flag = 1;
            ok = false;
          }
          ok = __all_sync(FULL_MASK, ok);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t col = tmem_base + ((uint32_t)(q * 32) << 16) + a * kAccCols + (uint32_t)half * kGroupRows;
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            const float w = __shfl_sync(FULL_MASK, ws[u], (kb0 + j) & 31);
            if (2 * u + half < t.n) {
              uint32_t v[32];
              tmem_ld32(col + (uint32_t)(2 * u) * kGroupRows, v);
              tmem_ld_wait();
              const float f = hs[j] * w;
#pragma unroll
              for (int k = 0; k < 16; ++k)
                acc[u][k] = fma2(make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), make_float2(f, f), acc[u][k]);
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(tempty + a);
          ++it;
        }
      }
      if (!ok) break;
      if (want_top && mine && b != best_row) {
        flush();
        best_row = b;
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (2 * u + half >= t.n || !mine) continue;
        float y[32];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          y[2 * k] = acc[u][k].x;
          y[2 * k + 1] = acc[u][k].y;
        }
        const int v0 = group[u] * kGroupRows;
        OutBits* out = p.logits ? static_cast<OutBits*>(p.logits) + b * p.logits_stride + v0 : nullptr;
        const unsigned long long key = finish_group<Out>(y, legal[u], out, vec, p.vocab - v0, p.vocab_offset + v0);
        best = key > best ? key : best;
      }
    }
    if (want_top) flush();
  }

  tc_fence_before_sync();
  __threadfence();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
  if (*abort_flag) {
    if (tid == 0 && p.device_error) atomicExch(p.device_error, 1);
    return;
  }
  if (!want_top) return;
  if (tid == 0) s_misc[1] = atomicAdd(p.tickets, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_misc[1]) return;
  __threadfence();
  for (int b = tid; b < p.batch; b += kGemmThreads) {
    const unsigned long long key = *(volatile unsigned long long*)(p.keys + b);
    if (p.top_value) p.top_value[b] = key_value(key);
    if (p.top_index) p.top_index[b] = key_index(key);
    if (p.top_key) p.top_key[b] = key_to_signed(key);
  }
}

// ---- host side --------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// Bytes [rows, cols] in boxes of 128 bytes x box_rows, 128-byte swizzle.
bool make_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {stride};
  const cuuint32_t box[2] = {kBlock, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
cudaError_t launch_prologue_typed(const Fp8Params& p, int builders, int blocks, cudaStream_t stream) {
  constexpr int kPer = DTypeTraits<T>::kPerVec;
  const bool vec = p.raw && p.hidden_dim % kPer == 0 && (reinterpret_cast<uintptr_t>(p.raw) & 15) == 0 &&
                   (p.batch == 1 || p.raw_stride % kPer == 0);  // (the values' buffer is aligned, its rows whole vectors)
  if (vec) fp8_prologue_kernel<T, true><<<(unsigned)(builders + blocks), kPrologueThreads, 0, stream>>>(p, builders);
  else fp8_prologue_kernel<T, false><<<(unsigned)(builders + blocks), kPrologueThreads, 0, stream>>>(p, builders);
  return cudaGetLastError();
}

cudaError_t launch_prologue(const Fp8Params& p, int builders, int sms, cudaStream_t stream) {
  const int64_t work = std::max<int64_t>(p.raw ? (int64_t)p.batch * p.blocks * 32 : (int64_t)p.batch * p.blocks, p.batch);
  const int blocks = (int)std::min<int64_t>((work + kPrologueThreads - 1) / kPrologueThreads, 2 * sms);
  if (p.raw_dtype == 2) return launch_prologue_typed<float>(p, builders, blocks, stream);
  if (p.raw_dtype == 1) return launch_prologue_typed<__nv_bfloat16>(p, builders, blocks, stream);
  return launch_prologue_typed<__half>(p, builders, blocks, stream);
}

template <typename Out, int kGroups>
cudaError_t launch_gemm(const Fp8Params& p, GemmConfig c, int dev, cudaStream_t stream) {
  int optin = 0;
  if (cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess || optin <= 0)
    optin = 227 * 1024;
  c.stages = kMaxStages;
  while (c.stages > 2 && GemmLayout<kGroups>(c).total + 1024 > (uint32_t)optin) --c.stages;
  const size_t smem = GemmLayout<kGroups>(c).total + 1024;
  CUtensorMap tw, tx;
  if (!make_map(&tw, p.weight, (uint64_t)p.vocab, (uint64_t)p.hidden_dim, (uint64_t)p.weight_stride, kGroupRows) ||
      !make_map(&tx, p.hidden, (uint64_t)p.batch, (uint64_t)p.hidden_dim, (uint64_t)p.hidden_stride, (uint32_t)c.xrows))
    return cudaErrorInvalidValue;
  auto k = fp8_gemm_kernel<Out, kGroups>;
  cudaError_t err = raise_smem_limit(reinterpret_cast<const void*>(k), smem, dev);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)num_sms(dev));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, tw, tx, p, c);
}

template <typename Out>
cudaError_t launch_typed(const Fp8Params& p, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  GemmConfig c{};
  c.chunks = (p.batch + kChunkRows - 1) / kChunkRows;
  c.xrows = c.chunks > 1 ? kChunkRows : (p.batch + 7) / 8 * 8;
  c.builders = p.dense ? 0 : (p.nw + kListGroups - 1) / kListGroups;
  if ((err = launch_prologue(p, c.builders, num_sms(dev), stream)) != cudaSuccess) return err;
  return c.chunks > 1 ? launch_gemm<Out, 8>(p, c, dev, stream) : launch_gemm<Out, 4>(p, c, dev, stream);
}

}  // namespace

cudaError_t launch_fp8_tensor(const Fp8Params& p, int out_dtype, cudaStream_t stream) {
  // TMA takes 16-byte aligned bases and row pitches, and the prefix table bounds the
  // vocabulary of the block route: otherwise the row-sparse kernel computes the same.
  const bool tma = p.hidden_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0 &&
                   (p.vocab == 1 || p.weight_stride % 16 == 0) && (reinterpret_cast<uintptr_t>(p.hidden) & 15) == 0 &&
                   (p.batch == 1 || p.hidden_stride % 16 == 0);
  if (!tma || (!p.dense && p.nw > kMaxBuilders * kListGroups)) return launch_fp8_row_sparse(p, out_dtype, stream);
  if (out_dtype == 2) return launch_typed<float>(p, stream);
  if (out_dtype == 1) return launch_typed<__nv_bfloat16>(p, stream);
  return launch_typed<__half>(p, stream);
}

}  // namespace gsp
