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
//   warps 4-11  epilogue, two per TMEM lane quadrant, alternating groups.
//
// A prologue kernel quantises (or turns round the scales of) the hidden states,
// clears the top-1 keys, and in block mode lists the 32-row groups that hold a legal
// token of some request; the -inf of the other groups is stored by the epilogue warps
// before their first accumulator.
//
// Measured (device, the prologue included): 64 x 151,936 x 1,024 bf16 48 us (floor 27),
// 32 requests x 248,320 x 2,048 at 5% in runs 105 us (66), 128 x 262,144 x 8,192 384-434 us on
// one state, 495-536 in turn over several (343: power and L2), 2,048 positions x 151,936 x
// 1,024 512-534 us eagerly on one state, 558-575 over several, 565-822 recorded in graphs (by
// bytes 121, by e4m3 products 191). Rows of logits that are not whole 32-byte sectors are
// stored an element at a time: 64 x 50,257 x 1,024 49 us, 50,272 20; 1,376 x 81,758 x 256 fp16
// 1,148 us, 81,760 118.
// Copies and tensor cores alone, without the epilogue, take 30, 334 and 240 us of these:
// what bounds the kernel is the epilogue warps' time a stage, 870 clocks for 128 columns
// (TMEM loads 100, the sums 265, scales and barriers the rest), and a tile's rounding and
// stores, which no accumulator is left to hide at N = 256.
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
// Eight epilogue warps, two per TMEM lane quadrant. Sixteen, with half the groups each,
// took longer (128 x 262,144 x 8,192: 477 us against 414): what a stage costs a warp
// besides its sums is then paid twice as often.
constexpr int kEpilogueWarps = 8, kQuadWarps = kEpilogueWarps / 4;
constexpr int kGemmThreads = 32 * (4 + kEpilogueWarps);  // (two of the first four warps only take part in the barriers)
// Registers: 168 a thread at launch (384 threads); the first four warps hand theirs to the
// epilogue: 4 * 56 + 8 * 224 = 12 * 168.
constexpr int kFewRegisters = 56, kManyRegisters = 224;
constexpr int kMaxStages = 10;
constexpr int kMaxAcc = 4;
constexpr int kMaxBuilders = 256;  // prefix sums that fit the CTA's table: 2^20 tokens; past it the row-sparse kernel takes the block route

constexpr int kAhead = 2, kScaleRing = 4;  // vectors of four scales that a thread loads ahead, and keeps

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
    if (i % U::kLanes == 0) p.scales[(int64_t)row * p.scales_stride + i / U::kLanes] = s.scale;
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
        const int64_t row = at / p.blocks;
        const int kb = (int)(at - row * p.blocks);
        p.scales[row * p.scales_stride + kb] = __ldg(p.hidden_scales + row * p.hidden_scales_stride + kb);
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
  uint32_t x, bars, tmem, misc, scales, prefix, total;
  __host__ __device__ GemmLayout(const GemmConfig& c) {
    x = (uint32_t)c.stages * kWBytes;
    // (the MMA reads 128 rows of a stage's hidden states, loaded or not)
    bars = x + (uint32_t)(c.stages - 1) * (uint32_t)c.xrows * kBlock + kChunkRows * kBlock;
    tmem = bars + 8 * (2 * kMaxStages + 2 * kMaxAcc);
    misc = tmem + 16;
    scales = misc + 16;  // of the hidden states: a ring of vectors per epilogue thread
    prefix = scales + 16 * kScaleRing * 32 * kEpilogueWarps;
    total = prefix + 4 * (kMaxBuilders + 1);
  }
};

// The CTA's tiles, one after another: `n` groups from compacted position `pos` on, for
// chunk `chunk` (n 0: past the last). One chunk: an even share of the positions. Several:
// (tile, chunk) pairs, chunks first, strided by the grid.
template <int kGroups>
struct Tiles {
  int chunk, pos, n;
  int end, chunks, tile_step, chunk_step;
  __device__ __forceinline__ Tiles(int total, int chunks_) : chunks(chunks_) {
    const int G = gridDim.x, cta = blockIdx.x;
    if (chunks == 1) {
      end = (int)((int64_t)total * (cta + 1) / G);
      chunk = chunk_step = 0;
      pos = (int)((int64_t)total * cta / G);
      tile_step = kGroups;
    } else {
      end = total;
      chunk = cta % chunks;
      chunk_step = G % chunks;
      pos = cta / chunks * kGroups;
      tile_step = G / chunks * kGroups;
    }
    n = max(0, min(kGroups, end - pos));
  }
  __device__ __forceinline__ void next() {
    pos += tile_step;
    chunk += chunk_step;
    if (chunk >= chunks) {  // (one chunk: never, chunk stays 0)
      chunk -= chunks;
      pos += kGroups;
    }
    n = max(0, min(kGroups, end - pos));
  }
};

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

// A request's largest logit so far, as a thread has seen them (ids rising).
struct Best {
  float value;
  unsigned long long key;
  int row;
};

// 32 bytes, a whole sector, in one store (`at` 32-byte aligned).
__device__ __forceinline__ void store_sector(void* at, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Larger of two, NaN above all.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

// One group's 32 logits of a request: rounded, masked, stored; and the largest of
// them, whose place is sought only when it passes the largest so far.
template <typename Out>
__device__ __forceinline__ void finish_group(const unsigned long long (&sums)[16], uint32_t legal, typename DTypeTraits<Out>::OutBits* out,
                                             bool vec, int left, int64_t first_id, bool want_top, Best& best) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  float top;
  float2 acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = unpack2(sums[k]);
  if constexpr (sizeof(OutBits) == 2) {
    using Out2 = typename std::conditional<std::is_same<Out, __half>::value, __half2, __nv_bfloat162>::type;
    uint32_t w[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      Out2 two;
      if constexpr (std::is_same<Out, __half>::value) two = __floats2half2_rn(acc[k].x, acc[k].y);
      else two = __floats2bfloat162_rn(acc[k].x, acc[k].y);
      w[k] = *reinterpret_cast<const uint32_t*>(&two);
    }
    if (legal != 0xffffffffu) {
      const uint32_t ninf = DTypeTraits<Out>::kNegInfBits * 0x00010001u;
      // bits 2k and 2k + 1 to the tops of a word's halves, whose signs spread over them
      const uint32_t lo = (legal & 0xffffu) | (legal << 15), hi = (legal >> 16) | ((legal >> 1) & 0xffff8000u);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t keep = spread_half_signs((k < 8 ? lo : hi) << (15 - 2 * (k & 7)));
        w[k] = (w[k] & keep) | (ninf & ~keep);
      }
    }
    if (out) {
      if (vec && left >= 32) {
#pragma unroll
        for (int k = 0; k < 2; ++k) store_sector(out + 16 * k, &w[8 * k]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < left) out[j] = (OutBits)(w[j / 2] >> (16 * (j & 1)));
      }
    }
    if (!want_top) return;
    Out2 m[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) m[k] = *reinterpret_cast<const Out2*>(&w[k]);
#pragma unroll
    for (int h = 8; h >= 1; h >>= 1) {
#pragma unroll
      for (int k = 0; k < h; ++k) m[k] = __hmax2_nan(m[k], m[k + h]);
    }
    const float2 two = DTypeTraits<Out>::pair_to_float2(*reinterpret_cast<const uint32_t*>(&m[0]));
    top = max_nan(two.x, two.y);
    if (!(top <= best.value)) {  // larger, or NaN
      // even elements that equal it in the low half, odd ones in the high half (NaN: those unordered with themselves)
      const uint32_t top_bits = (uint32_t)DTypeTraits<Out>::round_bits(top) * 0x00010001u;
      const Out2 same = *reinterpret_cast<const Out2*>(&top_bits);
      uint32_t equal = 0u;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const Out2 x = *reinterpret_cast<const Out2*>(&w[k]);
        equal |= (top != top ? __hneu2_mask(x, x) : __heq2_mask(x, same)) & (0x00010001u << k);
      }
      const int even = __ffs(equal & 0xffffu), odd = __ffs(equal >> 16);  // (from 1; 0: none)
      const int at = min(even ? 2 * even - 2 : 32, odd ? 2 * odd - 1 : 32);
      const unsigned long long key = top1_key(top, (uint64_t)(first_id + at));
      if (key > best.key) best.key = key;
      best.value = top;
    }
  } else {
    float y[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = (legal >> j) & 1u ? (j & 1 ? acc[j / 2].y : acc[j / 2].x) : -INFINITY;
    if (out) {
      if (vec && left >= 32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) store_sector(out + 8 * k, reinterpret_cast<const uint32_t*>(&y[8 * k]));
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < left) out[j] = __float_as_uint(y[j]);
      }
    }
    if (!want_top) return;
    top = y[0];
#pragma unroll
    for (int j = 1; j < 32; ++j) top = max_nan(top, y[j]);
    if (!(top <= best.value)) {
      int at = -1;
#pragma unroll
      for (int j = 31; j >= 0; --j)
        if (y[j] == top || (y[j] != y[j] && top != top)) at = j;
      const unsigned long long key = top1_key(top, (uint64_t)(first_id + at));
      if (key > best.key) best.key = key;
      best.value = top;
    }
  }
}

template <typename Out, int kGroups>
__global__ void __launch_bounds__(kGemmThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w4,
                    const __grid_constant__ CUtensorMap tmap_x,
                    const __grid_constant__ Fp8Params p, const GemmConfig c) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  constexpr int kUnits = kGroups / kQuadWarps;      // groups of an epilogue warp
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
    tma_prefetch_desc(&tmap_w4);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < c.stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(tfull + a, 1);
      mbar_init(tempty + a, kQuadWarps * (uint32_t)quads);
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

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
  }
  if (warp == 0) {
    if (elect_one()) {
      uint32_t parity = 1, issued = 0;
      int s = 0;
      for (Tiles<kGroups> t(total, c.chunks); t.n > 0 && !*abort_flag; t.next()) {
        int row[kGroups];
        bool whole[kGroups / 4];  // four groups side by side: one copy
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          row[g] = g < t.n ? group_at(p, s_prefix, c.builders, t.pos + g) * kGroupRows : 0;
#pragma unroll
        for (int h = 0; h < kGroups / 4; ++h) whole[h] = 4 * h + 4 <= t.n && row[4 * h + 3] - row[4 * h] == 3 * kGroupRows;
        const uint32_t bytes = (uint32_t)t.n * kGroupBytes + (uint32_t)c.xrows * kBlock;
        for (int kb = 0; kb < p.blocks; ++kb) {
          if (!mbar_wait(empty + s, parity, abort_flag)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(full + s, bytes);
          unsigned char* w = s_w + (size_t)s * GemmLayout<kGroups>::kWBytes;
#pragma unroll
          for (int h = 0; h < kGroups / 4; ++h) {
            if (whole[h]) {
              tma_load_2d(w + 4 * h * kGroupBytes, &tmap_w4, kb * kBlock, row[4 * h], full + s);
            } else {
#pragma unroll
              for (int g = 4 * h; g < 4 * h + 4; ++g)
                if (g < t.n) tma_load_2d(w + g * kGroupBytes, &tmap_w, kb * kBlock, row[g], full + s);
            }
          }
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
    if (elect_one()) {
      const uint64_t x_desc = tc_desc_sw128(s_x), w_desc = tc_desc_sw128(s_w);
      const uint32_t x_step = ((uint32_t)c.xrows * kBlock) >> 4, w_step = GemmLayout<kGroups>::kWBytes >> 4;
      uint32_t parity = 0, last_parity = 0, acc = 0, acc_parity = 1;  // (a fresh `tempty` lets parity 1 pass)
      int s = 0, last_stage = -1;
      bool ok = true;
      for (Tiles<kGroups> t(total, c.chunks); ok && t.n > 0 && !*abort_flag; t.next()) {
        const uint32_t idesc = tc_idesc_e4m3((uint32_t)(t.n * kGroupRows));
        for (int kb = 0; kb < p.blocks; ++kb) {
          if (!mbar_wait(tempty + acc, acc_parity, abort_flag) || !mbar_wait(full + s, parity, abort_flag)) {
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
          if (++acc == kAcc) {
            acc = 0;
            acc_parity ^= 1u;
          }
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
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int ew = warp - 4, q = warp & 3, part = ew >> 2;
    if (!p.dense && p.logits) fill_inactive<Out>(p, ew, lane);
    constexpr int kSector = 32 / (int)sizeof(OutBits);
    const bool vec = (reinterpret_cast<uintptr_t>(p.logits) & 31) == 0 && p.logits_stride % kSector == 0;
    Best best{-INFINITY, 0ull, -1};
    const auto flush = [&]() {
      if (best.key != 0ull && best.key > *(volatile unsigned long long*)(p.keys + best.row)) atomicMax(p.keys + best.row, best.key);
    };
    const uint32_t acc_base = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)part * kGroupRows;
    uint32_t a = 0, parity = 0, slot = 0;
    bool ok = q < quads;
    Tiles<kGroups> t(total, c.chunks);
    // The next tile's groups, mask words and first scales are loaded while a tile is
    // worked on: nothing else would hide their latency.
    int group_next[kUnits];
    uint32_t legal_next[kUnits];
    float ws_next[kUnits];
    // The scales of the thread's hidden state, four stages a vector, come through shared
    // memory: registers that wait for a load cannot be passed on in a loop.
    float4* s_scale = reinterpret_cast<float4*>(smem + L.scales) + (tid - 128);
    constexpr uint32_t kSlot = 32 * kEpilogueWarps, kSlots = kScaleRing * kSlot;
    Tiles<kGroups> ahead = t;
    const float* ahead_src;
    int ahead_left;  // stages of that tile
    bool ahead_valid;
    uint32_t ahead_slot = 0;
    const auto scales_of = [&]() {
      const int row = ahead.chunk * kChunkRows + q * 32 + lane;
      ahead_valid = ahead.n > 0 && row < p.batch;
      ahead_src = p.scales + (ahead_valid ? (int64_t)row * p.scales_stride : 0);
      ahead_left = p.blocks;
    };
    scales_of();
    const auto load_scales = [&]() {
      cp_async16(s_scale + ahead_slot, ahead_src, ahead_valid);
      cp_async_commit();
      ahead_slot = (ahead_slot + kSlot) & (kSlots - 1);
      ahead_src += 4;
      if ((ahead_left -= 4) <= 0) {
        ahead.next();
        scales_of();
      }
    };
    const auto load_ws = [&](int group, int kb) {
      return kb + lane < p.blocks ? __ldg(p.weight_scales + (int64_t)(group >> 2) * p.weight_scales_stride + kb + lane) : 0.f;
    };
    const auto load_tile = [&]() {  // of t; its hidden states' scales come with load_scales
      const int row = t.chunk * kChunkRows + q * 32 + lane;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int g = kQuadWarps * u + part;
        group_next[u] = g < t.n ? group_at(p, s_prefix, c.builders, t.pos + g) : 0;
        legal_next[u] = 0u;
        if (g < t.n && row < p.batch)
          legal_next[u] = p.mask ? __ldg(p.mask + (int64_t)row * p.mask_stride + group_next[u]) : 0xffffffffu;
        ws_next[u] = load_ws(group_next[u], 0);
      }
    };
    if (ok) {
      load_tile();
      for (int j = 0; j < kAhead; ++j) load_scales();
    }
    while (ok && t.n > 0) {
      const int b = t.chunk * kChunkRows + q * 32 + lane;
      const bool mine = b < p.batch;
      const int mine_n = (t.n - part + kQuadWarps - 1) / kQuadWarps;  // groups part, part + 2, ...
      int group[kUnits];
      uint32_t legal[kUnits];
      unsigned long long acc[kUnits][16];  // pairs of fp32 sums
      float ws[kUnits], ws_later[kUnits];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        group[u] = group_next[u];
        legal[u] = tail_clip(legal_next[u], group[u], p.vocab);
        ws[u] = ws_next[u];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[u][j] = 0ull;
      }
      t.next();
      load_tile();
#pragma unroll 1
      for (int kb = 0; kb < p.blocks; ++kb) {
        if ((kb & 3) == 0) {
          if (kb != 0) slot = (slot + kSlot) & (kSlots - 1);
          load_scales();
          cp_async_wait<kAhead>();
          if ((kb & 31) == 0) {  // the groups' scales: a lane each for 32 stages, the next 32 under way
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
              if (kb != 0) ws[u] = ws_later[u];
              ws_later[u] = load_ws(group[u], kb + 32);
            }
          }
        }
        const float h = reinterpret_cast<const float*>(s_scale + slot)[kb & 3];
        unsigned long long ff[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const uint32_t f = __float_as_uint(h * __shfl_sync(FULL_MASK, ws[u], kb & 31));
          ff[u] = pack2(f, f);
        }
        if (!mbar_wait(tfull + a, parity, abort_flag)) *abort_flag = 1;  // (seen below)
        tc_fence_after_sync();
        __syncwarp();
        const uint32_t col = acc_base + a * kAccCols;
        // (all of the warp's groups, whether the tile has them: their sums are not used)
#pragma unroll
        for (int u = 0; u < kUnits; u += 2) {
          uint32_t v[2][32];
          tmem_ld_2x32(col + (uint32_t)(kQuadWarps * u) * kGroupRows, col + (uint32_t)(kQuadWarps * (u + 1)) * kGroupRows,
                       v[0], v[1]);
          if (u + 2 >= kUnits) {  // all read: the accumulator is free
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty + a);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[u + e][k] = fma2(pack2(v[e][2 * k], v[e][2 * k + 1]), ff[u + e], acc[u + e][k]);
          }
        }
        if (++a == kAcc) {
          a = 0;
          parity ^= 1u;
        }
      }
      slot = (slot + kSlot) & (kSlots - 1);
      ok = !__any_sync(FULL_MASK, *abort_flag != 0);
      if (!ok) break;
      if (want_top && mine && b != best.row) {
        flush();
        best = Best{-INFINITY, 0ull, b};
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (u >= mine_n || !mine) continue;
        const int v0 = group[u] * kGroupRows;
        OutBits* out = p.logits ? static_cast<OutBits*>(p.logits) + b * p.logits_stride + v0 : nullptr;
        finish_group<Out>(acc[u], legal[u], out, vec, p.vocab - v0, p.vocab_offset + v0, want_top, best);
      }
    }
    if (want_top) flush();
    cp_async_wait<0>();
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
  CUtensorMap tw, tw4, tx;
  if (!make_map(&tw, p.weight, (uint64_t)p.vocab, (uint64_t)p.hidden_dim, (uint64_t)p.weight_stride, kGroupRows) ||
      !make_map(&tw4, p.weight, (uint64_t)p.vocab, (uint64_t)p.hidden_dim, (uint64_t)p.weight_stride, 4 * kGroupRows) ||
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
  return cudaLaunchKernelEx(&cfg, k, tw, tw4, tx, p, c);
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
