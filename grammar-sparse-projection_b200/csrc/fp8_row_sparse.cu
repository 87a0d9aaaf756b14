// The fp8 head's row-sparse route (sm_100a): only the legal rows of the weight are
// read.
//
//   y[b, v] = sum_kb ws[v / 128, kb] sum_{k in block kb} (hs[b, kb] q[b, k]) w[v, k]
//
// A request has `parts` CTAs (one or two SMs' worth over the batch). Each ranks the request's
// whole mask (one pass over its words, a prefix over the threads), takes an even share
// of the legal rows by rank, and streams them: a warp holds four rows, 16 bytes of each
// a lane, converts them to fp32 and multiplies with the hidden state, which lies in
// shared memory as hs q in fp32 (one rounding more than the product of integers has).
// A 16-byte vector lies in one block of 128 columns, so its sum is scaled once. -inf
// goes to the illegal tokens of an even share of the words. Bound by the legal rows'
// bytes where they are many, by latency (mask, list, rows, one after another) where
// they are few.
//
// Measured (device): one request, 248,320 x 2,048 fp16 at 1% 12-13 us (floor 0.9: launch of
// the clearing kernel, mask, prefix, list, rows, merge), 32 requests at 1% 57 us (24), one
// request at 20% 45 us (16).
//
// Hidden states that are not quantised yet are quantised here, each CTA its request's.
// The request's top-1 merges in scratch keys; its last CTA stores it.
#include <algorithm>

#include "fp8_head.cuh"

namespace gsp {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kListRows = 2048;  // legal rows listed at a time
constexpr int kRows = 4;         // rows a warp has under way

__global__ void __launch_bounds__(256) clear_keys_kernel(unsigned long long* keys, unsigned int* tickets, int batch) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int b = blockIdx.x * 256 + threadIdx.x; b < batch; b += gridDim.x * 256) {
    keys[b] = 0ull;
    tickets[b] = 0u;
  }
}

__device__ __forceinline__ float2 e4m3_pair(uint32_t two) {  // low 16 bits
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(__half2(h));
}

// The hidden state as fp32 (hs q), element k of 16-byte vector v at [k / 4][v] (kVec) or in order.
template <bool kVec>
__device__ __forceinline__ void put_state(float* s_x, int nvec, int k, float y) {
  if constexpr (kVec) s_x[((((k & 15) >> 2) * nvec) + (k >> 4)) * 4 + (k & 3)] = y;
  else s_x[k] = y;
}

template <typename T, bool kVec>
__device__ __forceinline__ void quantize_state(const Fp8Params& p, int b, int nvec, float* s_x) {
  using U = Units<T, false>;  // four elements 32 apart: a warp takes a block
  const auto* row = static_cast<const typename U::Bits*>(p.raw) + b * p.raw_stride;
  const int lane = threadIdx.x & 31;
  for (int kb = threadIdx.x >> 5; kb < p.blocks; kb += kWarps) {
    float f[4];
    U::load(row, kb * 32 + lane, p.hidden_dim, f);
    const BlockScale s = block_scale(lanes_max<32>(U::magnitude(f)));
    const uint32_t w = to_e4m3(f[0], f[1], f[2], f[3], s);
    const float2 lo = e4m3_pair(w & 0xffffu), hi = e4m3_pair(w >> 16);
    const float y[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = kb * kBlock + lane + 32 * j;
      if (k < p.hidden_dim) put_state<kVec>(s_x, nvec, k, y[j] * s.scale);
    }
  }
}

template <bool kVec>
__device__ __forceinline__ void load_state(const Fp8Params& p, int b, int nvec, float* s_x) {
  if (p.raw) {
    if (p.raw_dtype == 2) quantize_state<float, kVec>(p, b, nvec, s_x);
    else if (p.raw_dtype == 1) quantize_state<__nv_bfloat16, kVec>(p, b, nvec, s_x);
    else quantize_state<__half, kVec>(p, b, nvec, s_x);
    return;
  }
  const uint8_t* row = p.hidden + b * p.hidden_stride;
  const float* scales = p.hidden_scales + b * p.hidden_scales_stride;
  for (int k = threadIdx.x; k < p.hidden_dim; k += kThreads)
    put_state<kVec>(s_x, nvec, k, e4m3_pair(__ldg(row + k)).x * __ldg(scales + k / kBlock));
}

// Sum of 16 products: a weight vector with x[0..3] of the state.
__device__ __forceinline__ float dot16(const uint4& w, const float4 (&x)[4]) {
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 lo = e4m3_pair(word[k] & 0xffffu), hi = e4m3_pair(word[k] >> 16);
    a = fmaf(lo.x, x[k].x, a);
    b = fmaf(lo.y, x[k].y, b);
    a = fmaf(hi.x, x[k].z, a);
    b = fmaf(hi.y, x[k].w, b);
  }
  return a + b;
}

template <typename Out, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) fp8_row_sparse_kernel(const __grid_constant__ Fp8Params p, int parts) {
  using OutBits = typename DTypeTraits<Out>::OutBits;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_warp[kWarps], s_list[kListRows];
  __shared__ unsigned long long s_best;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / parts, part = blockIdx.x - b * parts;
  const int nw = p.nw, nvec = p.hidden_dim / 16;
  const uint32_t* mask = p.mask ? p.mask + (int64_t)b * p.mask_stride : nullptr;
  const bool want_top = (p.top_value != nullptr) | (p.top_index != nullptr) | (p.top_key != nullptr);
  float* s_x = reinterpret_cast<float*>(smem);
  const auto word_at = [&](int w) { return tail_clip(mask ? __ldg(mask + w) : 0xffffffffu, w, p.vocab); };

  // ranks: thread t has the words [w0, w1), whole 16-byte vectors of them
  const int per = (nw + 4 * kThreads - 1) / (4 * kThreads) * 4, w0 = min(nw, tid * per), w1 = min(nw, w0 + per);
  int count = 0, w = w0;
  if (mask && (reinterpret_cast<uintptr_t>(mask) & 15) == 0) {
#pragma unroll 4
    for (; w + 4 <= w1; w += 4) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(mask + w));
      count += __popc(tail_clip(q.x, w, p.vocab)) + __popc(tail_clip(q.y, w + 1, p.vocab)) +
               __popc(tail_clip(q.z, w + 2, p.vocab)) + __popc(tail_clip(q.w, w + 3, p.vocab));
    }
  }
  for (; w < w1; ++w) count += __popc(word_at(w));
  int incl = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(FULL_MASK, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (tid == 0) s_best = 0ull;
  load_state<kVec>(p, b, nvec, s_x);
  __syncthreads();
  int before = incl - count, total = 0;
  for (int k = 0; k < kWarps; ++k) {
    if (k < warp) before += s_warp[k];
    total += s_warp[k];
  }
  const int lo = (int)((int64_t)total * part / parts), hi = (int)((int64_t)total * (part + 1) / parts);
  OutBits* logits = p.logits ? static_cast<OutBits*>(p.logits) + b * p.logits_stride : nullptr;

  if (logits) {  // -inf: eight (fp32: four) tokens a lane
    constexpr int kPer = 16 / (int)sizeof(OutBits), kLanes = 32 / kPer;  // lanes of a word
    const OutBits ninf = DTypeTraits<Out>::kNegInfBits;
    const uint32_t x = sizeof(OutBits) == 2 ? (uint32_t)ninf * 0x00010001u : (uint32_t)ninf;
    const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    const int f0 = (int)((int64_t)nw * part / parts), f1 = (int)((int64_t)nw * (part + 1) / parts);
    for (int64_t u = (int64_t)f0 * kLanes + tid; u < (int64_t)f1 * kLanes; u += kThreads) {
      const int w = (int)(u / kLanes), v = w * 32 + (int)(u % kLanes) * kPer;
      const uint32_t bits = (word_at(w) >> (v & 31)) & ((1u << kPer) - 1u);
      if (vec && bits == 0u && v + kPer <= p.vocab) {
        *reinterpret_cast<uint4*>(logits + v) = make_uint4(x, x, x, x);
      } else {
        for (int j = 0; j < kPer && v + j < p.vocab; ++j)
          if (!((bits >> j) & 1u)) logits[v + j] = ninf;
      }
    }
  }

  unsigned long long best = 0ull;
  for (int r0 = lo; r0 < hi; r0 += kListRows) {
    const int r1 = min(hi, r0 + kListRows);
    if (before < r1 && before + count > r0) {
      int rank = before;
      for (int w = w0; w < w1 && rank < r1; ++w) {
        uint32_t bits = word_at(w);
        const int n = __popc(bits);
        if (rank + n > r0) {
          for (int k = rank; bits; ++k, bits &= bits - 1u)
            if (k >= r0 && k < r1) s_list[k - r0] = w * 32 + __ffs(bits) - 1;
        }
        rank += n;
      }
    }
    __syncthreads();
    const int n = r1 - r0;
    // (few rows: one or two a warp, so that all warps have some)
    const int share = min(kRows, (n + kWarps - 1) / kWarps);
    for (int i = warp * share; i < n; i += kWarps * share) {
      const int live = min(share, n - i);
      int row[kRows];
      const uint8_t* w[kRows];
      const float* ws[kRows];
      float acc[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        row[r] = s_list[min(i + r, n - 1)];  // (past `live`: not read)
        w[r] = p.weight + (int64_t)row[r] * p.weight_stride;
        ws[r] = p.weight_scales + (int64_t)(row[r] >> 7) * p.weight_scales_stride;
        acc[r] = 0.f;
      }
      if constexpr (kVec) {
        const float4* x4 = reinterpret_cast<const float4*>(s_x);
        for (int v0 = 0; v0 < nvec; v0 += 64) {  // two vectors of each row under way
          uint4 q[2][kRows];
          float scale[2][kRows];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int v = v0 + 32 * h + lane;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
              q[h][r] = v < nvec && r < live ? ld_stream_v4(reinterpret_cast<const uint4*>(w[r]) + v) : make_uint4(0u, 0u, 0u, 0u);
              scale[h][r] = v < nvec && r < live ? __ldg(ws[r] + (v >> 3)) : 0.f;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int v = v0 + 32 * h + lane;
            if (v >= nvec) continue;
            const float4 x[4] = {x4[v], x4[nvec + v], x4[2 * nvec + v], x4[3 * nvec + v]};
#pragma unroll
            for (int r = 0; r < kRows; ++r)
              if (r < live) acc[r] = fmaf(dot16(q[h][r], x), scale[h][r], acc[r]);
          }
        }
      } else {
        for (int kb = 0; kb < p.blocks; ++kb) {
          uint32_t q[4][kRows];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = kb * kBlock + lane + 32 * j;
#pragma unroll
            for (int r = 0; r < kRows; ++r) q[j][r] = k < p.hidden_dim && r < live ? (uint32_t)__ldg(w[r] + k) : 0u;
          }
          float x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = kb * kBlock + lane + 32 * j;
            x[j] = k < p.hidden_dim ? s_x[k] : 0.f;
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum = fmaf(e4m3_pair(q[j][r]).x, x[j], sum);
            acc[r] = fmaf(sum, __ldg(ws[r] + kb), acc[r]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) acc[r] = warp_sum(acc[r]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (lane != r || r >= live) continue;
        const OutBits bits = DTypeTraits<Out>::round_bits(acc[r]);
        if (logits) logits[row[r]] = bits;
        const float value = DTypeTraits<Out>::bits_to_float(bits);
        if (value == -INFINITY) continue;  // (rounded to what illegal tokens have: no key, as on the other routes)
        const unsigned long long key = top1_key(value, (uint64_t)(p.vocab_offset + row[r]));
        best = key > best ? key : best;
      }
    }
    __syncthreads();
  }
  if (!want_top) return;
  best = warp_max_u64(best);
  if (lane == 0 && best != 0ull) atomicMax(&s_best, best);
  __syncthreads();
  if (tid != 0) return;
  unsigned long long key = s_best;
  if (parts > 1) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the keys are cleared
    if (key != 0ull) atomicMax(p.keys + b, key);
    __threadfence();
    if (atomicAdd(p.tickets + b, 1u) != (unsigned)parts - 1u) return;
    __threadfence();
    key = *(volatile unsigned long long*)(p.keys + b);
  }
  if (p.top_value) p.top_value[b] = key_value(key);
  if (p.top_index) p.top_index[b] = key_index(key);
  if (p.top_key) p.top_key[b] = key_to_signed(key);
}

template <typename Out, bool kVec>
cudaError_t launch(const Fp8Params& p, cudaStream_t stream) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const int sms = num_sms(dev);
  // CTAs of a request, at least 64 mask words each: one per SM over a batch of up to 8,
  // whose time is that of ranking the masks (8 x 248,320 x 2,048 at 1%: 23.6 us, two per SM
  // 25.4), two per SM over a larger one (32: 59.7 and 57.4 us)
  int parts = std::max(1, (p.batch <= 8 ? 1 : 2) * sms / p.batch);
  parts = std::min(parts, std::max(1, p.nw / 64));
  if ((int64_t)p.batch * parts > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const bool keys = parts > 1 && (p.top_value || p.top_index || p.top_key);
  if (keys) {
    clear_keys_kernel<<<(unsigned)std::min(64, (p.batch + 255) / 256), 256, 0, stream>>>(p.keys, p.tickets, p.batch);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
  }
  auto k = fp8_row_sparse_kernel<Out, kVec>;
  const size_t smem = ((size_t)p.hidden_dim * sizeof(float) + 15) / 16 * 16;
  if ((err = raise_smem_limit(reinterpret_cast<const void*>(k), smem, dev)) != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.batch * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = keys ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, p, parts);
}

template <typename Out>
cudaError_t launch_typed(const Fp8Params& p, cudaStream_t stream) {
  const bool vec = p.hidden_dim % 16 == 0 && (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0 &&
                   (p.vocab == 1 || p.weight_stride % 16 == 0);
  return vec ? launch<Out, true>(p, stream) : launch<Out, false>(p, stream);
}

}  // namespace

cudaError_t launch_fp8_row_sparse(const Fp8Params& p, int out_dtype, cudaStream_t stream) {
  if (out_dtype == 2) return launch_typed<float>(p, stream);
  if (out_dtype == 1) return launch_typed<__nv_bfloat16>(p, stream);
  return launch_typed<__half>(p, stream);
}

}  // namespace gsp
