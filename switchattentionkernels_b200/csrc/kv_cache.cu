// Block-scaled 8-bit KV cache: writing new rows (append) and keeping the heaviest
// rows (evict).  The attention over the cache is in kv_decode_sm100.cu.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "kv_cache.h"
#include "mma_sync.cuh"
#include "sm100.cuh"

namespace swa {

namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------
// 8-bit formats
// ---------------------------------------------------------------------------
// Smallest power of two s (2^-126 .. 2^127) with s * qmax >= a, for qmax = (1 +
// mant_q / 2^23) 2^exp_q; 0 when a = 0.  Powers of two because then x / s, and the
// rescaling of a row when its block's scale grows, are exact before the one
// rounding to 8 bits: e4m3 loses nothing by it, int8 less than one bit, and rows
// rounded again at every growth (at most once per doubling) do not drift.
__device__ __forceinline__ float pow2_at_least(float a, int exp_q, uint32_t mant_q) {
  const uint32_t bits = __float_as_uint(a);
  if (bits == 0u) return 0.0f;
  const int e = static_cast<int>(bits >> 23) - 127 - exp_q + ((bits & 0x7FFFFFu) > mant_q ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23);
}

template <bool kInt8>
__device__ __forceinline__ float scale_for(float amax) {
  return kInt8 ? pow2_at_least(amax, 6, 0x7E0000u) : pow2_at_least(amax, 8, 0x600000u);  // 127, 448
}

// Four values to 8 bits (byte i = value i): to nearest even, saturating at 127 / 448;
// NaN becomes 0 (int8) or stays NaN (e4m3).
template <bool kInt8>
__device__ __forceinline__ uint32_t pack8(float a, float b, float c, float d) {
  if constexpr (kInt8) {
    auto q = [](float x) { return static_cast<uint32_t>(min(max(__float2int_rn(x), -127), 127)) & 0xFFu; };
    return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
  } else {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  }
}

// Four cached bytes times `ratio`, rounded back to 8 bits.
template <bool kInt8>
__device__ __forceinline__ uint32_t rescale8(uint32_t v, float ratio) {
  if constexpr (kInt8) {
    // a byte (offset by 128) as the low byte of 2^23 makes the float 2^23 + 128 + value, and the sum with
    // 1.5 * 2^23 rounds the product to a whole number in its low byte: no conversion instructions,
    // which run at a quarter of the rate (an eviction that rescales most rows: 28.8 -> 24.2 us)
    const uint32_t u = v ^ 0x80808080u;
    auto x = [u, ratio](uint32_t sel) {
      const float f = __uint_as_float(__byte_perm(u, 0x4B000000u, sel)) - 8388736.0f;
      return __float_as_uint(fmaf(fmaxf(f, -127.0f), ratio, 12582912.0f));
    };
    return __byte_perm(__byte_perm(x(0x7440), x(0x7441), 0x0040), __byte_perm(x(0x7442), x(0x7443), 0x0040), 0x5410);
  } else {
    uint32_t lo, hi;
    e4m3x4_to_f16x2x2(v, lo, hi);
    const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack8<false>(l.x * ratio, l.y * ratio, h.x * ratio, h.y * ratio);
  }
}

template <bool kInt8>
__device__ __forceinline__ uint4 rescale8(uint4 v, float ratio) {
  return make_uint4(rescale8<kInt8>(v.x, ratio), rescale8<kInt8>(v.y, ratio), rescale8<kInt8>(v.z, ratio),
                    rescale8<kInt8>(v.w, ratio));
}

// Largest |x| over the finite values of packed BF16 pairs, as the BF16's bits (the
// bits of non-negative BF16 values order as the values do).
__device__ __forceinline__ uint32_t finite_abs_max(uint32_t pair) {
  uint32_t lo = pair & 0x7FFFu, hi = (pair >> 16) & 0x7FFFu;
  lo = lo < 0x7F80u ? lo : 0u;
  hi = hi < 0x7F80u ? hi : 0u;
  return max(lo, hi);
}

// The same over N x 8 values, two at a time in packed 16-bit maxima; the values are
// looked at one by one only where an infinity or NaN is among them (`finite` false).
template <int N>
__device__ __forceinline__ uint32_t abs_max_bits(const uint4* v, bool& finite) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m = __vmaxu2(m, v[i].x & 0x7FFF7FFFu);
    m = __vmaxu2(m, v[i].y & 0x7FFF7FFFu);
    m = __vmaxu2(m, v[i].z & 0x7FFF7FFFu);
    m = __vmaxu2(m, v[i].w & 0x7FFF7FFFu);
  }
  m = max(m & 0xFFFFu, m >> 16);
  finite = m < 0x7F80u;
  if (!finite) {
    m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      m = max(max(m, max(finite_abs_max(v[i].x), finite_abs_max(v[i].y))), max(finite_abs_max(v[i].z), finite_abs_max(v[i].w)));
  }
  return m;
}

__device__ __forceinline__ float bf_lo(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf_hi(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }

// Eight BF16 values times `inv` (a power of two that brings finite ones within 127 /
// 448) to 8 bits.  The append is bound by instructions before it is by HBM, so:
//   e4m3: the product in packed BF16, which is exact (a result too small for BF16's
//   normal range is far below half of e4m3's smallest step);
//   int8: x inv + 1.5 * 2^23 in one FMA, whose low byte is x inv rounded to nearest even
//   (the sum's unit in the last place is 1); infinities and NaN go the long way.
template <bool kInt8>
__device__ __forceinline__ uint2 quantize8(uint4 v, float inv, bool finite) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
  if constexpr (kInt8) {
    if (finite) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        constexpr float kMagic = 12582912.0f;
        const uint32_t a = __float_as_uint(fmaf(bf_lo(w[2 * h]), inv, kMagic)), b = __float_as_uint(fmaf(bf_hi(w[2 * h]), inv, kMagic));
        const uint32_t c = __float_as_uint(fmaf(bf_lo(w[2 * h + 1]), inv, kMagic)), d = __float_as_uint(fmaf(bf_hi(w[2 * h + 1]), inv, kMagic));
        o[h] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[h] = pack8<true>(bf_lo(w[2 * h]) * inv, bf_hi(w[2 * h]) * inv, bf_lo(w[2 * h + 1]) * inv, bf_hi(w[2 * h + 1]) * inv);
    }
  } else {
    const __nv_bfloat162 f = __float2bfloat162_rn(inv);
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), f);
      y[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) o[h] = pack8<false>(bf_lo(y[2 * h]), bf_hi(y[2 * h]), bf_lo(y[2 * h + 1]), bf_hi(y[2 * h + 1]));
  }
  return make_uint2(o[0], o[1]);
}

struct RowRange {
  int start, end;
};
__device__ __forceinline__ RowRange append_range(const KvAppendParams& p, int b) {
  const int s = min(max(p.start[b], 0), p.Smax);
  const int n = p.new_lens != nullptr ? min(max(p.new_lens[b], 0), p.T) : p.T;
  return RowRange{s, min(n, p.Smax - s) + s};
}

// New scale of a block whose new rows reach `amax_bits`: the scale that its earlier
// rows need (none: 0), raised to what the new rows need.
template <bool kInt8>
__device__ __forceinline__ float grown_scale(uint32_t amax_bits, bool has_old, float old_scale) {
  const float need = scale_for<kInt8>(__uint_as_float(amax_bits << 16));
  return has_old ? fmaxf(pow2_at_least(old_scale, 0, 0u), need) : need;
}

// What a block's values are multiplied by (a power of two: exact).  A block with the scale 0 holds
// zeros, infinities and NaN.  e4m3: they are rounded as they are, so that infinities saturate
// (their value, 448 times the scale, is 0) and only NaN becomes NaN; infinity times 0 would be one
// too.  int8: times 0, where all of them become 0.
template <bool kInt8>
__device__ __forceinline__ float inverse_scale(float s) {
  return s > 0.0f ? 1.0f / s : (kInt8 ? 0.0f : 1.0f);
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
constexpr int kAppendRows = 128;  // rows that a CTA appends: one block or several

// Chunks of many rows: one CTA per (128 rows, KV head, K or V, sequence), whole blocks.  Each
// thread keeps its part of the new rows in registers (16 bytes a pass of 16 rows), so the
// rows are read once: maxima of the blocks, scales, rounding, store.  HBM-bound: 2 bytes read
// and 1 written per value (4 x 16384 rows of 8 heads: 60 us for 61 us of copying with blocks of
// 64 or 128, 63 with 32, 74 with 16 (int8 84), whose maxima cross the warps eight times a CTA;
// CTAs of 64 rows took 61, 67 and 76 us, CTAs of a single block 80 with 32 and 121 with 16).
constexpr int kAppendThreads = 256;

template <bool kInt8, int kBlock>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ KvAppendParams p) {
  constexpr int kRows = kAppendRows;
  constexpr int kPasses = kRows / 16;
  constexpr int kBlocks = kRows / kBlock;
  constexpr int kPer = kPasses / kBlocks;  // passes of a block
  constexpr int kWarps = kAppendThreads / 32;
  const int b = blockIdx.z, g = blockIdx.y >> 1, kv = blockIdx.y & 1;
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const RowRange rg = append_range(p, b);
  const int tid = threadIdx.x;
  if (!p.lens_after && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) p.seq_lens[b] = rg.end;
  const int row0 = (rg.start / kRows + static_cast<int>(blockIdx.x)) * kRows;
  if (rg.end <= rg.start || row0 >= rg.end) return;
  const int c = tid & 15;  // 8 values of a row
  const int64_t unit = static_cast<int64_t>(b) * p.Hkv + g;
  const __nv_bfloat16* x = p.x[kv] + b * p.sb[kv] + g * p.sh[kv] + 8 * c;
  uint8_t* cache = p.cache[kv] + unit * p.Smax * 128;
  float* scale = p.scale[kv] + unit * p.nblk + row0 / kBlock;
  uint4 v[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int pos = row0 + 16 * i + (tid >> 4);
    v[i] = make_uint4(0, 0, 0, 0);
    if (pos >= rg.start && pos < rg.end)
      v[i] = *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(pos - rg.start) * p.st[kv]);
  }
  // only the block of the first new row can hold earlier rows, whose scale counts
  const int past = max(0, rg.start - row0);
  const int old_block = past / kBlock;
  const bool any_old = past % kBlock != 0;
  const float old_scale = any_old ? scale[old_block] : 0.0f;
  __shared__ uint32_t warp_max[kBlocks][kWarps];
  bool finite[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const uint32_t amax = __reduce_max_sync(0xffffffffu, abs_max_bits<kPer>(v + j * kPer, finite[j]));
    if ((tid & 31) == 0) warp_max[j][tid >> 5] = amax;
  }
  __syncthreads();  // (also: every thread has the old scale before it is overwritten)
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int block0 = row0 + j * kBlock;
    if (block0 >= rg.end || block0 + kBlock <= rg.start) continue;  // no new row
    const uint32_t amax = __reduce_max_sync(0xffffffffu, warp_max[j][tid & (kWarps - 1)]);
    const bool has_old = any_old && j == old_block;
    const float s = grown_scale<kInt8>(amax, has_old, old_scale);
    const float inv = inverse_scale<kInt8>(s);
    if (has_old && s != old_scale) {
      const float ratio = old_scale / s;
      for (int i = tid; i < (rg.start - block0) * 8; i += kAppendThreads) {
        uint4* q = reinterpret_cast<uint4*>(cache + static_cast<int64_t>(block0) * 128) + i;
        *q = rescale8<kInt8>(*q, ratio);
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int pos = block0 + 16 * i + (tid >> 4);
      if (pos < rg.start || pos >= rg.end) continue;
      *reinterpret_cast<uint2*>(cache + static_cast<int64_t>(pos) * 128 + 8 * c) =
          quantize8<kInt8>(v[j * kPer + i], inv, finite[j]);
    }
    if (tid == 0) scale[j] = s;
  }
  if (kv == 0 && p.weights != nullptr && tid < kRows) {
    const int pos = row0 + tid;
    if (pos >= rg.start && pos < rg.end) p.weights[unit * p.Smax + pos] = 0.0f;
  }
}

__global__ void kv_advance_kernel(const __grid_constant__ KvAppendParams p) {
  cudaGridDependencySynchronize();  // the append has read the old lengths
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < p.B) p.seq_lens[b] = append_range(p, b).end;
}

// One new row per sequence: a CTA per sequence, a warp per (KV head, K or V), 4
// values per lane.  Latency-bound (a few KB in all); the CTA is the only one that
// reads its sequence's length, so it also writes the new one and the call is one
// launch.
template <bool kInt8>
__global__ void __launch_bounds__(1024) kv_append_token_kernel(const __grid_constant__ KvAppendParams p) {
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  cudaGridDependencySynchronize();
  const RowRange rg = append_range(p, b);
  if (rg.end > rg.start) {
    const int blk = rg.start / p.block, row0 = blk * p.block;
    for (int u = threadIdx.x >> 5; u < 2 * p.Hkv; u += blockDim.x >> 5) {
      const int g = u >> 1, kv = u & 1;
      const int64_t unit = static_cast<int64_t>(b) * p.Hkv + g;
      uint8_t* cache = p.cache[kv] + unit * p.Smax * 128;
      float* scale = p.scale[kv] + unit * p.nblk + blk;
      const uint2 v = *reinterpret_cast<const uint2*>(p.x[kv] + b * p.sb[kv] + g * p.sh[kv] + 4 * lane);
      const float old_scale = *scale;
      const uint32_t amax = __reduce_max_sync(0xffffffffu, max(finite_abs_max(v.x), finite_abs_max(v.y)));
      const bool has_old = rg.start > row0;
      const float s = grown_scale<kInt8>(amax, has_old, old_scale);
      const float inv = inverse_scale<kInt8>(s);
      if (has_old && s != old_scale) {
        const float ratio = old_scale / s;
        for (int i = lane; i < (rg.start - row0) * 8; i += 32) {
          uint4* q = reinterpret_cast<uint4*>(cache + static_cast<int64_t>(row0) * 128) + i;
          *q = rescale8<kInt8>(*q, ratio);
        }
      }
      reinterpret_cast<uint32_t*>(cache + static_cast<int64_t>(rg.start) * 128)[lane] =
          pack8<kInt8>(bf_lo(v.x) * inv, bf_hi(v.x) * inv, bf_lo(v.y) * inv, bf_hi(v.y) * inv);
      __syncwarp();
      if (lane == 0) {
        *scale = s;
        if (kv == 0 && p.weights != nullptr) p.weights[unit * p.Smax + rg.start] = 0.0f;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) p.seq_lens[b] = rg.end;
}

template <bool kInt8>
cudaError_t append_rows(const KvAppendParams& p, cudaStream_t stream) {
  void (*kernel)(KvAppendParams) = p.block == 16   ? kv_append_kernel<kInt8, 16>
                                   : p.block == 32 ? kv_append_kernel<kInt8, 32>
                                   : p.block == 64 ? kv_append_kernel<kInt8, 64>
                                                   : kv_append_kernel<kInt8, 128>;
  const dim3 grid((p.T - 1) / kAppendRows + 2, 2 * p.Hkv, p.B);
  cudaError_t e = launch_dependent(kernel, grid, dim3(kAppendThreads), 0, stream, p);
  if (e != cudaSuccess || !p.lens_after) return e;
  return launch_dependent(kv_advance_kernel, dim3((p.B + 127) / 128), dim3(128), 0, stream, p);
}

// ---------------------------------------------------------------------------
// evict: selection
// ---------------------------------------------------------------------------
// A cluster of 1 to 8 CTAs per (sequence, KV head), each CTA a contiguous part of the
// rows and each warp a contiguous part of that.  The k-th largest weight of the
// rows between the sink and the recent ones comes from a radix selection (digits
// of 11, 11 and 10 bits of the order-preserving integer form; the CTAs' histograms
// are added up through distributed shared memory), then the kept rows of each warp are
// counted and written in order, rows equal to the threshold from the lowest index on.
// Latency-bound (a chain of a dozen barriers over little data), so the weights are
// read once and stay in registers, kPerThread of them a thread; with kPerThread = 0
// (more rows than 8 CTAs can hold) every pass reads them again, from L2.
constexpr int kSelMaxCluster = 8;
constexpr int kSelBins = 2048;

// Order-preserving integer form of a weight; NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_bits(float w) {
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u ^ ((u >> 31) != 0u ? 0xFFFFFFFFu : 0x80000000u);
}

template <int kSelThreads, int kPerThread>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const __grid_constant__ KvEvictParams p) {
  constexpr int kSelWarps = kSelThreads / 32;
  constexpr int kPer = kSelBins / kSelThreads;  // bins of a thread
  __shared__ uint32_t hist[3][kSelBins];
  __shared__ uint32_t warp_sum[kSelWarps];
  __shared__ uint32_t found[2];
  __shared__ uint32_t warp_gt[kSelWarps], warp_eq[kSelWarps];
  __shared__ uint32_t cta_cnt[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int ncta = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t unit = blockIdx.x / ncta;
  const int b = static_cast<int>(unit / p.Hkv);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int L = min(max(p.seq_lens[b], 0), p.Smax);
  int32_t* slots = p.slots + unit * p.n;
  if (L <= p.keep) {  // nothing to evict (the whole cluster agrees)
    for (int i = rank * kSelThreads + tid; i < p.n; i += ncta * kSelThreads) slots[i] = i < L ? i : -1;
    return;
  }
  const float* w = p.src_weights + unit * p.Smax;
  const int all_warps = ncta * kSelWarps;
  const int per_warp = ((L + all_warps - 1) / all_warps + 31) & ~31;
  const int w0 = min(L, (rank * kSelWarps + warp) * per_warp), w1 = min(L, w0 + per_warp);
  const int lo = p.sink, hi = L - p.recent;  // candidates (L > keep >= sink + recent)
  uint32_t key[kPerThread > 0 ? kPerThread : 1];
  if constexpr (kPerThread > 0) {
    float x[kPerThread];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = w0 + 32 * j + lane;
      x[j] = i < w1 ? w[i] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) key[j] = order_bits(x[j]);
  }
  // calls f(row, key of the row if it is one of the warp's) for the warp's rows, 32 at a time
  auto each = [&](auto&& f) {
    if constexpr (kPerThread > 0) {
#pragma unroll
      for (int j = 0; j < kPerThread; ++j)
        if (w0 + 32 * j < w1) f(w0 + 32 * j + lane, key[j]);
    } else {
      for (int i0 = w0; i0 < w1; i0 += 32) f(i0 + lane, i0 + lane < w1 ? order_bits(w[i0 + lane]) : 0u);
    }
  };
  uint32_t need = static_cast<uint32_t>(p.keep - p.sink - p.recent);  // < hi - lo
  uint32_t thr = 0xFFFFFFFFu;  // need == 0: no weight is above it, and no equal one is taken
  if (need > 0) {
    for (int i = tid; i < 3 * kSelBins; i += kSelThreads) (&hist[0][0])[i] = 0u;
    __syncthreads();
    uint32_t pfx = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const uint32_t dmask = pass == 2 ? 1023u : 2047u;
      const int up = pass == 1 ? 21 : 10;  // the digits above: u >> up == pfx
      each([&](int i, uint32_t u) {
        if (i < w1 && i >= lo && i < hi && (pass == 0 || (u >> up) == pfx)) atomicAdd(&hist[pass][(u >> shift) & dmask], 1u);
      });
      if (ncta > 1) cluster.sync(); else __syncthreads();
      // bins kPer tid .. over the whole cluster, then the sum of the bins above them
      uint32_t bin[kPer] = {};
      for (int r = 0; r < ncta; ++r) {
        const uint2* h = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[pass][0], r)) + tid * (kPer / 2);
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j) {
          const uint2 x = h[j];
          bin[2 * j] += x.x;
          bin[2 * j + 1] += x.y;
        }
      }
      uint32_t total = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) total += bin[j];
      uint32_t suffix = total;  // over this lane and the lanes above it
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_down_sync(0xffffffffu, suffix, o);
        if (lane + o < 32) suffix += t;
      }
      if (lane == 0) warp_sum[warp] = suffix;
      __syncthreads();
      uint32_t above =
          __reduce_add_sync(0xffffffffu, lane > warp && lane < kSelWarps ? warp_sum[lane] : 0u) + suffix - total;
      if (above < need && above + total >= need) {  // exactly one thread
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j) {
          if (above < need && above + bin[j] >= need) {
            found[0] = static_cast<uint32_t>(kPer * tid + j);
            found[1] = need - above;
          }
          above += bin[j];
        }
      }
      __syncthreads();
      pfx = (pfx << (pass == 2 ? 10 : 11)) | found[0];
      need = found[1];
    }
    thr = pfx;
  }
  // rows above the threshold (and the sink and recent rows) and rows equal to it
  auto classify = [&](int i, uint32_t u, uint32_t& gt, uint32_t& eq) {
    const bool safe = i < lo || i >= hi;
    gt = __ballot_sync(0xffffffffu, i < w1 && (safe || u > thr));
    eq = __ballot_sync(0xffffffffu, i < w1 && !safe && u == thr);
  };
  uint32_t ngt = 0, neq = 0;
  each([&](int i, uint32_t u) {
    uint32_t gt, eq;
    classify(i, u, gt, eq);
    ngt += __popc(gt);
    neq += __popc(eq);
  });
  if (lane == 0) {
    warp_gt[warp] = ngt;
    warp_eq[warp] = neq;
  }
  __syncthreads();
  uint32_t gt_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_gt[lane] : 0u);
  uint32_t eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_eq[lane] : 0u);
  if (ncta > 1) {
    if (warp == kSelWarps - 1 && lane == 0) {
      cta_cnt[0] = gt_before + ngt;
      cta_cnt[1] = eq_before + neq;
    }
    cluster.sync();
    for (int r = 0; r < rank; ++r) {
      const uint32_t* other = cluster.map_shared_rank(&cta_cnt[0], r);
      gt_before += other[0];
      eq_before += other[1];
    }
    cluster.sync();  // the counts (and histograms) of a CTA are read no more: it may exit
  }
  const uint32_t below = (1u << lane) - 1u;
  each([&](int i, uint32_t u) {
    uint32_t gt, eq;
    classify(i, u, gt, eq);
    const uint32_t er = eq_before + __popc(eq & below);
    if (((gt >> lane) & 1u) != 0u || (((eq >> lane) & 1u) != 0u && er < need))
      slots[gt_before + __popc(gt & below) + min(er, need)] = i;
    gt_before += __popc(gt);
    eq_before += __popc(eq);
  });
}

// CTAs per (sequence, KV head), from the most rows a sequence can have.  Up to 2048 rows one
// CTA of 256 threads, several of which share an SM; more rows: CTAs of 1024 threads, each a
// whole SM, as few as hold the rows with 8 weights a thread where that fills at most the SMs once,
// else with 16.  Past 8 x 16 x 1024 rows no weight is held.  Measured, whole evictions: 512
// (sequence, KV head)s of 256 rows 29.1 us with 1024 threads, 13.0 us with 256; 32K rows with 8 against
// 16 weights a thread, 32 of them 35.7 / 39.3 us, 256 of them 155 / 118 us.
cudaError_t launch_select(const KvEvictParams& p, int num_sms, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(p.B) * p.Hkv;
  int cluster = 1, threads = 256;
  void (*kernel)(KvEvictParams) = kv_select_kernel<256, 8>;
  if (p.Smax > 256 * 8) {
    threads = 1024;
    while (cluster < kSelMaxCluster && p.Smax > cluster * 1024 * 8) cluster *= 2;
    if (cluster > 1 && units * cluster > num_sms && p.Smax <= cluster / 2 * 1024 * 16) cluster /= 2;
    kernel = p.Smax <= cluster * 1024 * 8    ? kv_select_kernel<1024, 8>
             : p.Smax <= cluster * 1024 * 16 ? kv_select_kernel<1024, 16>
                                             : kv_select_kernel<1024, 0>;
  }
  return launch_cluster_dependent(cluster, kernel, dim3(static_cast<unsigned>(units * cluster)), dim3(threads), 0, stream, p);
}

// ---------------------------------------------------------------------------
// evict: move
// ---------------------------------------------------------------------------
// A CTA gathers kRows destination rows of one (sequence, KV head), K and V, into
// registers (8 x 16 bytes per thread, 2 kRows threads), then rounds them to their destination
// block's scale (the largest of its rows' scales: rows of that scale keep their
// bytes) and stores them.  HBM-bound: each kept row is read and written once.
//   Out of place: one CTA per 128 rows.
//   In place: a cluster of 8 CTAs walks over the rows of its (sequence, KV head) 8 kRows
//   at a time; all eight have read their rows before any of them writes.  A kept row's
//   source lies at or behind its destination, so a later step's sources (rows and scales)
//   are never behind an earlier step's stores.  A step is a chain of some 4 us (slots, rows,
//   barrier).  Where it takes several, and the clusters of all (sequence, KV head)s fit on the SMs at
//   once, a CTA takes kBigRows rows a step (a whole SM's registers), else kMoveRows, so that several
//   clusters share the SMs.  Whole evictions in place, 512 / 128 rows: 2 x 131K rows of 4 heads
//   to 8K 36 / 55 us, 16 x 8K rows of 8 heads to 2K 65 / 37 us.
constexpr int kMoveRows = 128;
constexpr int kBigRows = 512;
constexpr int kMoveCluster = 8;

template <bool kInt8, bool kInPlace, int kRows>
__device__ __forceinline__ void move_rows(const KvEvictParams& p, int64_t unit, int base) {
  __shared__ int slot_sh[kRows];
  __shared__ float scale_sh[2][kRows];
  __shared__ float warp_max[2][kRows / 32];
  const int tid = threadIdx.x;
  // -1: no row, here or further on
  int slot = -1;
  float s[2] = {0.0f, 0.0f}, weight = 0.0f;
  bool moved = false;
  if (tid < kRows) {
    const int row = base + tid;
    if (row < p.n) slot = p.slots[unit * p.n + row];
    moved = slot != row && slot >= 0;
    if (slot >= 0) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) s[kv] = p.src_scale[kv][unit * p.nblk + slot / p.block];
      weight = p.src_weights[unit * p.Smax + slot];
    }
    slot_sh[tid] = slot;
  }
  const bool work = __syncthreads_or(kInPlace ? moved : slot >= 0) != 0;
  uint4 v[8];
  if (work) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = kRows / 4 * (i & 3) + (tid >> 3);
      const int src = slot_sh[r];
      v[i] = make_uint4(0, 0, 0, 0);
      if (src >= 0)  // (read once: the streaming load measured 5 % faster than a plain one)
        v[i] = __ldcs(reinterpret_cast<const uint4*>(p.src[i >> 2] + (unit * p.Smax + src) * 128 + 16 * (tid & 7)));
    }
    // destination scale of each row: the maximum over its block
    if (tid < kRows) {
      float m[2] = {s[0], s[1]};
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
          if (o < p.block) m[kv] = fmaxf(m[kv], __shfl_xor_sync(0xffffffffu, m[kv], o));
        if ((tid & 31) == 0) warp_max[kv][tid >> 5] = m[kv];
      }
      scale_sh[0][tid] = m[0];
      scale_sh[1][tid] = m[1];
    }
    __syncthreads();
    float d[2] = {0.0f, 0.0f};
    if (tid < kRows) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        d[kv] = scale_sh[kv][tid];
        if (p.block > 32) {
          const int per = p.block / 32, first = (tid >> 5) / per * per;
          for (int k = 0; k < per; ++k) d[kv] = fmaxf(d[kv], warp_max[kv][first + k]);
        }
      }
    }
    __syncthreads();
    if (tid < kRows) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) scale_sh[kv][tid] = s[kv] == d[kv] ? 1.0f : s[kv] / d[kv];
    }
    __syncthreads();
    if (kInPlace) cg::this_cluster().sync();
    if (tid < kRows && slot >= 0) {
      const int row = base + tid;
      p.dst_weights[unit * p.Smax_dst + row] = weight;
      if (tid % p.block == 0) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) p.dst_scale[kv][unit * p.nblk_dst + row / p.block] = d[kv];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = kRows / 4 * (i & 3) + (tid >> 3);
      if (slot_sh[r] < 0) continue;
      const float ratio = scale_sh[i >> 2][r];
      const uint4 o = ratio == 1.0f ? v[i] : rescale8<kInt8>(v[i], ratio);
      *reinterpret_cast<uint4*>(p.dst[i >> 2] + (unit * p.Smax_dst + base + r) * 128 + 16 * (tid & 7)) = o;
    }
  } else if (kInPlace) {
    cg::this_cluster().sync();
  }
}

__device__ __forceinline__ void write_kept_length(const KvEvictParams& p, int64_t unit) {
  if (unit % p.Hkv == 0 && threadIdx.x == 0) {
    const int b = static_cast<int>(unit / p.Hkv);
    p.dst_lens[b] = min(min(max(p.seq_lens[b], 0), p.Smax), p.keep);
  }
}

template <bool kInt8>
__global__ void __launch_bounds__(2 * kMoveRows) kv_move_kernel(const __grid_constant__ KvEvictParams p, int tiles) {
  const int64_t unit = blockIdx.x / tiles;
  const int tile = blockIdx.x % tiles;
  cudaGridDependencySynchronize();
  move_rows<kInt8, false, kMoveRows>(p, unit, tile * kMoveRows);
  if (tile == 0) write_kept_length(p, unit);
}

template <bool kInt8, int kRows>
__global__ void __launch_bounds__(2 * kRows)
    kv_move_in_place_kernel(const __grid_constant__ KvEvictParams p) {
  const int64_t unit = blockIdx.x / kMoveCluster;
  const int rank = blockIdx.x % kMoveCluster;
  cudaGridDependencySynchronize();
  for (int step = 0; step < p.n; step += kMoveCluster * kRows) {
    move_rows<kInt8, true, kRows>(p, unit, step + rank * kRows);
    __syncthreads();
  }
  if (rank == 0) write_kept_length(p, unit);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, bool int8, cudaStream_t stream) {
  if (p.T > 1) return int8 ? append_rows<true>(p, stream) : append_rows<false>(p, stream);
  const int threads = 32 * (2 * p.Hkv < 32 ? 2 * p.Hkv : 32);
  return launch_dependent(int8 ? kv_append_token_kernel<true> : kv_append_token_kernel<false>, dim3(p.B), dim3(threads), 0,
                          stream, p);
}

cudaError_t launch_kv_evict(const KvEvictParams& p, bool int8, bool in_place, int num_sms, cudaStream_t stream) {
  cudaError_t e = launch_select(p, num_sms, stream);
  if (e != cudaSuccess) return e;
  const int units = p.B * p.Hkv;
  if (in_place) {
    const bool big = units * kMoveCluster <= num_sms && p.n > kMoveCluster * kMoveRows;
    void (*kernel)(KvEvictParams) =
        big ? (int8 ? kv_move_in_place_kernel<true, kBigRows> : kv_move_in_place_kernel<false, kBigRows>)
            : (int8 ? kv_move_in_place_kernel<true, kMoveRows> : kv_move_in_place_kernel<false, kMoveRows>);
    return launch_cluster_dependent(kMoveCluster, kernel, dim3(units * kMoveCluster), dim3(2 * (big ? kBigRows : kMoveRows)), 0,
                                    stream, p);
  }
  const int tiles = (p.n + kMoveRows - 1) / kMoveRows;
  return launch_dependent(int8 ? kv_move_kernel<true> : kv_move_kernel<false>, dim3(units * tiles), dim3(2 * kMoveRows), 0,
                          stream, p, tiles);
}

}  // namespace swa
