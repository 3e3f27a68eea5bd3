// Decode attention over the block-scaled 8-bit KV cache on B200 (sm_100a): one query
// token per sequence attends to its cached keys [lo, L), lo = 0 (full) or
// max(0, L - window), with value = byte * scale[block of the key]:
//   s_hk = scale_log2 * ks_k * (q_h . k8_k)        (log2 domain)
//   O_h  = sum_k 2^(s_hk - lse_h) vs_k v8_k,  lse_h = log2 sum_k 2^s_hk
//   weights_k += sum over the heads h of the group of 2^(s_hk - lse_h)   (optional)
//
// HBM-bound: 256 bytes per (key, KV head).  The bytes go from TMA to the tensor cores
// as they are, with no conversion in between: the 8-bit operand is the M side,
//   S^T [128 keys x N]  = K tile [128 x 128 B] (K-major)  .  Qp^T
//   O^T [128 dims x N]  = V tile^T (MN-major)             .  Pp^T
// and the few query heads the N side.  Q and P, which have more than 8 bits, are cut
// into three 8-bit parts, a column each: e4m3 parts of 4 significant bits (kind::f8f6f4, 12 bits in
// all, P as FP16) or signed-byte digits (kind::i8, 23 bits and exact INT32 sums).  The parts'
// results are added up in FP32.  Q is scaled by its head's largest |q|: e4m3 parts hold BF16 exactly
// down to 2^-18 of that and to within 2^-25 of it below, digits all of it to within 2^-23.9.
// P's FP16 rounding is 2^-11 of a weight at most, an eighth of O's to BF16, and differs from key to
// key: O's error against 64 bits is that of an FP32 step to four digits.
//
// Roles of a CTA (192 threads): warps 0-3 softmax, warp 4 TMA producer, warp 5 MMA issuer.
// A softmax thread owns one key of a tile (TMEM lane) when it reads S^T, and one of the
// 128 dims when it reads O^T: O is kept in its registers, one value per head, and each
// tile's O^T is added with the tile's own factor, so P and the V scales enter as
// 2^(s - m) vs / max vs (never above 1), m the tile's largest score of the head.  The parts' last
// step is a fixed fraction of 1, and keys under a large scale that get no weight must not take
// the digits of those that do: where a tile's V scales do not lie within 2^4 of one another
// (hardly ever), m is lowered by head until the largest of these products is 1, which takes a second
// exchange between the softmax warps (all tiles so: 64 sequences of up to 32K keys 62.2 against
// 61.0 us, 16 int8 ones with weights 36.2 against 32.2).
//
// Measured (B200, graph of ten calls): 64 sequences of 16K-32K keys, an eighth routed full, 359 MB
// of legal bytes, 61 to 67 us (5.4 to 5.9 TB/s; the e4m3 cache with one scale per head, whose bytes are
// converted in registers, takes 154 us); 536 MB of full sequences 85 us (6.3 TB/s).  Reading alone,
// tiles of this size stream at 7.1 TB/s with 96 to 128 KB in flight per SM and at 6.5 to 7.0 with
// 192 KB; two CTAs an SM with two K and two V tiles each hold 128 KB (three tiles each: 75.2
// against 73.5 us on the 64 sequences; three CTAs: 81 us, their registers spill).  The
// tensor pipe is 8 % busy.  What is left is the start (about 4 us to the first scores), the
// uneven end and the second kernel (about 3 us).  With more than 8 query heads per KV head every
// tile is taken once per 8 heads, and the softmax warps' chain per tile (about 2400 cycles)
// bounds: 8 x 32K keys, 16 heads per KV head, 80 us for 41 us of bytes.
#include <atomic>

#include <cuda_fp16.h>

#include "kv_cache.h"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include "swattn_internal.h"

namespace swa {

namespace {

constexpr int kTile = 128;                 // keys of a tile
constexpr int kTileBytes = kTile * 128;
constexpr int kStages = 2;                 // K tiles and V tiles in flight
constexpr int kScaleRing = 8;              // tiles whose block scales are held
constexpr int kThreads = 192;
constexpr int kParts = 3;
constexpr float kE4m3Step = 16.0f;         // weight of an e4m3 part against the next
constexpr float kEvenScales = 1.0f / 16.0f;  // V scales down to this share of a tile's largest one are near it
constexpr float kInt8One = 127.0f * 65536.0f;  // 1.0 as three signed-byte digits

// What the softmax warps have to agree on for a tile: the (up to) 8 heads' largest scores by warp, and
// the largest V scale (the issuer warp's finding, negative where others are not near it).
struct __align__(16) KvTileMax {
  float top[4][8], vref, pad[3];
};

template <int kHeads>
struct KvSmem {
  static constexpr int cols = kHeads <= 4 ? 16 : 32;  // N: parts x heads, padded
  static constexpr uint32_t k = 0;
  static constexpr uint32_t v = k + kStages * kTileBytes;
  static constexpr uint32_t q = v + kStages * kTileBytes;          // [cols][128 B]
  static constexpr uint32_t p = q + cols * 128;                    // 2 x [cols][128 B]
  static constexpr uint32_t red = p + 2 * cols * 128;              // [2] KvTileMax
  static constexpr uint32_t lred = red + 2 * sizeof(KvTileMax);    // [2][4 warps][8] floats
  static constexpr uint32_t off = lred + 2 * 4 * 8 * 4;            // [4 warps][8] floats
  static constexpr uint32_t qf = off + 4 * 8 * 4;                  // [2][8] floats
  static constexpr uint32_t sc = qf + 64;                          // [kScaleRing][2][16] floats: K, V scales of a tile
  static constexpr uint32_t bars = sc + kScaleRing * 128;
  static constexpr uint32_t misc = bars + 32 * 8;                  // tmem holder, abort flag, the share
  static constexpr uint32_t total = misc + 16 + 64;
  static constexpr uint32_t bytes = total + 1024;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// x[h] over the warp's lanes for every head h, halving the heads with each of the first
// steps (9 shuffles for 8 heads, 7 for 4, instead of 5 a head): lanes (32 / kHeads) h and on
// return head h's.  x is overwritten.
template <int kHeads, typename Op>
__device__ __forceinline__ float reduce_heads(float* x, int lane, Op op) {
  int d = 16;
#pragma unroll
  for (int k = kHeads / 2; k >= 1; k >>= 1, d >>= 1) {
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int j = 0; j < k; ++j) {
      const float give = up ? x[j] : x[j + k];
      x[j] = op(up ? x[j + k] : x[j], __shfl_xor_sync(0xffffffffu, give, d));
    }
  }
#pragma unroll
  for (; d >= 1; d >>= 1) x[0] = op(x[0], __shfl_xor_sync(0xffffffffu, x[0], d));
  return x[0];
}

struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const KvDecodeParams& p, int b) {
  const int L = min(max(p.seq_lens[b], 0), p.Smax);
  return KeyRange{p.route[b] != 0 ? 0 : max(0, L - p.window), L};
}
__device__ __forceinline__ int seq_tiles(const KvDecodeParams& p, int b) {
  const KeyRange r = key_range(p, b);
  return (r.hi - r.lo + kTile - 1) / kTile;
}

// First step of share c of the axis of work, and the share that step v lies on.
__device__ __forceinline__ int share_start(int c, int per, int longer) { return c * per + min(c, longer); }
__device__ __forceinline__ int share_of(int v, int per, int longer) {
  const int w = v - longer * (per + 1);
  return w < 0 ? v / (per + 1) : longer + w / per;
}

// Steps for starting a unit (its Q, its first tile's latency, the sums and the output at
// its end), in half tiles.  On 64 sequences a CTA with six segments took 1.5 us more
// per segment than one with a single one, at 1.2 us a tile: without these steps the CTAs of the
// short units ended 8 us of 62 after the others.  With few tiles a CTA they do not
// matter and every CTA takes whole tiles only.
constexpr int kUnitSteps = 3;
constexpr int kFewTiles = 4;

// A CTA's share, segment by segment.
struct Segments {
  int hb, b, g, off, left;  // of the next segment: head block, sequence, KV head, first step in the unit; steps left
  int vbase, tbase;     // steps and tiles before that unit
  int lo, hi, all;      // legal keys of sequence b, tiles of its units
  int omega;
  // the current segment
  int cur_hb, cur_b, cur_g, cur_vbase, cur_tbase, cur_lo, cur_hi, cur_all, first, n;

  __device__ __forceinline__ void start(const KvShare& s) {
    hb = s.hb;
    b = s.b;
    g = s.g;
    off = s.off;
    left = s.left;
    vbase = s.vbase;
    tbase = s.tbase;
    lo = s.lo;
    hi = s.hi;
    all = (hi - lo + kTile - 1) / kTile;
    omega = s.omega;
  }
  // the next segment with a tile of this share; false when there is none
  __device__ __forceinline__ bool next(const KvDecodeParams& p) {
    while (left > 0) {
      const int length = all > 0 ? omega + all * kTileSteps : 0;
      const int take = min(length - off, left);
      cur_hb = hb;
      cur_b = b;
      cur_g = g;
      cur_vbase = vbase;
      cur_tbase = tbase;
      cur_lo = lo;
      cur_hi = hi;
      cur_all = all;
      first = max(0, off - omega + kTileSteps - 1) / kTileSteps;
      n = max(0, off + take - omega + kTileSteps - 1) / kTileSteps - first;
      left -= take;
      off += take;
      if (off == length && left > 0) {
        off = 0;
        vbase += length;
        tbase += all;
        if (all == 0 || ++g == p.Hkv) {  // (a sequence without a key has no unit)
          g = 0;
          if (++b == p.B) {
            b = 0;
            ++hb;
          }
          const KeyRange r = key_range(p, b);
          lo = r.lo;
          hi = r.hi;
          all = (r.hi - r.lo + kTile - 1) / kTile;
        }
      }
      if (n > 0) return true;
    }
    return false;
  }
};

__device__ __forceinline__ float pow2_at_least_448th(float a) {  // smallest 2^e with 448 * 2^e >= a
  const uint32_t bits = __float_as_uint(a);
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23);
}

__device__ __forceinline__ uint16_t f16x2_to_e4m3x2(uint32_t h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h));
  return r;
}
__device__ __forceinline__ __half2 e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return *reinterpret_cast<__half2*>(&r);
}

// Two values (|x| <= 448) as three e4m3 parts each: x = p0 + p1 / 16 + p2 / 256, the
// parts' pairs as bytes (low byte: first value).  e4m3 has 4 significant bits, so the
// rest left by a part is at most 1/16 of its value's binade and 16 times it is in
// range again: together the parts hold the 11 bits of an FP16 x, down to steps of 2^-17
// (the last part's smallest, 2^-9 / 256).
__device__ __forceinline__ void split_e4m3(__half2 x, uint16_t* part) {
  part[0] = f16x2_to_e4m3x2(*reinterpret_cast<uint32_t*>(&x));
  const __half2 r1 = __hsub2(x, e4m3x2_to_f16x2(part[0]));
  __half2 y = __hmul2(r1, __float2half2_rn(kE4m3Step));
  part[1] = f16x2_to_e4m3x2(*reinterpret_cast<uint32_t*>(&y));
  y = __hmul2(__hsub2(y, e4m3x2_to_f16x2(part[1])), __float2half2_rn(kE4m3Step));
  part[2] = f16x2_to_e4m3x2(*reinterpret_cast<uint32_t*>(&y));
}

// A value in [-1, 1] in steps of 1 / (127 * 65536) as three signed bytes (byte 2 the highest).
__device__ __forceinline__ uint32_t split_int8(float x) {
  return static_cast<uint32_t>(__float2int_rn(x * kInt8One) + 0x008080) ^ 0x008080u;
}

// Sum of the parts' results of head h (accumulator columns part * kHeads + h).
template <bool kInt8, int kHeads>
__device__ __forceinline__ float join_parts(const uint32_t* c, int h) {
  if constexpr (kInt8) {
    return fmaf(static_cast<float>(static_cast<int>(c[h])), 65536.0f,
                fmaf(static_cast<float>(static_cast<int>(c[kHeads + h])), 256.0f,
                     static_cast<float>(static_cast<int>(c[2 * kHeads + h]))));
  } else {
    return fmaf(__uint_as_float(c[2 * kHeads + h]), 1.0f / (kE4m3Step * kE4m3Step),
                fmaf(__uint_as_float(c[kHeads + h]), 1.0f / kE4m3Step, __uint_as_float(c[h])));
  }
}

template <int kCols>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t* c) {
  if constexpr (kCols == 16) {
    tmem_ld_x16(addr, c);
    tmem_ld_wait();
    reg_fence16(c);
  } else {
    tmem_ld_x32(addr, c);
    tmem_ld_wait();
    reg_fence32(c);
  }
}

// kWeights: also stores every legal key's scores for the second kernel.
template <bool kInt8, int kHeads, bool kWeights>
__global__ void __launch_bounds__(kThreads, kKvDecodeCtasPerSm)
    kv_decode_kernel(const __grid_constant__ KvDecodeParams p) {
  using Sm = KvSmem<kHeads>;
  constexpr int kCols = Sm::cols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + Sm::bars);
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;  // [2] scores of a tile in TMEM
  uint64_t* p_full = s_full + 2;         // [2] P of a tile in shared memory (and its scores read)
  uint64_t* o_full = p_full + 2;         // [2] O^T of a tile in TMEM
  uint64_t* red_full = o_full + 2;       // [2] a tile's KvTileMax
  uint64_t* q_full = red_full + 2;       // Q parts of a segment
  uint64_t* l_full = q_full + 1;         // the four warps' row sums of a segment
  uint64_t* done = l_full + 1;
  uint64_t* sc_full = done + 1;          // [kScaleRing] block scales of a tile in shared memory
  uint64_t* off_full = sc_full + kScaleRing;  // the four warps' `off` of a tile with V scales far apart
  static_assert(4 * kStages + 4 * 2 + 3 + kScaleRing + 1 <= 32, "barrier space");
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + Sm::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Sm::misc + 4);
  KvShare* share = reinterpret_cast<KvShare*>(smem + Sm::misc + 16);
  KvTileMax* red = reinterpret_cast<KvTileMax*>(smem + Sm::red);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  // set up what needs no global memory while the kernel before this one ends
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&red_full[i], 5);
    }
    mbar_init(q_full, 128);
    mbar_init(l_full, 4);
    mbar_init(off_full, 4);
    mbar_init(done, 1);
    for (int i = 0; i < kScaleRing; ++i) mbar_init(&sc_full[i], 32);
    *abort_flag = 0;
    share->left = 0;
    fence_barrier_init();
  }
  if (tid == 128) {
    tma_prefetch_desc(&p.map[0]);
    tma_prefetch_desc(&p.map[1]);
  }
  // unused columns of Q and P are zero
  for (int i = tid; i < 3 * kCols * 8; i += kThreads)
    reinterpret_cast<uint4*>(smem + Sm::q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();  // the second kernel waits for this one's end by itself
  // (tensor memory only from here on: a CTA that held some while it waits for the kernel before
  // could keep that one from getting its own)
  if (warp == 5) {
    __syncwarp();
    tmem_alloc(tmem_holder, 4 * kCols);
    tmem_relinquish();
  }
  {
    // this CTA's share: thread t sums a run of sequences' tiles and counts those that have any, then
    // a scan of both (packed into 64 bits) over the threads
    int64_t* scan = reinterpret_cast<int64_t*>(smem + Sm::red);
    constexpr int64_t kOne = int64_t{1} << 32;
    const int run = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * run), b1 = min(p.B, b0 + run);
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = seq_tiles(p, b);
      sum += n > 0 ? kOne + n : 0;
    }
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int64_t before = incl - sum, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    const int tiles = static_cast<int>(total & (kOne - 1)) * p.Hkv;  // of one head block
    const int omega = tiles * p.nhb >= kFewTiles * p.ctas ? kUnitSteps : 0;
    auto steps_of = [&](int64_t x) {  // of x's sequences and tiles, all KV heads
      return (static_cast<int>(x >> 32) * omega + static_cast<int>(x & (kOne - 1)) * kTileSteps) * p.Hkv;
    };
    const int block_steps = steps_of(total), steps = block_steps * p.nhb;
    // every share holds the first step of a tile: they lie at most omega + kTileSteps apart
    const int ctas = max(1, min(p.ctas, steps / (omega + kTileSteps)));
    KvShare sh{};
    sh.omega = omega;
    sh.per = steps / ctas;
    sh.longer = steps % ctas;
    sh.block_steps = block_steps;
    sh.block_tiles = tiles;
    const int v0 = share_start(cta, sh.per, sh.longer), v1 = share_start(cta + 1, sh.per, sh.longer);
    sh.hb = block_steps > 0 ? v0 / block_steps : 0;
    const int w0 = v0 - sh.hb * block_steps;  // in its head block
    if (cta >= ctas || v0 >= v1) {
      if (tid == 0) {
        p.share[cta] = sh;
        *share = sh;
      }
    } else if (w0 >= steps_of(before) && w0 < steps_of(before + sum)) {  // exactly one thread
      int64_t at = before;
      for (int b = b0;; ++b) {
        const int n = seq_tiles(p, b);
        const int64_t next = at + (n > 0 ? kOne + n : 0);
        if (w0 < steps_of(next)) {
          const KeyRange kr = key_range(p, b);
          const int length = omega + n * kTileSteps, in = w0 - steps_of(at);
          sh.b = b;
          sh.g = in / length;
          sh.off = in % length;
          sh.left = v1 - v0;
          sh.vbase = v0 - sh.off;
          sh.tbase = sh.hb * tiles + static_cast<int>(at & (kOne - 1)) * p.Hkv + sh.g * n;
          sh.lo = kr.lo;
          sh.hi = kr.hi;
          break;
        }
        at = next;
      }
      p.share[cta] = sh;
      *share = sh;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;  // S: columns 0 and kCols, O: 2 kCols and 3 kCols
  Segments seg{};
  seg.start(*share);

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    // Lane 0 issues the tiles; the warp copies the tile's block scales (at most 9 of K and 9 of V)
    // along with K, so that they are there when the scores are: softmax threads that loaded their
    // key's scales themselves, one tile ahead, waited for them behind the tiles that fill the
    // memory queues (64 sequences: 72.4 against 71.4 us).  K and V leave L2 first: a step reads
    // them once, and the scores that the second kernel reads stay in it (two 131K-token sequences
    // with weights: 50.0 against 45.2 us).  Slot t % kScaleRing is free: k_empty of tile t - kStages
    // says that the scores of that tile are done, so that P of the tile two before is written
    // and the scales up to there are read.
    static_assert(kScaleRing >= kStages + 2, "scale ring");
    const uint64_t once = l2_policy_evict_first();
    int it = 0, iv = 0;  // K and V tiles issued
    bool ok = true;
    const int withheld = p.test_withhold != 0 && cta == 0 ? 1 : -1;  // K tile that is not loaded
    while (ok && seg.next(p)) {
      const int row = seg.cur_b * p.Hkv + seg.cur_g;
      const float* scales = p.scale[lane >> 4] + static_cast<int64_t>(row) * p.nblk;
      for (int i = 0; i < seg.n; ++i) {
        const int s = it % kStages;
        const uint32_t ph = ((it / kStages) & 1) ^ 1;
        const int key0 = seg.cur_lo + (seg.first + i) * kTile;
        if (!(ok = warp_wait(&k_empty[s], ph, abort_flag))) break;
        if (lane == 0 && it != withheld) {
          mbar_arrive_expect_tx(&k_full[s], kTileBytes);
          tma_load_3d_hint(smem + Sm::k + s * kTileBytes, &p.map[0], &k_full[s], 0, key0, row, once);
        }
        const int blk = (key0 >> p.block_shift) + (lane & 15);
        if (blk <= (min(key0 + kTile, seg.cur_hi) - 1) >> p.block_shift)
          cp_async_4(smem_u32(smem + Sm::sc + (it % kScaleRing) * 128 + lane * 4), scales + blk);
        cp_async_arrive(&sc_full[it % kScaleRing]);
        ++it;
        if (!(ok = warp_wait(&v_empty[s], ph, abort_flag))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&v_full[s], kTileBytes);
          tma_load_3d_hint(smem + Sm::v + s * kTileBytes, &p.map[1], &v_full[s], 0, key0, row, once);
        }
        ++iv;
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
    if (*abort_flag && lane == 0) {
      // let the loads already issued land before the CTA's shared memory is released
      volatile int dummy = 0;
      for (int t = max(0, it - kStages); t < it; ++t)
        if (t != withheld) mbar_wait(&k_full[t % kStages], (t / kStages) & 1, &dummy);
      for (int t = max(0, iv - kStages); t < iv; ++t) mbar_wait(&v_full[t % kStages], (t / kStages) & 1, &dummy);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_s = make_idesc_8bit(kInt8, 128, kCols, false, false);
    constexpr uint32_t idesc_o = make_idesc_8bit(kInt8, 128, kCols, true, false);
    const uint64_t q_desc = make_smem_desc_sw128(smem_u32(smem + Sm::q), 16, 1024);
    bool ok = true;
    int pv = 0;  // tiles whose PV product has been issued
    auto issue_pv = [&]() {
      const int s = pv % kStages;
      if (!warp_wait(&v_full[s], (pv / kStages) & 1, abort_flag)) return false;
      if (!warp_wait(&p_full[pv & 1], (pv >> 1) & 1, abort_flag)) return false;
      tc_fence_after();
      const uint64_t v_desc = make_smem_desc_sw128(smem_u32(smem + Sm::v + s * kTileBytes), kTileBytes, 1024);
      const uint64_t p_desc = make_smem_desc_sw128(smem_u32(smem + Sm::p + (pv & 1) * kCols * 128), 16, 1024);
      umma8_ss_k128_warp<kInt8>(tmem + (2 + (pv & 1)) * kCols, v_desc, p_desc, 32 * 128 / 16, 2, idesc_o);
      tc_commit_warp(&o_full[pv & 1]);
      tc_commit_warp(&v_empty[s]);
      ++pv;
      return true;
    };
    int it = 0, nseg = 0;
    while (ok && seg.next(p)) {
      // (a segment's Q is written once the last scores of the one before are there, so before that
      // segment's last P)
      ok = warp_wait(q_full, nseg & 1, abort_flag);
      ++nseg;
      for (int i = 0; i < seg.n && ok; ++i, ++it) {
        const int s = it % kStages;
        if (!(ok = warp_wait(&k_full[s], (it / kStages) & 1, abort_flag))) break;
        tc_fence_after();
        // score buffer it & 1 was read before P of tile it - 2, whose product is issued
        const uint64_t k_desc = make_smem_desc_sw128(smem_u32(smem + Sm::k + s * kTileBytes), 16, 1024);
        umma8_ss_k128_warp<kInt8>(tmem + (it & 1) * kCols, k_desc, q_desc, 2, 2, idesc_s);
        tc_commit_warp(&s_full[it & 1]);
        tc_commit_warp(&k_empty[s]);
        while (ok && pv < it) ok = issue_pv();
        if (!ok) break;
        // the tile's V scales, a lane each: their largest, and whether the others above 0 are near it
        // (the softmax warps have read those of tile it - 2: its P is there)
        if (!(ok = warp_wait(&sc_full[it % kScaleRing], (it / kScaleRing) & 1, abort_flag))) break;
        const int key0 = seg.cur_lo + (seg.first + i) * kTile;
        const int blocks = ((min(key0 + kTile, seg.cur_hi) - 1) >> p.block_shift) - (key0 >> p.block_shift) + 1;
        const float* sc = reinterpret_cast<const float*>(smem + Sm::sc + (it % kScaleRing) * 128) + 16;
        const float vs = lane < blocks ? sc[lane] : 0.0f, vref = warp_max(vs);
        const bool wide = __any_sync(0xffffffffu, vs > 0.0f && vs < vref * kEvenScales);
        if (lane == 0) {
          red[it & 1].vref = wide ? -vref : vref;
          mbar_arrive(&red_full[it & 1]);
        }
      }
    }
    while (ok && pv < it) ok = issue_pv();
    tc_commit_warp(done);  // every MMA issued, before the CTA frees its tensor memory
    volatile int dummy = 0;
    mbar_wait(done, 0, &dummy);
  } else {
    // ------------------------------------------------------------ softmax warps
    const uint32_t lane_off = static_cast<uint32_t>(32 * warp) << 16;
    float* off = reinterpret_cast<float*>(smem + Sm::off);
    float* lred = reinterpret_cast<float*>(smem + Sm::lred);
    float* qf = reinterpret_cast<float*>(smem + Sm::qf);
    bool ok = true;
    int it = 0, nseg = 0, nwide = 0;
    // Q of a segment: 16 threads per head, 8 dims each
    auto load_q = [&](const Segments& sg) {
      const int h = tid >> 4, hb = sg.cur_hb;
      if (h >= min(kHeads, p.r - hb * kHeads)) return make_uint4(0, 0, 0, 0);
      const int head = sg.cur_g * p.r + hb * kHeads + h;
      return *reinterpret_cast<const uint4*>(p.q + sg.cur_b * p.q_sb + head * p.q_sh + 8 * (tid & 15));
    };
    // its parts into shared memory, once the scores of the segment before are done
    auto write_q = [&](uint4 w, int parity) {
      const int h = tid >> 4, c = tid & 15;
      const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
      float x[8];
      float amax = 0.0f;
      bool finite = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __uint_as_float((i & 1) ? (wd[i >> 1] & 0xFFFF0000u) : (wd[i >> 1] << 16));
        finite = finite && fabsf(x[i]) < INFINITY;
        amax = fmaxf(amax, fabsf(x[i]));
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        finite = __shfl_xor_sync(0xffffffffu, finite ? 1 : 0, o) != 0 && finite;
      }
      if (h < kHeads) {
        uint32_t lo[kParts], hi[kParts];  // bytes of dims 0-3 and 4-7
        float unit;                       // value of one step of the parts' sum
        if constexpr (kInt8) {
          unit = amax / kInt8One;
          const float inv = (amax > 0.0f && finite) ? 1.0f / amax : 0.0f;
#pragma unroll
          for (int pt = 0; pt < kParts; ++pt) lo[pt] = hi[pt] = 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t v = split_int8(x[i] * inv);
#pragma unroll
            for (int pt = 0; pt < kParts; ++pt) {
              const uint32_t byte = (v >> (16 - 8 * pt)) & 0xFFu;
              if (i < 4) lo[pt] |= byte << (8 * i); else hi[pt] |= byte << (8 * (i - 4));
            }
          }
        } else {
          unit = amax > 0.0f ? pow2_at_least_448th(amax) : 1.0f;  // a power of two: x / unit is exact
          const float inv = finite ? 1.0f / unit : 0.0f;
          uint16_t pr[4][kParts];
#pragma unroll
          for (int i = 0; i < 4; ++i) split_e4m3(__floats2half2_rn(x[2 * i] * inv, x[2 * i + 1] * inv), pr[i]);
#pragma unroll
          for (int pt = 0; pt < kParts; ++pt) {
            lo[pt] = pr[0][pt] | (static_cast<uint32_t>(pr[1][pt]) << 16);
            hi[pt] = pr[2][pt] | (static_cast<uint32_t>(pr[3][pt]) << 16);
          }
        }
#pragma unroll
        for (int pt = 0; pt < kParts; ++pt) {
          const int n = pt * kHeads + h;
          *reinterpret_cast<uint2*>(smem + Sm::q + n * 128 + (((c >> 1) ^ (n & 7)) << 4) + 8 * (c & 1)) =
              make_uint2(lo[pt], hi[pt]);
        }
        // a query with an infinity or NaN has no finite score: NaN all through
        if (c == 0) qf[8 * parity + h] = finite ? p.scale_log2 * unit : __uint_as_float(0x7FC00000u);
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    };
    Segments ahead = seg;  // one segment further on, whose Q is loaded while this one runs
    bool more = ahead.next(p);
    if (more) write_q(load_q(ahead), 0);
    while (ok && more) {
      seg = ahead;
      more = ahead.next(p);
      const uint4 q_next = more ? load_q(ahead) : make_uint4(0, 0, 0, 0);
      const int head0 = seg.cur_g * p.r + seg.cur_hb * kHeads;  // first query head of the block
      const int nh = min(kHeads, p.r - seg.cur_hb * kHeads);    // heads that exist
      if (!(ok = warp_wait(q_full, nseg & 1, abort_flag))) break;
      float f[kHeads], m[kHeads], l[kHeads], o[kHeads], alpha[kHeads], beta[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        f[h] = qf[8 * (nseg & 1) + h];
        m[h] = -INFINITY;
        l[h] = o[h] = alpha[h] = beta[h] = 0.0f;
      }
      // adds O^T of tile t (relative to that tile's maximum and V scale)
      auto take_o = [&](int t) {
        if (!warp_wait(&o_full[t & 1], (t >> 1) & 1, abort_flag)) return false;
        tc_fence_after();
        uint32_t c[kCols];
        tmem_ld_cols<kCols>(tmem + (2 + (t & 1)) * kCols + lane_off, c);
#pragma unroll
        for (int h = 0; h < kHeads; ++h) o[h] = fmaf(join_parts<kInt8, kHeads>(c, h), beta[h], o[h] * alpha[h]);
        return true;
      };
      for (int i = 0; i < seg.n && ok; ++i, ++it) {
        const int key0 = seg.cur_lo + (seg.first + i) * kTile;
        const bool legal = key0 + tid < seg.cur_hi;
        const int buf = it & 1;
        if (!(ok = warp_wait(&sc_full[it % kScaleRing], (it / kScaleRing) & 1, abort_flag))) break;
        const float* sc = reinterpret_cast<const float*>(smem + Sm::sc + (it % kScaleRing) * 128) +
                          ((min(key0 + tid, seg.cur_hi - 1) >> p.block_shift) - (key0 >> p.block_shift));
        const float ks = sc[0], vs = legal ? sc[16] : 0.0f;
        KvTileMax& rb = red[buf];
        if (!(ok = warp_wait(&s_full[buf], (it >> 1) & 1, abort_flag))) break;
        tc_fence_after();
        float s[kHeads];
        {
          uint32_t c[kCols];
          tmem_ld_cols<kCols>(tmem + buf * kCols + lane_off, c);
#pragma unroll
          for (int h = 0; h < kHeads; ++h) s[h] = legal ? join_parts<kInt8, kHeads>(c, h) * (f[h] * ks) : -INFINITY;
        }
        if (more && i + 1 == seg.n) write_q(q_next, (nseg + 1) & 1);  // the last scores with this Q are done
        if constexpr (kWeights) {
          float* dst = p.scores + static_cast<int64_t>(seg.cur_tbase + seg.first + i) * kHeads * kTile + tid;
#pragma unroll
          for (int h = 0; h < kHeads; ++h) dst[h * kTile] = s[h];
        }
        // maxima of the tile over its keys
        const auto larger = [](float a, float b) { return fmaxf(a, b); };
        float mt[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) mt[h] = s[h];
        const float top = reduce_heads<kHeads>(mt, lane, larger);
        if (lane % (32 / kHeads) == 0) rb.top[warp][lane / (32 / kHeads)] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_full[buf]);
        // (while the other warps' maxima come in: O of the tile before, whose product has been issued
        // since that tile's P)
        if (i > 0 && !(ok = take_o(it - 1))) break;
        if (!(ok = warp_wait(&red_full[buf], (it >> 1) & 1, abort_flag))) break;
#pragma unroll
        for (int h = 0; h < kHeads; h += 4) {
          const float4 a = *reinterpret_cast<const float4*>(&rb.top[0][h]), b = *reinterpret_cast<const float4*>(&rb.top[1][h]);
          const float4 c = *reinterpret_cast<const float4*>(&rb.top[2][h]), d = *reinterpret_cast<const float4*>(&rb.top[3][h]);
          mt[h] = fmaxf(fmaxf(a.x, b.x), fmaxf(c.x, d.x));
          mt[h + 1] = fmaxf(fmaxf(a.y, b.y), fmaxf(c.y, d.y));
          mt[h + 2] = fmaxf(fmaxf(a.z, b.z), fmaxf(c.z, d.z));
          mt[h + 3] = fmaxf(fmaxf(a.w, b.w), fmaxf(c.w, d.w));
        }
        // P relative to the tile's maximum, V scales relative to the tile's largest
        const float vref = fabsf(rb.vref);
        const float vrel = vref > 0.0f ? vs / vref : 0.0f;
        if (rb.vref < 0.0f) {  // (the same for all threads)
          // the maximum is lowered by as much as the head's largest 2^(s - m) vs lies below the largest V
          // scale, to 2^-100 at most, so that all factors stay within FP32
          const float lv = lg2_approx(vrel);
          float x[kHeads];
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            x[h] = s[h] - mt[h] + lv;
            const float mn = fmaxf(m[h], mt[h]), a = ex2_approx(m[h] - mn);  // (the row's maximum is the true one)
            m[h] = mn;
            l[h] *= a;
            o[h] *= a;
          }
          const float mine = reduce_heads<kHeads>(x, lane, larger);
          if (lane % (32 / kHeads) == 0) off[8 * warp + lane / (32 / kHeads)] = mine;
          __syncwarp();
          if (lane == 0) mbar_arrive(off_full);
          if (!(ok = warp_wait(off_full, nwide & 1, abort_flag))) break;
          ++nwide;
          const int lh = lane % kHeads;
          const float low = fminf(fmaxf(fmaxf(fmaxf(off[lh], off[8 + lh]), fmaxf(off[16 + lh], off[24 + lh])), -100.0f), 0.0f);
          // (rounded up: a product above 1 would not fit the signed-byte digits)
#pragma unroll
          for (int h = 0; h < kHeads; ++h) mt[h] = __fadd_ru(mt[h], __shfl_sync(0xffffffffu, low, h));
        }
        float pr[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float mn = fmaxf(m[h], mt[h]);
          alpha[h] = ex2_approx(m[h] - mn);  // (0 at the first tile)
          const float be = ex2_approx(mt[h] - mn);
          m[h] = mn;
          const float e = ex2_approx(s[h] - mt[h]);
          l[h] = fmaf(e, be, l[h] * alpha[h]);
          beta[h] = be * (vref * (kInt8 ? 1.0f / kInt8One : 1.0f / 256.0f));
          pr[h] = e * vrel;
        }
        uint8_t* pb = smem + Sm::p + buf * kCols * 128;
        auto put = [&](int part, int h, uint32_t byte) {
          const int n = part * kHeads + h;
          pb[n * 128 + (((tid >> 4) ^ (n & 7)) << 4) + (tid & 15)] = static_cast<uint8_t>(byte);
        };
#pragma unroll
        for (int h = 0; h < kHeads; h += 2) {
          if constexpr (kInt8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t v = split_int8(pr[h + e]);
#pragma unroll
              for (int pt = 0; pt < kParts; ++pt) put(pt, h + e, v >> (16 - 8 * pt));
            }
          } else {
            uint16_t part[kParts];
            split_e4m3(__floats2half2_rn(pr[h] * 256.0f, pr[h + 1] * 256.0f), part);
#pragma unroll
            for (int pt = 0; pt < kParts; ++pt) {
              put(pt, h, part[pt] & 0xFFu);
              put(pt, h + 1, part[pt] >> 8);
            }
          }
        }
        if (key0 + kTile > seg.cur_hi) {
          // rows past the legal keys: whatever the cache holds there (a NaN byte, say) must not
          // meet P = 0 in the product
          const int st = it % kStages;
          if (!(ok = warp_wait(&v_full[st], (it / kStages) & 1, abort_flag))) break;
          if (!legal) {
            uint4* row = reinterpret_cast<uint4*>(smem + Sm::v + st * kTileBytes + tid * 128);
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[buf]);
      }
      if (ok) ok = take_o(it - 1);
      if (!ok) break;
      // row sums over the keys (threads)
      float* lb = lred + (nseg & 1) * 32;
      const float lw = reduce_heads<kHeads>(l, lane, [](float a, float b) { return a + b; });
      if (lane % (32 / kHeads) == 0) lb[warp * 8 + lane / (32 / kHeads)] = lw;
      __syncwarp();
      if (lane == 0) mbar_arrive(l_full);
      if (!(ok = warp_wait(l_full, nseg & 1, abort_flag))) break;
      const int64_t slot = (static_cast<int64_t>(seg.cur_hb) * p.B + seg.cur_b) * p.Hkv + seg.cur_g + cta;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float sum = (lb[h] + lb[8 + h]) + (lb[16 + h] + lb[24 + h]);
        if (tid == h) reinterpret_cast<float2*>(p.part_ml)[slot * kHeads + h] = make_float2(m[h], sum);
        if (h >= nh) continue;
        if (seg.n == seg.cur_all) {  // the whole unit: no merge
          const int64_t row = static_cast<int64_t>(seg.cur_b) * p.Hq + head0 + h;
          p.out[row * 128 + tid] = __float2bfloat16_rn(o[h] / sum);
          if (tid == h) p.lse[row] = lg2_approx(sum) + m[h];
        } else {
          p.part_o[(slot * kHeads + h) * 128 + tid] = o[h];
        }
      }
      ++nseg;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 4 * kCols);
  }
  if (tid == 0) p.cta_status[cta] = *abort_flag ? kStatusTimeout : 0;
}

// Second kernel, blocks (c, y) for each CTA c of the first.
// The last kHeads values of y: where c's share holds the last but not the first tile of a
// unit, a block merges the segments of one of that unit's heads; the blocks also
// write the rows of sequences without a key.
// The y before those (with weights; they are dispatched first): the attention weights 2^(s - lse) of the keys of c's tiles,
// summed over the group's heads in a fixed order and added to the accumulated ones.  A
// warp takes a tile at a time, with all of its scores (4 keys a lane, kHeads heads) in
// flight at once: the pass is a chain of L2 latencies (share, sums, scores) over little data.
constexpr int kMergeThreads = 128;
constexpr int kWeightBlocks = 2;  // blocks over a CTA's tiles

template <int kHeads, bool kWeights>
__global__ void __launch_bounds__(kMergeThreads, kWeights ? 6 : 8) kv_decode_merge_kernel(const __grid_constant__ KvDecodeParams p) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = blockIdx.x, y = blockIdx.y;
  cudaGridDependencySynchronize();
  const KvShare sh = p.share[c];
  Segments seg{};
  seg.start(sh);
  constexpr int kFirstMerge = kWeights ? kWeightBlocks : 0;
  const auto gave_up = [&]() {  // whether a CTA of the first kernel did
    int st = 0;
    for (int i = tid; i < p.ctas; i += kMergeThreads) st |= p.cta_status[i];
    return __syncthreads_or(st) != 0;
  };
  if (y >= kFirstMerge) {
    const int h = y - kFirstMerge;
    if (c == 0 && h == 0) {
      const bool st = gave_up();
      if (tid == 0) *p.status = st ? kStatusTimeout : 0;
    }
    for (int b = c; b < p.B; b += p.ctas) {
      if (p.seq_lens[b] > 0) continue;
      // no key: 0 / 0 and log2 0, as the prefill writes a row without a legal key
      for (int hq = h; hq < p.Hq; hq += kHeads) {
        const int64_t row = static_cast<int64_t>(b) * p.Hq + hq;
        p.out[row * 128 + tid] = __float2bfloat16_rn(__uint_as_float(0x7FC00000u));
        if (tid == 0) p.lse[row] = -INFINITY;
      }
    }
    if (!seg.next(p) || seg.first == 0 || seg.first + seg.n < seg.cur_all) return;
    const int b = seg.cur_b, hb = seg.cur_hb;
    if (h >= min(kHeads, p.r - hb * kHeads)) return;
    const int first = share_of(seg.cur_vbase + sh.omega, sh.per, sh.longer);
    const int nseg = c - first + 1;
    const int64_t slot0 = (static_cast<int64_t>(hb) * p.B + b) * p.Hkv + seg.cur_g + first;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + slot0 * kHeads + h;
    // 32 segments at a time, a lane each for their maxima and sums; their O rows are on the way meanwhile
    const float* po = p.part_o + (slot0 * kHeads + h) * 128 + tid;
    float M = -INFINITY, L = 0.0f, acc = 0.0f;
    for (int i0 = 0; i0 < nseg; i0 += 32) {
      const int cnt = min(32, nseg - i0);
      const float2 x = lane < cnt ? ml[static_cast<int64_t>(i0 + lane) * kHeads] : make_float2(-INFINITY, 0.0f);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < cnt ? po[static_cast<int64_t>(i0 + j) * kHeads * 128] : 0.0f;
      const float mn = fmaxf(M, warp_max(x.x));
      const float w = lane < cnt ? ex2_approx(x.x - mn) : 0.0f;
      const float scale = M == -INFINITY ? 0.0f : ex2_approx(M - mn);
      float sum = x.y * w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      L = fmaf(L, scale, sum);
      acc *= scale;
      M = mn;
      for (int j0 = 0; j0 < cnt; j0 += 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc = fmaf(v[j], __shfl_sync(0xffffffffu, w, j0 + j), acc);
          const int k = j0 + 8 + j;
          v[j] = k < cnt ? po[static_cast<int64_t>(i0 + k) * kHeads * 128] : 0.0f;
        }
      }
    }
    const int64_t row = static_cast<int64_t>(b) * p.Hq + seg.cur_g * p.r + hb * kHeads + h;
    p.out[row * 128 + tid] = __float2bfloat16_rn(acc / L);
    if (tid == 0) p.lse[row] = lg2_approx(L) + M;
    return;
  }
  if constexpr (kWeights) {
    // Unlike O and LSE, accumulated weights cannot be computed again: a step that failed leaves them as they
    // are (0.7 us of 32 to 42; the same read warp by warp, in fewer words or beside the sums took as long).
    if (gave_up()) return;
    constexpr int kStep = kWeightBlocks * (kMergeThreads / 32);  // warps of the share
    int mine = y * (kMergeThreads / 32) + warp;                  // this warp's next tile, from the segment's first on
    while (seg.next(p)) {
      if (seg.cur_hb != 0) break;  // a key's tile of the first head block stands for the others' too
      const int64_t unit = static_cast<int64_t>(seg.cur_b) * p.Hkv + seg.cur_g;
      float* dst = p.weights + unit * p.Smax;
      float lse = 0.0f;  // of head lane % kHeads of head block `of`
      int of = -1;
      for (int i = mine; i < seg.n; i += kStep) {
        const int key0 = seg.cur_lo + (seg.first + i) * kTile + lane;
        float old[4], w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) old[j] = key0 + 32 * j < seg.cur_hi ? dst[key0 + 32 * j] : 0.0f;
        for (int hb = 0; hb < p.nhb; ++hb) {
          const int nh = min(kHeads, p.r - hb * kHeads);
          const float* sc = p.scores + static_cast<int64_t>(seg.cur_tbase + hb * sh.block_tiles + seg.first + i) * kHeads * kTile + lane;
          float s[kHeads][4];
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[h][j] = h < nh ? sc[h * kTile + 32 * j] : -INFINITY;
          }
          if (of != hb) {  // from the unit's segments, 32 / kHeads of them at a time
            of = hb;
            const int v0 = seg.cur_vbase + sh.omega + hb * sh.block_steps;  // the unit's first tile
            const int first = share_of(v0, sh.per, sh.longer);
            const int nseg = share_of(v0 + (seg.cur_all - 1) * kTileSteps, sh.per, sh.longer) - first + 1;
            const float2* ml = reinterpret_cast<const float2*>(p.part_ml) +
                               (static_cast<int64_t>(hb) * p.B * p.Hkv + unit + first) * kHeads;
            float M = -INFINITY, L = 0.0f;
#pragma unroll 4
            for (int k = lane; k < nseg * kHeads; k += 32) {
              const float2 x = ml[k];
              const float mn = fmaxf(M, x.x);
              L = fmaf(x.y, ex2_approx(x.x - mn), M == -INFINITY ? L : L * ex2_approx(M - mn));
              M = mn;
            }
#pragma unroll
            for (int o = kHeads; o < 32; o <<= 1) {
              const float mo = __shfl_xor_sync(0xffffffffu, M, o), lo = __shfl_xor_sync(0xffffffffu, L, o);
              const float mn = fmaxf(M, mo);
              L = (M == -INFINITY ? L : L * ex2_approx(M - mn)) + (mo == -INFINITY ? lo : lo * ex2_approx(mo - mn));
              M = mn;
            }
            lse = lg2_approx(L) + M;
          }
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            const float z = __shfl_sync(0xffffffffu, lse, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] += h < nh ? ex2_approx(s[h][j] - z) : 0.0f;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key0 + 32 * j < seg.cur_hi) dst[key0 + 32 * j] = old[j] + w[j];
      }
      mine -= seg.n;
      while (mine < 0) mine += kStep;
    }
  }
}

template <bool kInt8, int kHeads, bool kWeights>
cudaError_t launch_main(const KvDecodeParams& p, cudaStream_t stream) {
  static std::atomic<bool> attr_set[64];  // host threads may call at once; setting it twice does no harm
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kv_decode_kernel<kInt8, kHeads, kWeights>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             KvSmem<kHeads>::bytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev].store(true, std::memory_order_release);
  }
  e = launch_dependent(kv_decode_kernel<kInt8, kHeads, kWeights>, dim3(p.ctas), dim3(kThreads), KvSmem<kHeads>::bytes, stream, p);
  if (e != cudaSuccess) return e;
  return launch_dependent(kv_decode_merge_kernel<kHeads, kWeights>, dim3(p.ctas, kHeads + (kWeights ? kWeightBlocks : 0)),
                          dim3(kMergeThreads), 0, stream, p);
}

template <bool kInt8>
cudaError_t launch_for(const KvDecodeParams& p, cudaStream_t stream) {
  const bool w = p.weights != nullptr;
  if (p.heads == 4) return w ? launch_main<kInt8, 4, true>(p, stream) : launch_main<kInt8, 4, false>(p, stream);
  return w ? launch_main<kInt8, 8, true>(p, stream) : launch_main<kInt8, 8, false>(p, stream);
}

}  // namespace

cudaError_t launch_kv_decode(const KvDecodeParams& p, bool int8, cudaStream_t stream) {
  return int8 ? launch_for<true>(p, stream) : launch_for<false>(p, stream);
}

}  // namespace swa
