// Block-scaled 8-bit KV cache: parameters shared by its kernels and entry points.
//
// K and V are [B, Hkv, Smax, 128] bytes (e4m3 or int8): the rows of one KV head lie
// together, so 128 keys are one contiguous 16 KB tile (the token-major layout of
// the BF16 cache would make it 128 pieces of 128 bytes).  Every block of `block`
// rows (16, 32, 64 or 128) of a head has one FP32 scale for K and one for V,
// [B, Hkv, nblk], nblk = ceil(Smax / block): value = byte * scale.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>

namespace swa {

// Launches `kernel` as the dependent of the kernel before it on the stream: its CTAs may
// start while that one still runs, and wait (cudaGridDependencySynchronize) for its
// end before they touch global memory.  Every kernel launched this way does so in every
// CTA, so that its own end implies the end of all kernels before it.
// cluster > 1: clusters of that many CTAs along x.
template <typename... Params, typename... Args>
cudaError_t launch_cluster_dependent(int cluster, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                                     cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                             Args&&... args) {
  return launch_cluster_dependent(1, kernel, grid, block, smem, stream, static_cast<Args&&>(args)...);
}

struct KvAppendParams {
  const __nv_bfloat16* x[2];  // new K, V rows: element (b, t, g, d) at b * sb + t * st + g * sh + d
  int64_t sb[2], st[2], sh[2];
  uint8_t* cache[2];          // [B, Hkv, Smax, 128]
  float* scale[2];            // [B, Hkv, nblk]
  float* weights;             // [B, Hkv, Smax] or null; new rows start at 0
  const int32_t* start;       // [B] rows already cached (may be seq_lens)
  const int32_t* new_lens;    // [B] new rows of each sequence, or null: T
  int32_t* seq_lens;          // [B] written: rows cached after the call
  bool lens_after;            // start (or new_lens) is seq_lens: written once every CTA has read it
  int B, T, Hkv, Smax, nblk, block;
};
cudaError_t launch_kv_append(const KvAppendParams& p, bool int8, cudaStream_t stream);

struct KvEvictParams {
  const uint8_t* src[2];      // K, V caches [B, Hkv, Smax, 128]
  const float* src_scale[2];  // [B, Hkv, nblk]
  const float* src_weights;   // [B, Hkv, Smax]
  uint8_t* dst[2];            // [B, Hkv, Smax_dst, 128]; in place: the same pointers
  float* dst_scale[2];        // [B, Hkv, nblk_dst]
  float* dst_weights;         // [B, Hkv, Smax_dst]
  const int32_t* seq_lens;    // [B]
  int32_t* dst_lens;          // [B] written: min(length, keep); in place: seq_lens
  int32_t* slots;             // [B, Hkv, n] written: source row of each kept row, -1 past the count
  int B, Hkv, Smax, Smax_dst, nblk, nblk_dst, block, n, keep, sink, recent;
};
cudaError_t launch_kv_evict(const KvEvictParams& p, bool int8, bool in_place, int num_sms, cudaStream_t stream);

// Decode over the cache.  The (sequence, KV head, head block) units' legal keys are
// cut into tiles of 128 keys.  All units of the batch are laid end to end along one axis
// of work, in the order (head block, sequence, KV head), each as `omega` steps for
// starting it and kTileSteps for every tile, and the axis is cut into equal shares, one
// a CTA: a tile belongs to the CTA on whose share its first step lies.  (The head blocks
// are outermost so that the CTAs that read the same keys for different heads do so at
// the same time, all but one of them from L2.)  A CTA's part of one unit is a segment; its
// partial result lies in slot unit + cta (both grow along the axis and each new segment
// moves one of them, so slots are distinct).
constexpr int kTileSteps = 2;

// What CTA c's share begins with, and the whole plan.
struct __align__(16) KvShare {
  int hb, b, g;           // head block, sequence, KV head
  int off, left;          // first step in the unit, steps of the share
  int vbase, tbase;       // steps and tiles before the unit
  int lo, hi;             // legal keys of the sequence
  int omega;              // of the batch, as are
  int per, longer;        // steps of a share; the first `longer` shares have one more
  int block_steps, block_tiles;  // steps and tiles of one head block's units
  int pad[2];
};

struct __align__(64) KvDecodeParams {
  CUtensorMap map[2];         // K, V bytes: 3-D {128, Smax, B * Hkv}, box {128, 128, 1}, 128B swizzle
  const __nv_bfloat16* q;     // element (b, h, d) at b * q_sb + h * q_sh + d
  int64_t q_sb, q_sh;
  const float* scale[2];      // [B, Hkv, nblk]
  const int32_t* seq_lens;    // [B] cached keys, the new token's included
  const uint8_t* route;       // [B] non-zero = full attention
  __nv_bfloat16* out;         // [B, Hq, 128]
  float* lse;                 // [B, Hq]
  float* weights;             // [B, Hkv, Smax] added to, or null
  // workspace
  KvShare* share;             // [ctas]
  int32_t* cta_status;        // [ctas]
  int32_t* status;
  float* part_ml;             // [slots, heads, 2] maximum and sum of each partial row
  float* part_o;              // [slots, heads, 128]
  float* scores;              // [tiles, heads, 128] log2-domain scores (with weights)
  int B, Smax, Hq, Hkv, r, nblk, block_shift, window;
  int heads;                  // query heads of a head block: 4 or 8
  int nhb;                    // head blocks per KV head
  int ctas;
  float scale_log2;
  int test_withhold;          // failure-detection test hook: CTA 0 withholds its second K tile
};
cudaError_t launch_kv_decode(const KvDecodeParams& p, bool int8, cudaStream_t stream);
// Resident CTAs of the decode kernel per SM (what its shared memory allows).
constexpr int kKvDecodeCtasPerSm = 2;

}  // namespace swa
