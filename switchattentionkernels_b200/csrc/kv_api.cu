// C ABI of the block-scaled 8-bit KV cache (declared in include/swattn_b200.h).
#include <algorithm>
#include <atomic>
#include <string>

#include "../../include/swattn_b200.h"
#include "kv_cache.h"
#include "swattn_internal.h"
#include "tma_host.h"

namespace {

int fail(int code, const std::string& msg) {
  swa::set_last_error(msg.c_str());
  return code;
}
int cuda_fail(cudaError_t e, const char* what) {
  return fail(SWA_E_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// SMs of the current device, asked once for each device.
int device_sms(int* nsm) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 64 && (*nsm = known[dev].load(std::memory_order_relaxed)) > 0) return SWA_OK;
  int major = 0;
  e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(nsm, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
  if (major != 10) return fail(SWA_E_UNSUPPORTED, "this library targets sm_100 (B200) devices");
  if (dev < 64) known[dev].store(*nsm, std::memory_order_relaxed);
  return SWA_OK;
}

// Shape checks shared by the three entry points.
int check_cache(int dtype, int B, int Hkv, int Smax, int block) {
  if (dtype != SWA_KV_E4M3 && dtype != SWA_KV_INT8) return fail(SWA_E_INVALID, "cache dtype must be e4m3 or int8");
  if (B <= 0 || Hkv <= 0 || Smax <= 0) return fail(SWA_E_INVALID, "empty or negative shape");
  if (block != 16 && block != 32 && block != 64 && block != 128)
    return fail(SWA_E_INVALID, "block_size must be 16, 32, 64 or 128");
  if (Smax > (1 << 30)) return fail(SWA_E_UNSUPPORTED, "more than 2^30 rows in a sequence");
  return SWA_OK;
}

// Head blocks of the decode kernel: 4 query heads fill its 16-column tiles, 8 its
// 32-column ones.
struct KvDecodePlan {
  int heads, nhb, ctas;
  int64_t slots, tiles;
  size_t share, cta_status, ml, o, scores, bytes;  // offsets of the workspace's parts, and its size
};

KvDecodePlan plan_decode(int B, int Smax, int Hq, int Hkv, bool weights, int nsm) {
  KvDecodePlan d{};
  const int r = Hq / Hkv;
  d.heads = r <= 4 ? 4 : 8;
  d.nhb = (r + d.heads - 1) / d.heads;
  const int64_t units = static_cast<int64_t>(B) * Hkv * d.nhb;
  d.tiles = units * ((static_cast<int64_t>(Smax) + 127) / 128);
  d.ctas = static_cast<int>(std::min<int64_t>(d.tiles, static_cast<int64_t>(nsm) * swa::kKvDecodeCtasPerSm));
  d.slots = units + d.ctas;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  d.share = 256;  // the status word first
  d.cta_status = up(d.share + static_cast<size_t>(d.ctas) * sizeof(swa::KvShare));
  d.ml = up(d.cta_status + static_cast<size_t>(d.ctas) * 4);
  d.o = up(d.ml + static_cast<size_t>(d.slots) * d.heads * 8);
  d.scores = up(d.o + static_cast<size_t>(d.slots) * d.heads * 512);
  d.bytes = d.scores + (weights ? static_cast<size_t>(d.tiles) * d.heads * 512 : 0);
  return d;
}

}  // namespace

extern "C" {

int swa_kv_append(const void* k_new, const void* v_new, int64_t k_stride_b, int64_t k_stride_t, int64_t k_stride_h,
                  int64_t v_stride_b, int64_t v_stride_t, int64_t v_stride_h, const int32_t* start, const int32_t* new_lens, void* k_cache, void* v_cache, float* k_scale,
                  float* v_scale, float* key_weights, int32_t* seq_lens, int B, int T, int Hkv, int Smax,
                  int head_dim, int block_size, int dtype, void* stream) {
  if (head_dim != 128) return fail(SWA_E_UNSUPPORTED, "head_dim must be 128");
  int rc = check_cache(dtype, B, Hkv, Smax, block_size);
  if (rc != SWA_OK) return rc;
  if (T <= 0) return fail(SWA_E_INVALID, "empty or negative shape");
  if (k_new == nullptr || v_new == nullptr || start == nullptr ||
      k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || seq_lens == nullptr)
    return fail(SWA_E_INVALID, "null pointer");
  if (!aligned16(k_new) || !aligned16(v_new) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(SWA_E_INVALID, "k/v and the caches must be 16-byte aligned");
  if (k_cache == v_cache || k_scale == v_scale) return fail(SWA_E_INVALID, "K and V must not share a cache");
  const int64_t strides[2][3] = {{k_stride_b, k_stride_t, k_stride_h}, {v_stride_b, v_stride_t, v_stride_h}};
  for (const auto& s : strides)
    if (s[0] % 8 != 0 || s[1] % 8 != 0 || s[2] % 8 != 0)
      return fail(SWA_E_INVALID, "strides of k/v must be multiples of 8 elements");
  for (const int32_t* t : {start, new_lens})
    if (t != nullptr && t != seq_lens && t < seq_lens + B && seq_lens < t + B)
      return fail(SWA_E_INVALID, "start and new_lens may be seq_lens but not overlap it otherwise");
  if (T > 1 && (B > 65535 || 2 * static_cast<int64_t>(Hkv) > 65535))
    return fail(SWA_E_UNSUPPORTED, "append grid: at most 65535 sequences and 32767 KV heads");
  int nsm = 0;
  rc = device_sms(&nsm);
  if (rc != SWA_OK) return rc;
  swa::KvAppendParams p{};
  p.x[0] = static_cast<const __nv_bfloat16*>(k_new);
  p.x[1] = static_cast<const __nv_bfloat16*>(v_new);
  for (int kv = 0; kv < 2; ++kv) {
    p.sb[kv] = strides[kv][0];
    p.st[kv] = strides[kv][1];
    p.sh[kv] = strides[kv][2];
  }
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.weights = key_weights;
  p.start = start;
  p.new_lens = new_lens;
  p.seq_lens = seq_lens;
  p.lens_after = start == seq_lens || new_lens == seq_lens;
  p.B = B;
  p.T = std::min(T, Smax);  // later rows are dropped wherever they start; row numbers stay below 2^31
  p.Hkv = Hkv;
  p.Smax = Smax;
  p.block = block_size;
  p.nblk = (Smax + block_size - 1) / block_size;
  cudaError_t e = swa::launch_kv_append(p, dtype == SWA_KV_INT8, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "KV append launch");
  return SWA_OK;
}

size_t swa_kv_decode_workspace_bytes(int B, int Smax, int Hq, int Hkv, int with_weights) {
  if (B <= 0 || Smax <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) {
    swa::set_last_error("empty or negative shape");
    return 0;
  }
  int nsm = 0;
  if (device_sms(&nsm) != SWA_OK) return 0;
  return plan_decode(B, Smax, Hq, Hkv, with_weights != 0, nsm).bytes;
}

int swa_kv_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache, const void* v_cache,
                  const float* k_scale, const float* v_scale, const int32_t* seq_lens, const uint8_t* route,
                  void* out, float* lse, float* key_weights, int B, int Smax, int Hq, int Hkv, int head_dim,
                  int block_size, int window, float scale_log2, int dtype, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (head_dim != 128) return fail(SWA_E_UNSUPPORTED, "head_dim must be 128");
  int rc = check_cache(dtype, B, Hkv, Smax, block_size);
  if (rc != SWA_OK) return rc;
  if (Hq <= 0) return fail(SWA_E_INVALID, "empty or negative shape");
  if (Hq % Hkv != 0) return fail(SWA_E_INVALID, "query heads must be divisible by KV heads");
  if (window <= 0) return fail(SWA_E_INVALID, "window_size must be positive");
  if (!(scale_log2 > 0.0f)) return fail(SWA_E_INVALID, "softmax scale must be positive");
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr ||
      seq_lens == nullptr || route == nullptr || out == nullptr || lse == nullptr || workspace == nullptr)
    return fail(SWA_E_INVALID, "null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
    return fail(SWA_E_INVALID, "q/k/v/workspace must be 16-byte aligned");
  if (q_stride_b % 8 != 0 || q_stride_h % 8 != 0)
    return fail(SWA_E_INVALID, "strides of q must be multiples of 8 elements");
  int nsm = 0;
  rc = device_sms(&nsm);
  if (rc != SWA_OK) return rc;
  const KvDecodePlan d = plan_decode(B, Smax, Hq, Hkv, key_weights != nullptr, nsm);
  if (d.tiles >= (int64_t(1) << 28) || static_cast<int64_t>(B) * Hq + d.ctas >= (int64_t(1) << 31))
    return fail(SWA_E_UNSUPPORTED, "KV cache too large for 32-bit tile indices");
  if (workspace_bytes < d.bytes) return fail(SWA_E_INVALID, "workspace too small");
  swa::KvDecodeParams p{};
  const uint64_t dims[3] = {128, static_cast<uint64_t>(Smax), static_cast<uint64_t>(B) * Hkv};
  const uint64_t strides[2] = {128, static_cast<uint64_t>(Smax) * 128};
  const uint32_t box[3] = {128, 128, 1};
  if (!swa::make_u8_map_sw128(&p.map[0], k_cache, 3, dims, strides, box)) return fail(SWA_E_TMA, "k tensor map");
  if (!swa::make_u8_map_sw128(&p.map[1], v_cache, 3, dims, strides, box)) return fail(SWA_E_TMA, "v tensor map");
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.seq_lens = seq_lens;
  p.route = route;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.weights = key_weights;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.status = reinterpret_cast<int32_t*>(ws);
  p.share = reinterpret_cast<swa::KvShare*>(ws + d.share);
  p.cta_status = reinterpret_cast<int32_t*>(ws + d.cta_status);
  p.part_ml = reinterpret_cast<float*>(ws + d.ml);
  p.part_o = reinterpret_cast<float*>(ws + d.o);
  p.scores = reinterpret_cast<float*>(ws + d.scores);
  p.B = B;
  p.Smax = Smax;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.r = Hq / Hkv;
  p.nblk = (Smax + block_size - 1) / block_size;
  p.block_shift = block_size == 16 ? 4 : (block_size == 32 ? 5 : (block_size == 64 ? 6 : 7));
  p.window = window;
  p.heads = d.heads;
  p.nhb = d.nhb;
  p.ctas = d.ctas;
  p.scale_log2 = scale_log2;
  p.test_withhold = swa::test_withhold();
  cudaError_t e = swa::launch_kv_decode(p, dtype == SWA_KV_INT8, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "KV decode launch");
  return SWA_OK;
}

int swa_kv_evict(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                 const float* key_weights, const int32_t* seq_lens, void* k_out, void* v_out, float* k_scale_out,
                 float* v_scale_out, float* key_weights_out, int32_t* seq_lens_out, int32_t* slots, int B, int Hkv,
                 int Smax, int Smax_out, int head_dim, int block_size, int keep, int sink, int recent, int dtype,
                 void* stream) {
  if (head_dim != 128) return fail(SWA_E_UNSUPPORTED, "head_dim must be 128");
  int rc = check_cache(dtype, B, Hkv, Smax, block_size);
  if (rc != SWA_OK) return rc;
  if (keep <= 0 || sink < 0 || recent < 0 || static_cast<int64_t>(sink) + recent > keep)
    return fail(SWA_E_INVALID, "keep must be positive and at least sink + recent, both non-negative");
  if (k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || key_weights == nullptr ||
      seq_lens == nullptr || k_out == nullptr || v_out == nullptr || k_scale_out == nullptr ||
      v_scale_out == nullptr || key_weights_out == nullptr || seq_lens_out == nullptr || slots == nullptr)
    return fail(SWA_E_INVALID, "null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return fail(SWA_E_INVALID, "the caches must be 16-byte aligned");
  if (k_out == v_out || k_scale_out == v_scale_out) return fail(SWA_E_INVALID, "K and V must not share a cache");
  const int n = std::min(keep, Smax);
  if (Smax_out < n) return fail(SWA_E_INVALID, "the destination holds fewer rows than are kept");
  const bool same[6] = {k_cache == k_out, v_cache == v_out, k_scale == k_scale_out, v_scale == v_scale_out,
                        key_weights == key_weights_out, seq_lens == seq_lens_out};
  const int n_same = static_cast<int>(std::count(same, same + 6, true));
  if ((n_same != 0 && n_same != 6) || (n_same == 6 && Smax_out != Smax))
    return fail(SWA_E_INVALID, "the destination must be the source (in place) or share nothing with it");
  const int64_t tiles = static_cast<int64_t>(B) * Hkv * std::max<int64_t>(8, (static_cast<int64_t>(n) + 127) / 128);
  if (tiles >= (int64_t(1) << 31)) return fail(SWA_E_UNSUPPORTED, "KV cache too large for 32-bit tile indices");
  int nsm = 0;
  rc = device_sms(&nsm);
  if (rc != SWA_OK) return rc;
  swa::KvEvictParams p{};
  p.src[0] = static_cast<const uint8_t*>(k_cache);
  p.src[1] = static_cast<const uint8_t*>(v_cache);
  p.src_scale[0] = k_scale;
  p.src_scale[1] = v_scale;
  p.src_weights = key_weights;
  p.dst[0] = static_cast<uint8_t*>(k_out);
  p.dst[1] = static_cast<uint8_t*>(v_out);
  p.dst_scale[0] = k_scale_out;
  p.dst_scale[1] = v_scale_out;
  p.dst_weights = key_weights_out;
  p.seq_lens = seq_lens;
  p.dst_lens = seq_lens_out;
  p.slots = slots;
  p.B = B;
  p.Hkv = Hkv;
  p.Smax = Smax;
  p.Smax_dst = Smax_out;
  p.nblk = (Smax + block_size - 1) / block_size;
  p.nblk_dst = (Smax_out + block_size - 1) / block_size;
  p.block = block_size;
  p.n = n;
  p.keep = keep;
  p.sink = sink;
  p.recent = recent;
  cudaError_t e = swa::launch_kv_evict(p, dtype == SWA_KV_INT8, n_same == 6, nsm, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "KV evict launch");
  return SWA_OK;
}

}  // extern "C"
