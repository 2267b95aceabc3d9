// Writing the 8-bit KV cache and reading it back (format: mxfp8.h).
//
// Store: token t's [Hkv, D] rows of key and value are quantised into slot slot_mapping[t] (page slot / block_size, row
// slot % block_size), tokens with a slot outside the cache are skipped: store_kvcache.hip's contract. A lane takes 8
// elements (one 16-byte load, one 8-byte store), 4 lanes a block of 32, whose largest magnitude is two DPP steps; nothing
// else is shared. Load: the tokens of sequence b, cu[b] .. cu[b+1] - 1 of the output, from the pages of block_table row b,
// in bf16.
//
// Both are bound by HBM. Their lanes run over (token group, K / V, head, token, element): consecutive tokens of a head
// are neighbours in the cache, so a block's codes are one run of 32 x 128 bytes and its scales whole lines.
#include <algorithm>

#include "mxfp8.h"

namespace nvhip {
namespace {

constexpr int kThreads = 256;

struct MxCache {
  uint8_t* code[2];   // k, v
  uint8_t* scale[2];
  int64_t bs, num_blocks;
  int Hkv;
};

// Row of (slot, head) in the caches.
__device__ __forceinline__ int64_t cache_row(const MxCache& c, int64_t blk, int64_t off, int h) {
  return (blk * c.Hkv + h) * c.bs + off;
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_row8(const void* base, int64_t elem, float* x) {
  if constexpr (std::is_same_v<T, float>) {
    const float* p = static_cast<const float*>(base) + elem;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    if constexpr (ALIGNED) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  } else {
    const u32x4 w = load8<ALIGNED>(static_cast<const uint16_t*>(base) + elem);
    if constexpr (std::is_same_v<T, _Float16>) {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t word = w[i];  // a bit_cast of the vector's element itself takes element 0
        const f16x2 h = __builtin_bit_cast(f16x2, word);
        x[2 * i] = float(h[0]), x[2 * i + 1] = float(h[1]);
      }
    } else {
      unpack8(w, x);
    }
  }
}

struct StoreArgs {
  MxCache c;
  const void* src[2];
  int64_t stride[2];  // elements between tokens
  const int32_t* slots;
  int64_t n, threads;  // tokens; lanes of work
  int group;           // tokens per group
};

template <typename T, int D, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void store_mxfp8_kernel(const StoreArgs g) {
  constexpr int LPR = D / 8;  // lanes per row
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= g.threads) return;  // whole rows leave together
  const int sub = int(i % LPR);
  const int64_t row = i / LPR, rest = row / g.group;
  const int hk = int(rest % (2 * g.c.Hkv)), kv = hk >= g.c.Hkv, h = hk - kv * g.c.Hkv;
  const int64_t t = rest / (2 * g.c.Hkv) * g.group + row % g.group;
  if (t >= g.n) return;
  const int64_t slot = g.slots[t];
  float x[8];
  load_row8<T, ALIGNED>(g.src[kv], t * g.stride[kv] + int64_t(h) * D + sub * 8, x);
  if (slot < 0 || slot >= g.c.num_blocks * g.c.bs) return;
  float a = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = fmaxf(a, finite_abs(x[e]));
  const uint32_t byte = mx_scale_byte(quad_max(a));
  const int64_t blk = slot / g.c.bs, r = cache_row(g.c, blk, slot - blk * g.c.bs, h);
  *reinterpret_cast<u32x2*>(g.c.code[kv] + r * D + sub * 8) = mx_encode8(x, mx_scale(byte));
  if (sub % 4 == 0) g.c.scale[kv][r * (D / kMxBlock) + sub / 4] = uint8_t(byte);
}

struct LoadArgs {
  MxCache c;
  uint16_t* out[2];  // [total, Hkv, D]
  const int32_t* bt;
  const int32_t* cu;
  int64_t total, threads;
  int num_seqs, max_blocks, group;
};

template <int D>
__global__ __launch_bounds__(kThreads) void load_mxfp8_kernel(const LoadArgs g) {
  constexpr int LPR = D / 8;
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= g.threads) return;
  const int sub = int(i % LPR);
  const int64_t row = i / LPR, rest = row / g.group;
  const int hk = int(rest % (2 * g.c.Hkv)), kv = hk >= g.c.Hkv, h = hk - kv * g.c.Hkv;
  const int64_t t = rest / (2 * g.c.Hkv) * g.group + row % g.group;
  if (t >= g.total) return;
  int lo = 0, hi = g.num_seqs;  // the last sequence that begins at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (g.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int64_t pos = t - g.cu[lo], page = pos / g.c.bs;
  int64_t blk = -1;
  if (pos >= 0 && t < g.cu[lo + 1] && page < g.max_blocks) blk = g.bt[int64_t(lo) * g.max_blocks + page];
  u32x4 v = {};  // a row behind the last sequence or in no valid page is 0
  if (blk >= 0 && blk < g.c.num_blocks) {
    const int64_t r = cache_row(g.c, blk, pos - page * g.c.bs, h);
    const u32x2 w = *reinterpret_cast<const u32x2*>(g.c.code[kv] + r * D + sub * 8);
    v = mx_decode8(w[0], w[1], mx_scale(g.c.scale[kv][r * (D / kMxBlock) + sub / 4]));
  }
  *reinterpret_cast<u32x4*>(g.out[kv] + (t * g.c.Hkv + h) * D + sub * 8) = v;
}

// Tokens per group: 32 (the codes of a head's group then fill 32 rows in a run) unless that leaves CUs without a block.
int group_of(int64_t tokens) { return tokens >= 512 ? 32 : tokens >= 64 ? 8 : 1; }

int check_cache(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int64_t num_blocks,
                int64_t block_size, int64_t Hkv, int64_t D) {
  const std::string w(what);
  if (num_blocks < 0 || block_size < 1 || Hkv < 1 || Hkv > (1 << 20)) return invalid(w + ": bad size");
  if (D != 64 && D != 128 && D != 256) return invalid(w + ": head_dim must be 64, 128 or 256");
  if (num_blocks > INT32_MAX || block_size > INT32_MAX || num_blocks * block_size > INT32_MAX)
    return invalid(w + ": size too large");
  if (num_blocks > 0 && (!kc || !vc || !ks || !vs)) return invalid(w + ": null pointer");
  if (!aligned16(kc) || !aligned16(vc) || !aligned16(ks) || !aligned16(vs))
    return invalid(w + ": the caches and scales must be 16-byte aligned");
  return NVHIP_OK;
}

}  // namespace
}  // namespace nvhip

extern "C" int nvhip_store_kvcache_mxfp8(void* k_cache, void* v_cache, void* k_scales, void* v_scales, const void* key,
                                         const void* value, int64_t key_stride, int64_t value_stride,
                                         const int32_t* slot_mapping, int64_t num_blocks, int64_t block_size, int64_t n,
                                         int64_t Hkv, int64_t D, int dtype, void* stream) {
  using namespace nvhip;
  clear_error();
  if (int rc = check_cache("store_kvcache_mxfp8", k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, Hkv, D))
    return rc;
  if (n < 0 || n > INT32_MAX) return invalid("store_kvcache_mxfp8: bad number of tokens");
  if (dtype != NVHIP_DTYPE_F32 && dtype != NVHIP_DTYPE_BF16 && dtype != NVHIP_DTYPE_F16)
    return invalid("store_kvcache_mxfp8: unsupported dtype");
  if (key_stride < Hkv * D || value_stride < Hkv * D) return invalid("store_kvcache_mxfp8: row stride < row size");
  if (n == 0 || num_blocks == 0) return NVHIP_OK;
  if (!key || !value || !slot_mapping) return invalid("store_kvcache_mxfp8: null pointer");
  StoreArgs g{};
  g.c = MxCache{{static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache)},
                {static_cast<uint8_t*>(k_scales), static_cast<uint8_t*>(v_scales)}, block_size, num_blocks, int(Hkv)};
  g.src[0] = key, g.src[1] = value, g.stride[0] = key_stride, g.stride[1] = value_stride;
  g.slots = slot_mapping, g.n = n, g.group = group_of(n);
  g.threads = (n + g.group - 1) / g.group * g.group * 2 * Hkv * (D / 8);
  const int64_t blocks = (g.threads + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return invalid("store_kvcache_mxfp8: size too large");
  const int64_t per16 = dtype == NVHIP_DTYPE_F32 ? 4 : 8;  // elements in 16 bytes
  const bool aligned = aligned16(key) && aligned16(value) && key_stride % per16 == 0 && value_stride % per16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int d = decltype(dim)::value;
    if (aligned) hipLaunchKernelGGL((store_mxfp8_kernel<T, d, true>), dim3(unsigned(blocks)), dim3(kThreads), 0, s, g);
    else hipLaunchKernelGGL((store_mxfp8_kernel<T, d, false>), dim3(unsigned(blocks)), dim3(kThreads), 0, s, g);
    return check_launch("store_kvcache_mxfp8");
  };
  auto by_dim = [&](auto type) {
    if (D == 64) return launch(type, std::integral_constant<int, 64>{});
    if (D == 128) return launch(type, std::integral_constant<int, 128>{});
    return launch(type, std::integral_constant<int, 256>{});
  };
  if (dtype == NVHIP_DTYPE_F32) return by_dim(float{});
  if (dtype == NVHIP_DTYPE_F16) return by_dim(_Float16{});
  return by_dim(uint16_t{});
}

extern "C" int nvhip_load_kvcache_mxfp8(void* k, void* v, const void* k_cache, const void* v_cache, const void* k_scales,
                                        const void* v_scales, const int32_t* block_table, const int32_t* cu_seqlens_k,
                                        int64_t num_seqs, int64_t total, int64_t Hkv, int64_t D, int64_t block_size,
                                        int64_t num_blocks, int64_t max_blocks, void* stream) {
  using namespace nvhip;
  clear_error();
  if (int rc = check_cache("load_kvcache_mxfp8", k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, Hkv, D))
    return rc;
  if (num_seqs < 0 || num_seqs >= INT32_MAX || total < 0 || total > INT32_MAX || max_blocks < 0 || max_blocks > INT32_MAX)
    return invalid("load_kvcache_mxfp8: bad size");
  if (total == 0) return NVHIP_OK;
  if (!k || !v || !cu_seqlens_k || (num_seqs > 0 && max_blocks > 0 && !block_table))
    return invalid("load_kvcache_mxfp8: null pointer");
  if (num_seqs == 0) return invalid("load_kvcache_mxfp8: rows to read but no sequence");
  if (!aligned16(k) || !aligned16(v)) return invalid("load_kvcache_mxfp8: outputs must be 16-byte aligned");
  LoadArgs g{};
  auto bytes = [](const void* p) { return static_cast<uint8_t*>(const_cast<void*>(p)); };
  g.c = MxCache{{bytes(k_cache), bytes(v_cache)}, {bytes(k_scales), bytes(v_scales)}, block_size, num_blocks, int(Hkv)};
  g.out[0] = static_cast<uint16_t*>(k), g.out[1] = static_cast<uint16_t*>(v);
  g.bt = block_table, g.cu = cu_seqlens_k, g.total = total;
  g.num_seqs = int(num_seqs), g.max_blocks = int(max_blocks), g.group = group_of(total);
  g.threads = (total + g.group - 1) / g.group * g.group * 2 * Hkv * (D / 8);
  const int64_t blocks = (g.threads + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return invalid("load_kvcache_mxfp8: size too large");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
  if (D == 64) hipLaunchKernelGGL(load_mxfp8_kernel<64>, grid, block, 0, s, g);
  else if (D == 128) hipLaunchKernelGGL(load_mxfp8_kernel<128>, grid, block, 0, s, g);
  else hipLaunchKernelGGL(load_mxfp8_kernel<256>, grid, block, 0, s, g);
  return check_launch("load_kvcache_mxfp8");
}
