// Writing the 8-bit KV cache and reading it back (format: mxfp8.h).
//
// Store: token t's [Hkv, D] rows of key and value are quantised into slot slot_mapping[t] (page slot / block_size, row
// slot % block_size), tokens with a slot outside the cache are skipped: store_kvcache.hip's contract. A lane takes 8
// elements (one 16-byte load, one 8-byte store), 4 lanes a block of 32, whose largest magnitude is two DPP steps; nothing
// else is shared. Load: the tokens of sequence b, cu[b] .. cu[b+1] - 1 of the output, from the pages of block_table row b,
// in bf16, 8 elements a lane.
//
// Both are bound by HBM. blockIdx.y is a head of K or V, a block takes consecutive tokens of it: they are neighbours in the
// cache, so its codes are runs of 128-byte rows and its scales whole lines. Each lane has U tokens' loads on the way at
// once. Times (8 heads of 128, pages of 256; both launches of a write and read-back): 11.9k tokens written and read 30.5 us
// (148 MB, 4.9 TB/s), 27.9k read and 1250 written 35 us (181 MB, 5.2 TB/s); with a flat grid and six 64-bit divisions a
// lane 43.5 and 68.
#include <algorithm>

#include "mxfp8.h"

namespace nvhip {
namespace {

constexpr int kThreads = 256;

struct MxCache {
  uint8_t* code[2];   // k, v
  uint8_t* scale[2];
  uint32_t bs, slots;  // rows of a page, rows of all pages
  int Hkv;
};

// Row of (page, row in the page, head) in the caches.
__device__ __forceinline__ int64_t cache_row(const MxCache& c, uint32_t blk, uint32_t off, int h) {
  return (int64_t(blk) * c.Hkv + h) * c.bs + off;
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
  int n;
};

template <typename T, int D, bool ALIGNED, int U>
__global__ __launch_bounds__(kThreads) void store_mxfp8_kernel(const StoreArgs g) {
  constexpr int LPR = D / 8, TPP = kThreads / LPR;  // lanes per row, tokens per pass
  const int sub = threadIdx.x % LPR, kv = int(blockIdx.y) >= g.c.Hkv, h = int(blockIdx.y) - kv * g.c.Hkv;
  const int t0 = int(blockIdx.x) * (TPP * U) + threadIdx.x / LPR;
  float x[U][8];
  uint32_t slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u * TPP;
    slot[u] = UINT32_MAX;
    if (t >= g.n) continue;  // whole rows
    slot[u] = uint32_t(g.slots[t]);  // a negative one is past the last, too
    load_row8<T, ALIGNED>(g.src[kv], t * g.stride[kv] + int64_t(h) * D + sub * 8, x[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (slot[u] >= g.c.slots) continue;
    float a = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, finite_abs(x[u][e]));
    const uint32_t byte = mx_scale_byte(quad_max(a)), blk = slot[u] / g.c.bs;
    const int64_t r = cache_row(g.c, blk, slot[u] - blk * g.c.bs, h);
    *reinterpret_cast<u32x2*>(g.c.code[kv] + r * D + sub * 8) = mx_encode8(x[u], mx_scale(byte));
    if (sub % 4 == 0) g.c.scale[kv][r * (D / kMxBlock) + sub / 4] = uint8_t(byte);
  }
}

struct LoadArgs {
  MxCache c;
  uint16_t* out[2];  // [total, Hkv, D]
  const int32_t* bt;
  const int32_t* cu;
  int total, num_seqs, max_blocks, num_blocks;
};

template <int D, int U>
__global__ __launch_bounds__(kThreads) void load_mxfp8_kernel(const LoadArgs g) {
  constexpr int LPR = D / 8, TPP = kThreads / LPR;
  const int sub = threadIdx.x % LPR, kv = int(blockIdx.y) >= g.c.Hkv, h = int(blockIdx.y) - kv * g.c.Hkv;
  const int first = int(blockIdx.x) * (TPP * U);
  // the last sequence that begins at or before the block's first token
  int lo = 0, hi = g.num_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (load_uniform(g.cu + mid) <= first) lo = mid;
    else hi = mid;
  }
  int64_t row[U];
  u32x2 code[U];
  uint32_t scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = first + u * TPP + int(threadIdx.x) / LPR;
    row[u] = -1;
    if (t >= g.total) continue;
    int b = lo;
    while (b + 1 < g.num_seqs && g.cu[b + 1] <= t) ++b;  // this token's: few steps, unless sequences are very short
    const int pos = t - g.cu[b];
    const uint32_t page = uint32_t(pos) / g.c.bs;
    int blk = -1;
    if (pos >= 0 && t < g.cu[b + 1] && page < uint32_t(g.max_blocks)) blk = g.bt[int64_t(b) * g.max_blocks + page];
    if (blk >= 0 && blk < g.num_blocks) row[u] = cache_row(g.c, blk, uint32_t(pos) - page * g.c.bs, h);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] < 0) continue;
    code[u] = *reinterpret_cast<const u32x2*>(g.c.code[kv] + row[u] * D + sub * 8);
    scale[u] = g.c.scale[kv][row[u] * (D / kMxBlock) + sub / 4];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = first + u * TPP + int(threadIdx.x) / LPR;
    if (t >= g.total) continue;
    // a row behind the last sequence or in no valid page is 0
    const u32x4 v = row[u] < 0 ? u32x4{} : mx_decode8(code[u][0], code[u][1], mx_scale(scale[u]));
    // with the nontemporal hint: 27.9k tokens 57.7 -> 34.8 us (written through the L2 60.9)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(g.out[kv] + (int64_t(t) * g.c.Hkv + h) * D + sub * 8));
  }
}

// Tokens a lane has on the way: 2 where that leaves every CU two blocks, else 1 (27.9k tokens read back: 1, 2, 4, 8 tokens
// 37.8, 34.8, 35.5, 38.6 us; 3.7k tokens 9.4, 9.6, 10.5, 12.8).
bool two_tokens(int64_t tokens, int64_t Hkv, int64_t D) { return tokens * 2 * Hkv * D >= int64_t(512) * 2 * kThreads * 8; }

int check_cache(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int64_t num_blocks,
                int64_t block_size, int64_t Hkv, int64_t D) {
  const std::string w(what);
  if (num_blocks < 0 || block_size < 1 || Hkv < 1) return invalid(w + ": bad size");
  if (D != 64 && D != 128 && D != 256) return invalid(w + ": head_dim must be 64, 128 or 256");
  if (num_blocks > INT32_MAX || block_size > INT32_MAX || num_blocks * block_size > INT32_MAX || Hkv > 32767)
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
  if (n < 0 || n > INT32_MAX - 1024) return invalid("store_kvcache_mxfp8: bad number of tokens");
  if (dtype != NVHIP_DTYPE_F32 && dtype != NVHIP_DTYPE_BF16 && dtype != NVHIP_DTYPE_F16)
    return invalid("store_kvcache_mxfp8: unsupported dtype");
  if (key_stride < Hkv * D || value_stride < Hkv * D) return invalid("store_kvcache_mxfp8: row stride < row size");
  if (n == 0 || num_blocks == 0) return NVHIP_OK;
  if (!key || !value || !slot_mapping) return invalid("store_kvcache_mxfp8: null pointer");
  StoreArgs g{};
  g.c = MxCache{{static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache)},
                {static_cast<uint8_t*>(k_scales), static_cast<uint8_t*>(v_scales)}, uint32_t(block_size),
                uint32_t(num_blocks * block_size), int(Hkv)};
  g.src[0] = key, g.src[1] = value, g.stride[0] = key_stride, g.stride[1] = value_stride;
  g.slots = slot_mapping, g.n = int(n);
  const int64_t per16 = dtype == NVHIP_DTYPE_F32 ? 4 : 8;  // elements in 16 bytes
  const bool aligned = aligned16(key) && aligned16(value) && key_stride % per16 == 0 && value_stride % per16 == 0;
  const bool two = two_tokens(n, Hkv, D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int d = decltype(dim)::value;
    const int64_t per = kThreads / (d / 8) * (two ? 2 : 1);
    const dim3 grid(unsigned((n + per - 1) / per), unsigned(2 * Hkv)), block(kThreads);
    if (aligned && two) hipLaunchKernelGGL((store_mxfp8_kernel<T, d, true, 2>), grid, block, 0, s, g);
    else if (aligned) hipLaunchKernelGGL((store_mxfp8_kernel<T, d, true, 1>), grid, block, 0, s, g);
    else if (two) hipLaunchKernelGGL((store_mxfp8_kernel<T, d, false, 2>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((store_mxfp8_kernel<T, d, false, 1>), grid, block, 0, s, g);
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
  if (num_seqs < 0 || num_seqs >= INT32_MAX || total < 0 || total > INT32_MAX - 1024 || max_blocks < 0 || max_blocks > INT32_MAX)
    return invalid("load_kvcache_mxfp8: bad size");
  if (total == 0) return NVHIP_OK;
  if (!k || !v || !cu_seqlens_k || (num_seqs > 0 && max_blocks > 0 && !block_table))
    return invalid("load_kvcache_mxfp8: null pointer");
  if (num_seqs == 0) return invalid("load_kvcache_mxfp8: rows to read but no sequence");
  if (!aligned16(k) || !aligned16(v)) return invalid("load_kvcache_mxfp8: outputs must be 16-byte aligned");
  LoadArgs g{};
  auto bytes = [](const void* p) { return static_cast<uint8_t*>(const_cast<void*>(p)); };
  g.c = MxCache{{bytes(k_cache), bytes(v_cache)}, {bytes(k_scales), bytes(v_scales)}, uint32_t(block_size),
                uint32_t(num_blocks * block_size), int(Hkv)};
  g.out[0] = static_cast<uint16_t*>(k), g.out[1] = static_cast<uint16_t*>(v);
  g.bt = block_table, g.cu = cu_seqlens_k, g.total = int(total);
  g.num_seqs = int(num_seqs), g.max_blocks = int(max_blocks), g.num_blocks = int(num_blocks);
  const bool two = two_tokens(total, Hkv, D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto dim) {
    constexpr int d = decltype(dim)::value;
    const int64_t per = kThreads / (d / 8) * (two ? 2 : 1);
    const dim3 grid(unsigned((total + per - 1) / per), unsigned(2 * Hkv)), block(kThreads);
    if (two) hipLaunchKernelGGL((load_mxfp8_kernel<d, 2>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((load_mxfp8_kernel<d, 1>), grid, block, 0, s, g);
    return check_launch("load_kvcache_mxfp8");
  };
  if (D == 64) return launch(std::integral_constant<int, 64>{});
  if (D == 128) return launch(std::integral_constant<int, 128>{});
  return launch(std::integral_constant<int, 256>{});
}
