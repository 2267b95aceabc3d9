// Attention of a few query tokens per sequence over a paged cache, bf16 or MXFP8 (mxfp8.h): the decode step of the 8-bit
// cache, and the verification of a tree of drafted tokens over either cache.
//
// Sequence b has ctx cached tokens, the last n of them the query tokens themselves (their keys and values are stored
// before the call), and query i attends to
//   the tokens before them, t < ctx - n, and
//   of the n last ones, token ctx - n + j where bit j of its mask is set: with a tree, mask = tree_mask[b, i] (the node's
//   ancestors and itself); causal, bits 0 .. i; otherwise all.
// A query that sees nothing (no token, no valid page, every score -inf) gets zeros.
//
// The G = Hq / Hkv query heads of a kv head times the n query tokens are R = G n rows (row = i G + head); a block takes 16
// of them (a unit: sequence, kv head, row tile) over a range of the context. Its 4 waves take 32-token chunks in turn:
//   S^T [16 tokens x 16 rows] = K Q^T, two v_mfma_f32_16x16x32_bf16 tiles a chunk: the A operand comes straight from the
//     cache (lane l: token l % 16, 16 bytes of its row), codes converted in registers with their scale; the order of the
//     dims within a K step is free as long as Q, in registers, has the same: for codes a lane's 16 bytes are two steps;
//   online softmax in base 2 with a reference maximum that moves only when a score exceeds it by more than 8;
//   O^T [16 dims x 16 rows] += V^T P^T: p stays in the lanes it was computed in as the B operand (a bf16 head and a bf16
//     remainder, ~17 bits of p), V^T comes from the wave's own slice of LDS by the transpose read; V's codes are
//     converted to bf16 (exactly) on the way into the slice.
// The waves' (max, sum, O) are merged through LDS in wave order.
//
// Work split: the chunks of all units, one behind the other, are dealt evenly to the blocks whatever the lengths: block p
// of N takes chunks [p C / N, (p + 1) C / N) of C (each block counts the context lengths itself), so that one long
// sequence among short ones costs no more than its share. A unit that lies in several blocks is merged by the last of them to
// arrive: each writes its (max, sum, O) record through the L2 (device-scope stores; the XCDs' L2s are not coherent),
// waits for the stores and counts itself in; the one that completes the count reads the records back and sums them in
// block order, so the result does not depend on which it is.
// The count is a word of the workspace that needs no initialisation: it holds a number of the call in its upper 48 bits,
// and a word with another number counts as 0. The word is left at 0 for the replays of a captured call. Calls may run
// at the same time on several streams as long as each has its own workspace.
#include <algorithm>
#include <atomic>
#include <random>
#include <string>

#include "mxfp8.h"

namespace nvhip {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kChunk = 32;   // tokens per wave step
constexpr int kWaves = 4;    // waves per block
constexpr int kRows = 16;    // query rows per unit
constexpr int kMaxQ = 64;    // query tokens per sequence (bits of a mask)
constexpr int kBlocks = 1024;  // blocks of a split launch: 4 per CU

struct TreeArgs {
  uint16_t* out;
  const uint16_t* q;
  const uint8_t* kc;  // bf16 [num_blocks, bs, Hkv, D] or codes [num_blocks, Hkv, bs, D]
  const uint8_t* vc;
  const uint8_t* ks;  // scales [num_blocks, Hkv, bs, D / 32]
  const uint8_t* vs;
  const int32_t* bt;
  const int32_t* ctx_lens;
  const int64_t* mask;  // [num_seqs, n] or null
  int n, Hkv, G, bs, num_blocks, max_blocks, num_seqs, tiles;  // tiles: row tiles per kv head
  int64_t q_st, q_sh, o_st, o_sh;
  float scale_log2;  // softmax scale * log2(e)
  int causal;
  // split launch (ws != null): gridDim.x blocks share all chunks; otherwise block u takes unit u
  unsigned long long* counts;  // one word per unit
  float* ws;                   // two records per block of rows x (2 + D) floats
  unsigned long long call;     // this call's number, in the upper 48 bits
};

// The part of a unit that a block takes.
struct Piece {
  int b, h, tile, ch0, ch1;  // sequence, kv head, row tile, chunks [ch0, ch1)
  int first, parts;          // blocks that share the unit: first .. first + parts - 1
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ int context(const TreeArgs& g, int b) {
  return min(max(load_uniform(g.ctx_lens + b), 0), g.max_blocks * g.bs);
}
// Chunks of a unit; a sequence without tokens has one, so that some block writes its zeros.
__device__ __forceinline__ int chunks_of(int ctx) { return max(1, (ctx + kChunk - 1) / kChunk); }

constexpr int lds_bytes(int D) {  // the waves' V slices, or their partial O; then their row maxima and sums
  const int v = kWaves * kChunk * (D + 16) * 2, o = kWaves * kRows * D * 4;
  return (v > o ? v : o) + 2 * kWaves * kRows * 4;
}

template <int D, bool MX, bool ALIGNED>
__device__ __forceinline__ void run_piece(const TreeArgs& g, const Piece& pc, int block, unsigned char* lds) {
  constexpr int VP = D + 16;              // LDS row pitch of a V chunk: the 4 rows of a transpose read hit 32 distinct banks
  constexpr int KL = MX ? D / 64 : D / 32;  // 16-byte loads of a K row's lane
  constexpr int KC = D / 32;              // K steps of Q K^T
  constexpr int EPL = MX ? 16 : 8;        // elements in 16 bytes
  constexpr int LPT = D / EPL, TPI = 64 / LPT, PVI = kChunk / TPI;  // V: lanes per row, rows per load, loads per chunk
  constexpr int DT = D / 16;              // 16-dim tiles of O^T
  constexpr int SB = D / kMxBlock;        // scale bytes of a row
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int l16 = lane % 16, h4 = lane / 16;
  const int b = pc.b, h = pc.h, ctx = context(g, b), R = g.G * g.n, r0 = pc.tile * kRows;
  const int32_t* bt_row = g.bt + int64_t(b) * g.max_blocks;

  // this lane's query row, its dims in the order of the K operand's steps, and which of the last n tokens it sees
  const int row = r0 + l16, qi = min(row, R - 1) / g.G;
  bf16x8_t qf[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) qf[c] = bf16x8_t{};
  uint64_t see = 0;
  if (row < R) {
    const uint16_t* qp = g.q + (int64_t(b) * g.n + qi) * g.q_st + int64_t(h * g.G + row - qi * g.G) * g.q_sh;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int dim = MX ? 64 * (c / 2) + 16 * h4 + 8 * (c % 2) : 32 * c + 8 * h4;
      qf[c] = *reinterpret_cast<const bf16x8_t*>(qp + dim);
    }
    see = g.mask != nullptr ? uint64_t(g.mask[int64_t(b) * g.n + qi]) : g.causal ? (2ull << qi) - 1 : ~0ull;
  }
  const int before = ctx - g.n;  // the query tokens' positions begin here (below 0: the first of them are not cached)

  float m_run = -INFINITY, l_run = 0.0f;  // reference maximum of the row, this lane's part of its sum
  f32x4_t acc[DT];                        // O^T dims 16 t + 4 h4 + r of the row
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x4_t{0, 0, 0, 0};
  uint16_t* vl = reinterpret_cast<uint16_t*>(lds) + wave * kChunk * VP;  // this wave's V slice
  const int vt = lane / LPT, vd = lane % LPT;  // V: row and 16-byte piece of this lane

  for (int ch = pc.ch0 + wave; ch < pc.ch1; ch += kWaves) {
    const int t0 = ch * kChunk;
    if (t0 >= ctx) break;
    // cache row (in rows of D) of token t0 + j
    int64_t base = 0;
    uint32_t valid = ctx - t0 >= kChunk ? ~0u : (1u << (ctx - t0)) - 1;  // tokens of the chunk that take part
    if constexpr (ALIGNED) {  // a chunk lies in one page, whose rows behind the context may be read
      const int page = t0 / g.bs, blk = load_uniform(bt_row + page);
      if (blk < 0 || blk >= g.num_blocks) continue;
      base = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + (t0 - page * g.bs)
                : (int64_t(blk) * g.bs + (t0 - page * g.bs)) * g.Hkv + h;
    } else {
      const int t = t0 + lane % 32, page = t / g.bs;
      const int blk = t < ctx ? bt_row[page] : -1;
      valid = uint32_t(__ballot(blk >= 0 && blk < g.num_blocks));
      if (valid == 0) continue;
      base = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + (t - page * g.bs)
                : (int64_t(blk) * g.bs + (t - page * g.bs)) * g.Hkv + h;
      if (!((valid >> (lane % 32)) & 1)) base = -1;
    }
    auto row_of = [&](int j) -> int64_t {  // of token t0 + j; unaligned: a row of an invalid token is that of a valid one
      if constexpr (ALIGNED) {
        return base + int64_t(j) * (MX ? 1 : g.Hkv);
      } else {
        const int from = (valid >> j) & 1 ? j : __builtin_ctz(valid);
        const uint32_t lo = __shfl(uint32_t(base), from), hi = __shfl(uint32_t(base >> 32), from);
        return int64_t((uint64_t(hi) << 32) | lo);
      }
    };
    u32x4 kraw[2][KL], vraw[PVI];
    uint64_t kscale[2] = {};
    uint32_t vscale[PVI] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t r = row_of(16 * u + l16);
      if constexpr (MX) {
        const uint8_t* p = g.kc + r * D + 16 * h4;
#pragma unroll
        for (int c = 0; c < KL; ++c) kraw[u][c] = *reinterpret_cast<const u32x4*>(p + 64 * c);
        if constexpr (SB == 2) kscale[u] = *reinterpret_cast<const uint16_t*>(g.ks + r * SB);
        if constexpr (SB == 4) kscale[u] = *reinterpret_cast<const uint32_t*>(g.ks + r * SB);
        if constexpr (SB == 8) kscale[u] = *reinterpret_cast<const uint64_t*>(g.ks + r * SB);
      } else {
        const uint8_t* p = g.kc + (r * D + 8 * h4) * 2;
#pragma unroll
        for (int c = 0; c < KL; ++c) kraw[u][c] = *reinterpret_cast<const u32x4*>(p + 64 * c);
      }
    }
#pragma unroll
    for (int it = 0; it < PVI; ++it) {
      const int64_t r = row_of(it * TPI + vt);
      vraw[it] = *reinterpret_cast<const u32x4*>(g.vc + (MX ? r * D : r * D * 2) + 16 * vd);
      if constexpr (MX) vscale[it] = g.vs[r * SB + vd / 2];
    }
    const bool masked = t0 + kChunk > before || valid != ~0u;  // some row may not see some token of the chunk

    // V into the wave's slice
    uint64_t odd = 0;  // tokens with a value that is not finite (masked chunks)
#pragma unroll
    for (int it = 0; it < PVI; ++it) {
      uint16_t* dst = vl + (it * TPI + vt) * VP + EPL * vd;
      u32x4 w[MX ? 2 : 1];
      if constexpr (MX) {
        const float sc = mx_scale(vscale[it]);
        w[0] = mx_decode8(vraw[it][0], vraw[it][1], sc);
        w[1] = mx_decode8(vraw[it][2], vraw[it][3], sc);
      } else {
        w[0] = vraw[it];
      }
      if (masked) {
        const bool keep = (valid >> (it * TPI + vt)) & 1;
        bool bad = false;
#pragma unroll
        for (int x = 0; x < (MX ? 2 : 1); ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!keep) w[x][e] = 0;
            bad |= (w[x][e] & 0x7f80u) == 0x7f80u || (w[x][e] & 0x7f800000u) == 0x7f800000u;
          }
        uint64_t m = __ballot(bad);  // lanes of rows: fold each row's lanes onto its bit
        while (m != 0) {
          const int j = __builtin_ctzll(m) / LPT;
          odd |= 1ull << (it * TPI + j);
          m &= ~(((LPT == 64 ? 0ull : 1ull << LPT) - 1) << (j * LPT));
        }
      }
#pragma unroll
      for (int x = 0; x < (MX ? 2 : 1); ++x) *reinterpret_cast<u32x4*>(dst + 8 * x) = w[x];
    }

    // scores: this lane's tokens t0 + 16 u + 4 h4 + r of its row
    f32x4_t s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        bf16x8_t a;
        if constexpr (MX) {
          const float sc = mx_scale((uint32_t(kscale[u] >> (16 * (c / 2))) >> (8 * (h4 / 2))) & 0xffu);
          a = __builtin_bit_cast(bf16x8_t, mx_decode8(kraw[u][c / 2][2 * (c % 2)], kraw[u][c / 2][2 * (c % 2) + 1], sc));
        } else {
          a = __builtin_bit_cast(bf16x8_t, kraw[u][c]);
        }
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[c], s[u], 0, 0, 0);
      }
    }
    float tmax = -INFINITY;
    uint32_t sees = 0xff;  // bit 4 u + r
    if (masked) {
      sees = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * u + 4 * h4 + r, k = t0 + j - before;  // k: which of the query tokens, if it is one
          const bool yes = ((valid >> j) & 1) && row < R && (k < 0 || ((see >> (k & 63)) & 1));
          sees |= uint32_t(yes) << (4 * u + r);
          if (!yes) s[u][r] = -INFINITY;
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, s[u][r]);
    tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
    tmax = pair32_max(tmax) * g.scale_log2;  // the scale is positive
    const bool move = tmax > m_run + 8.0f;   // also true for the first finite maximum (m_run = -inf)
    if (__ballot(move) != 0) {
      const float alpha = move ? exp2f(m_run - tmax) : 1.0f;  // 0 from m_run = -inf
      if (move) m_run = tmax;
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.0f : m_run;
    float p[8];  // P^T as the B operand: k slots 0..3 = tokens 4 h4 + r, 4..7 = tokens 16 + 4 h4 + r
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[4 * u + r] = exp2f(__builtin_fmaf(s[u][r], g.scale_log2, -m_use));
        l_run += p[4 * u + r];
      }
    wave_sync();  // the slice is written
    // Values that are not finite, in tokens that some rows do not see: 0 times them would be NaN there. Such a token is
    // added row by row to the rows that see it, and leaves the product below as zeros.
    while (odd != 0) {
      const int j = __builtin_ctzll(odd);
      odd &= odd - 1;
      float pj = 0.0f;
      uint32_t yes = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e == 4 * (j / 16) + j % 4) pj = p[e], yes = (sees >> e) & 1;
      const int from = l16 + 16 * ((j % 16) / 4);
      pj = __shfl(pj, from);
      yes = __shfl(yes, from);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = bf16_to_f32(vl[j * VP + 16 * t + 4 * h4 + r]);
          if (yes) acc[t][r] = __builtin_fmaf(pj, v, acc[t][r]);
        }
      wave_sync();
      for (int d = lane; d < D; d += 64) vl[j * VP + d] = 0;
      wave_sync();
    }
    const u32x4 phi = pack8(p);
    float ph[8];
    unpack8(phi, ph);
#pragma unroll
    for (int e = 0; e < 8; ++e) ph[e] = p[e] - ph[e];
    const bf16x8_t pk = __builtin_bit_cast(bf16x8_t, phi), pr = __builtin_bit_cast(bf16x8_t, pack8(ph));
    // V^T fragments: the lanes of group h4 address rows 4 h4 + i / 4 (slots 0..3) and 16 + 4 h4 + i / 4 (slots 4..7),
    // dims 16 t + 4 (i % 4)
    const uint16_t* v0 = vl + (4 * h4 + l16 / 4) * VP + 4 * (l16 % 4);
    const uint16_t* v1 = v0 + 16 * VP;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const u32x2 lo = lds_read_tr16(v0 + 16 * t), hi = lds_read_tr16(v1 + 16 * t);
      const bf16x8_t va = __builtin_bit_cast(bf16x8_t, u32x4{lo[0], lo[1], hi[0], hi[1]});
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pk, acc[t], 0, 0, 0);
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pr, acc[t], 0, 0, 0);
    }
    wave_sync();  // the next chunk rewrites the slice
  }

  // the waves' results through LDS
  l_run += __shfl_xor(l_run, 16);
  l_run = pair32_sum(l_run);
  constexpr int VB = kWaves * kChunk * VP * 2, OB = kWaves * kRows * D * 4;
  float (*red_m)[kRows] = reinterpret_cast<float (*)[kRows]>(lds + (VB > OB ? VB : OB));
  float (*red_l)[kRows] = red_m + kWaves;
  float (*red_o)[kRows][D] = reinterpret_cast<float (*)[kRows][D]>(lds);
  __syncthreads();  // every wave is done with its slice
#pragma unroll
  for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4_t*>(&red_o[wave][l16][16 * t + 4 * h4]) = acc[t];
  if (h4 == 0) red_m[wave][l16] = m_run, red_l[wave][l16] = l_run;
  __syncthreads();
  const int rows = min(kRows, R - r0);
  const int64_t record = int64_t(kRows) * (2 + D);
  // a block's record of the unit that it finishes, and of the one that it begins and does not finish
  float* rec = pc.parts > 1 ? g.ws + (2 * int64_t(block) + (block == pc.first ? 1 : 0)) * record : nullptr;
  auto write = [&](int r, int d, float o) {
    const int rr = r0 + r, i = rr / g.G;
    g.out[(int64_t(b) * g.n + i) * g.o_st + int64_t(h * g.G + rr - i * g.G) * g.o_sh + d] = f32_to_bf16(o);
  };
  for (int idx = threadIdx.x; idx < rows * D; idx += kWaves * 64) {
    const int r = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, red_m[w][r]);
    float num = 0.0f, den = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = red_m[w][r] == -INFINITY ? (red_l[w][r] == 0.0f ? 0.0f : 1.0f) : exp2f(red_m[w][r] - M);
      num = __builtin_fmaf(red_o[w][r][d], f, num);
      den = __builtin_fmaf(red_l[w][r], f, den);
    }
    if (pc.parts == 1) {
      write(r, d, den == 0.0f ? 0.0f : num / den);
    } else {
      if (d == 0) {
        __hip_atomic_store(rec + r * (2 + D), M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(rec + r * (2 + D) + 1, den, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __hip_atomic_store(rec + r * (2 + D) + 2 + d, num, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (pc.parts == 1) return;
  __builtin_amdgcn_s_waitcnt(0);  // this wave's record stores have reached memory
  __syncthreads();
  int* flag = reinterpret_cast<int*>(red_m);
  if (threadIdx.x == 0) {
    unsigned long long* word = g.counts + (int64_t(b) * g.Hkv + h) * g.tiles + pc.tile;
    unsigned long long old = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), next;
    bool last;
    do {  // a failed exchange means that another block has counted itself in: at most parts - 1 times
      const unsigned long long before_me = (old & ~0xffffull) == g.call ? old & 0xffffull : 0;
      last = before_me + 1 == (unsigned long long)pc.parts;
      next = g.call | (last ? 0 : before_me + 1);
    } while (!__hip_atomic_compare_exchange_strong(word, &old, next, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT));
    *flag = last;
  }
  __syncthreads();
  if (!*flag) return;
  auto get = [&](int part, int at) {  // float `at` of the record of the unit's part
    const float* p = g.ws + (2 * int64_t(pc.first + part) + (part == 0 ? 1 : 0)) * record + at;
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  for (int idx = threadIdx.x; idx < rows * D; idx += kWaves * 64) {
    const int r = idx / D, d = idx % D, at = r * (2 + D);
    float M = -INFINITY;
    for (int k = 0; k < pc.parts; ++k) M = fmaxf(M, get(k, at));
    float num = 0.0f, den = 0.0f;
    for (int k = 0; k < pc.parts; ++k) {
      const float m = get(k, at), l = get(k, at + 1);
      const float f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - M);
      num = __builtin_fmaf(get(k, at + 2 + d), f, num);
      den = __builtin_fmaf(l, f, den);
    }
    write(r, d, den == 0.0f ? 0.0f : num / den);
  }
}

template <int D, bool MX, bool ALIGNED>
__global__ __launch_bounds__(kWaves * 64) void tree_attention_kernel(const TreeArgs g) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[lds_bytes(D)];
  const int U = g.Hkv * g.tiles;  // units of a sequence
  if (g.ws == nullptr) {
    const int u = blockIdx.x, b = u / U, v = u - b * U;
    run_piece<D, MX, ALIGNED>(g, Piece{b, v / g.tiles, v % g.tiles, 0, chunks_of(context(g, b)), 0, 1}, 0, lds);
    return;
  }
  // chunks of a unit of each sequence: lane l sums sequences [l S, (l + 1) S)
  const int lane = threadIdx.x % 64, S = (g.num_seqs + 63) / 64;
  int sum = 0;
  for (int j = 0; j < S; ++j) {
    const int b = lane * S + j;
    if (b < g.num_seqs) sum += chunks_of(min(max(g.ctx_lens[b], 0), g.max_blocks * g.bs));
  }
  int incl = sum;  // inclusive scan over the lanes
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(incl, off);
    if (lane >= off) incl += v;
  }
  const int64_t C = int64_t(__shfl(incl, 63)) * U;
  const int64_t N = min(int64_t(gridDim.x), C);
  // blocks p of one XCD (blockIdx.x % 8) are neighbours: row tiles of a kv head read the same rows through one L2
  const int64_t per = (N + 7) / 8, p = int64_t(blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || p >= N) return;
  int64_t at = p * C / N;
  const int64_t end = (p + 1) * C / N;
  // the sequence that holds chunk `at`: the lane that holds it, then its sequences one by one
  const int from = __popcll(__ballot(int64_t(incl) * U <= at));
  int b = from * S;
  int64_t begin = int64_t(__shfl(incl - sum, from)) * U;  // first chunk of sequence b
  while (at < end) {
    const int c = chunks_of(context(g, b));
    if (at >= begin + int64_t(c) * U) {
      begin += int64_t(c) * U;
      ++b;
      continue;
    }
    const int u = int((at - begin) / c);
    const int64_t u0 = begin + int64_t(u) * c;
    const int64_t stop = min(end, u0 + c);
    const int64_t first = ((u0 + 1) * N - 1) / C, last = ((u0 + c) * N - 1) / C;  // the blocks of its first and last chunk
    run_piece<D, MX, ALIGNED>(g, Piece{b, u / g.tiles, u % g.tiles, int(at - u0), int(stop - u0), int(first),
                                       int(last - first) + 1}, int(p), lds);
    at = stop;
    if (at < end) __syncthreads();  // the next piece reuses the LDS
  }
}

template <int D, bool MX>
int launch(const TreeArgs& g, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWaves * 64);
  if (g.bs % kChunk == 0) hipLaunchKernelGGL((tree_attention_kernel<D, MX, true>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((tree_attention_kernel<D, MX, false>), grid, block, 0, s, g);
  return check_launch("tree_attention");
}

int64_t tiles_of(int64_t q_len, int64_t Hq, int64_t Hkv) { return (Hq / Hkv * q_len + kRows - 1) / kRows; }

// Blocks of the split launch: at most 4 per CU, and none without a chunk at the longest possible context.
int64_t split_blocks(int64_t num_seqs, int64_t units, int64_t max_ctx) {
  const int64_t most = units * std::max<int64_t>(1, (max_ctx + kChunk - 1) / kChunk);
  return std::min<int64_t>(kBlocks, (most + 7) / 8 * 8);
}
struct Workspace {
  int64_t count_bytes, bytes;
};
Workspace workspace_of(int64_t units, int64_t blocks, int64_t D) {
  const int64_t counts = (units * 8 + 255) / 256 * 256;
  return {counts, counts + blocks * 2 * kRows * (2 + D) * 4};
}

// A number for each call, from a random start, in the upper 48 bits of a word; never 0.
unsigned long long next_call() {
  static std::atomic<unsigned long long> n{(static_cast<unsigned long long>(std::random_device{}()) << 16) ^
                                           std::random_device{}()};
  unsigned long long c;
  do c = n.fetch_add(1, std::memory_order_relaxed) << 16;
  while (c == 0);
  return c;
}

}  // namespace
}  // namespace nvhip

extern "C" int64_t nvhip_tree_attention_workspace_size(int64_t num_seqs, int64_t q_len, int64_t Hq, int64_t Hkv,
                                                       int64_t D, int64_t block_size, int64_t max_blocks) {
  using namespace nvhip;
  if (num_seqs <= 0 || q_len < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || D < 1 || block_size < 1 || max_blocks < 0)
    return 0;
  const int64_t units = num_seqs * Hkv * tiles_of(q_len, Hq, Hkv);
  return workspace_of(units, split_blocks(num_seqs, units, max_blocks * block_size), D).bytes;
}

extern "C" int nvhip_tree_attention(void* out, const void* q, const void* k_cache, const void* v_cache,
                                    const void* k_scales, const void* v_scales, const int32_t* block_table,
                                    const int32_t* context_lens, const int64_t* tree_mask, int64_t num_seqs,
                                    int64_t q_len, int64_t Hq, int64_t Hkv, int64_t D, int64_t block_size,
                                    int64_t num_blocks, int64_t max_blocks, int64_t q_stride_token,
                                    int64_t q_stride_head, int64_t out_stride_token, int64_t out_stride_head,
                                    float scale, int causal, void* workspace, int64_t workspace_size, void* stream) {
  using namespace nvhip;
  clear_error();
  if (num_seqs < 0 || q_len < 1 || Hq < 1 || Hkv < 1 || block_size < 1 || num_blocks < 0 || max_blocks < 0)
    return invalid("tree_attention: bad size");
  if (q_len > kMaxQ) return invalid("tree_attention: at most 64 query tokens per sequence");
  if (Hq % Hkv != 0) return invalid("tree_attention: Hq must be a multiple of Hkv");
  if (D != 64 && D != 128 && D != 256) return invalid("tree_attention: head_dim must be 64, 128 or 256");
  if (q_stride_head < D || q_stride_token < Hq * q_stride_head || out_stride_head < D ||
      out_stride_token < Hq * out_stride_head || q_stride_head % 8 != 0 || q_stride_token % 8 != 0)
    return invalid("tree_attention: bad q / out strides (rows of D contiguous, 16-byte aligned)");
  if (!(scale > 0.0f) || scale > 3e38f) return invalid("tree_attention: softmax_scale must be positive and finite");
  if ((k_scales == nullptr) != (v_scales == nullptr))
    return invalid("tree_attention: k_scales and v_scales must be given together");
  if (Hq > (1 << 20) || num_seqs > (1 << 24) || num_blocks > INT32_MAX || block_size > INT32_MAX ||
      max_blocks > INT32_MAX || max_blocks * block_size > INT32_MAX - 64)
    return invalid("tree_attention: size too large");
  if (num_seqs == 0) return NVHIP_OK;
  if (!out || !q || !context_lens || (max_blocks > 0 && !block_table) || (num_blocks > 0 && (!k_cache || !v_cache)))
    return invalid("tree_attention: null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scales) || !aligned16(v_scales))
    return invalid("tree_attention: q, the caches and the scales must be 16-byte aligned");
  TreeArgs g{};
  g.out = static_cast<uint16_t*>(out), g.q = static_cast<const uint16_t*>(q);
  g.kc = static_cast<const uint8_t*>(k_cache), g.vc = static_cast<const uint8_t*>(v_cache);
  g.ks = static_cast<const uint8_t*>(k_scales), g.vs = static_cast<const uint8_t*>(v_scales);
  g.bt = block_table, g.ctx_lens = context_lens, g.mask = tree_mask;
  g.n = int(q_len), g.Hkv = int(Hkv), g.G = int(Hq / Hkv), g.bs = int(block_size), g.num_blocks = int(num_blocks);
  g.max_blocks = int(max_blocks), g.num_seqs = int(num_seqs), g.tiles = int(tiles_of(q_len, Hq, Hkv));
  g.q_st = q_stride_token, g.q_sh = q_stride_head, g.o_st = out_stride_token, g.o_sh = out_stride_head;
  g.scale_log2 = scale * 1.4426950408889634f;
  g.causal = causal ? 1 : 0;
  const int64_t units = num_seqs * Hkv * g.tiles;
  // the chunk counts are 32-bit sums over the sequences and 64-bit products with the units and blocks
  if (units > INT32_MAX || num_seqs * ((max_blocks * block_size) / kChunk + 1) > INT32_MAX)
    return invalid("tree_attention: size too large");
  int64_t blocks = units;
  const int64_t split = split_blocks(num_seqs, units, max_blocks * block_size);
  const Workspace w = workspace_of(units, split, D);
  if (workspace != nullptr && workspace_size >= w.bytes) {
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return invalid("tree_attention: workspace must be 16-byte aligned");
    blocks = split;
    g.counts = static_cast<unsigned long long*>(workspace);
    g.ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.count_bytes);
    g.call = next_call();
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto by_dim = [&](auto mx) {
    constexpr bool MX = decltype(mx)::value;
    if (D == 64) return launch<64, MX>(g, blocks, s);
    if (D == 128) return launch<128, MX>(g, blocks, s);
    return launch<256, MX>(g, blocks, s);
  };
  return k_scales != nullptr ? by_dim(std::true_type{}) : by_dim(std::false_type{});
}
