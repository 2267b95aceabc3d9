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
// The G = Hq / Hkv query heads of a kv head times the n query tokens are R = G n rows (row = i G + head), cut into units of
// 16, 32 or 64 of them (Shape). A block of 4 waves takes a unit over a range of the context:
//   S^T [16 tokens x 16 rows] = K Q^T with v_mfma_f32_16x16x32_bf16 (A: token l % 16 of lane l, B: row l % 16);
//   online softmax in base 2 with a reference maximum that moves only when a score exceeds it by more than 8;
//   O^T [16 dims x 16 rows] += V^T P^T: p stays in the lanes it was computed in as the B operand, as a bf16 head and a bf16
//   remainder (~17 bits of p, so that the output's own rounding to bf16 is the only one that shows); V^T comes from LDS by
//   the transpose read.
// Codes are converted to the bf16 numbers that they stand for, exactly, by v_cvt_scalef32_pk_bf16_fp8: 2 elements and their
// scale an instruction.
//   Up to 32 rows (run_piece): each wave takes 32-token chunks on its own, K straight from the cache into the A operand (the
//   order of the dims within a K step is free as long as Q, in registers, has the same: a lane's 16 codes are two steps), V
//   through the wave's slice of LDS, the next chunk's loads on the way during softmax and second product. The waves'
//   (max, sum, O) are merged through LDS in wave order.
//   64 rows (run_wide): a wave has 16 of them, and all waves bring 64 tokens at a time into LDS in bf16.
//
// Work split: the chunks of all units, one behind the other, are dealt evenly to as many blocks as are resident at once,
// whatever the lengths (each block counts the context lengths itself), with what a piece costs beside its chunks counted in:
// one long sequence among short ones costs no more than its share. The parts of a unit that lies in several blocks are merged
// in block order, so the result does not depend on timing:
//   up to 32 rows by the last of them to arrive. Each writes its (max, sum, O) record through the L2 (device-scope stores;
//   the XCDs' L2s are not coherent), waits for the stores and counts itself in; the one that completes the count reads the
//   records back. The count is a word of the workspace that needs no initialisation: it holds a number of the call in its
//   upper 48 bits, and a word with another number counts as 0. It is left at 0 for the replays of a captured call.
//   Of 64 rows a record is 33 KB, and one block took longer to merge them (up to 20 us) than a second launch does (9 us for
//   512 units), which reads them with the whole card.
// Short units are not split (Shape::whole).
// Calls may run at the same time on several streams as long as each has its own workspace.
//
// Times (8 kv heads of 128, G = 2, pages of 256; replayed from a graph). 8-bit decode step of 1 sequence of 700 tokens 10.5 us
// (the chain of loads: lengths, pages, rows, records), of 32 sequences of 512 .. 2048 25 us (3.8 TB/s), of 250 up to 4096
// 187 .. 193 us (5.4 TB/s; while streaming the blocks read at the card's rate, the rest is each piece's start and end). Trees
// of 33 nodes for 8 sequences of 1000 .. 4000, bf16, 33.0 us (2.5 TB/s); of 64 nodes for 32 sequences of 512 .. 2048, 8 bit,
// 67 us (0.35 PFLOP/s): products, softmax, staging, loads and the merge take what they take one after the other (leaving one
// out saves 27, 11, 8, 8 and 10 us) although none fills its unit: vector issue 38 %, matrix cores 26 %, LDS 35 % of the
// clocks. Two, three or four waves per SIMD, waves of 32 rows that read half as much of LDS, 128 rows to a block, and two LDS
// buffers with one barrier a step took the same time within 3 %.
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
constexpr int kStep = 64;    // tokens per step of a block with more than 32 rows
constexpr int kMaxQ = 64;    // query tokens per sequence (bits of a mask)
constexpr int kCountStride = 16;  // words between two units' counts: a 128-byte line each

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
  int once;  // the rows are read with the nontemporal hint
  // split launch (ws != null): gridDim.x blocks share all chunks; otherwise block u takes unit u
  unsigned long long* counts;  // one word per unit
  float* ws;                   // two records per block of rows x (2 + D) floats
  int2* plan;                  // of each unit of more than 32 rows: the first of its blocks, and how many
  unsigned long long call;     // this call's number, in the upper 48 bits
};

// The part of a unit that a block takes.
struct Piece {
  int b, h, tile, ch0, ch1;  // sequence, kv head, row tile, chunks [ch0, ch1)
  int first, parts;          // blocks that share the unit: first .. first + parts - 1
};

// max / sum of v over lanes l and l ^ 16, in both lanes (v_permlane16_swap of v with itself: rows 0, 0, 2, 2 and 1, 1, 3, 3).
__device__ __forceinline__ float pair16_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair16_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Inclusive scan of v over the wave by DPP: within rows of 16, then across them.
template <class F>
__device__ __forceinline__ int wave_scan(int v, F&& f) {
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast 15 into rows 1 and 3
  return f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast 31 into rows 2 and 3
}

// 2^x by the hardware (within an ulp; below 2^-126 it is 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <bool ONCE = false>  // ONCE: with the nontemporal hint
__device__ __forceinline__ u32x4 load16(const uint8_t* base, uint32_t offset) {
  const u32x4* p = reinterpret_cast<const u32x4*>(base + offset);
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
}

__device__ __forceinline__ int context(const TreeArgs& g, int b) {
  return min(max(load_uniform(g.ctx_lens + b), 0), g.max_blocks * g.bs);
}
// Which of the 64 tokens from t0 on a row sees, `ahead` = the query tokens' first position - t0: all before them, then by
// the bits of `see`.
__device__ __forceinline__ uint64_t visible(int ahead, uint64_t see) {
  if (ahead >= 64) return ~0ull;
  return ahead > 0 ? ((1ull << ahead) - 1) | (see << ahead) : ahead > -64 ? see >> -ahead : 0;
}

// Bytes of LDS: the waves' V slices, or a step's K and V (and which tokens take part); afterwards the waves' O, row maxima
// and sums.
constexpr int lds_bytes(int D, bool wide) {
  const int v = wide ? kStep * (2 * D + 24) * 2 + kStep * 4 + 16 : kWaves * kChunk * (D + 16) * 2;
  const int o = kWaves * 16 * D * 4 + 2 * kWaves * 16 * 4;
  return v > o ? v : o;
}

// 2^(m - M) for a maximum m of the overall M, and 1 for a sum that is NaN without any maximum (every score NaN).
__device__ __forceinline__ float share(float m, float l, float M) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2_fast(m - M);
}

// The waves' (max, sum, O^T) of a piece through LDS: to the output, or into a record, and by the last of the unit's blocks
// all records into the output. A wave holds RT tiles of 16 rows: lane l has row l % 16, dims 16 t + 4 (l / 16) + r. chunks: of
// the piece; of a single one, the first wave's result is the unit's (1464 units of 18 rows and up to 23 tokens 31.5 -> 24.6 us).
template <int D, int RT>
__device__ __forceinline__ void finish(const TreeArgs& g, const Piece& pc, int block, int chunks, unsigned char* lds,
                                       const f32x4_t (&acc)[RT][D / 16], const float (&m_run)[RT], const float (&l_run)[RT]) {
  constexpr int RU = 16 * RT;  // rows of a unit
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int l16 = lane % 16, h4 = lane / 16;
  const int r0 = pc.tile * RU, rows = min(RU, g.G * g.n - r0);
  if (chunks <= 1 && pc.parts == 1) {
    if (wave != 0) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float l = pair32_sum(pair16_sum(l_run[rt]));
      const int rr = r0 + 16 * rt + l16, i = rr / g.G;
      if (rr - r0 >= rows) continue;
      uint16_t* out = g.out + (int64_t(pc.b) * g.n + i) * g.o_st + int64_t(pc.h * g.G + rr - i * g.G) * g.o_sh + 4 * h4;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const f32x4_t o = acc[rt][t];
        *reinterpret_cast<u32x2*>(out + 16 * t) =
            l == 0.0f ? u32x2{} : u32x2{pack_bf16x2(o[0] / l, o[1] / l), pack_bf16x2(o[2] / l, o[3] / l)};
      }
    }
    return;
  }
  float (*red_o)[16][D] = reinterpret_cast<float (*)[16][D]>(lds);
  float (*red_m)[16] = reinterpret_cast<float (*)[16]>(lds + kWaves * 16 * D * 4);
  float (*red_l)[16] = red_m + kWaves;
  // record: (max, sum) of each row, then O [row][D]
  constexpr int64_t kRecord = int64_t(RU) * (2 + D);
  // a block's record of the unit that it finishes, and of the one that it begins and does not finish
  float* rec = pc.parts > 1 ? g.ws + (2 * int64_t(block) + (block == pc.first ? 1 : 0)) * kRecord : nullptr;
  // the unit's count, asked for early: what it says is only tried below, an old value does no harm
  unsigned long long* word = g.counts + ((int64_t(pc.b) * g.Hkv + pc.h) * g.tiles + pc.tile) * kCountStride;
  unsigned long long old = 0;
  if (pc.parts > 1 && threadIdx.x == 0) old = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  auto write = [&](int r, int d, float o0, float o1) {
    const int rr = r0 + r, i = rr / g.G;
    const int64_t at = (int64_t(pc.b) * g.n + i) * g.o_st + int64_t(pc.h * g.G + rr - i * g.G) * g.o_sh + d;
    *reinterpret_cast<uint32_t*>(g.out + at) = pack_bf16x2(o0, o1);
  };
  auto put = [&](int at, float a, float b) {  // two floats of the record, through the L2
    const f32x2 v = {a, b};
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(rec + at), __builtin_bit_cast(unsigned long long, v),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto get = [&](int part, int at) {  // two floats of the record of the unit's part
    const float* q = g.ws + (2 * int64_t(pc.first + part) + (part == 0 ? 1 : 0)) * kRecord + at;
    return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<unsigned long long*>(const_cast<float*>(q)),
                                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  };
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    __syncthreads();  // every wave is done with what the LDS held
    if (rt * 16 + l16 < rows) {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4_t*>(&red_o[wave][l16][16 * t + 4 * h4]) = acc[rt][t];
    }
    const float l = pair32_sum(pair16_sum(l_run[rt]));
    if (h4 == 0) red_m[wave][l16] = m_run[rt], red_l[wave][l16] = l;
    __syncthreads();
    for (int idx = threadIdx.x; idx < min(16, rows - 16 * rt) * (D / 2); idx += kWaves * 64) {
      const int y = idx / (D / 2), d = idx % (D / 2) * 2, r = 16 * rt + y;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, red_m[w][y]);
      float n0 = 0.0f, n1 = 0.0f, den = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = share(red_m[w][y], red_l[w][y], M);
        n0 = __builtin_fmaf(red_o[w][y][d], f, n0);
        n1 = __builtin_fmaf(red_o[w][y][d + 1], f, n1);
        den = __builtin_fmaf(red_l[w][y], f, den);
      }
      if (pc.parts == 1) {
        write(r, d, den == 0.0f ? 0.0f : n0 / den, den == 0.0f ? 0.0f : n1 / den);
      } else {
        if (d == 0) put(2 * r, M, den);
        put(2 * RU + r * D + d, n0, n1);
      }
    }
  }
  if (pc.parts == 1) return;
  __builtin_amdgcn_s_waitcnt(0);  // this wave's record stores have reached memory
  __syncthreads();
  int* flag = reinterpret_cast<int*>(red_m);
  if (threadIdx.x == 0) {
    // the first to find another number (a later one's exchange fails: the number is there) puts this call's in its place,
    // itself counted; everybody else adds one
    if ((old & ~0xffffull) == g.call ||
        !__hip_atomic_compare_exchange_strong(word, &old, g.call | 1, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT))
      old = __hip_atomic_fetch_add(word, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else
      old = g.call;
    const bool last = int(old & 0xffffull) == pc.parts - 1;
    if (last) __hip_atomic_store(word, g.call, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for a replay
    *flag = last;
  }
  __syncthreads();
  if (!*flag) return;
  // 4 pairs of elements a thread and 4 parts at a time, 16 loads on the way, the first of them with the parts' (max, sum)
  const int pairs = rows * (D / 2);
  f32x2 o[4][4];
  auto load_parts = [&](int i0, int k0) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int idx = min(i0 + y * kWaves * 64, pairs - 1);
        o[u][y] = get(min(k0 + u, pc.parts - 1), 2 * RU + idx / (D / 2) * D + idx % (D / 2) * 2);
      }
  };
  load_parts(threadIdx.x, 0);
  // every part's (max, sum) of every row; from them each part's share of the row's O
  f32x2* ml = reinterpret_cast<f32x2*>(lds);  // [part][row]; the waves' O is no longer needed
  for (int i = threadIdx.x; i < pc.parts * rows; i += kWaves * 64) ml[i] = get(i / rows, 2 * (i % rows));
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += kWaves * 64) {
    float M = -INFINITY, den = 0.0f;
    for (int k = 0; k < pc.parts; ++k) M = fmaxf(M, ml[k * rows + r][0]);
    for (int k = 0; k < pc.parts; ++k) {
      const f32x2 v = ml[k * rows + r];
      const float f = share(v[0], v[1], M);
      ml[k * rows + r][0] = f;
      den = __builtin_fmaf(v[1], f, den);
    }
    ml[r][1] = den;
  }
  __syncthreads();
  for (int i0 = threadIdx.x; i0 < pairs; i0 += 4 * kWaves * 64) {
    f32x2 sum[4] = {};
    for (int k0 = 0; k0 < pc.parts; k0 += 4) {
      if (k0 != 0 || i0 != int(threadIdx.x)) load_parts(i0, k0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (k0 + u >= pc.parts) break;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float f = ml[(k0 + u) * rows + min(i0 + y * kWaves * 64, pairs - 1) / (D / 2)][0];
          sum[y][0] = __builtin_fmaf(o[u][y][0], f, sum[y][0]);
          sum[y][1] = __builtin_fmaf(o[u][y][1], f, sum[y][1]);
        }
      }
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int idx = i0 + y * kWaves * 64, r = idx / (D / 2), d = idx % (D / 2) * 2;
      if (idx >= pairs) break;
      const float den = ml[r][1];
      write(r, d, den == 0.0f ? 0.0f : sum[y][0] / den, den == 0.0f ? 0.0f : sum[y][1] / den);
    }
  }
}

// V^T fragments from LDS rows of pitch VP, two 16-dim tiles at a time, the next ones' reads issued before the products with
// the ones at hand: f(tile, fragment). v: this lane's place in the first 4 x 16 block (row 4 (l / 16) + l % 16 / 4, dims
// 4 (l % 4) ..): the transpose read hands the lanes of group l / 16 rows 4 (l / 16) .. + 3 (k slots 0..3), and 16 more (4..7).
// TS: from a tile to the next in LDS.
template <int DT, int VP, int TS = 16>
struct VFragments {
  static constexpr int TP = 2;
  u32x4 f[2][TP];
  __device__ __forceinline__ void load(const uint16_t* v, int group) {
#pragma unroll
    for (int i = 0; i < TP; ++i) {
      const u32x2 lo = lds_read_tr16(v + TS * (TP * group + i)), hi = lds_read_tr16(v + 16 * VP + TS * (TP * group + i));
      f[group % 2][i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
  // after load(v, 0); `next` is the rows to go on with (their first group is loaded), or null
  template <class F>
  __device__ __forceinline__ void run(const uint16_t* v, const uint16_t* next, F&& mul) {
    static_assert(DT / TP % 2 == 0, "an even number of groups");
#pragma unroll
    for (int group = 0; group < DT / TP; ++group) {
      if (group + 1 < DT / TP) load(v, group + 1);
      else if (next != nullptr) load(next, 0);
      __builtin_amdgcn_sched_barrier(0);
      mul(TP * group, f[group % 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// acc[rt][t + i] += f[i] P^T of the row tiles, for the two V^T fragments at tile t: p's heads, then its remainders.
template <int RT, int DT>
__device__ __forceinline__ void multiply(f32x4_t (&acc)[RT][DT], int t, const u32x4* f, const u32x4* phi, const u32x4* plo) {
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc[rt][t + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f[i]),
                                                                  __builtin_bit_cast(bf16x8_t, part ? plo[rt] : phi[rt]),
                                                                  acc[rt][t + i], 0, 0, 0);
}

// p = 2^(s scale - m) of N scores of a row with the reference maximum m_run, which first moves up (and sum and O with it) if
// a score is more than 8 above it: p <= 256, and few chunks move it. Adds p to the lane's part of the row's sum; hi, lo: p
// as a bf16 head and a bf16 remainder (together ~17 bits; the sums take p itself).
template <int N, int DT>
__device__ __forceinline__ void softmax(const float* s, float scale_log2, float& m_run, float& l_run, f32x4_t (&acc)[DT],
                                        u32x4* hi, u32x4* lo) {
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < N; ++e) top = fmaxf(top, s[e]);
  top = pair32_max(pair16_max(top)) * scale_log2;  // over the row's four lanes; the scale is positive
  const bool move = top > m_run + 8.0f;   // also true for the first finite maximum (m_run = -inf)
  if (__ballot(move) != 0) {
    const float alpha = move ? exp2_fast(m_run - top) : 1.0f;  // 0 from m_run = -inf
    if (move) m_run = top;
    l_run *= alpha;
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] *= alpha;
  }
  const float m = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
  for (int y = 0; y < N / 8; ++y) {
    float p[8], head[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = exp2_fast(__builtin_fmaf(s[8 * y + e], scale_log2, -m));
      l_run += p[e];
    }
    hi[y] = pack8(p);
    unpack8(hi[y], head);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] -= head[e];
    lo[y] = pack8(p);
  }
}

// -inf for the scores (tokens 16 u + r of a row, N = 4 u + r) whose bit 16 u + r of vis is not set.
template <int N, class V>
__device__ __forceinline__ void hide(float* s, V vis) {
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = (vis >> (16 * (e / 4) + e % 4)) & 1 ? s[e] : -INFINITY;
}

// Whether one of 8 bf16 is not finite.
__device__ __forceinline__ bool not_finite(const u32x4& w) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// Query token k's contribution to the rows that see it, for a value that is not finite (the products leave such tokens out:
// 0 times their value would be NaN in the rows that do not see them). Its score is computed again, from cache row r.
// qf in the order of the dims that DIM gives.
template <int D, bool MX, int RT, class DIM>
__device__ __forceinline__ void add_token(const TreeArgs& g, int64_t r, int k, const bf16x8_t (&qf)[RT][D / 32],
                                          const uint64_t (&see)[RT], const float (&m_run)[RT],
                                          f32x4_t (&acc)[RT][D / 16], DIM dim) {
  constexpr int SB = D / kMxBlock;
  const int h4 = threadIdx.x % 64 / 16;
  auto values = [&](const uint8_t* cache, const uint8_t* scales, int d, float* x) {  // 4 elements of the row
    u32x2 w;
    if constexpr (MX) {
      const u32x4 y = mx_decode8(*reinterpret_cast<const uint32_t*>(cache + r * D + d), 0,
                                 mx_scale(scales[r * SB + d / kMxBlock]));
      w = u32x2{y[0], y[1]};
    } else {
      w = *reinterpret_cast<const u32x2*>(cache + 2 * (r * D + d));
    }
    x[0] = bf16_lo(w[0]), x[1] = bf16_hi(w[0]), x[2] = bf16_lo(w[1]), x[3] = bf16_hi(w[1]);
  };
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float s = 0.0f;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        float kk[4];
        values(g.kc, g.ks, dim(x) + e, kk);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = __builtin_fmaf(float(qf[rt][x][e + i]), kk[i], s);
      }
    s = pair32_sum(pair16_sum(s)) * g.scale_log2;
    const bool yes = (see[rt] >> k) & 1;
    const float p = exp2_fast(s - (m_run[rt] == -INFINITY ? 0.0f : m_run[rt]));
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      float v[4];
      values(g.vc, g.vs, 16 * t + 4 * h4, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[rt][t][i] = yes ? __builtin_fmaf(p, v[i], acc[rt][t][i]) : acc[rt][t][i];
    }
  }
}

template <int D, bool MX, bool ALIGNED, int RT>
__device__ __forceinline__ void run_piece(const TreeArgs& g, const Piece& pc, int block, unsigned char* lds) {
  constexpr int VP = D + 16;              // LDS row pitch of a V chunk: the 4 rows of a transpose read hit 32 distinct banks
  constexpr int KL = MX ? D / 64 : D / 32;  // 16-byte loads of a K row's lane
  constexpr int KC = D / 32;              // K steps of Q K^T
  constexpr int EPL = MX ? 16 : 8;        // elements in 16 bytes
  constexpr int LPT = D / EPL, TPI = 64 / LPT, PVI = kChunk / TPI;  // V: lanes per row, rows per load, loads per chunk
  constexpr int DT = D / 16;              // 16-dim tiles of O^T
  constexpr int RB = MX ? D : 2 * D, SB = D / kMxBlock;  // bytes of a row, and of its scales
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int l16 = lane % 16, h4 = lane / 16;
  const int b = pc.b, h = pc.h, ctx = context(g, b), R = g.G * g.n;
  const int32_t* bt_row = g.bt + int64_t(b) * g.max_blocks;
  const int ch0 = pc.ch0 + wave, ch_end = min(pc.ch1, (ctx + kChunk - 1) / kChunk);

  // The table's entry for the wave's next chunk, asked for one chunk ahead of its rows: aligned, of its page `at` (and `off`,
  // where in the page it begins); else of token lane % 32.
  const int last_page = (max(ctx, 1) - 1) / g.bs;
  int at = ch0 * kChunk / g.bs, off = ch0 * kChunk - at * g.bs, page = 0;
  auto ask_page = [&](int ch) {
    if constexpr (ALIGNED) page = load_uniform(bt_row + min(at, last_page));
    else page = bt_row[min(ch * kChunk + lane % 32, ctx - 1) / g.bs];
  };
  if (ch0 < ch_end) ask_page(ch0);

  // this lane's query rows, their dims in the order of the K operand's steps, and which of the last n tokens they see
  bf16x8_t qf[RT][KC];
  uint64_t see[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = (pc.tile * RT + rt) * 16 + l16, qi = min(row, R - 1) / g.G;
#pragma unroll
    for (int x = 0; x < KC; ++x) qf[rt][x] = bf16x8_t{};
    see[rt] = 0;
    if (row < R) {
      const uint16_t* qp = g.q + (int64_t(b) * g.n + qi) * g.q_st + int64_t(h * g.G + row - qi * g.G) * g.q_sh;
#pragma unroll
      for (int x = 0; x < KC; ++x) {
        const int dim = MX ? 64 * (x / 2) + 16 * h4 + 8 * (x % 2) : 32 * x + 8 * h4;
        qf[rt][x] = *reinterpret_cast<const bf16x8_t*>(qp + dim);
      }
      see[rt] = g.mask != nullptr ? uint64_t(g.mask[int64_t(b) * g.n + qi]) : g.causal ? (2ull << qi) - 1 : ~0ull;
    }
  }
  const int before = ctx - g.n;  // the query tokens' positions begin here (below 0: the first of them are not cached)

  float m_run[RT], l_run[RT];  // reference maximum of the row, this lane's part of its sum
  f32x4_t acc[RT][DT];         // O^T dims 16 t + 4 h4 + r of the row
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m_run[rt] = -INFINITY, l_run[rt] = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[rt][t] = f32x4_t{0, 0, 0, 0};
  }
  uint16_t* vl = reinterpret_cast<uint16_t*>(lds) + wave * kChunk * VP;  // this wave's V slice
  const int vt = lane / LPT, vd = lane % LPT;  // V: row and 16-byte piece of this lane

  using scale_t = std::conditional_t<SB == 2, uint16_t, std::conditional_t<SB == 4, uint32_t, uint64_t>>;
  // A chunk's rows in registers. Its loads are issued as soon as the chunk before has left these registers, so that they
  // are in flight during that chunk's softmax and second product.
  struct Chunk {
    u32x4 k[2][KL], v[PVI];
    scale_t kscale[2];
    uint32_t vscale[PVI];
    uint32_t valid;  // tokens that take part
  } c;
  // Of a chunk with tokens < ctx, and the page of the next one; a token in no valid page reads the row's place in page 0.
  auto load_chunk = [&](int ch) {
    const int t0 = ch * kChunk;
    int blk = page;
    if constexpr (ALIGNED) {  // a chunk lies in one page, whose rows behind the context may be read: one base, small offsets
      c.valid = ctx - t0 >= kChunk ? ~0u : (1u << (ctx - t0)) - 1;
      if (blk < 0 || blk >= g.num_blocks) blk = 0, c.valid = 0;
      const int64_t base = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + off : (int64_t(blk) * g.bs + off) * g.Hkv + h;
      const uint8_t *kb = g.kc + base * RB, *vb = g.vc + base * RB;
      const uint32_t step = MX ? RB : RB * g.Hkv;  // bytes between a head's rows
      auto load_rows = [&](auto once) {
        constexpr bool ONCE = decltype(once)::value;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < KL; ++x) c.k[u][x] = load16<ONCE>(kb, (16 * u + l16) * step + 16 * h4 + 64 * x);
#pragma unroll
        for (int it = 0; it < PVI; ++it) c.v[it] = load16<ONCE>(vb, (it * TPI + vt) * step + 16 * vd);
      };
      if (g.once) load_rows(std::true_type{});
      else load_rows(std::false_type{});
      if constexpr (MX) {
        const uint8_t *ksb = g.ks + base * SB, *vsb = g.vs + base * SB;
#pragma unroll
        for (int u = 0; u < 2; ++u) c.kscale[u] = *reinterpret_cast<const scale_t*>(ksb + uint32_t((16 * u + l16) * SB));
#pragma unroll
        for (int it = 0; it < PVI; ++it) c.vscale[it] = vsb[uint32_t((it * TPI + vt) * SB + vd / 2)];
      }
    } else {
      const int t = t0 + lane % 32, in_page = min(t, ctx - 1) % g.bs;
      if (t >= ctx) blk = -1;
      c.valid = uint32_t(__ballot(blk >= 0 && blk < g.num_blocks));
      if (blk < 0 || blk >= g.num_blocks) blk = 0;
      const int64_t base = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + in_page
                              : (int64_t(blk) * g.bs + in_page) * g.Hkv + h;
      auto row_of = [&](int j) -> int64_t {  // cache row of token t0 + j
        const uint32_t lo = __shfl(uint32_t(base), j), hi = __shfl(uint32_t(base >> 32), j);
        return int64_t((uint64_t(hi) << 32) | lo);
      };
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t r = row_of(16 * u + l16);
#pragma unroll
        for (int x = 0; x < KL; ++x) c.k[u][x] = load16(g.kc + r * RB, 16 * h4 + 64 * x);
        if constexpr (MX) c.kscale[u] = *reinterpret_cast<const scale_t*>(g.ks + r * SB);
      }
#pragma unroll
      for (int it = 0; it < PVI; ++it) {
        const int64_t r = row_of(it * TPI + vt);
        c.v[it] = load16(g.vc + r * RB, 16 * vd);
        if constexpr (MX) c.vscale[it] = g.vs[r * SB + vd / 2];
      }
    }
    if constexpr (ALIGNED)
      for (off += kWaves * kChunk; off >= g.bs; off -= g.bs) ++at;
    ask_page(ch + kWaves);
  };

  uint64_t odd = 0;  // query tokens of this wave's chunks with a value that is not finite
  auto step = [&](int ch) {  // takes chunk ch, which c holds, and loads the wave's next one into it
    const int t0 = ch * kChunk;
    const uint32_t valid = c.valid;
    const bool masked = t0 + kChunk > before || valid != ~0u;  // some row may not see some token of the chunk

    // V into the wave's slice
#pragma unroll
    for (int it = 0; it < PVI; ++it) {
      uint16_t* dst = vl + (it * TPI + vt) * VP + EPL * vd;
      if constexpr (MX) {
        const float sc = mx_scale(c.vscale[it]);
        *reinterpret_cast<u32x4*>(dst) = mx_decode8(c.v[it][0], c.v[it][1], sc);
        *reinterpret_cast<u32x4*>(dst + 8) = mx_decode8(c.v[it][2], c.v[it][3], sc);
      } else {
        *reinterpret_cast<u32x4*>(dst) = c.v[it];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // scores: this lane's tokens t0 + 16 u + 4 h4 + r of its rows
    float s[RT][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u && RT > 1) __builtin_amdgcn_sched_barrier(0);
      f32x4_t d[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) d[rt] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < KC; ++x) {
        bf16x8_t a;
        if constexpr (MX) {
          const float sc = mx_scale((uint32_t(c.kscale[u] >> (16 * (x / 2))) >> (8 * (h4 / 2))) & 0xffu);
          a = __builtin_bit_cast(bf16x8_t, mx_decode8(c.k[u][x / 2][2 * (x % 2)], c.k[u][x / 2][2 * (x % 2) + 1], sc));
        } else {
          a = __builtin_bit_cast(bf16x8_t, c.k[u][x]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          d[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[rt][x], d[rt], 0, 0, 0);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[rt][4 * u + r] = d[rt][r];
    }
    __builtin_amdgcn_sched_barrier(0);
    if (ch + kWaves < ch_end) load_chunk(ch + kWaves);
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) hide<8>(s[rt], (uint32_t(visible(before - t0, see[rt])) & valid) >> (4 * h4));
    }
    wave_sync();  // the slice is written
    if (masked) {
      // Values of tokens that take no part, and of query tokens with a value that is not finite, become zeros: some rows
      // may not see them, and 0 times them would be NaN there.
      constexpr int LPR = D / 8, RPS = 64 / LPR;  // lanes per row, rows per step
#pragma unroll 1
      for (int j0 = 0; j0 < kChunk; j0 += RPS) {
        const int j = j0 + lane / LPR;
        u32x4* at = reinterpret_cast<u32x4*>(vl + j * VP + 8 * (lane % LPR));
        const u32x4 w = *at;
        const bool in = (valid >> j) & 1;
        const uint64_t m = __ballot(in && t0 + j >= before && not_finite(w));
        if (!in || ((m >> (lane / LPR * LPR)) & (~0ull >> (64 - LPR))) != 0) *at = u32x4{};
#pragma unroll
        for (int r = 0; r < RPS; ++r)
          if ((m >> (r * LPR)) & (~0ull >> (64 - LPR))) odd |= 1ull << (t0 + j0 + r - before);
      }
      wave_sync();
    }
    const uint16_t* v0 = vl + (4 * h4 + l16 / 4) * VP + 4 * (l16 % 4);
    VFragments<DT, VP> vf;
    vf.load(v0, 0);
    u32x4 phi[RT], plo[RT];  // P^T as the B operand: k slots 0..3 = tokens 4 h4 + r, 4..7 = tokens 16 + 4 h4 + r
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) softmax<8>(s[rt], g.scale_log2, m_run[rt], l_run[rt], acc[rt], &phi[rt], &plo[rt]);
    vf.run(v0, nullptr, [&](int t, const u32x4* f) { multiply(acc, t, f, phi, plo); });
    wave_sync();  // the next chunk rewrites the slice
  };
  if (ch0 < ch_end) load_chunk(ch0);
  for (int ch = ch0; ch < ch_end; ch += kWaves) step(ch);
  for (; odd != 0; odd &= odd - 1) {
    const int k = __builtin_ctzll(odd), t = before + k, blk = bt_row[t / g.bs], off = t % g.bs;  // a valid page
    add_token<D, MX, RT>(g, MX ? (int64_t(blk) * g.Hkv + h) * g.bs + off : (int64_t(blk) * g.bs + off) * g.Hkv + h, k, qf,
                         see, m_run, acc, [&](int x) { return MX ? 64 * (x / 2) + 16 * h4 + 8 * (x % 2) : 32 * x + 8 * h4; });
  }
  finish<D, RT>(g, pc, block, ch_end - pc.ch0, lds, acc, m_run, l_run);
}

// A unit of up to 64 rows: wave w has rows 16 w .. + 15, and a step is 64 tokens, which all waves bring into LDS in bf16
// together (16 bytes of a row a lane, the next step's on the way meanwhile) and all read: what a step costs of the L2 and of
// conversions is shared by all rows. Of the waves on a SIMD the one furthest in its step goes first, but scores before
// softmaxes (products of one wave beside the softmax of another): 3 % off 32 sequences with 128 rows, 1 .. 3 off others.
// 8 bits: 16 codes become 32 bytes of bf16, and 8 lanes that wrote those one behind the other would meet on half of the
// banks. The first 8 of each 16 elements lie in the first half of a row in LDS instead, the others in the second, so that 8
// lanes write 128 bytes in a row; the rows of q are read in that order, and V's fragments from both halves (32 sequences of
// 512 .. 2048 tokens with 128 rows: 73.0 -> 68.3 us).
template <int D, bool MX, bool ALIGNED>
__device__ __forceinline__ void run_wide(const TreeArgs& g, const Piece& pc, int block, unsigned char* lds) {
  constexpr int NU = kStep / 16;                // 16-token tiles of a step
  constexpr int KP = D + 8, VP = D + (MX ? 8 : 16);  // LDS row pitches: fragment reads on distinct banks
  constexpr int HALF = MX ? D / 2 : 8;          // in LDS, from 8 elements to the next 8 of the row
  constexpr int KC = D / 32, DT = D / 16, EPL = MX ? 16 : 8, RB = MX ? D : 2 * D, SB = D / kMxBlock;
  constexpr int LPR = D / EPL, RPP = kWaves * 64 / LPR, NP = kStep / RPP;  // lanes per row, rows per pass, passes
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int l16 = lane % 16, h4 = lane / 16;
  const int b = pc.b, h = pc.h, ctx = context(g, b), R = g.G * g.n, r0 = pc.tile * 64;
  const bool active = r0 + 16 * wave < R;  // otherwise the wave has no row, and only helps to bring the rows in
  const int32_t* bt_row = g.bt + int64_t(b) * g.max_blocks;
  uint16_t* ks = reinterpret_cast<uint16_t*>(lds);
  uint16_t* vs = ks + kStep * KP;
  uint32_t* there = reinterpret_cast<uint32_t*>(vs + kStep * VP);  // unaligned: which of the step's tokens take part

  const int row = r0 + 16 * wave + l16, qi = min(row, R - 1) / g.G;
  bf16x8_t qf[1][KC];
#pragma unroll
  for (int x = 0; x < KC; ++x) qf[0][x] = bf16x8_t{};
  uint64_t see[1] = {0};
  // the dims of a K or q fragment: 8 elements at 32 x + 8 h4 of a row in LDS
  auto dim = [&](int x) { return MX ? 16 * ((4 * x + h4) % LPR) + 8 * (4 * x / LPR) : 32 * x + 8 * h4; };
  if (row < R) {
    const uint16_t* qp = g.q + (int64_t(b) * g.n + qi) * g.q_st + int64_t(h * g.G + row - qi * g.G) * g.q_sh;
#pragma unroll
    for (int x = 0; x < KC; ++x) qf[0][x] = *reinterpret_cast<const bf16x8_t*>(qp + dim(x));
    see[0] = g.mask != nullptr ? uint64_t(g.mask[int64_t(b) * g.n + qi]) : g.causal ? (2ull << qi) - 1 : ~0ull;
  }
  const int before = ctx - g.n;

  float m_run[1] = {-INFINITY}, l_run = 0.0f;
  f32x4_t acc[1][DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[0][t] = f32x4_t{0, 0, 0, 0};

  // this thread's pieces of the next step's rows
  const int prow = tid / LPR, piece = tid % LPR;
  u32x4 kraw[NP], vraw[NP];
  uint32_t kscale[NP], vscale[NP];
  uint64_t valid = 0;  // aligned: which of the step's tokens take part
  uint32_t mine = 0;   // unaligned: bit p, this thread's row of pass p does
  uint64_t odd = 0;    // query tokens among this thread's rows with a value that is not finite
  const int ch_end = min(pc.ch1, (ctx + kStep - 1) / kStep);
  // the table's entries for the next step, asked for one step ahead of its rows (aligned: its page `at`, which it begins
  // `off` tokens into)
  const int last_page = (max(ctx, 1) - 1) / g.bs;
  int page[ALIGNED ? 1 : NP], at = pc.ch0 * kStep / g.bs, off = pc.ch0 * kStep - at * g.bs;
  auto ask_pages = [&](int ch) {
    if constexpr (ALIGNED) {
      page[0] = load_uniform(bt_row + min(at, last_page));
    } else {
#pragma unroll
      for (int p = 0; p < NP; ++p) page[p] = bt_row[min(ch * kStep + p * RPP + prow, ctx - 1) / g.bs];
    }
  };
  auto load_step = [&](int ch) {
    const int t0 = ch * kStep;
    if constexpr (ALIGNED) {
      int blk = page[0];
      valid = ctx - t0 >= 64 ? ~0ull : (1ull << (ctx - t0)) - 1;
      if (blk < 0 || blk >= g.num_blocks) blk = 0, valid = 0;
      const int64_t base = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + off
                              : (int64_t(blk) * g.bs + off) * g.Hkv + h;
      const uint8_t *kb = g.kc + base * RB, *vb = g.vc + base * RB;
      const uint32_t step = MX ? RB : RB * g.Hkv;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kraw[p] = load16(kb, (p * RPP + prow) * step + 16 * piece);
        vraw[p] = load16(vb, (p * RPP + prow) * step + 16 * piece);
      }
      if constexpr (MX) {
        const uint8_t *ksb = g.ks + base * SB, *vsb = g.vs + base * SB;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          kscale[p] = ksb[uint32_t((p * RPP + prow) * SB + piece / 2)];
          vscale[p] = vsb[uint32_t((p * RPP + prow) * SB + piece / 2)];
        }
      }
    } else {
      mine = 0;
      int64_t rows[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int t = t0 + p * RPP + prow, in_page = min(t, ctx - 1) % g.bs;
        int blk = t < ctx ? page[p] : -1;
        if (blk < 0 || blk >= g.num_blocks) blk = 0;
        else mine |= 1u << p;
        rows[p] = MX ? (int64_t(blk) * g.Hkv + h) * g.bs + in_page : (int64_t(blk) * g.bs + in_page) * g.Hkv + h;
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kraw[p] = load16(g.kc + rows[p] * RB, 16 * piece);
        vraw[p] = load16(g.vc + rows[p] * RB, 16 * piece);
        if constexpr (MX) {
          kscale[p] = g.ks[rows[p] * SB + piece / 2];
          vscale[p] = g.vs[rows[p] * SB + piece / 2];
        }
      }
    }
    if constexpr (ALIGNED)
      if ((off += kStep) == g.bs) off = 0, ++at;
    ask_pages(ch + 1);
  };
  // The loaded rows into LDS. Of tokens that take no part, and of query tokens with a value that is not finite, the value is
  // zeros there: some rows may not see them, and 0 times them would be NaN.
  auto stage = [&](int t0) {
    const bool masked = t0 + kStep > before || (ALIGNED && valid != ~0ull) || !ALIGNED;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int j = p * RPP + prow;
      uint16_t *kd = ks + j * KP + 8 * piece, *vd = vs + j * VP + 8 * piece;
      u32x4 v[MX ? 2 : 1];
      if constexpr (MX) {
        const float ka = mx_scale(kscale[p]), va = mx_scale(vscale[p]);
        *reinterpret_cast<u32x4*>(kd) = mx_decode8(kraw[p][0], kraw[p][1], ka);
        *reinterpret_cast<u32x4*>(kd + HALF) = mx_decode8(kraw[p][2], kraw[p][3], ka);
        v[0] = mx_decode8(vraw[p][0], vraw[p][1], va), v[1] = mx_decode8(vraw[p][2], vraw[p][3], va);
      } else {
        *reinterpret_cast<u32x4*>(kd) = kraw[p];
        v[0] = vraw[p];
      }
      if (masked) {
        const bool in = ALIGNED ? (valid >> j) & 1 : (mine >> p) & 1;
        const bool bad = in && t0 + j >= before && (not_finite(v[0]) || (MX && not_finite(v[MX ? 1 : 0])));
        const uint64_t odd_row = (__ballot(bad) >> (lane / LPR * LPR)) & (~0ull >> (64 - LPR));  // of the row's lanes
        if (!in || odd_row != 0) {
#pragma unroll
          for (int x = 0; x < (MX ? 2 : 1); ++x) v[x] = u32x4{};
        }
        if (odd_row != 0) odd |= 1ull << (t0 + j - before);
        if constexpr (!ALIGNED)
          if (piece == 0) there[j] = in;
      }
#pragma unroll
      for (int x = 0; x < (MX ? 2 : 1); ++x) *reinterpret_cast<u32x4*>(vd + HALF * x) = v[x];
    }
  };

  auto compute = [&](int t0, uint64_t live) {  // of a step that is in LDS
    const bool masked = t0 + kStep > before || live != ~0ull;
    // scores: this lane's tokens 16 u + 4 h4 + r of its row, a tile's fragments read while the one before is multiplied
    float s[4 * NU];
    __builtin_amdgcn_s_setprio(1);
    bf16x8_t kf[2][KC];
    auto load_k = [&](int u) {
#pragma unroll
      for (int x = 0; x < KC; ++x)
        kf[u % 2][x] = *reinterpret_cast<const bf16x8_t*>(ks + (16 * u + l16) * KP + 32 * x + 8 * h4);
    };
    load_k(0);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (u + 1 < NU) load_k(u + 1);
      __builtin_amdgcn_sched_barrier(0);
      f32x4_t d = {0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < KC; ++x) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[u % 2][x], qf[0][x], d, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * u + r] = d[r];
    }
    const uint16_t* v0 = vs + (4 * h4 + l16 / 4) * VP + l16 % 4 / 2 * HALF + 4 * (l16 % 2);
    VFragments<DT, VP, MX ? 8 : 16> vf;
    vf.load(v0, 0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (masked) hide<4 * NU>(s, (visible(before - t0, see[0]) & live) >> (4 * h4));
    u32x4 phi[NU / 2], plo[NU / 2];
    softmax<4 * NU>(s, g.scale_log2, m_run[0], l_run, acc[0], phi, plo);
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int y = 0; y < NU / 2; ++y)
      vf.run(v0 + 32 * y * VP, y + 1 < NU / 2 ? v0 + 32 * (y + 1) * VP : nullptr,
             [&](int t, const u32x4* f) { multiply(acc, t, f, phi + y, plo + y); });
    __builtin_amdgcn_s_setprio(3);
  };
  if (pc.ch0 < ch_end) {
    ask_pages(pc.ch0);
    load_step(pc.ch0);
  }
  for (int ch = pc.ch0; ch < ch_end; ++ch) {
    const int t0 = ch * kStep;
    __syncthreads();  // every wave is done with the step before
    stage(t0);
    uint64_t live = valid;
    if (ch + 1 < ch_end) load_step(ch + 1);
    __syncthreads();
    if constexpr (!ALIGNED) live = __ballot(there[lane] != 0);
    if (active) compute(t0, live);
  }
  if (before < pc.ch1 * kStep) {  // the unit's last steps: every wave needs all threads' findings
    uint64_t* all = reinterpret_cast<uint64_t*>(there + kStep);
    __syncthreads();
    if (tid == 0) *all = 0;
    __syncthreads();
    if (odd != 0) atomicOr(reinterpret_cast<unsigned long long*>(all), static_cast<unsigned long long>(odd));
    __syncthreads();
    for (odd = *all; odd != 0; odd &= odd - 1) {
      const int k = __builtin_ctzll(odd), t = before + k, blk = bt_row[t / g.bs], off = t % g.bs;  // a valid page
      if (t / kStep < pc.ch0 || t / kStep >= pc.ch1) continue;
      add_token<D, MX, 1>(g, MX ? (int64_t(blk) * g.Hkv + h) * g.bs + off : (int64_t(blk) * g.bs + off) * g.Hkv + h, k, qf,
                           see, m_run, acc, dim);
    }
  }
  // to the output, or into a record that tree_combine_kernel merges with the other blocks' (through plain stores: that is
  // another launch): (max, sum) of each row, then O [row][D]
  if (g.ws != nullptr && tid == 0 && block == pc.first)
    g.plan[(b * g.Hkv + h) * g.tiles + pc.tile] = int2{pc.first, pc.parts};
  const float l = pair32_sum(pair16_sum(l_run));
  if (row >= R) return;
  if (pc.parts == 1) {
    uint16_t* out = g.out + (int64_t(b) * g.n + qi) * g.o_st + int64_t(h * g.G + row - qi * g.G) * g.o_sh + 4 * h4;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const f32x4_t o = acc[0][t];
      *reinterpret_cast<u32x2*>(out + 16 * t) =
          l == 0.0f ? u32x2{} : u32x2{pack_bf16x2(o[0] / l, o[1] / l), pack_bf16x2(o[2] / l, o[3] / l)};
    }
  } else {
    float* rec = g.ws + (2 * int64_t(block) + (block == pc.first ? 1 : 0)) * (int64_t(64) * (2 + D));
    const int r = 16 * wave + l16;
    if (h4 == 0) *reinterpret_cast<f32x2*>(rec + 2 * r) = f32x2{m_run[0], l};
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4_t*>(rec + 128 + r * D + 16 * t + 4 * h4) = acc[0][t];
  }
}

// The units of a kernel: 16 or 32 rows (run_piece), or 64 (run_wide).
template <int ROWS>
struct Shape {
  static constexpr int rows = ROWS;
  static constexpr bool wide = ROWS == 64;
  static constexpr int tokens = wide ? kStep : kChunk;          // of a chunk
  // What starting and finishing a piece costs beside its chunks, in chunks (measured per block: 4.4 us of 0.57 us a chunk, 10
  // of 0.6, and 4 us of 2 us): without it the blocks with many short units end last (250 sequences 218 -> 187 us).
  static constexpr int start = wide ? 2 : ROWS == 32 ? 16 : 8;
  // Units of no more chunks than a start costs are not split: a second start and the merge took longer (484 units of 6 chunks
  // 23.9 -> 20.0 us, 258 of 24 rows 22.3 -> 18.7; units of twice as many gain from the split: 208 of 10 .. 15 13.8 -> 13.2).
  static constexpr int whole = 2 * start;
  // chunks that a block takes at least (64 rows: a unit of one step; with 4, 5 sequences of up to 34 tokens 8.0 -> 11.5 us)
  static constexpr int least = wide ? start + 1 : 8;
  static constexpr int max_parts = wide ? 64 : 2048 / rows;     // of a unit (not wide: their maxima and sums fit the LDS)
  // What the registers are laid out for. bf16 rows of 256 elements: a chunk's rows and the sums take 390 registers; as two
  // waves with 256 each, and the rest in scratch memory, 1 sequence of 11k tokens with 40 rows took 34.6 us for 20.8, 169 of 50
  // with 4 rows 37.4 for 26.7.
  static constexpr int waves_per_simd(int D, bool MX) { return D == 256 ? (MX ? 2 : 1) : wide ? 3 : 2; }
  static constexpr int blocks(int D, bool MX) { return 256 * waves_per_simd(D, MX); }  // of a split launch: all resident at once
};

template <int D, bool MX, bool ALIGNED, class S>
__global__ __launch_bounds__(kWaves * 64, S::waves_per_simd(D, MX)) void tree_attention_kernel(const TreeArgs g) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[lds_bytes(D, S::wide)];
  auto chunks_of = [](int ctx) { return max(1, (ctx + S::tokens - 1) / S::tokens); };
  const int U = g.Hkv * g.tiles;  // units of a sequence
  int p = 0, at, end, b, begin = 0, quota = INT32_MAX, more = 0;  // without a split: one block has everything
  if (g.ws == nullptr) {
    b = int(blockIdx.x) / U;
    const int w = S::start + chunks_of(context(g, b));
    at = (int(blockIdx.x) - b * U) * w, end = at + w;
  } else {
    // a unit's chunks of each sequence: lane l sums those of sequences [l per_lane, (l + 1) per_lane)
    const int lane = threadIdx.x % 64, per_lane = (g.num_seqs + 63) / 64;
    int sum = 0, longest = 0;
    for (int j = lane * per_lane; j < min((lane + 1) * per_lane, g.num_seqs); ++j) {
      const int w = S::start + chunks_of(min(max(g.ctx_lens[j], 0), g.max_blocks * g.bs));
      sum += w, longest = max(longest, w);
    }
    const int incl = wave_scan(sum, [](int x, int y) { return x + y; });
    const int C = __builtin_amdgcn_readlane(incl, 63) * U;
    longest = __builtin_amdgcn_readlane(wave_scan(longest, [](int x, int y) { return max(x, y); }), 63);
    // A block takes enough that no unit lies in more than max_parts of them (one at either end), and, where the last of a
    // unit's blocks merges them alone, about the square root of (chunks x merging a part / a chunk): c chunks in P parts
    // take c / P of 0.4 us and P of 0.27 us (32 rows of 64; less with fewer rows).
    int least = max(S::least, (longest + S::max_parts - 3) / (S::max_parts - 2));
    if (!S::wide) least = max(least, int(__builtin_sqrtf(float(longest) * float(min(g.G * g.n, S::rows) * D) / 1536.0f)));
    const int N = max(1, min(int(gridDim.x), C / least));
    quota = C / N, more = C - quota * N;  // the first `more` blocks take quota + 1 chunks
    // blocks p of one XCD (blockIdx.x % 8) are neighbours: row tiles of a kv head read the same rows through one L2
    const int per = (N + 7) / 8;
    p = int(blockIdx.x % 8) * per + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per || p >= N) return;
    at = p * quota + min(p, more);
    end = at + quota + (p < more ? 1 : 0);
    // the sequence that holds chunk `at`: the lane that holds it, then its sequences one by one
    const int from = __builtin_amdgcn_readfirstlane(__popcll(__ballot(incl * U <= at)));
    b = from * per_lane;
    begin = __builtin_amdgcn_readlane(incl - sum, from) * U;  // first chunk of sequence b
  }
  auto block_of = [&](int x) {  // the block that takes chunk x
    return x < more * (quota + 1) ? x / (quota + 1) : more + (x - more * (quota + 1)) / quota;
  };
  while (at < end) {
    const int c = chunks_of(context(g, b)), w = S::start + c;
    if (at >= begin + w * U) {
      begin += w * U;
      ++b;
      continue;
    }
    const int u = (at - begin) / w, u0 = begin + u * w + S::start;  // u0: its first chunk
    const bool whole = w <= S::whole, mine = !whole || at == u0 - S::start;  // a whole unit is of the block it begins in
    const int stop = whole ? u0 + c : min(end, u0 + c);
    const int first = whole ? p : block_of(u0), last = whole ? p : block_of(u0 + c - 1);
    if (mine && stop > u0) {
      const Piece pc{b, u / g.tiles, u % g.tiles, max(at, u0) - u0, stop - u0, first, last - first + 1};
      if constexpr (S::wide) run_wide<D, MX, ALIGNED>(g, pc, p, lds);
      else run_piece<D, MX, ALIGNED, S::rows / 16>(g, pc, p, lds);
      if (stop < end) __syncthreads();  // the next piece reuses the LDS
    }
    at = stop;
  }
}

// The records of 64-row units that several blocks share: a lane has 4 elements of O. SPLIT waves share them, each with every
// SPLIT-th record in the blocks' order, kAhead on the way at a time; their sums are joined in LDS.
template <int D, int SPLIT>
__global__ __launch_bounds__(kWaves * 64) void tree_combine_kernel(const TreeArgs g) {
  constexpr int RU = 64, kSlices = RU * D * SPLIT / 1024, kAhead = SPLIT == 1 ? 4 : 8;  // rows, blocks of a unit
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), k_first = wave % SPLIT;
  const int unit = int(blockIdx.x) / kSlices;
  const int at = ((int(blockIdx.x) % kSlices * kWaves + wave) / SPLIT * 64 + lane) * 4;
  const int2 plan = g.plan[unit];
  const int tile = unit % g.tiles, bh = unit / g.tiles, b = bh / g.Hkv, h = bh % g.Hkv;
  const int r = at / D, d = at % D, row = tile * RU + r;
  if (plan.y == 1) return;
  float M = -INFINITY, den = 0.0f;
  f32x4_t sum = {0, 0, 0, 0};
  if (row < g.G * g.n) {
    for (int k0 = k_first; k0 < plan.y; k0 += SPLIT * kAhead) {
      f32x2 ml[kAhead];
      f32x4_t o[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + SPLIT * u;
        ml[u] = f32x2{-INFINITY, 0.0f};
        o[u] = f32x4_t{0, 0, 0, 0};
        if (k >= plan.y) continue;
        const float* rec = g.ws + (2 * int64_t(plan.x + k) + (k == 0 ? 1 : 0)) * (int64_t(RU) * (2 + D));
        ml[u] = *reinterpret_cast<const f32x2*>(rec + 2 * r);
        o[u] = *reinterpret_cast<const f32x4_t*>(rec + 2 * RU + r * D + d);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) top = fmaxf(top, ml[u][0]);
      const float keep = share(M, den, top);
      M = top, den *= keep;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] *= keep;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float f = share(ml[u][0], ml[u][1], M);
        den = __builtin_fmaf(ml[u][1], f, den);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(o[u][e], f, sum[e]);
      }
    }
  }
  if constexpr (SPLIT > 1) {
    static_assert(SPLIT == kWaves, "the block's waves");
    __shared__ float part[kWaves][6][64];
    part[wave][0][lane] = M, part[wave][1][lane] = den;
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][2 + e][lane] = sum[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, part[w][0][lane]);
    den = 0.0f, sum = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = share(part[w][0][lane], part[w][1][lane], M);
      den = __builtin_fmaf(part[w][1][lane], f, den);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(part[w][2 + e][lane], f, sum[e]);
    }
  }
  if (row >= g.G * g.n) return;
  const int i = row / g.G;
  uint16_t* out = g.out + (int64_t(b) * g.n + i) * g.o_st + int64_t(h * g.G + row - i * g.G) * g.o_sh + d;
  *reinterpret_cast<u32x2*>(out) = den == 0.0f ? u32x2{} : u32x2{pack_bf16x2(sum[0] / den, sum[1] / den),
                                                                pack_bf16x2(sum[2] / den, sum[3] / den)};
}

template <int D, bool MX, class S>
int launch(const TreeArgs& g, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWaves * 64);
  if (g.bs % S::tokens == 0) hipLaunchKernelGGL((tree_attention_kernel<D, MX, true, S>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((tree_attention_kernel<D, MX, false, S>), grid, block, 0, s, g);
  if (int rc = check_launch("tree_attention")) return rc;
  if (!S::wide || g.ws == nullptr) return NVHIP_OK;
  // Few units: many records each, which the waves of a block share (8 units of up to 64 records 51.4 -> 45.0 us; 512 units
  // of two or three 69.3 -> 73.2).
  const int64_t units = int64_t(g.num_seqs) * g.Hkv * g.tiles, slices = units * (64 * D / 1024);
  const dim3 one(static_cast<unsigned>(slices)), shared(static_cast<unsigned>(kWaves * slices));
  if (units * 16 > blocks) hipLaunchKernelGGL((tree_combine_kernel<D, 1>), one, block, 0, s, g);
  else hipLaunchKernelGGL((tree_combine_kernel<D, kWaves>), shared, block, 0, s, g);
  return check_launch("tree_attention (combine)");
}

// Rows of a unit for R = (Hq / Hkv) q_len rows of a kv head. 33 .. 64 rows as two units of 32 (8 sequences of 1000 .. 4000
// tokens with 66 rows) took 53 us, as units of 64 rows 37 at that time.
// Heads of 256 have no registers for two row tiles in a wave.
int unit_rows(int64_t R, int64_t D) { return R <= 16 ? 16 : R <= 32 && D < 256 ? 32 : 64; }

// Blocks of the split launch: none without a chunk at the longest possible context.
int64_t split_blocks(int64_t units, int64_t rows, int64_t D, bool mx, int64_t max_ctx) {
  const int64_t most = units * std::max<int64_t>(1, (max_ctx + kChunk - 1) / kChunk);
  return std::min<int64_t>(rows == 64 ? Shape<64>::blocks(int(D), mx) : Shape<16>::blocks(int(D), mx), (most + 7) / 8 * 8);
}
struct Workspace {
  int64_t count_bytes, bytes;
};
Workspace workspace_of(int64_t units, int64_t blocks, int64_t rows, int64_t D) {
  const int64_t counts = units * kCountStride * 8;
  return {counts, counts + blocks * 2 * rows * (2 + D) * 4};
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
  const int64_t R = Hq / Hkv * q_len, rows = unit_rows(R, D), units = num_seqs * Hkv * ((R + rows - 1) / rows);
  // 8 bit: the launch with more blocks
  return workspace_of(units, split_blocks(units, rows, D, true, max_blocks * block_size), rows, D).bytes;
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
      out_stride_token < Hq * out_stride_head || q_stride_head % 8 != 0 || q_stride_token % 8 != 0 ||
      out_stride_head % 4 != 0 || out_stride_token % 4 != 0 || reinterpret_cast<uintptr_t>(out) % 8 != 0)
    return invalid("tree_attention: bad q / out strides (rows of D contiguous; q 16-byte, out 8-byte aligned)");
  if (!(scale > 0.0f) || scale > 3e38f) return invalid("tree_attention: softmax_scale must be positive and finite");
  if ((k_scales == nullptr) != (v_scales == nullptr))
    return invalid("tree_attention: k_scales and v_scales must be given together");
  // (a head's rows of a page step lie up to 63 Hkv 2 D bytes apart, counted in 32 bits)
  if (Hq > (1 << 16) || num_seqs > (1 << 24) || num_blocks > INT32_MAX || block_size > INT32_MAX ||
      max_blocks > INT32_MAX || max_blocks * block_size > INT32_MAX - 64)
    return invalid("tree_attention: size too large");
  if (num_seqs == 0) return NVHIP_OK;
  if (!out || !q || !context_lens || (max_blocks > 0 && !block_table) || (num_blocks > 0 && (!k_cache || !v_cache)))
    return invalid("tree_attention: null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scales) || !aligned16(v_scales))
    return invalid("tree_attention: q, the caches and the scales must be 16-byte aligned");
  const int64_t R = Hq / Hkv * q_len, rows = unit_rows(R, D);
  TreeArgs g{};
  g.out = static_cast<uint16_t*>(out), g.q = static_cast<const uint16_t*>(q);
  g.kc = static_cast<const uint8_t*>(k_cache), g.vc = static_cast<const uint8_t*>(v_cache);
  g.ks = static_cast<const uint8_t*>(k_scales), g.vs = static_cast<const uint8_t*>(v_scales);
  g.bt = block_table, g.ctx_lens = context_lens, g.mask = tree_mask;
  g.n = int(q_len), g.Hkv = int(Hkv), g.G = int(Hq / Hkv), g.bs = int(block_size), g.num_blocks = int(num_blocks);
  g.max_blocks = num_blocks > 0 ? int(max_blocks) : 0;  // without pages every context is empty
  g.num_seqs = int(num_seqs), g.tiles = int((R + rows - 1) / rows);
  g.q_st = q_stride_token, g.q_sh = q_stride_head, g.o_st = out_stride_token, g.o_sh = out_stride_head;
  g.scale_log2 = scale * 1.4426950408889634f;
  g.causal = causal ? 1 : 0;
  // Rows that are read once (one row tile) and cannot all stay in the 256 MB Infinity Cache for the next call are read past
  // it: 250 sequences (1 GB) 193 -> 187 us; 32 sequences (94 MB, part of which is still there) 25.3 us without, 28.9 with.
  const int64_t row_bytes = k_scales != nullptr ? D + D / kMxBlock : 2 * D;
  g.once = g.tiles == 1 && double(num_seqs) * double(max_blocks * block_size) * double(2 * Hkv * row_bytes) > 512e6;
  const int64_t units = num_seqs * Hkv * g.tiles;
  // chunks are counted in 32 bits
  if (units > INT32_MAX / 1024 || double(units) * double(max_blocks * block_size / kChunk + 2 + 64) > double(INT32_MAX))
    return invalid("tree_attention: size too large");
  int64_t blocks = units;
  const int64_t split = split_blocks(units, rows, D, k_scales != nullptr, max_blocks * block_size);
  const Workspace w = workspace_of(units, split, rows, D);
  if (workspace != nullptr && workspace_size >= w.bytes) {
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return invalid("tree_attention: workspace must be 16-byte aligned");
    blocks = split;
    g.counts = static_cast<unsigned long long*>(workspace);  // or, of units of more than 32 rows, the plan
    g.plan = static_cast<int2*>(workspace);
    g.ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.count_bytes);
    g.call = next_call();
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto by_rows = [&](auto mx, auto dim) {
    constexpr bool MX = decltype(mx)::value;
    constexpr int d = decltype(dim)::value;
    if (rows == 16) return launch<d, MX, Shape<16>>(g, blocks, s);
    if constexpr (d < 256)
      if (rows == 32) return launch<d, MX, Shape<32>>(g, blocks, s);
    return launch<d, MX, Shape<64>>(g, blocks, s);
  };
  auto by_dim = [&](auto mx) {
    if (D == 64) return by_rows(mx, std::integral_constant<int, 64>{});
    if (D == 128) return by_rows(mx, std::integral_constant<int, 128>{});
    return by_rows(mx, std::integral_constant<int, 256>{});
  };
  return k_scales != nullptr ? by_dim(std::true_type{}) : by_dim(std::false_type{});
}
