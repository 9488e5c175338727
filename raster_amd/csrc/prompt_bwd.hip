// prompt_bwd.hip — gradient of the attention over packed prompts (prompt.hip).
//
// With P the forward's weights, recomputed as exp(s - L) from its log-sum-exp L:
//   D_i  = dO_i . O_i
//   dV_j = sum_i p_ij dO_i
//   dS_ij = p_ij (dO_i . V_j - D_i)
//   dQ_i = scale sum_j dS_ij K_j      dK_j = scale sum_i dS_ij Q_i
// the sums over i of dK and dV also over the query heads of the KV head.
//
// Three parts, none with an atomic, so results do not depend on scheduling: D; dK
// and dV (a wave owns 32 keys and walks the queries of every head of its group); dQ
// (a wave owns 32 queries and walks the keys). The scores and dO V^T are formed
// in both of the last two: 7 products for the 5 that a single kernel would need, which
// would have to add dQ from many workgroups.
//
// Bound by the matrix instructions and the chain product - exponential - product of a step, with two waves a
// SIMD: 2048, 777, 1500, 331, 1999 and 64 tokens, bf16, 32/8 heads x 128: 19 + 5.5 us for D, 433 for the rest
// (dQ alone 195, dK and dV alone 350), 0.73 PFLOP/s of the 7 products, matrix pipe busy 0.34. f32, 129, 300, 64
// and 511 tokens, 16/2 heads x 64: 4.8 + 53 + 6.8 us (the parts' sum).
//
// With a window (WIN) each walk is of the tiles that the window or the sinks reach: 4096, 777, 1500, 331, 1999 and 64
// tokens, bf16, 32/8 heads x 128, window 1024 and 4 sinks: 25 + 6 us for D, 600 for the rest, 5 for the sinks' sum
// (160 the forward), 0.5 PFLOP/s of the pairs that count: shorter walks, in
// which the first loads and the masked tiles at both edges weigh more.
//
// Rounded to bf16 in the bf16 kernels: P for dV, dS for dK and dQ (operands of their products), and the results.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "attn_tile.h"
#include "prompt.h"

namespace rq {

namespace {

// L in base 2; +inf, which makes every weight 0, where no key had one (L = -inf)
__device__ __forceinline__ float base2_lse(float lse) {
  return lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
}

// D of a row and head: LANES lanes a (row, head), 16 bytes each at a time.
constexpr int kDeltaLanes = 16;
template <typename T>
__global__ __launch_bounds__(256) void prompt_delta_kernel(PromptArgs a) {
  constexpr int E = TileType<T>::kPiece;
  typedef T TE __attribute__((ext_vector_type(E)));
  const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kDeltaLanes;
  const int sub = threadIdx.x % kDeltaLanes;
  if (id >= a.rows_q * a.n_q) return;
  const int64_t row = id / a.n_q;
  if (row < clamp_cu(a.cu_q, 0, a.rows_q) || row >= clamp_cu(a.cu_q, a.batch, a.rows_q)) return;  // of no sequence
  const int hq = (int)(id % a.n_q);
  const T* o = static_cast<const T*>(a.out) + row * a.out_stride + hq * a.head_dim;
  const T* d = static_cast<const T*>(a.dout) + row * a.dout_stride + hq * a.head_dim;
  float sum = 0.0f;
  for (int e = sub * E; e < a.head_dim; e += kDeltaLanes * E) {
    const TE x = *reinterpret_cast<const TE*>(o + e), y = *reinterpret_cast<const TE*>(d + e);
#pragma unroll
    for (int j = 0; j < E; j++) sum += (float)x[j] * (float)y[j];
  }
#pragma unroll
  for (int k = kDeltaLanes / 2; k >= 1; k >>= 1) sum += __shfl_xor(sum, k, 64);
  if (sub == 0) a.delta[(int64_t)hq * a.rows_q + row] = sum;
}

// D of the queries that see at most kExactKeys keys, anew. In bf16 O has been rounded, and what D is off by
// reaches dQ and dK through every weight of its row: little where many keys share the weight, but for
// the first queries of a sequence as much as all other roundings together (error of dQ of 37, 5 and 12
// tokens, in roundings of the result: 1.60; of 777, 1500, 331 and 64: 1.50). Here D is formed from the
// weights, sum_j p_ij dO_i . V_j (1.42 and 1.43; with 256 keys 1.43).
// This kernel takes a sequence's first queries, those with at most kExactKeys keys up to themselves; with a window and
// sinks of no more than that in all, every query is one of few keys, and prompt_delta_few_kernel's.
// One workgroup a sequence and head (without a causal mask several, for its many queries): a wave
// 32 queries and 32 keys. 5.5 us beside the other kernel's 19 at 6719 tokens in six sequences, 32/8 heads x 128
// (from registers, each lane its row, 15: 64 cache lines a load).
constexpr int kExactKeys = 64, kExactTiles = 8;
template <typename T, int HD>
__global__ __launch_bounds__(256) void prompt_delta_exact_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  constexpr int kTile = TL::bytes(64);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float part[4][32];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, i = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), qb = 32 * (wave & 1), kb = 32 * (wave >> 1);
  const int hq = blockIdx.x % a.n_q, hkv = hq / (a.n_q / a.n_kv), rest = blockIdx.x / a.n_q;
  const int b = rest % a.batch, tile = rest / a.batch;
  const int64_t q0 = clamp_cu(a.cu_q, b, a.rows_q), q1 = clamp_cu(a.cu_q, b + 1, a.rows_q);
  const int64_t k0 = clamp_cu(a.cu_k, b, a.rows_k), k1 = clamp_cu(a.cu_k, b + 1, a.rows_k);
  const int lq = (int)(q1 > q0 ? q1 - q0 : 0), lk = (int)(k1 > k0 ? k1 - k0 : 0), off = lk - lq;
  // (queries before -off see no key: out is 0 there, and so is D already)
  const int begin = a.causal ? max(-off, 0) : 0, end = a.causal ? min(lq, kExactKeys - off) : lk <= kExactKeys ? lq : 0;
  for (int row0 = begin + 64 * tile; row0 < end; row0 += 64 * kExactTiles) {
    const int64_t first = q0 + row0;
    {
      Stage<T, HD, 64, 256> x, y;
      x.load(static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim, a.k_stride, lk, a.head_dim, tid);
      y.load(static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim, a.v_stride, lk, a.head_dim, tid);
      x.store(lds, tid);
      y.store(lds + kTile, tid);
      x.load(static_cast<const T*>(a.q) + first * a.q_stride + hq * a.head_dim, a.q_stride, end - row0, a.head_dim, tid);
      y.load(static_cast<const T*>(a.dout) + first * a.dout_stride + hq * a.head_dim, a.dout_stride, end - row0,
             a.head_dim, tid);
      x.store(lds + 2 * kTile, tid);
      y.store(lds + 3 * kTile, tid);
    }
    const int r = qb + i, see = a.causal ? min(lk - 1, row0 + r + off) : lk - 1;
    const int from = a.window > 0 ? row0 + r + off - a.window + 1 : 0;
    const float lse = base2_lse(a.lse[(int64_t)hq * a.rows_q + first + min(r, end - row0 - 1)]);
    __syncthreads();
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int d = 0; d < HD / 16; d++) {
      s = tile_mma(TL::frag(lds, kb + i, d, h), TL::frag(lds + 2 * kTile, r, d, h), s);
      dp = tile_mma(TL::frag(lds + kTile, kb + i, d, h), TL::frag(lds + 3 * kTile, r, d, h), dp);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const int key = kb + 8 * (j >> 2) + 4 * h + (j & 3);
      if (key <= see && (key >= from || key < a.sinks))
        sum += __builtin_amdgcn_exp2f(fmaf(s[j], a.scale2, -lse)) * dp[j];
    }
    sum += __shfl_xor(sum, 32, 64);
    if (h == 0) part[wave][i] = sum;
    __syncthreads();
    if (tid < 64 && row0 + tid < end)
      a.delta[(int64_t)hq * a.rows_q + first + tid] = part[tid >> 5][tid & 31] + part[2 + (tid >> 5)][tid & 31];
    __syncthreads();
  }
}

// D of all queries from their weights where window + sinks <= kExactKeys: 64 queries a workgroup, its sinks' tile and
// those that its window reaches, a wave 32 queries and 32 keys of each. It takes the place of both others. Error of dQ
// of its norm, D from the rounded O and this way, queries from 64 on: window 2 0.0037 / 0.0023, 8 and 4 sinks 0.0026 /
// 0.0023, 32 0.0025 / 0.0024, 60 and 4 sinks 0.0025 / 0.0024 (100 and 4 sinks, O: 0.0024). us of the whole gradient, so:
// 4096, 777, 1500, 331, 1999 and 64 tokens, 32/8 heads x 128, window 2 213 / 230, 60 and 4 sinks 275 / 302; 1000 and
// 500, 16/4 x 256, 2 57 / 61; 512, 16/2 x 64, 2 41 / 39; 37, 5 and 12, 32/8 x 128, 33 / 30.
static bool few_keys(const PromptArgs& a) { return a.window > 0 && a.window + a.sinks <= kExactKeys; }
template <typename T, int HD>
__global__ __launch_bounds__(256) void prompt_delta_few_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  constexpr int kTile = TL::bytes(64);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float part[4][32];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, i = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), qb = 32 * (wave & 1), kb = 32 * (wave >> 1);
  const int group = a.n_q / a.n_kv, hkv = blockIdx.x % a.n_kv, rest = blockIdx.x / a.n_kv, hq = hkv * group + rest % group;
  const TileSpan tq = tile_of_slot(a.cu_q, a.batch, a.rows_q, 64, rest / group);
  if (tq.len == 0) return;
  const int64_t k0 = clamp_cu(a.cu_k, tq.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tq.seq + 1, a.rows_k);
  const int lk = (int)(k1 > k0 ? k1 - k0 : 0), n = min(tq.len - tq.row0, 64), pos = tq.row0 + lk - tq.len;
  const int64_t first = tq.begin + tq.row0;
  Walk<true> walk;
  const int nk = min(max(pos + n, 0), lk) - walk.leave_out(a, pos, 64);
  const T* kbase = static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim;
  const T* vbase = static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim;
  Stage<T, HD, 64, 256> x, y;
  auto load = [&](int key) {
    x.load(kbase + (int64_t)key * a.k_stride, a.k_stride, walk.rows_from(key, lk), a.head_dim, tid);
    y.load(vbase + (int64_t)key * a.v_stride, a.v_stride, walk.rows_from(key, lk), a.head_dim, tid);
  };
  x.load(static_cast<const T*>(a.q) + first * a.q_stride + hq * a.head_dim, a.q_stride, n, a.head_dim, tid);
  y.load(static_cast<const T*>(a.dout) + first * a.dout_stride + hq * a.head_dim, a.dout_stride, n, a.head_dim, tid);
  x.store(lds + 2 * kTile, tid);
  y.store(lds + 3 * kTile, tid);
  if (nk > 0) load(walk.key(0));
  const int r = qb + i;
  Seen<true> see;
  see.init(a, tq.row0 + r, lk - tq.len, lk);
  const float lse = base2_lse(a.lse[(int64_t)hq * a.rows_q + first + min(r, n - 1)]);
  float sum = 0.0f;
  for (int at = 0; at < nk; at += 64) {
    x.store(lds, tid);
    y.store(lds + kTile, tid);
    if (at + 64 < nk) load(walk.key(at + 64));
    __syncthreads();
    const int key = walk.key(at) + kb;
    if (key <= pos + qb + 31 && window_any<true>(a, pos + qb, key, 32)) {
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int d = 0; d < HD / 16; d++) {
        s = tile_mma(TL::frag(lds, kb + i, d, h), TL::frag(lds + 2 * kTile, r, d, h), s);
        dp = tile_mma(TL::frag(lds + kTile, kb + i, d, h), TL::frag(lds + 3 * kTile, r, d, h), dp);
      }
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (see.sees(key + 8 * (j >> 2) + 4 * h + (j & 3)))
          sum += __builtin_amdgcn_exp2f(fmaf(s[j], a.scale2, -lse)) * dp[j];
    }
    __syncthreads();
  }
  sum += __shfl_xor(sum, 32, 64);
  if (h == 0) part[wave][i] = sum;
  __syncthreads();
  if (tid < n) a.delta[(int64_t)hq * a.rows_q + first + tid] = part[tid >> 5][tid & 31] + part[2 + (tid >> 5)][tid & 31];
}

template <typename T, int HD>
__device__ __forceinline__ void store_rows(T* row, const f32x16 (&acc)[HD / 32], float f, int h, int hd) {
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int e = 32 * d + 2 * i + 4 * h;
      if (e >= hd) continue;
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y;
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = (T)(acc[d][i + j] * f);
      *reinterpret_cast<T4*>(row + e) = y;
    }
}

// Weights on their way from one wave to another, 16 a lane: f32 as they are; in the bf16 kernel their
// upper 24 bits (cut off at 2^-16 of the value), for which there is just room in LDS. Rounded to bf16 here
// and again as gradients, dK would be off by 0.0030 of its norm instead of 0.0025.
template <typename T>
struct Handover {
  static constexpr int N = sizeof(T) == 4 ? 4 : 3;  // 16-byte pieces a lane
  static __device__ __forceinline__ void put(char* at, const float* x) {
    u32x4 w[N];
    uint32_t* o = reinterpret_cast<uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t a = __float_as_uint(x[4 * i]), b = __float_as_uint(x[4 * i + 1]),
                     c = __float_as_uint(x[4 * i + 2]), d = __float_as_uint(x[4 * i + 3]);
      if constexpr (N == 4) {
        o[4 * i] = a, o[4 * i + 1] = b, o[4 * i + 2] = c, o[4 * i + 3] = d;
      } else {
        o[3 * i] = __builtin_amdgcn_perm(b, a, 0x05030201);
        o[3 * i + 1] = __builtin_amdgcn_perm(c, b, 0x06050302);
        o[3 * i + 2] = __builtin_amdgcn_perm(d, c, 0x07060503);
      }
    }
#pragma unroll
    for (int k = 0; k < N; k++) *reinterpret_cast<u32x4*>(at + k * 64 * 16) = w[k];
  }
  static __device__ __forceinline__ void take(const char* at, float* x) {
    u32x4 w[N];
#pragma unroll
    for (int k = 0; k < N; k++) w[k] = *reinterpret_cast<const u32x4*>(at + k * 64 * 16);
    const uint32_t* o = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t y[4];
      if constexpr (N == 4) {
        y[0] = o[4 * i], y[1] = o[4 * i + 1], y[2] = o[4 * i + 2], y[3] = o[4 * i + 3];
      } else {
        y[0] = o[3 * i] << 8;
        y[1] = __builtin_amdgcn_perm(o[3 * i + 1], o[3 * i], 0x0504030C);
        y[2] = __builtin_amdgcn_perm(o[3 * i + 2], o[3 * i + 1], 0x0403020C);
        y[3] = o[3 * i + 2] & 0xFFFFFF00u;
      }
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * i + j] = __uint_as_float(y[j]);
    }
  }
};

// The slot of a sequence's first chunk, the others behind it. All sequences cut: as in tile_of_slot, one each and one for
// each chunk of rows. Only those of more than a chunk (few_cut): two chunks and more have room in slots of half a
// chunk before the next sequence's. (Which, by an argument and not the template: 8767 tokens in six sequences 595 -> 601 us.)
template <bool FEW_CUT>
__device__ __forceinline__ int64_t sink_slot0(const PromptArgs& a, int b) {
  const int64_t q0 = clamp_cu(a.cu_q, b, a.rows_q);
  return FEW_CUT ? q0 / (a.sink_chunk / 2) : q0 / a.sink_chunk + b;
}

// dK and dV of 64 keys: query tiles of 32 or 64 rows through LDS, two waves for each 32
// keys. One holds K and dV: it forms S = Q K^T and P, and adds dO^T P to dV; the
// other holds V and dK: it forms dO V^T meanwhile, takes P over through LDS and adds
// Q^T dS to dK. So a wave needs the registers of one operand and one result only
// (two to three waves a SIMD instead of one), and both do the same two products in
// each half of a step.
//
// The steps of a workgroup go from the sequence's last queries down, every query head of the group at each
// tile: workgroups that began together read the same tiles at the same time, from their L2.
// us, dK/dV alone, bf16, 32/8 heads x 128, 8192 queries: 1333 (heads outside, queries upwards: 1386).
// The steps are one of nsplit parts;
// with more than one the parts' f32 sums go to a.part and prompt_dkv_sum_kernel adds them in
// order.
constexpr int kDkvKeys = 64, kDqQueries = 128;
// 64 queries a step halve the barriers (the whole gradient of 2048, 777, 1500, 331, 1999 and 64 tokens:
// 461 us, with 32 480); f32 and heads past 128 have no registers for them.
template <typename T, int HD>
constexpr int dkv_queries() {
  return sizeof(T) == 2 && HD <= 128 ? 64 : 32;
}
template <typename T, int HD>
constexpr int dkv_lds() {  // twice Q, dO, L and D of a step, and two pairs' weights
  return 2 * (2 * Tile<T, HD>::bytes(dkv_queries<T, HD>()) + 2 * dkv_queries<T, HD>() * 4) +
         2 * Handover<T>::N * 16 * 64 * dkv_queries<T, HD>() / 32;
}

//
// With `sink` (WIN) one of the first keys' tiles, which all later queries see, and one chunk of the queries; the sums
// go to a.sink_part and prompt_sink_sum_kernel adds them in order. As one workgroup's steps those tiles would be the
// last to end, long after the others, which see the queries of the window only: forward and gradient of 4096, 777,
// 1500, 331, 1999 and 64 tokens, bf16, 32/8 heads x 128, window 1024 and 4 sinks: 1181 us, by chunks 740 to 780.
template <typename T, int HD, bool WIN, bool FEW_CUT>
__device__ __forceinline__ void dkv_body(const PromptArgs& a, int block, bool sink, char* lds) {
  using TL = Tile<T, HD>;
  using Frag = typename TL::Frag;
  constexpr int THREADS = 256, BQ = dkv_queries<T, HD>(), NT = BQ / 32;
  constexpr int kTile = TL::bytes(BQ);
  constexpr int kBuf = 2 * kTile + 2 * BQ * 4;  // Q, dO, then L and D of the rows
  constexpr int kShare = Handover<T>::N * 16 * 64, kPair = NT * kShare;  // weights of 32 keys and 32 or all queries
  const int group = a.n_q / a.n_kv;
  const int hkv = block % a.n_kv, rest = block / a.n_kv, split = rest % a.nsplit;
  const int sink_tile = WIN && sink ? rest / a.nsplit % a.sink_tiles : 0;
  // a sequence's first keys, which most queries see, first
  const int64_t slot = WIN && sink ? rest / a.nsplit / a.sink_tiles : rest / a.nsplit;
  TileSpan tk;
  int chunk = 0;  // first query of the chunk
  if (WIN && sink) {
    if constexpr (FEW_CUT) {
      tk.seq = count_first(a.batch, [&](int b) { return sink_slot0<true>(a, b) <= slot; }) - 1;
      if (tk.seq < 0) return;
    } else {
      tk = tile_of_slot(a.cu_q, a.batch, a.rows_q, a.sink_chunk, slot);
      if (tk.len == 0) return;
      chunk = tk.row0;
    }
    const int64_t k0 = clamp_cu(a.cu_k, tk.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tk.seq + 1, a.rows_k);
    tk.begin = k0;
    tk.len = (int)(k1 > k0 ? k1 - k0 : 0);
    tk.row0 = sink_tile * kDkvKeys;
    if (tk.row0 >= tk.len) return;
  } else {
    tk = tile_of_slot(a.cu_k, a.batch, a.rows_k, kDkvKeys, slot);
    if (tk.len == 0 || (WIN && !FEW_CUT && tk.row0 < a.sink_tiles * kDkvKeys)) return;
  }
  const int64_t q0 = clamp_cu(a.cu_q, tk.seq, a.rows_q), q1 = clamp_cu(a.cu_q, tk.seq + 1, a.rows_q);
  const int lq = (int)(q1 > q0 ? q1 - q0 : 0), off = tk.len - lq;
  if constexpr (FEW_CUT) {
    const int64_t c = slot - sink_slot0<true>(a, tk.seq);
    if (sink && (lq <= a.sink_chunk || c < 0 || c * a.sink_chunk >= lq)) return;
    if (!sink && tk.row0 < a.sink_tiles * kDkvKeys && lq > a.sink_chunk) return;
    if (sink) chunk = (int)c * a.sink_chunk;
  }
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool is_k = wave & 1;  // this wave forms dK
  const int w_key = tk.row0 + (wave >> 1) * 32, kj = w_key + (lane & 31);
  const bool live = kj < tk.len;
  char* pair = lds + 2 * kBuf + (wave >> 1) * kPair + lane * 16;

  const T* src = static_cast<const T*>(is_k ? a.v : a.k);
  const int64_t src_stride = is_k ? a.v_stride : a.k_stride;
  const T* row = live ? src + (tk.begin + kj) * src_stride + hkv * a.head_dim : nullptr;
  Frag f[HD / 16];
#pragma unroll
  for (int s = 0; s < HD / 16; s++) f[s] = TL::frag_global(row, s, h, a.head_dim);
  settle(f);
  f32x16 acc[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++) acc[d] = f32x16{};

  // the first query that sees the tile's first key, down to a whole query tile
  const int qstart = max(a.causal ? max(tk.row0 - off, 0) / BQ * BQ : 0, chunk);
  // behind the last one that does
  const int qend = WIN && sink ? min(lq, chunk + a.sink_chunk)
                        : WIN && tk.row0 >= a.sinks ? min(lq, tk.row0 + kDkvKeys - 1 - off + a.window) : lq;
  const int per_head = qend > qstart ? (qend - qstart + BQ - 1) / BQ : 0;
  const int64_t steps = (int64_t)per_head * group;
  const int s0 = (int)(steps * split / a.nsplit), s1 = (int)(steps * (split + 1) / a.nsplit);
  Stage<T, HD, BQ, THREADS> qs, os;
  float rowv = 0.0f;  // L (the first BQ threads) or D (as many more) of the next tile's rows
  auto load = [&](int hq, int r) {
    qs.load(static_cast<const T*>(a.q) + (q0 + r) * a.q_stride + hq * a.head_dim, a.q_stride, lq - r, a.head_dim, tid);
    os.load(static_cast<const T*>(a.dout) + (q0 + r) * a.dout_stride + hq * a.head_dim, a.dout_stride, lq - r,
            a.head_dim, tid);
    if (tid < 2 * BQ) {
      const int64_t at = (int64_t)hq * a.rows_q + q0 + min(r + (tid & (BQ - 1)), lq - 1);
      rowv = tid < BQ ? base2_lse(a.lse[at]) : a.delta[at];
    }
  };
  auto store = [&](char* b) {
    qs.store(b, tid);
    os.store(b + kTile, tid);
    if (tid < 2 * BQ) reinterpret_cast<float*>(b + 2 * kTile)[tid] = rowv;
  };
  int hq = hkv * group, r = qstart;  // of the step
  if (s0 < s1) {
    hq += s0 % group;
    r += (per_head - 1 - s0 / group) * BQ;
    load(hq, r);
    store(lds);
  }
  // From the last queries down. Of a tile with sinks first those that see nothing else of the wave's keys: what they
  // gave to keys that are no sinks is 0 times their rows, and a NaN in one must not stay there.
  int behind = s0;
  if (WIN && tk.row0 < a.sinks) {
    const int near = (w_key + 31 + a.window - off - qstart + BQ - 1) / BQ;  // query tiles before those
    behind = min(max((per_head - min(max(near, 0), per_head)) * group, s0), s1);
  }
  int step = s0, buf = 0;
#pragma unroll 1
  for (int part = WIN ? 0 : 1; part < 2; part++) {
    const int stop = part == 0 ? behind : s1;
    for (; step < stop; step++, buf ^= 1) {
      const char* qt = lds + buf * kBuf;
      const char* ot = qt + kTile;
      const float* rows = reinterpret_cast<const float*>(qt + 2 * kTile) + (is_k ? BQ : 0) + 4 * h;
      int next_hq = hq + 1, next_r = r;
      if (next_hq == (hkv + 1) * group) next_hq = hkv * group, next_r -= BQ;
      if (step + 1 < s1) load(next_hq, next_r);
      __syncthreads();
      const bool seen = (!a.causal || r + BQ - 1 + off >= w_key) && window_any<WIN>(a, r + off, w_key, 32);
      const bool whole = r + BQ <= lq && w_key + 32 <= tk.len && (!a.causal || w_key + 31 <= r + off) &&
                         window_all<WIN>(a, r + BQ - 1 + off, w_key, 32);
      // value i of product t: query r + 32 t + 8 (i / 4) + 4 h + i % 4, the lane's key
      auto see = [&](int t, int i) {
        const int qi = r + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
        return qi < lq && live && (!a.causal || kj <= qi + off) && window_any<WIN>(a, qi + off, kj, 1);
      };
      float x[NT][16];
      Frag pf[NT][2];  // bf16: weights and their gradients rounded to nearest for the products
      if (seen) {
        const char* t1 = is_k ? ot : qt;
        f32x16 s[NT] = {};
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int d = 0; d < HD / 16; d++) s[t] = tile_mma(TL::frag(t1, 32 * t + (lane & 31), d, h), f[d], s[t]);
        if constexpr (sizeof(T) == 2) order_products<NT * HD / 16, 1>();
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const f32x4 c = *reinterpret_cast<const f32x4*>(rows + 32 * t + 8 * g);
#pragma unroll
            for (int j = 0; j < 4; j++)
              x[t][4 * g + j] = is_k ? s[t][4 * g + j] - c[j] : fmaf(s[t][4 * g + j], a.scale2, -c[j]);
          }
          if (!is_k) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[t][i] = __builtin_amdgcn_exp2f(x[t][i]);
            if (!whole)
#pragma unroll
              for (int i = 0; i < 16; i++) x[t][i] = see(t, i) ? x[t][i] : 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++) tile_pack(x[t] + 8 * u, pf[t][u]);
            Handover<T>::put(pair + t * kShare, x[t]);
          }
        }
      }
      __syncthreads();
      if (seen) {
        if (is_k) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float p[16];
            Handover<T>::take(pair + t * kShare, p);
#pragma unroll
            for (int i = 0; i < 16; i++) x[t][i] *= p[i];
            if (!whole)  // what is masked has weight 0, and its other factor may be anything
#pragma unroll
              for (int i = 0; i < 16; i++) x[t][i] = see(t, i) ? x[t][i] : 0.0f;
            tile_pack(x[t], pf[t][0]);
            tile_pack(x[t] + 8, pf[t][1]);
          }
        }
        const char* t2 = is_k ? qt : ot;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int d = 0; d < HD / 32; d++)
              acc[d] = tile_mma(TL::frag_t(t2, 32 * t + 16 * u, d, lane), pf[t][u], acc[d]);
        if constexpr (sizeof(T) == 2) order_products<NT * HD / 16, 2>();
      }
      if (step + 1 < s1) store(lds + (buf ^ 1) * kBuf);
      hq = next_hq, r = next_r;
    }
    if (WIN && part == 0 && tk.row0 < a.sinks && kj >= a.sinks)
#pragma unroll
      for (int d = 0; d < HD / 32; d++) acc[d] = f32x16{};
  }
  if (!live) return;
  const float factor = is_k ? a.scale : 1.0f;
  const int64_t at = tk.begin + kj;
  if (WIN && sink) {
    float* part = a.sink_part + ((((slot * a.nsplit + split) * a.sink_tiles + sink_tile) * a.n_kv + hkv) * 2 + is_k) *
                                   (kDkvKeys * a.head_dim);
    store_rows<float, HD>(part + (kj - tk.row0) * a.head_dim, acc, factor, h, a.head_dim);
  } else if (a.nsplit > 1) {
    float* part = a.part + ((int64_t)(2 * split + is_k) * a.rows_k + at) * (a.n_kv * a.head_dim) + hkv * a.head_dim;
    store_rows<float, HD>(part, acc, factor, h, a.head_dim);
  } else {
    store_rows<T, HD>(static_cast<T*>(is_k ? a.dk : a.dv) + at * (is_k ? a.dk_stride : a.dv_stride) + hkv * a.head_dim,
                      acc, factor, h, a.head_dim);
  }
}

// dK and dV from their parts: a thread 4 elements of both.
template <typename T>
__global__ __launch_bounds__(256) void prompt_dkv_sum_kernel(PromptArgs a) {
  const int width = a.n_kv * a.head_dim, per_row = width / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / per_row;
  const int e = (int)(id - row * per_row) * 4;
  if (row < clamp_cu(a.cu_k, 0, a.rows_k) || row >= clamp_cu(a.cu_k, a.batch, a.rows_k)) return;
  const int64_t part = a.rows_k * width, at = row * width + e;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f}, k = v;
  for (int s = 0; s < a.nsplit; s++) {
    v += *reinterpret_cast<const f32x4*>(a.part + 2 * s * part + at);
    k += *reinterpret_cast<const f32x4*>(a.part + (2 * s + 1) * part + at);
  }
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 yv, yk;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    yv[j] = (T)v[j];
    yk[j] = (T)k[j];
  }
  *reinterpret_cast<T4*>(static_cast<T*>(a.dv) + row * a.dv_stride + e) = yv;
  *reinterpret_cast<T4*>(static_cast<T*>(a.dk) + row * a.dk_stride + e) = yk;
}

// dK and dV of the first keys from their chunks: `wgs` workgroups the 64 keys of a sequence and KV head, one where there
// are too many sequences for more (the limit on D's workgroups keeps those within one launch's).
int64_t sink_sum_parts(int64_t batch, int64_t n_kv, int64_t tiles) {
  return batch * n_kv * tiles * 16 <= kMaxGroups ? 16 : 1;
}
template <typename T>
__global__ __launch_bounds__(256) void prompt_sink_sum_kernel(PromptArgs a, int wgs) {
  const int part_of = blockIdx.x % wgs, hkv = blockIdx.x / wgs % a.n_kv;
  const int rest = blockIdx.x / wgs / a.n_kv, tile = rest % a.sink_tiles, b = rest / a.sink_tiles;
  const int64_t q0 = clamp_cu(a.cu_q, b, a.rows_q), q1 = clamp_cu(a.cu_q, b + 1, a.rows_q);
  const int64_t k0 = clamp_cu(a.cu_k, b, a.rows_k), k1 = clamp_cu(a.cu_k, b + 1, a.rows_k);
  const int lq = (int)(q1 > q0 ? q1 - q0 : 0), keys = (int)min(k1 - k0 - tile * kDkvKeys, (int64_t)kDkvKeys);
  if (a.few_cut && lq <= a.sink_chunk) return;
  const int64_t slot = a.few_cut ? sink_slot0<true>(a, b) : sink_slot0<false>(a, b);
  const int parts = (lq + a.sink_chunk - 1) / a.sink_chunk * a.nsplit, hd = a.head_dim;
  const int64_t step = (int64_t)a.sink_tiles * a.n_kv * 2 * kDkvKeys * hd;
  typedef T T4 __attribute__((ext_vector_type(4)));
  for (int i = part_of * 256 + threadIdx.x; i < 2 * keys * (hd / 4); i += wgs * 256) {
    const int is_k = i >= keys * (hd / 4), j = is_k ? i - keys * (hd / 4) : i, row = j / (hd / 4), e = 4 * (j % (hd / 4));
    const float* part =
        a.sink_part + slot * a.nsplit * step + ((tile * a.n_kv + hkv) * 2 + is_k) * (kDkvKeys * hd) + row * hd + e;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < parts; c++) x += *reinterpret_cast<const f32x4*>(part + c * step);
    T4 y;
#pragma unroll
    for (int n = 0; n < 4; n++) y[n] = (T)x[n];
    T* out = static_cast<T*>(is_k ? a.dk : a.dv) + (k0 + tile * kDkvKeys + row) * (is_k ? a.dk_stride : a.dv_stride);
    *reinterpret_cast<T4*>(out + hkv * hd + e) = y;
  }
}

// dQ of a wave's 32 queries += their share of the 32 keys from row `r` of the staged tiles on,
// keys `key` and on of the sequence.
template <typename T, int HD, bool WIN>
__device__ __forceinline__ void dq_tile(const char* kt, const char* vt, int r, int key, bool whole,
                                        const Seen<WIN>& see, float lse, float del, float scale2, int lane,
                                        const typename Tile<T, HD>::Frag (&qf)[HD / 16],
                                        const typename Tile<T, HD>::Frag (&of)[HD / 16], f32x16 (&dq)[HD / 32]) {
  using TL = Tile<T, HD>;
  const int h = lane >> 5;
  f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
  for (int d = 0; d < HD / 16; d++) s = tile_mma(TL::frag(kt, r + (lane & 31), d, h), qf[d], s);
#pragma unroll
  for (int d = 0; d < HD / 16; d++) dp = tile_mma(TL::frag(vt, r + (lane & 31), d, h), of[d], dp);
  if constexpr (sizeof(T) == 2) order_products<HD / 8, 1>();
  float ds[16];
#pragma unroll
  for (int i = 0; i < 16; i++) ds[i] = __builtin_amdgcn_exp2f(fmaf(s[i], scale2, -lse)) * (dp[i] - del);
  if (!whole)
#pragma unroll
    for (int i = 0; i < 16; i++) ds[i] = see.sees(key + 8 * (i >> 2) + 4 * h + (i & 3)) ? ds[i] : 0.0f;
  typename TL::Frag sf[2];
  tile_pack(ds, sf[0]);
  tile_pack(ds + 8, sf[1]);
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int d = 0; d < HD / 32; d++) dq[d] = tile_mma(TL::frag_t(kt, r + 16 * u, d, lane), sf[u], dq[d]);
  if constexpr (sizeof(T) == 2) order_products<HD / 16, 2>();
}

// dQ: four waves of 32 queries each, key tiles of BK rows through LDS.
template <typename T, int HD, int BK, bool WIN>
__device__ __forceinline__ void dq_body(const PromptArgs& a, int block, char* lds) {
  using TL = Tile<T, HD>;
  using Frag = typename TL::Frag;
  constexpr int THREADS = 256, BQ = kDqQueries;
  constexpr int kTile = TL::bytes(BK);
  // f32 heads past 128: no registers are left to hold the next tile of both while this one is used
  constexpr bool kOneStage = sizeof(T) == 4 && HD > 128;
  const int group = a.n_q / a.n_kv;
  const int hkv = block % a.n_kv, rest = block / a.n_kv, hq = hkv * group + rest % group;
  const int64_t slot = a.q_slots - 1 - rest / group;
  const TileSpan tq = tile_of_slot(a.cu_q, a.batch, a.rows_q, BQ, slot);
  if (tq.len == 0) return;
  const int64_t k0 = clamp_cu(a.cu_k, tq.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tq.seq + 1, a.rows_k);
  const int lk = (int)(k1 > k0 ? k1 - k0 : 0), off = lk - tq.len;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w_row = tq.row0 + wave * 32, qi = w_row + (lane & 31);
  const bool live = qi < tq.len;
  const int q_last = min(tq.row0 + BQ, tq.len) - 1;
  Walk<WIN> walk;
  const int nk = (a.causal ? min(max(q_last + off + 1, 0), lk) : lk) - walk.leave_out(a, tq.row0 + off, BK);

  const T* kbase = static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim;
  const T* vbase = static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim;
  Stage<T, HD, BK, THREADS> ks, vs;
  auto load_k = [&](int key) {
    ks.load(kbase + (int64_t)key * a.k_stride, a.k_stride, walk.rows_from(key, lk), a.head_dim, tid);
  };
  auto load_v = [&](int key) {
    vs.load(vbase + (int64_t)key * a.v_stride, a.v_stride, walk.rows_from(key, lk), a.head_dim, tid);
  };
  if (nk > 0) {
    load_k(walk.key(0));
    load_v(walk.key(0));
  }
  const T* qrow = live ? static_cast<const T*>(a.q) + (tq.begin + qi) * a.q_stride + hq * a.head_dim : nullptr;
  const T* orow = live ? static_cast<const T*>(a.dout) + (tq.begin + qi) * a.dout_stride + hq * a.head_dim : nullptr;
  Frag qf[HD / 16], of[HD / 16];
#pragma unroll
  for (int s = 0; s < HD / 16; s++) {
    qf[s] = TL::frag_global(qrow, s, h, a.head_dim);
    of[s] = TL::frag_global(orow, s, h, a.head_dim);
  }
  settle(qf);
  settle(of);
  const int64_t at = (int64_t)hq * a.rows_q + tq.begin + min(qi, tq.len - 1);
  const float lse = base2_lse(a.lse[at]), del = a.delta[at];
  f32x16 dq[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++) dq[d] = f32x16{};
  if (nk > 0) {
    ks.store(lds, tid);
    vs.store(lds + kTile, tid);
  }
  Seen<WIN> see;
  see.init(a, qi, off, lk);
  if (!live) see.last = -1;
  for (int kb = 0, buf = 0; kb < nk; kb += BK, buf ^= 1) {
    const char* kt = lds + buf * 2 * kTile;
    const char* vt = kt + kTile;
    const bool more = kb + BK < nk;
    char* next = lds + (buf ^ 1) * 2 * kTile;
    if (more) {
      load_k(walk.key(kb + BK));
      if constexpr (!kOneStage) load_v(walk.key(kb + BK));
    }
    __syncthreads();
    const int key = walk.key(kb);
    if ((!a.causal || key <= w_row + 31 + off) && window_any<WIN>(a, w_row + off, key, BK)) {
      const bool whole = key + BK <= lk && w_row + 32 <= tq.len && (!a.causal || key + BK - 1 <= w_row + off) &&
                         window_all<WIN>(a, w_row + 31 + off, key, BK);
#pragma unroll
      for (int t = 0; t < BK / 32; t++)
        dq_tile<T, HD, WIN>(kt, vt, 32 * t, key + 32 * t, whole, see, lse, del, a.scale2, lane, qf, of, dq);
    }
    if (more) {
      ks.store(next, tid);
      if constexpr (kOneStage) load_v(walk.key(kb + BK));
      vs.store(next + kTile, tid);
    }
  }
  if (live)
    store_rows<T, HD>(static_cast<T*>(a.dq) + (tq.begin + qi) * a.dq_stride + hq * a.head_dim, dq, a.scale, h,
                      a.head_dim);
}

// dQ of 32 QG queries, 4 / QG waves over the same ones, each with its own 32 of the keys that are
// staged at a time, and their sums added at the end: for grids that would leave CUs idle.
template <typename T, int HD, int QG, bool WIN>
__device__ __forceinline__ void dq_split_body(const PromptArgs& a, int block, char* lds) {
  using TL = Tile<T, HD>;
  using Frag = typename TL::Frag;
  constexpr int THREADS = 256, KG = 4 / QG, BQ = 32 * QG, BK = 32 * KG, kTile = TL::bytes(BK);
  constexpr int kCol = HD + 4;  // floats from query to query of the sums
  const int group = a.n_q / a.n_kv;
  const int hkv = block % a.n_kv, rest = block / a.n_kv, hq = hkv * group + rest % group;
  const TileSpan tq = tile_of_slot(a.cu_q, a.batch, a.rows_q, BQ, a.q_slots - 1 - rest / group);
  if (tq.len == 0) return;
  const int64_t k0 = clamp_cu(a.cu_k, tq.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tq.seq + 1, a.rows_k);
  const int lk = (int)(k1 > k0 ? k1 - k0 : 0), off = lk - tq.len;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave % KG;
  const int w_row = tq.row0 + wave / KG * 32, qi = w_row + (lane & 31);
  const bool live = qi < tq.len;
  const int q_last = min(tq.row0 + BQ, tq.len) - 1;
  Walk<WIN> walk;
  const int nk = (a.causal ? min(max(q_last + off + 1, 0), lk) : lk) - walk.leave_out(a, tq.row0 + off, BK);
  const T* kbase = static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim;
  const T* vbase = static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim;
  Stage<T, HD, BK, THREADS> ks, vs;
  auto load = [&](int key) {
    ks.load(kbase + (int64_t)key * a.k_stride, a.k_stride, walk.rows_from(key, lk), a.head_dim, tid);
    vs.load(vbase + (int64_t)key * a.v_stride, a.v_stride, walk.rows_from(key, lk), a.head_dim, tid);
  };
  if (nk > 0) load(walk.key(0));
  const T* qrow = live ? static_cast<const T*>(a.q) + (tq.begin + qi) * a.q_stride + hq * a.head_dim : nullptr;
  const T* orow = live ? static_cast<const T*>(a.dout) + (tq.begin + qi) * a.dout_stride + hq * a.head_dim : nullptr;
  Frag qf[HD / 16], of[HD / 16];
#pragma unroll
  for (int s = 0; s < HD / 16; s++) {
    qf[s] = TL::frag_global(qrow, s, h, a.head_dim);
    of[s] = TL::frag_global(orow, s, h, a.head_dim);
  }
  settle(qf);
  settle(of);
  const int64_t at = (int64_t)hq * a.rows_q + tq.begin + min(qi, tq.len - 1);
  const float lse = base2_lse(a.lse[at]), del = a.delta[at];
  f32x16 dq[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++) dq[d] = f32x16{};
  Seen<WIN> see;
  see.init(a, qi, off, lk);
  if (!live) see.last = -1;
  for (int kb = 0; kb < nk; kb += BK) {
    ks.store(lds, tid);
    vs.store(lds + kTile, tid);
    if (kb + BK < nk) load(walk.key(kb + BK));
    __syncthreads();
    const int mine = walk.key(kb) + 32 * kg;
    if (kb + 32 * kg < nk && (!a.causal || mine <= w_row + 31 + off) && window_any<WIN>(a, w_row + off, mine, 32)) {
      const bool whole = mine + 32 <= lk && w_row + 32 <= tq.len && (!a.causal || mine + 31 <= w_row + off) &&
                         window_all<WIN>(a, w_row + 31 + off, mine, 32);
      dq_tile<T, HD, WIN>(lds, lds + kTile, 32 * kg, mine, whole, see, lse, del, a.scale2, lane, qf, of, dq);
    }
    __syncthreads();
  }
  float* st = reinterpret_cast<float*>(lds);
  store_rows<float, HD>(st + (wave * 32 + (lane & 31)) * kCol, dq, a.scale, h, HD);
  __syncthreads();
  // 8 / QG threads a query, 4 values each at a time; the query's sums are 32 apart
  constexpr int kSub = 8 / QG;
  const int qn = tid / kSub, row = tq.row0 + qn;
  if (row >= tq.len) return;
  st += ((qn >> 5) * KG * 32 + (qn & 31)) * kCol;
  T* out = static_cast<T*>(a.dq) + (tq.begin + row) * a.dq_stride + hq * a.head_dim;
  for (int e = 4 * (tid % kSub); e < a.head_dim; e += 4 * kSub) {
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < KG; u++) y += *reinterpret_cast<const f32x4*>(st + u * 32 * kCol + e);
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 z;
#pragma unroll
    for (int j = 0; j < 4; j++) z[j] = (T)y[j];
    *reinterpret_cast<T4*>(out + e) = z;
  }
}

// Both in one launch, so that the short workgroups of one fill the compute units that the
// last long ones of the other leave idle.
template <typename T, int HD, int BK, int QG, bool WIN, bool FEW_CUT>
__global__ __launch_bounds__(256, sizeof(T) == 2 && HD <= 128 ? 2 : 1) void prompt_grad_kernel(PromptArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int block = blockIdx.x;
  const int sinks = WIN ? (int)(a.sink_slots * a.sink_tiles * a.n_kv * a.nsplit) : 0;
  const int dkv = sinks + (int)(a.k_slots * a.n_kv * a.nsplit);
  if (block < dkv)
    dkv_body<T, HD, WIN, FEW_CUT>(a, block < sinks ? block : block - sinks, block < sinks, lds);
  else if constexpr (QG == 4)
    dq_body<T, HD, BK, WIN>(a, block - dkv, lds);
  else
    dq_split_body<T, HD, QG, WIN>(a, block - dkv, lds);
}

template <typename T, int HD, int BK, int QG, bool WIN>
hipError_t run_bwd(PromptArgs a, hipStream_t stream) {
  using TL = Tile<T, HD>;
  const bool few = WIN && sizeof(T) == 2 && few_keys(a);
  if (a.rows_q > 0 && !few) {
    const int64_t n = a.rows_q * a.n_q * kDeltaLanes;
    hipLaunchKernelGGL(prompt_delta_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (a.rows_q > 0 && sizeof(T) == 2) {
    constexpr int lds = 4 * Tile<__bf16, HD>::bytes(64);
    const auto kernel = few ? prompt_delta_few_kernel<__bf16, HD> : prompt_delta_exact_kernel<__bf16, HD>;
    static std::atomic<uint64_t> allowed[2];
    if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds, &allowed[few])) return e;
    const int64_t groups = few ? tile_slots(a.rows_q, a.batch, 64) * a.n_q
                               : (int64_t)a.batch * a.n_q * (a.causal ? 1 : kExactTiles);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), lds, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
  }
  constexpr int dq_lds = QG == 4 ? 4 * TL::bytes(BK) : std::max(2 * TL::bytes(128 / QG), 4 * 32 * (HD + 4) * 4);
  constexpr int lds = std::max(dkv_lds<T, HD>(), dq_lds);
  a.k_slots = a.rows_k > 0 ? tile_slots(a.rows_k, a.batch, kDkvKeys) : 0;
  a.q_slots = a.rows_q > 0 ? tile_slots(a.rows_q, a.batch, 32 * QG) : 0;
  const bool few_cut = WIN && a.few_cut;
  const auto kernel = few_cut ? prompt_grad_kernel<T, HD, BK, QG, WIN, WIN> : prompt_grad_kernel<T, HD, BK, QG, WIN, false>;
  static std::atomic<uint64_t> allowed[2];
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds, &allowed[few_cut])) return e;
  const int64_t sinks = a.sink_slots * a.sink_tiles * a.n_kv * a.nsplit;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(sinks + a.k_slots * a.n_kv * a.nsplit + a.q_slots * a.n_q)), dim3(256),
                     lds, stream, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.nsplit > 1 && a.rows_k > 0) {
    const int64_t n = a.rows_k * (a.n_kv * a.head_dim / 4);
    hipLaunchKernelGGL(prompt_dkv_sum_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
  }
  if (WIN && a.sink_tiles > 0) {  // (after the parts' sums, which know nothing of these keys and write what was there)
    const int64_t wgs = sink_sum_parts(a.batch, a.n_kv, a.sink_tiles);
    hipLaunchKernelGGL(prompt_sink_sum_kernel<T>, dim3((unsigned)(a.batch * a.sink_tiles * a.n_kv * wgs)), dim3(256), 0,
                       stream, a, (int)wgs);
    return hipGetLastError();
  }
  return hipSuccess;
}

}  // namespace

// Parts of the (head, query tile) steps of the keys' gradients: enough that the grid is
// 768 workgroups, while a part keeps 4 query tiles of the longest sequence that the rows allow.
// With a window, whose keys all have about as many queries, fewer and longer parts: us of forward and gradient, 768
// and 4 / 512 and 5: 129, 300, 64, 511 (f32, 16/2 x 64, window 100) 72 / 68 | 2048 (f32, 16/2 x 64, 64) 131 / 117 |
// 2048 (f32, 32/8 x 128, 64) 408 / 386 | 2048 (bf16, 32/8 x 128, 256) 151 / 141
PromptBwdPlan plan_prompt_bwd(const PromptArgs& a) {
  const int64_t batch = a.batch, rows_q = a.rows_q, rows_k = a.rows_k, n_q = a.n_q, n_kv = a.n_kv, head_dim = a.head_dim;
  const int64_t groups = std::max<int64_t>(1, (rows_k + kDkvKeys - 1) / kDkvKeys * n_kv);
  const int64_t most = a.window > 0 ? 512 : 768, least_steps = a.window > 0 ? 5 : 4;
  int64_t longest = rows_q / std::max<int64_t>(batch, 1);
  if (a.window > 0) longest = std::min<int64_t>(longest, a.window + kDkvKeys);
  const int64_t steps = longest / 32 * (n_q / n_kv);
  PromptBwdPlan p;
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({most / groups, steps / least_steps, 16}));
  // Chunks of the first keys' queries, of about as many steps as the other keys have and in as many parts, where a
  // sequence can be longer than the window and a chunk; with many sinks their tiles are workgroups enough.
  p.sink_tiles = p.sink_chunk = p.few_cut = 0;
  p.sink_slots = 0;
  const int tiles = (a.sinks + kDkvKeys - 1) / kDkvKeys;
  const int chunk = std::min(std::max((a.window + 63) / 64 * 64, 256), 2048);
  if (a.window > 0 && tiles > 0 && tiles <= 8 && rows_q > a.window + chunk) {
    p.sink_tiles = tiles;
    p.sink_chunk = chunk;
    // Where most sequences are shorter than a chunk, a slot for each would be most of the workspace (64 KV heads x 256, 10000
    // sequences, 500 sinks: 671 GB), so those of one chunk stay whole, which is faster there too. us, a slot a
    // sequence at least / so, bf16, 4 sinks: 500 of 100 (8/4 x 128, window 40) 479 / 433, 100 of 60 and one of 3000 (32/8,
    // 256) 315 / 296; but 16 of 500 (32/8, 256) 280 / 307, 4 of 2047 (32/8, 1024) 571 / 580.
    p.few_cut = batch > rows_q / chunk;
    p.sink_slots = p.few_cut ? rows_q / (chunk / 2) + 1 : tile_slots(rows_q, batch, chunk);
  }
  const int64_t sinks = p.sink_slots * p.sink_tiles * n_kv * p.nsplit;
  p.groups = std::max(sinks + tile_slots(rows_k, batch, kDkvKeys) * n_kv * p.nsplit + tile_slots(rows_q, batch, 64) * n_q,
                      std::max<int64_t>({(rows_q * n_q * kDeltaLanes + 255) / 256, batch * n_q * kExactTiles,
                                         batch * n_kv * p.sink_tiles * sink_sum_parts(batch, n_kv, p.sink_tiles)}));
  p.delta_bytes = ((size_t)(n_q * rows_q) * sizeof(float) + 255) & ~(size_t)255;
  p.part_bytes = p.nsplit > 1 ? (size_t)(2 * p.nsplit * rows_k * n_kv * head_dim) * sizeof(float) : 0;
  p.work = p.delta_bytes + p.part_bytes + (size_t)(sinks * 2 * kDkvKeys * head_dim) * sizeof(float);
  return p;
}

// dQ of 64 queries a workgroup (two waves over the same 32) or of 128. f32 products are long enough
// that the finer grid is all that counts; in bf16 128 queries read keys and values half as often,
// which is the better from about two workgroups a CU on (one and a quarter past 128 elements). us of the whole
// gradient, 128 / 64 queries, causal, 16/16 heads x 128 unless said (workgroups of 128 queries):
//   bf16  512 tokens (80) 47 / 42   2048 (272) 102 / 87   2048 (32/8 heads, 544) 188 / 183   8 x 512 (640) 78 / 79
//         8 x 512 (32/8, 1280) 123 / 127   16/2 x 64: 2048 (272) 75 / 67
//   bf16  x 256: 512 (80) 90 / 78   2048 (272) 276 / 245   64/8 heads, 512 (320) 136 / 132   8 x 256 (384) 86 / 90
//   f32   512 (80) 156 / 111   2048 (272) 760 / 601   2048 (32/8, 544) 1207 / 1186   8 x 512 (32/8, 1280) 738 / 727
//         16/2 x 64: 129, 300, 64, 511 (176) 88 / 65   2048 (272) 480 / 341   8 x 512 (640) 215 / 194
template <bool WIN>
static hipError_t launch_bwd(int dtype, const PromptArgs& a, hipStream_t stream) {
  if (dtype == RQ_BF16) {
    const int64_t most = a.head_dim > 128 ? 320 : 576;
    const bool wide = tile_slots(a.rows_q, a.batch, 128) * a.n_q * 256 > most * a.cu_count;
    if (a.head_dim > 128)
      return wide ? run_bwd<__bf16, 256, 32, 4, WIN>(a, stream) : run_bwd<__bf16, 256, 32, 2, WIN>(a, stream);
    if (a.head_dim <= 64)
      return wide ? run_bwd<__bf16, 64, 64, 4, WIN>(a, stream) : run_bwd<__bf16, 64, 64, 2, WIN>(a, stream);
    return wide ? run_bwd<__bf16, 128, 32, 4, WIN>(a, stream) : run_bwd<__bf16, 128, 32, 2, WIN>(a, stream);
  }
  if (a.head_dim <= 64) return run_bwd<float, 64, 32, 2, WIN>(a, stream);
  if (a.head_dim <= 128) return run_bwd<float, 128, 32, 2, WIN>(a, stream);
  return run_bwd<float, 256, 32, 4, WIN>(a, stream);
}

hipError_t launch_prompt_bwd(int dtype, const PromptArgs& a, hipStream_t stream) {
  return a.window > 0 ? launch_bwd<true>(dtype, a, stream) : launch_bwd<false>(dtype, a, stream);
}

}  // namespace rq
