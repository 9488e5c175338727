// prompt.hip — attention over whole prompts: packed sequences, grouped heads.
//
//   s_ij = scale q_i . k_j, p_ij = exp(s_ij - L_i), L_i = log sum_j exp(s_ij), o_i = sum_j p_ij v_j
//
// over the keys j of i's own sequence, with a causal mask those with
// j <= i + (keys - queries): the last query sees every key (the queries may be the
// end of a longer sequence). One pass over the keys: each query keeps its running
// maximum m and sum l, and what it has summed is scaled by exp(m - m') when the
// maximum rises to m'. Scores are kept in base 2 (scale log2 e folded into one
// factor), so that a weight is one exp2.
//
// One workgroup takes kWaves x 32 queries of one head, a wave 32 of them, the
// query on the lane: the wave forms S^T = K Q^T (rows keys, columns queries), so a
// query's scores lie in two lanes, its maximum needs one exchange, and the weights
// are the B operand of O^T += V^T P^T as they lie. Keys and values pass through LDS
// in tiles of BK rows for all waves, the next tile's loads in flight meanwhile.
//
// Bound by the matrix instructions: 4 head_dim operations for every (query, key) pair that sees the other
// against a few bytes. Measured, causal: bf16, 8192 tokens, 32/8 heads x 128, 502 to 511 us, 1.08 PFLOP/s, 558 us on a
// card warm from other work (a library's 8192^3 product reaches 1.3); 2048, 777, 1500, 331, 1999 and 64 tokens
// 124 us, 0.74; 37 tokens 6.0 us, a launch and one tile's latencies. f32, 613, 1, 1024, 250 and 89 queries, 16/16
// heads x 128, 117 us, 59 TFLOP/s (product 153): the matrix pipe is busy 0.40 of the time, a third of that on the
// masked halves of cut tiles, the rest is one wave a SIMD waiting for its tiles.
//
// With a window (WIN) j > i - window too, or j < sinks. A workgroup walks the sinks' tiles and those from its first
// query's window on, so the work is queries times window, and a tile is masked where an edge runs through it. 16384
// tokens, 32/8 heads x 128, bf16, window 4096 and 4 sinks: 970 to 1030 us by card, 0.94 to 0.99 PFLOP/s of the pairs
// that count; a tile more at each edge than that is computed, one part in 32. The f32 prompts above with windows of
// 256: 77 to 81 us, 44 TFLOP/s: shorter walks, so a larger part of each is cut tiles, the first loads and the join of
// the waves.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "attn_tile.h"
#include "prompt.h"

namespace rq {

namespace {

// The two halves' values of lanes l and l ^ 32, in both.
struct Halves {
  float lo, hi;
};
__device__ __forceinline__ Halves halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// A wave's 32 queries: the lane's column of S^T and O^T, and its softmax state.
constexpr float kSlack = 8.0f;

template <typename T, int HD, int BK>
struct Queries {
  using TL = Tile<T, HD>;
  using Frag = typename TL::Frag;
  Frag q[HD / 16];
  f32x16 acc[HD / 32], s[BK / 32];
  Frag p[BK / 16];
  float m = -INFINITY, l = 0.0f;  // m: in base 2; l: of the lane's half of the keys
  int h, lane;

  __device__ __forceinline__ void init(const T* row, int hd, int lane_) {
    lane = lane_;
    h = lane >> 5;
#pragma unroll
    for (int d = 0; d < HD / 16; d++) q[d] = TL::frag_global(row, d, h, hd);
#pragma unroll
    for (int d = 0; d < HD / 32; d++) acc[d] = f32x16{};
  }

  // S^T of a tile of keys
  __device__ __forceinline__ void scores(const char* kt) {
#pragma unroll
    for (int t = 0; t < BK / 32; t++) s[t] = f32x16{};
#pragma unroll
    for (int d = 0; d < HD / 16; d++)
#pragma unroll
      for (int t = 0; t < BK / 32; t++) s[t] = tile_mma(TL::frag(kt, 32 * t + (lane & 31), d, h), q[d], s[t]);
    if constexpr (sizeof(T) == 2) order_products<HD / 16 * (BK / 32), 1>();
  }

  // The weights of the tile's keys from kb on; those that `v` does not see are masked when `cut`.
  template <bool WIN>
  __device__ __forceinline__ void softmax(int kb, const Seen<WIN>& v, bool cut, float scale2) {
    if (cut)
#pragma unroll
      for (int t = 0; t < BK / 32; t++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (!v.sees(kb + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3))) s[t][i] = -INFINITY;
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < BK / 32; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[t][i]);
    const Halves both = halves(mx);
    mx = fmaxf(both.lo, both.hi) * scale2;
    // The reference m moves only when some query's maximum is past it by kSlack: below that
    // the weights are at most 2^kSlack, which costs no digits, and nothing is rescaled.
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack || m == -INFINITY)) {
      const float mn = fmaxf(m, mx), alpha = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < HD / 32; d++) acc[d] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.0f : m;  // nothing seen yet: every weight 0
#pragma unroll
    for (int t = 0; t < BK / 32; t++) {
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        w[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], scale2, -ref));
        l += w[i];
      }
      // bf16: rounded to nearest; their sum l is of the unrounded ones
      tile_pack(w, p[2 * t]);
      tile_pack(w + 8, p[2 * t + 1]);
    }
  }

  __device__ __forceinline__ void add_values(const char* vt) {
#pragma unroll
    for (int u = 0; u < BK / 16; u++)
#pragma unroll
      for (int d = 0; d < HD / 32; d++) acc[d] = tile_mma(TL::frag_t(vt, 16 * u, d, lane), p[u], acc[d]);
    if constexpr (sizeof(T) == 2) order_products<HD / 32 * (BK / 16), 2>();
  }

  // add_values(vt), then scores(kt), the reads of the second under way in the first
  __device__ __forceinline__ void add_values_and_scores(const char* vt, const char* kt) {
#pragma unroll
    for (int u = 0; u < BK / 16; u++)
#pragma unroll
      for (int d = 0; d < HD / 32; d++) acc[d] = tile_mma(TL::frag_t(vt, 16 * u, d, lane), p[u], acc[d]);
#pragma unroll
    for (int t = 0; t < BK / 32; t++) s[t] = f32x16{};
#pragma unroll
    for (int d = 0; d < HD / 16; d++)
#pragma unroll
      for (int t = 0; t < BK / 32; t++) s[t] = tile_mma(TL::frag(kt, 32 * t + (lane & 31), d, h), q[d], s[t]);
    order_products<HD / 32 * (BK / 16), 2, HD / 16 * (BK / 32), 1>();
  }

  __device__ __forceinline__ void finish(const PromptArgs& a, int hq, int64_t row, bool live) {
    const Halves both = halves(l);
    l = both.lo + both.hi;
    if (!live) return;
    if (a.lse && h == 0)
      a.lse[(int64_t)hq * a.rows_q + row] = l == 0.0f ? -INFINITY : m * 0.6931471805599453f + __logf(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a query that sees nothing: zeros
    T* out = static_cast<T*>(a.out) + row * a.out_stride + hq * a.head_dim;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int e = 32 * d + 2 * i + 4 * h;
        if (e >= a.head_dim) continue;
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (T)(acc[d][i + j] * inv);
        *reinterpret_cast<T4*>(out + e) = y;
      }
  }
};

// What a workgroup and a wave of it work on. BK: keys of its steps. nk: keys that it walks over, which are the
// sequence's first ones or, with a window, w.key() of them.
template <typename T, int BQ, int BK, bool WIN>
struct Work : Walk<WIN> {
  TileSpan tq;
  int hq, lk, off, nk, q_first, qi;
  Seen<WIN> see;
  bool live;
  const T *k, *v, *q;
  // false: nothing to do
  __device__ __forceinline__ bool init(const PromptArgs& a, int wave, int lane) {  // wave: of 32 queries each
    const int group = a.n_q / a.n_kv;
    // ids next to each other go to different XCDs: a KV head's tiles stay on as few as can be
    const int hkv = blockIdx.x % a.n_kv, rest = blockIdx.x / a.n_kv;
    hq = hkv * group + rest % group;
    // a long sequence's last tiles, which see most keys, first
    tq = tile_of_slot(a.cu_q, a.batch, a.rows_q, BQ, a.slots - 1 - rest / group);
    if (tq.len == 0) return false;
    const int64_t k0 = clamp_cu(a.cu_k, tq.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tq.seq + 1, a.rows_k);
    lk = (int)(k1 > k0 ? k1 - k0 : 0);
    off = lk - tq.len;
    q_first = tq.row0 + wave * 32;
    qi = q_first + (lane & 31);  // the lane's query
    live = qi < tq.len;
    see.init(a, qi, off, lk);
    const int q_last = min(tq.row0 + BQ, tq.len) - 1;
    nk = a.causal ? min(max(q_last + off + 1, 0), lk) : lk;  // keys that the tile sees
    nk -= this->leave_out(a, tq.row0 + off, BK);
    k = static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim;
    v = static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim;
    q = live ? static_cast<const T*>(a.q) + (tq.begin + qi) * a.q_stride + hq * a.head_dim : nullptr;
    return true;
  }
  // whether the wave sees any of the bk keys from kb on, and whether it sees less than all of them
  __device__ __forceinline__ bool any(const PromptArgs& a, int kb, int bk) const {
    return q_first < tq.len && (!a.causal || kb <= q_first + 31 + off) && window_any<WIN>(a, q_first + off, kb, bk);
  }
  __device__ __forceinline__ bool cut(const PromptArgs& a, int kb, int bk) const {
    return kb + bk > lk || (a.causal && kb + bk - 1 > q_first + off) || !window_all<WIN>(a, q_first + 31 + off, kb, bk);
  }
};

template <typename T, int HD, int BK, bool WIN>
__global__ __launch_bounds__(256) void prompt_fwd_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  constexpr int THREADS = 256, kTile = TL::bytes(BK);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Work<T, 128, BK, WIN> w;
  if (!w.init(a, wave, lane)) return;
  Stage<T, HD, BK, THREADS> ks, vs;
  auto load = [&](int key) {
    ks.load(w.k + (int64_t)key * a.k_stride, a.k_stride, w.rows_from(key, w.lk), a.head_dim, tid);
    vs.load(w.v + (int64_t)key * a.v_stride, a.v_stride, w.rows_from(key, w.lk), a.head_dim, tid);
  };
  if (w.nk > 0) load(w.key(0));
  Queries<T, HD, BK> x;
  x.init(w.q, a.head_dim, lane);
  settle(x.q);
  if (w.nk > 0) {
    ks.store(lds, tid);
    vs.store(lds + kTile, tid);
  }
  for (int kb = 0, buf = 0; kb < w.nk; kb += BK, buf ^= 1) {
    const char* kt = lds + buf * 2 * kTile;
    const bool more = kb + BK < w.nk;
    if (more) load(w.key(kb + BK));
    __syncthreads();
    const int key = w.key(kb);
    if (w.any(a, key, BK)) {
      // products first, the other wave's softmax in their gaps: 131 us of the six sequences above, else 140
      __builtin_amdgcn_s_setprio(1);
      x.scores(kt);
      __builtin_amdgcn_s_setprio(0);
      x.softmax(key, w.see, w.cut(a, key, BK), a.scale2);
      __builtin_amdgcn_s_setprio(1);
      x.add_values(kt + kTile);
      __builtin_amdgcn_s_setprio(0);
    }
    if (more) {
      char* next = lds + (buf ^ 1) * 2 * kTile;
      ks.store(next, tid);
      vs.store(next + kTile, tid);
    }
  }
  x.finish(a, w.hq, w.tq.begin + w.qi, w.live);
}

// Eight waves, two a SIMD, in two groups half a step apart: while one group's waves
// are in their products (the values of the last tile, the scores of the next), the other's
// are in their softmax, so that the matrix pipe and the vector pipe of a SIMD are
// both in use. Without the barriers between the halves the two waves of a SIMD fall
// into step and take turns at both.
//
// Time slots end at a barrier. Group g has its products of tile i in slot 2 i + g, in whose
// shadow it also stores its share of tile i + 1 and asks for that of tile i + 2, and its softmax
// in the next slot. Tile t is complete before slot 2 t; its keys are read in slots 2 t and
// 2 t + 1, its values two later: rings of 2 and 3 tiles.
template <typename T, int HD, int BK, bool WIN>
__global__ __launch_bounds__(512, 2) void prompt_fwd_pair_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  constexpr int THREADS = 512, kTile = TL::bytes(BK);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = wave >> 2;
  Work<T, 256, BK, WIN> w;
  if (!w.init(a, wave, lane)) return;
  const int n = (w.nk + BK - 1) / BK;
  Stage<T, HD, BK, THREADS> ks, vs;
  auto load = [&](int t) {
    const int key = w.key(t * BK);
    ks.load(w.k + (int64_t)key * a.k_stride, a.k_stride, w.rows_from(key, w.lk), a.head_dim, tid);
    vs.load(w.v + (int64_t)key * a.v_stride, a.v_stride, w.rows_from(key, w.lk), a.head_dim, tid);
  };
  auto k_tile = [&](int t) { return lds + (t & 1) * kTile; };
  auto v_tile = [&](int t) { return lds + (2 + t % 3) * kTile; };
  auto store = [&](int t) {
    ks.store(k_tile(t), tid);
    vs.store(v_tile(t), tid);
  };
  auto slot_end = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };
  if (n > 0) load(0);
  Queries<T, HD, BK> x;
  x.init(w.q, a.head_dim, lane);
  settle(x.q);
  if (n > 0) store(0);
  if (n > 1) load(1);
  slot_end();
  if (g == 1) slot_end();
  if (n > 1) store(1);
  if (n > 2) load(2);
  if (n > 0) x.scores(k_tile(0));
  slot_end();
  char *kn = lds + kTile, *vc = lds + 2 * kTile;  // keys of the next tile, values of this one
#pragma unroll 1
  for (int i = 0; i < n; i++) {
    // A tile that none of the wave's queries see is left out: a NaN in its values must not reach them, and
    // the wave's matrix pipe is the other group's (4200 tokens, 32/8 heads 165 -> 160 us, 8192 517 -> 511).
    const int key = w.key(i * BK);
    const bool any = w.any(a, key, BK);
    if (any) {
      x.softmax(key, w.see, w.cut(a, key, BK), a.scale2);
      settle(x.p);  // (else the exponentials sink past the barrier, to the products)
    }
    slot_end();
    __builtin_amdgcn_s_setprio(1);
    if (i + 2 < n) store(i + 2);
    if (i + 3 < n) load(i + 3);
    if (any)
      x.add_values_and_scores(vc, kn);  // (after the last tile the scores are of an old one, not used)
    else if (WIN && i + 1 < n && w.any(a, w.key((i + 1) * BK), BK))  // a window begins with the next tile
      x.scores(kn);
    __builtin_amdgcn_s_setprio(0);
    slot_end();
    kn = kn == lds ? lds + kTile : lds;
    vc = vc == lds + 4 * kTile ? lds + 2 * kTile : vc + kTile;
  }
  if (g == 0) slot_end();
  x.finish(a, w.hq, w.tq.begin + w.qi, w.live);
}

// Fewer queries a workgroup, for grids that would leave CUs idle with 128: QG groups of 32,
// and 4 / QG waves over the same queries, each with its own 32 of the keys that are staged at
// a time, their states joined at the end. One tile in LDS, the next on its way in registers.
template <typename T, int HD, int QG, bool WIN>
__global__ __launch_bounds__(256) void prompt_fwd_split_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  constexpr int THREADS = 256, KG = 4 / QG, BK = 32 * KG, kTile = TL::bytes(BK);
  constexpr int kCol = HD + 4;  // floats from query to query of a joined state
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave % KG;
  Work<T, 32 * QG, BK, WIN> w;
  if (!w.init(a, wave / KG, lane)) return;
  Stage<T, HD, BK, THREADS> ks, vs;
  auto load = [&](int key) {
    ks.load(w.k + (int64_t)key * a.k_stride, a.k_stride, w.rows_from(key, w.lk), a.head_dim, tid);
    vs.load(w.v + (int64_t)key * a.v_stride, a.v_stride, w.rows_from(key, w.lk), a.head_dim, tid);
  };
  if (w.nk > 0) load(w.key(0));
  Queries<T, HD, 32> x;
  x.init(w.q, a.head_dim, lane);
  settle(x.q);
  for (int kb = 0; kb < w.nk; kb += BK) {
    ks.store(lds, tid);
    vs.store(lds + kTile, tid);
    if (kb + BK < w.nk) load(w.key(kb + BK));
    __syncthreads();
    const int mine = w.key(kb) + 32 * kg;
    if (kb + 32 * kg < w.nk && w.any(a, mine, 32)) {
      const char* kt = lds + 32 * kg * TL::kPitch;
      x.scores(kt);
      x.softmax(mine, w.see, w.cut(a, mine, 32), a.scale2);
      x.add_values(kt + kTile);
    }
    __syncthreads();
  }
  // state of wave u: [query][HD weighted values, maximum, sum of the half's keys x 2]
  float* st = reinterpret_cast<float*>(lds);
  float* own = st + (wave * 32 + (lane & 31)) * kCol;
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<f32x4*>(own + 32 * d + 2 * i + 4 * h) =
          f32x4{x.acc[d][i], x.acc[d][i + 1], x.acc[d][i + 2], x.acc[d][i + 3]};
  if (h == 0) own[HD] = x.m;
  own[HD + 1 + h] = x.l;
  __syncthreads();
  // 8 / QG threads a query, 4 values each at a time; the query's states are 32 apart
  constexpr int kSub = 8 / QG;
  const int qn = tid / kSub, sub = tid % kSub, qi = w.tq.row0 + qn;
  if (qi >= w.tq.len) return;
  st += ((qn >> 5) * KG * 32 + (qn & 31)) * kCol;
  float m = -INFINITY, l = 0.0f, f[KG];
#pragma unroll
  for (int u = 0; u < KG; u++) m = fmaxf(m, st[u * 32 * kCol + HD]);
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int u = 0; u < KG; u++) {
    const float* s = st + u * 32 * kCol + HD;
    f[u] = __builtin_amdgcn_exp2f(s[0] - ref);
    l += f[u] * (s[1] + s[2]);
  }
  const int64_t row = w.tq.begin + qi;
  if (a.lse && sub == 0)
    a.lse[(int64_t)w.hq * a.rows_q + row] = l == 0.0f ? -INFINITY : m * 0.6931471805599453f + __logf(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a query that sees nothing: zeros
  T* out = static_cast<T*>(a.out) + row * a.out_stride + w.hq * a.head_dim;
  for (int e = 4 * sub; e < a.head_dim; e += 4 * kSub) {
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < KG; u++) y += f[u] * *reinterpret_cast<const f32x4*>(st + u * 32 * kCol + e);
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 z;
#pragma unroll
    for (int j = 0; j < 4; j++) z[j] = (T)(y[j] * inv);
    *reinterpret_cast<T4*>(out + e) = z;
  }
}

template <typename T, int HD, int BK, bool WIN>
hipError_t run_fwd(PromptArgs a, hipStream_t stream) {
  constexpr int lds = 4 * Tile<T, HD>::bytes(BK);
  a.slots = tile_slots(a.rows_q, a.batch, 128);
  const auto kernel = prompt_fwd_kernel<T, HD, BK, WIN>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.slots * a.n_q)), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <typename T, int HD, int BK, bool WIN>
hipError_t run_fwd_pair(PromptArgs a, hipStream_t stream) {
  constexpr int lds = 5 * Tile<T, HD>::bytes(BK);
  a.slots = tile_slots(a.rows_q, a.batch, 256);
  const auto kernel = prompt_fwd_pair_kernel<T, HD, BK, WIN>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.slots * a.n_q)), dim3(512), lds, stream, a);
  return hipGetLastError();
}

template <typename T, int HD, int QG, bool WIN>
hipError_t run_fwd_split(PromptArgs a, hipStream_t stream) {
  constexpr int lds = std::max(2 * Tile<T, HD>::bytes(128 / QG), 4 * 32 * (HD + 4) * 4);
  a.slots = tile_slots(a.rows_q, a.batch, 32 * QG);
  const auto kernel = prompt_fwd_split_kernel<T, HD, QG, WIN>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.slots * a.n_q)), dim3(256), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

// The split kernel's groups of 32 queries a workgroup, or 0 for the kernel of 128 queries: that reads
// keys and values least often, the others fill the CUs with fewer queries. By the 128-query
// kernel's workgroups for every 256 CUs; us, 128 / 64 / 32 queries, causal, 16/16 heads x 128 unless said:
//   bf16  256 tokens (32/8 heads, 96) 11.7 / 11.0 / 10.1   512 (32/8, 160) 17.4 / 15.4 / 19.8   613, 1, 1024,
//         250, 89 (320) 28.9 / 25.2 / 46.5   8 x 256 (384) 14.5 / 13.9 / 29.7   2048 (32/8, 544) 55 / 64 / 138
//         4 x 64 after 4032 (32/8, 192) 80 / 71 / 60
//   bf16  16/2 x 64: 1024 (144) 22.7 / 17.5 / 13.7   2048 (272) 41 / 29 / 29   4096 (528) 78 / 60 / 74
//         8 x 512 (640) 16.6 / 17.5 / 24.6
//   bf16  x 256, 128 / 64 queries: 512 (80) 34.8 / 26.5   2048 (272) 115 / 91   64/8 heads, 512 (320) 37.6 / 37.7
//         8 x 256 (384) 25.9 / 34.4   4 x 64 after 4032 (64/8, 384) 201 / 147
//   f32   (x 256: 64 queries do not fit the registers)   37 tokens (16) 15.0 / 12.4 / 14.7   512 (80) 81 / 49 / 38   512 (32/8, 160) 82 / 50 / 51   613, 1, 1024,
//         250, 89 (320) 156 / 111 / 138   8 x 256 (384) 48 / 56 / 75   2048 (32/8, 544) 327 / 363 / 532
//   f32   16/2 x 64: 1024 (144) 86 / 48 / 37   2048 (272) 164 / 113 / 101   8 x 256 (384) 31 / 24 / 31
//         8 x 512 (640) 80 / 69 / 77
// f32 with few queries after many keys: every workgroup walks about all keys, so a tile's time is its rounds of
// workgroups (two a CU to 64 elements, one past them) times that of a round, by the tiles of a sequence of
// average length. us, 128 / 64 / 32 queries:
//   x 128   4 x 64 after 4032 (32/8 heads) 569 / 334 / 242   (64/8) 570 / 334 / 479   8 x 16 after 984 (32/8) 146 / 88 / 70
//           8 x 64 after 1984 (32/8) 289 / 173 / 247   8 x 128 after 896 (16/16) 153 / 91 / 132   2 x 300 after 2700
//           (32/8) 429 / 466 / 512
//   x 64    4 x 64 after 4032 (64/8) 523 / 290 / 164   8 x 64 after 1984 (64/8) 267 / 151 / 166   16 x 64 after 960 (64/8)
//           269 / 155 / 176   16 x 20 after 1004 (64/8) 158 / 150 / 89   2 x 300 after 2700 (32/8) 231 / 208 / 177
static int f32_few_queries_groups(const PromptArgs& a, bool narrow) {
  const int64_t len = (a.rows_q + a.batch - 1) / a.batch, places = (int64_t)a.cu_count * (narrow ? 2 : 1);
  const int64_t round[2][3] = {{242, 334, 569}, {41, 75, 134}};  // of 32, 64 and 128 queries
  int64_t best = 0;
  int tile = 0;
  for (int i = 0; i < 3; i++) {
    const int64_t groups = a.batch * ((len + (32 << i) - 1) / (32 << i)) * a.n_q;
    const int64_t time = (groups + places - 1) / places * round[narrow][i];
    if (i == 0 || time < best) best = time, tile = i;
  }
  return tile == 2 ? 0 : tile + 1;
}

static int fwd_split_groups(int dtype, const PromptArgs& a) {
  const bool f32 = dtype == RQ_F32, narrow = a.head_dim <= 64, broad = a.head_dim > 128;
  if (f32 && broad) return 0;
  if (a.rows_k < 64 * (int64_t)a.batch) return f32 ? 2 : 0;  // hardly a tile of keys to split
  const bool few_queries = a.rows_k >= 4 * a.rows_q;  // every tile sees most keys
  if (f32 && few_queries) return f32_few_queries_groups(a, narrow);
  int one = broad ? 0 : narrow ? (f32 ? 320 : 256) : few_queries ? 256 : f32 ? 152 : 128;
  int two = broad && !few_queries ? 320 : narrow ? (f32 ? 640 : 576) : f32 ? 352 : 448;
  // With a window a workgroup walks it and its own queries' keys: fewer queries a workgroup cost more of them, the
  // sooner the shorter the window. us, windows of 32 / 128 / 400, 128, 64 and 32 queries:
  //   f32   x 128: 512 (80) 38, 26, 32 / 53, 31, 33 / 85, 51, 39   1024 (144) 39, 27, 53 / 54, 33, 61 / 95, 58, 81
  //         1024 (32/8, 288) 41, 50, 99 / 56, 61, 110 / 97, 107, 144
  //         2048 (272), 64 / 256 / 1024: 47, 53, 103 / 75, 84, 147 / 185, 194, 240
  //         16/2 x 64: 1024 (144) 25, 17, 22 / 34, 20, 23 / 56, 33, 33   4096 (528) 39, 42, 69 / 51, 52, 78 / 89, 95, 121
  //   bf16  x 128: 512 (80) 17, 12, 14 / 20, 14, 14 / 22, 18, 15   1024 (144) 17, 13, 23 / 20, 14, 25 / 28, 20, 29
  //         16/2 x 64: 1024 (144) 15, 11, 12 / 18, 11, 12 / 24, 16, 15
  if (a.window > 0 && !few_queries) {
    if (f32)
      one = 96, two = narrow ? 400 : 256;
    else if (a.window <= 256)
      one = 0;
  }
  const int64_t groups = tile_slots(a.rows_q, a.batch, 128) * a.n_q * 256;
  return groups <= (int64_t)one * a.cu_count ? 1 : groups <= (int64_t)two * a.cu_count ? 2 : 0;
}

template <int QG, bool WIN>
static hipError_t launch_fwd_split(int dtype, const PromptArgs& a, hipStream_t stream) {
  if constexpr (QG == 2)
    if (a.head_dim > 128) return run_fwd_split<__bf16, 256, QG, WIN>(a, stream);
  if (dtype == RQ_BF16)
    return a.head_dim <= 64 ? run_fwd_split<__bf16, 64, QG, WIN>(a, stream) : run_fwd_split<__bf16, 128, QG, WIN>(a, stream);
  return a.head_dim <= 64 ? run_fwd_split<float, 64, QG, WIN>(a, stream) : run_fwd_split<float, 128, QG, WIN>(a, stream);
}

int prompt_fwd_tile(int dtype, const PromptArgs& a) {
  if (const int qg = fwd_split_groups(dtype, a)) return 32 * qg;
  // The pair kernel reads keys and values half as often but cuts the queries in tiles of 256.
  // us, this / the other, bf16, causal: 32/8 heads x 128: 8 x 512 tokens 52 / 43, 4 x 1024 68 / 58, 4 x 3000
  // 314 / 312, 4 x 4096 548 / 548, 4096 139 / 142, 8192 502 / 520, 16384 1919 / 2021; 16/16 heads: 4096
  // 106 / 103, 4 x 4096 279 / 281, 8192 256 / 267.
  // With a window the wider tile has more at both of its edges: 16384 tokens, 32/8 heads, windows of 256, 1024 and
  // 4096 301 / 196, 457 / 367, 1010 / 970; 32768, 16/4 heads, 8192 1816 / 1847, 16384 2957 / 3065.
  const bool pair = dtype == RQ_BF16 && a.head_dim > 64 && a.head_dim <= 128 && a.rows_q / a.batch > 4096 &&
                    (a.window == 0 || a.window >= 8192);
  return pair ? 256 : 128;
}

template <bool WIN>
static hipError_t launch_fwd(int dtype, const PromptArgs& a, hipStream_t stream) {
  const int tile = prompt_fwd_tile(dtype, a);
  if (tile == 32) return launch_fwd_split<1, WIN>(dtype, a, stream);
  if (tile == 64) return launch_fwd_split<2, WIN>(dtype, a, stream);
  if (tile == 256) return run_fwd_pair<__bf16, 128, 64, WIN>(a, stream);
  if (dtype == RQ_BF16) {
    if (a.head_dim <= 64) return run_fwd<__bf16, 64, 64, WIN>(a, stream);
    if (a.head_dim <= 128) return run_fwd<__bf16, 128, 64, WIN>(a, stream);
    return run_fwd<__bf16, 256, 32, WIN>(a, stream);
  }
  if (a.head_dim <= 64) return run_fwd<float, 64, 32, WIN>(a, stream);
  if (a.head_dim <= 128) return run_fwd<float, 128, 32, WIN>(a, stream);
  return run_fwd<float, 256, 32, WIN>(a, stream);
}

hipError_t launch_prompt_fwd(int dtype, const PromptArgs& a, hipStream_t stream) {
  return a.window > 0 ? launch_fwd<true>(dtype, a, stream) : launch_fwd<false>(dtype, a, stream);
}

}  // namespace rq
