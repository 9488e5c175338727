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
#include <algorithm>
#include <cmath>

#include "attn_tile.h"
#include "prompt.h"

namespace rq {

namespace {

// v of lane ^ 32
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

constexpr float kSlack = 8.0f;

template <typename T, int HD, int NW, int BK>
__global__ __launch_bounds__(NW * 64) void prompt_fwd_kernel(PromptArgs a) {
  using TL = Tile<T, HD>;
  using Frag = typename TL::Frag;
  constexpr int THREADS = NW * 64, BQ = NW * 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kTile = TL::bytes(BK);
  const int group = a.n_q / a.n_kv;
  // ids next to each other go to different XCDs: a KV head's tiles stay on as few as can be
  const int hkv = blockIdx.x % a.n_kv, rest = blockIdx.x / a.n_kv, hq = hkv * group + rest % group;
  const int64_t slot = a.slots - 1 - rest / group;  // a long sequence's last tiles, which see most keys, first
  const TileSpan tq = tile_of_slot(a.cu_q, a.batch, a.rows_q, BQ, slot);
  if (tq.len == 0) return;
  const int64_t k0 = clamp_cu(a.cu_k, tq.seq, a.rows_k), k1 = clamp_cu(a.cu_k, tq.seq + 1, a.rows_k);
  const int lk = (int)(k1 > k0 ? k1 - k0 : 0), off = lk - tq.len;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = tq.row0 + wave * 32 + (lane & 31);  // the lane's query
  const bool live = qi < tq.len;
  const int q_last = min(tq.row0 + BQ, tq.len) - 1;
  const int nk = a.causal ? min(max(q_last + off + 1, 0), lk) : lk;  // keys that the tile sees

  const T* kbase = static_cast<const T*>(a.k) + k0 * a.k_stride + hkv * a.head_dim;
  const T* vbase = static_cast<const T*>(a.v) + k0 * a.v_stride + hkv * a.head_dim;
  Stage<T, HD, BK, THREADS> ks, vs;
  if (nk > 0) {
    ks.load(kbase, a.k_stride, lk, a.head_dim, tid);
    vs.load(vbase, a.v_stride, lk, a.head_dim, tid);
  }
  const T* qrow = live ? static_cast<const T*>(a.q) + (tq.begin + qi) * a.q_stride + hq * a.head_dim : nullptr;
  Frag qf[HD / 16];
#pragma unroll
  for (int s = 0; s < HD / 16; s++) qf[s] = TL::frag_global(qrow, s, h, a.head_dim);

  f32x16 acc[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; d++) acc[d] = f32x16{};
  float m = -INFINITY, l = 0.0f;  // m: base-2 units; l: of the lane's half of the keys
  if (nk > 0) {
    ks.store(lds, tid);
    vs.store(lds + kTile, tid);
  }
  for (int kb = 0, buf = 0; kb < nk; kb += BK, buf ^= 1) {
    const char* kt = lds + buf * 2 * kTile;
    const char* vt = kt + kTile;
    const bool more = kb + BK < nk;
    if (more) {
      ks.load(kbase + (int64_t)(kb + BK) * a.k_stride, a.k_stride, lk - kb - BK, a.head_dim, tid);
      vs.load(vbase + (int64_t)(kb + BK) * a.v_stride, a.v_stride, lk - kb - BK, a.head_dim, tid);
    }
    __syncthreads();
    const int w_first = tq.row0 + wave * 32 + off;  // the last key that the wave's first query sees (causal)
    if (!a.causal || kb <= w_first + 31) {
      f32x16 s[BK / 32];
#pragma unroll
      for (int t = 0; t < BK / 32; t++) {
        s[t] = f32x16{};
#pragma unroll
        for (int d = 0; d < HD / 16; d++) s[t] = tile_mma(TL::frag(kt, 32 * t + (lane & 31), d, h), qf[d], s[t]);
      }
      if (kb + BK > lk || (a.causal && kb + BK - 1 > w_first)) {
        const int see = a.causal ? min(lk - 1, qi + off) : lk - 1;  // the last key that this query sees
#pragma unroll
        for (int t = 0; t < BK / 32; t++)
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (kb + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > see) s[t][i] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < BK / 32; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[t][i]);
      mx = fmaxf(mx, other_half(mx)) * a.scale2;
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
        float p[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], a.scale2, -ref));
          l += p[i];
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
          Frag pf;  // bf16: the weights, at most 1, rounded to nearest; their sum l is of the unrounded ones
          tile_pack(p + 8 * u, pf);
#pragma unroll
          for (int d = 0; d < HD / 32; d++) acc[d] = tile_mma(TL::frag_t(vt, 32 * t + 16 * u, d, lane), pf, acc[d]);
        }
      }
    }
    if (more) {
      char* next = lds + (buf ^ 1) * 2 * kTile;
      ks.store(next, tid);
      vs.store(next + kTile, tid);
    }
  }
  l += other_half(l);
  if (!live) return;
  if (a.lse && h == 0)
    a.lse[(int64_t)hq * a.rows_q + tq.begin + qi] =
        l == 0.0f ? -INFINITY : m * 0.6931471805599453f + __logf(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a query that sees nothing: zeros
  T* orow = static_cast<T*>(a.out) + (tq.begin + qi) * a.out_stride + hq * a.head_dim;
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
      *reinterpret_cast<T4*>(orow + e) = y;
    }
}

template <typename T, int HD, int NW, int BK>
hipError_t run_fwd(PromptArgs a, hipStream_t stream) {
  constexpr int lds = 4 * Tile<T, HD>::bytes(BK);
  a.slots = tile_slots(a.rows_q, a.batch, NW * 32);
  const auto kernel = prompt_fwd_kernel<T, HD, NW, BK>;
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.slots * a.n_q)), dim3(NW * 64), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t allow_lds(const void* kernel, int bytes) {
  if (bytes <= 65536) return hipSuccess;
  return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

hipError_t launch_prompt_fwd(int dtype, const PromptArgs& a, hipStream_t stream) {
  if (dtype == RQ_BF16) {
    if (a.head_dim <= 64) return run_fwd<__bf16, 64, 4, 64>(a, stream);
    if (a.head_dim <= 128) return run_fwd<__bf16, 128, 4, 64>(a, stream);
    return run_fwd<__bf16, 256, 4, 32>(a, stream);
  }
  if (a.head_dim <= 64) return run_fwd<float, 64, 4, 32>(a, stream);
  if (a.head_dim <= 128) return run_fwd<float, 128, 4, 32>(a, stream);
  return run_fwd<float, 256, 4, 32>(a, stream);
}

}  // namespace rq
