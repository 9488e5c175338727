// paged.hip — a key-value cache in pages: one new token of every sequence (RoPE,
// append, attention), a packed prompt's RoPE and append, pages copied.
//
// The batched form of attention.hip's decode step. A sequence's rows lie in pages
// of 2^b rows, found through its row of the page table. Pages hold at least 16 rows, so 16
// rows that start at a multiple of 16 lie in one page: a page number is looked up once
// for them, by the whole wave.
#include <algorithm>
#include <cmath>

#include "attn_tile.h"
#include "paged.h"

namespace rq {

namespace {

// cos and sin of pos * theta^(-2 i / head_dim). The angle is formed in double in turns
// and its whole turns taken off there, so far positions keep their digits.
__device__ __forceinline__ void rope_angle(int64_t pos, int i, int head_dim, double log2_theta, float* c, float* s) {
  double t = (double)pos * exp2(-2.0 * (double)i / (double)head_dim * log2_theta) * 0.15915494309189535;
  t -= rint(t);
  double sd, cd;
  sincospi(2.0 * t, &sd, &cd);
  *c = (float)cd;
  *s = (float)sd;
}

constexpr int kPagedThreads = 256, kPagedWaves = 4, kRec = 4;

__device__ __forceinline__ uint32_t low16_pair(uint32_t a, uint32_t b) {  // a.lo | b.lo << 16
  return __builtin_amdgcn_perm(b, a, 0x05040100);
}
__device__ __forceinline__ uint32_t high16_pair(uint32_t a, uint32_t b) {  // a.hi | b.hi << 16
  return __builtin_amdgcn_perm(b, a, 0x07060302);
}

// The bf16 terms of x: x = t0 + t1 + t2 within 2^-24 |x|
template <int NT>
__device__ __forceinline__ void split_terms(float x, __bf16 (&t)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; n++) {
    t[n] = (__bf16)x;
    x -= (float)t[n];
  }
}

}  // namespace

// One workgroup: up to 16 query heads of a KV head, one range of a sequence's
// cached rows; its four waves take tiles of 32 rows in turn. With 16x16 MFMAs (operand: lane
// l row l % 16, k slots of group g = l / 16; result: column l % 16, rows 4 g + i) the wave forms
// S^T = K Q^T, rows keys, columns heads, so a head's softmax state sits in its lanes,
// and its 4 scores a lane of each 16 rows are the B operand of O^T += V^T P^T when slot
// j of group g stands for rows 4 g + j % 4 (of the first 16 for j < 4, of the second above).
// The other operands come straight from memory: K rows as they lie; of V a lane reads
// E = HD / 16 neighbouring elements of the 8 rows of its group, so 16 lanes read a
// row of the head, and takes its elements' columns apart in registers (bf16: one v_perm a
// pair; f32, one row a slot: nothing). Row i of result tile t is element E i + t.
// Nothing of the cache passes through LDS.
//
// The queries and, over a bf16 cache, the weights P go in as NT bf16 terms: 3 for
// f32 activations (to 2^-24), 1 for bf16 ones (rounded). An f32 cache is multiplied in f32.
template <typename A, typename C, int HD, bool PART>
__global__ __launch_bounds__(kPagedThreads) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr bool F32 = sizeof(C) == 4;
  constexpr int NT = F32 || sizeof(A) == 2 ? 1 : 3;
  constexpr int E = HD / 16, KS = F32 ? HD / 16 : HD / 32, PE = 16 / (int)sizeof(C);
  constexpr int VP = E > PE ? E / PE : 1;     // 16-byte pieces of a lane's V elements
  constexpr int VW = E * (int)sizeof(C) / 4 / VP;  // words of a piece: 2 or 4
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const PagesArgs& p = a.p;
  const int hd = p.head_dim, half = hd / 2, group = p.n_q / p.n_kv, htiles = (group + 15) / 16;
  float* qr = sm;              // [16][HD]
  float* kr = qr + 16 * HD;    // [HD]
  float* vn = kr + HD;         // [HD]
  float* wacc = vn + HD;       // [waves][16][HD]; before that cos and sin [2][HD / 2]
  float* wm = wacc + kPagedWaves * 16 * HD;  // [waves][16]
  float* wl = wm + kPagedWaves * 16;
  float* ns = wl + kPagedWaves * 16;  // [16]
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x;
  const int ht = id % htiles;
  id /= htiles;
  const int hkv = id % p.n_kv;
  id /= p.n_kv;
  const int b = id % p.batch, split = id / p.batch;
  const int hq0 = hkv * group + ht * 16, heads = min(group - ht * 16, 16);
  const int len = a.lens[b];
  const bool add = p.k != nullptr;
  A* orow = static_cast<A*>(a.out) + (int64_t)b * a.out_stride + hq0 * hd;
  const int64_t rows = (int64_t)len + add;
  const bool bad = rows > a.max_len || rows > p.table_stride << p.page_bits;
  if (len < 0 || bad || rows == 0) {  // idle slot or nothing to see: zeros; more rows than the call allows: NaN
    if (split == 0)
      for (int i = tid; i < heads * hd; i += kPagedThreads) orow[i] = (A)(bad && len >= 0 ? NAN : 0.0f);
    return;
  }
  const int nsplit = max(1, (len + a.split_rows - 1) / a.split_rows);
  if (split >= nsplit) return;
  const int r0 = split * a.split_rows, r1 = min(r0 + a.split_rows, len);
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  const int kvd = p.n_kv * hd;
  bool lost = false;  // a page number out of range

  // the page rows of 16 rows from r (a multiple of 16; past the end: of the range's first)
  auto base_of = [&](int r) -> int64_t {
    r = r < r1 ? r : r0;
    const int page = trow[r >> p.page_bits];
    const bool ok = (uint32_t)page < (uint64_t)p.pages;
    lost |= !ok;
    return ((int64_t)(ok ? page : 0) << p.page_bits) + (r & ((1 << p.page_bits) - 1));
  };
  const C* kb = static_cast<const C*>(p.kpages) + hkv * hd;
  const C* vb = static_cast<const C*>(p.vpages) + hkv * hd;
  typedef uint32_t VPiece __attribute__((ext_vector_type(VW)));
  struct Rows {
    u32x4 k[2][KS];
    VPiece v[8][VP];
  };
  constexpr int VE = E / VP;  // elements of a piece; past the head's end it forms rows that nobody stores
  auto load = [&](Rows& x, int r) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const int64_t base = base_of(r + 16 * t);
      const C* kp = kb + (base + col) * kvd;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const int d = (F32 ? 16 * s : 32 * s) + PE * g;
        x.k[t][s] = *reinterpret_cast<const u32x4*>(kp + (PART ? min(d, hd - PE) : d));
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int q = 0; q < VP; q++)
          x.v[4 * t + j][q] = *reinterpret_cast<const VPiece*>(
              vb + (base + 4 * g + j) * kvd + (PART ? min(E * col + VE * q, hd - VE) : E * col + VE * q));
    }
  };
  constexpr int KT = 32, STEP = KT * kPagedWaves;
  Rows x[2];
  const int first = r0 + wave * KT;
  if (first < r1) load(x[0], first);

  // the rotated queries (zeros for heads and elements past the end), and the new row as it is stored
  float* cs = wacc;
  if (p.rope)
    for (int i = tid; i < half; i += kPagedThreads) rope_angle(len, i, hd, p.log2_theta, cs + i, cs + HD / 2 + i);
  for (int i = tid; i < 16 * HD; i += kPagedThreads) qr[i] = 0.0f;
  __syncthreads();
  const A* qrow = static_cast<const A*>(p.q) + (int64_t)b * p.q_stride + hq0 * hd;
  for (int i = tid; i < heads * half; i += kPagedThreads) {
    const int hh = i / half, e = i - hh * half;
    const float c = p.rope ? cs[e] : 1.0f, s = p.rope ? cs[HD / 2 + e] : 0.0f;
    const float x0 = (float)qrow[hh * hd + e], x1 = (float)qrow[hh * hd + e + half];
    qr[hh * HD + e] = x0 * c - x1 * s;
    qr[hh * HD + e + half] = x1 * c + x0 * s;
  }
  const bool last = split == nsplit - 1;
  if (add) {
    const int page = trow[len >> p.page_bits];
    const bool ok = (uint32_t)page < (uint64_t)p.pages;
    lost |= !ok;
    const int64_t at = (((int64_t)(ok ? page : 0) << p.page_bits) + (len & ((1 << p.page_bits) - 1))) * kvd + hkv * hd;
    const bool write = ok && split == 0 && ht == 0;
    const A* krow = static_cast<const A*>(p.k) + (int64_t)b * p.k_stride + hkv * hd;
    const A* vrow = static_cast<const A*>(p.v) + (int64_t)b * p.v_stride + hkv * hd;
    for (int e = tid; e < half; e += kPagedThreads) {
      const float c = p.rope ? cs[e] : 1.0f, s = p.rope ? cs[HD / 2 + e] : 0.0f;
      const float x0 = (float)krow[e], x1 = (float)krow[e + half];
      const C k0 = (C)(x0 * c - x1 * s), k1 = (C)(x1 * c + x0 * s), v0 = (C)(float)vrow[e],
              v1 = (C)(float)vrow[e + half];
      kr[e] = (float)k0;
      kr[e + half] = (float)k1;
      vn[e] = (float)v0;
      vn[e + half] = (float)v1;
      if (write) {
        C *ko = static_cast<C*>(p.kpages) + at, *vo = static_cast<C*>(p.vpages) + at;
        ko[e] = k0;
        ko[e + half] = k1;
        vo[e] = v0;
        vo[e + half] = v1;
      }
    }
  }
  __syncthreads();

  // query fragments: elements 32 s + 8 g .. (bf16), 16 s + 4 g .. (f32) of head `col`
  bf16x8 qb[F32 ? 1 : KS][NT];
  f32x4 qf[F32 ? KS : 1];
  if constexpr (F32) {
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const f32x4*>(qr + col * HD + 16 * s + 4 * g);
  } else {
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        __bf16 t[NT];
        split_terms<NT>(qr[col * HD + 32 * s + 8 * g + j], t);
#pragma unroll
        for (int n = 0; n < NT; n++) qb[s][n][j] = t[n];
      }
  }

  f32x4 acc[E];
#pragma unroll
  for (int t = 0; t < E; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  auto compute = [&](Rows& y, int r) {
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        u32x4 kw = y.k[t][ks];
        if (PART && (F32 ? 16 * ks : 32 * ks) + PE * g >= hd) kw = u32x4{0, 0, 0, 0};
        if constexpr (F32) {
          const f32x4 kf = __builtin_bit_cast(f32x4, kw);
#pragma unroll
          for (int j = 0; j < 4; j++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[ks][j], d, 0, 0, 0);
        } else {
#pragma unroll
          for (int n = 0; n < NT; n++)
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kw), qb[ks][n], d, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) s[4 * t + i] = r + 16 * t + 4 * g + i < r1 ? d[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale2;
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale2, -ref));
      l += s[i];
    }
#pragma unroll
    for (int t = 0; t < E; t++) acc[t] *= alpha;
    if (r + KT > r1) {  // rows past the end hold anything: 0 times it must stay 0
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (r + 16 * (j >> 2) + 4 * g + (j & 3) >= r1)
#pragma unroll
          for (int q = 0; q < VP; q++)
#pragma unroll
            for (int w = 0; w < VW; w++) y.v[j][q][w] = 0;
    }
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < E; t++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(y.v[j][t / PE][t % PE]), s[j], acc[t], 0, 0, 0);
    } else {
      bf16x8 pb[NT];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        __bf16 t[NT];
        split_terms<NT>(s[j], t);
#pragma unroll
        for (int n = 0; n < NT; n++) pb[n][j] = t[n];
      }
#pragma unroll
      for (int w = 0; w < E / 2; w++) {  // elements 2 w and 2 w + 1 of the lane
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t e0 = y.v[2 * j][w / VW][w % VW], e1 = y.v[2 * j + 1][w / VW][w % VW];
          lo[j] = low16_pair(e0, e1);
          hi[j] = high16_pair(e0, e1);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          acc[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lo), pb[n], acc[2 * w], 0, 0, 0);
          acc[2 * w + 1] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, hi), pb[n], acc[2 * w + 1], 0, 0, 0);
        }
      }
    }
  };
  for (int r = first; r < r1; r += 2 * STEP) {
    if (r + STEP < r1) load(x[1], r + STEP);
    compute(x[0], r);
    if (r + STEP >= r1) break;
    if (r + 2 * STEP < r1) load(x[0], r + 2 * STEP);
    compute(x[1], r + STEP);
  }

  // the waves' states, then the new row (last range)
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int t = 0; t < E; t++) wacc[(wave * 16 + col) * HD + E * (4 * g + i) + t] = acc[t][i];
  if (g == 0) {
    wm[wave * 16 + col] = m;
    wl[wave * 16 + col] = l;
  }
  if (add && last)
    for (int hh = wave; hh < heads; hh += kPagedWaves) {
      float dot = 0.0f;
      for (int d = lane; d < hd; d += 64) dot += qr[hh * HD + d] * kr[d];
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off, 64);
      if (lane == 0) ns[hh] = dot * a.scale2;
    }
  const bool any_lost = __syncthreads_or(lost);
  for (int i = tid; i < heads * hd; i += kPagedThreads) {
    const int hh = i / hd, d = i - hh * hd;
    const float sn = add && last ? ns[hh] : -INFINITY;
    float mx = sn;
#pragma unroll
    for (int w = 0; w < kPagedWaves; w++) mx = fmaxf(mx, wm[w * 16 + hh]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float o = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kPagedWaves; w++) {
      const float f = __builtin_amdgcn_exp2f(wm[w * 16 + hh] - ref);
      sum += f * wl[w * 16 + hh];
      o += f * wacc[(w * 16 + hh) * HD + d];
    }
    if (add && last) {
      const float e = __builtin_amdgcn_exp2f(sn - ref);
      sum += e;
      o += e * vn[d];
    }
    if (any_lost) sum = NAN;
    if (nsplit == 1) {
      orow[i] = (A)(sum == 0.0f ? 0.0f : o / sum);
    } else {
      float* rec = a.part + (((int64_t)b * p.n_q + hq0 + hh) * a.nsplit + split) * (kRec + hd);
      rec[kRec + d] = o;
      if (d == 0) {
        rec[0] = mx;
        rec[1] = sum;
      }
    }
  }
}

// Joins the ranges' records of a (sequence, head), one workgroup each: head_dim / 4 lanes
// a record, the lane groups' sums added in order.
template <typename A>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
  const PagesArgs& p = a.p;
  const int hq = blockIdx.x % p.n_q, b = blockIdx.x / p.n_q, hd = p.head_dim, len = a.lens[b];
  const int64_t rows = (int64_t)len + (p.k != nullptr);
  if (len < 0 || rows > a.max_len || rows > p.table_stride << p.page_bits) return;
  const int n = (len + a.split_rows - 1) / a.split_rows;
  if (n <= 1) return;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float sums[256 * 4];
  __shared__ float lsum[128];
  const int tid = threadIdx.x, dl = hd / 4, groups = 256 / dl, grp = tid / dl, d = tid % dl;
  const int64_t rs = kRec + hd;
  const float* rec = a.part + (int64_t)(b * p.n_q + hq) * a.nsplit * rs;
  float mx = -INFINITY;
  for (int r = tid; r < n; r += 256) mx = fmaxf(mx, rec[r * rs]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = mx == -INFINITY ? 0.0f : mx;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f;
  if (grp < groups) {
    for (int r = grp; r < n; r += groups) {
      const float f = __builtin_amdgcn_exp2f(rec[r * rs] - ref);
      sum += f * rec[r * rs + 1];
      o += f * *reinterpret_cast<const f32x4*>(rec + r * rs + kRec + 4 * d);
    }
    *reinterpret_cast<f32x4*>(&sums[4 * tid]) = o;
    if (d == 0) lsum[grp] = sum;
  }
  __syncthreads();
  if (tid < dl) {
    for (int k = 1; k < groups; k++) {
      o += *reinterpret_cast<const f32x4*>(&sums[4 * (k * dl + tid)]);
      sum += lsum[k];
    }
    A* out = static_cast<A*>(a.out) + (int64_t)b * a.out_stride + hq * hd + 4 * tid;
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = (A)(sum == 0.0f ? 0.0f : o[e] / sum);
  }
}

// RoPE and append of packed rows: a workgroup a row. The row's angles are formed once
// for all heads; a thread takes 16-byte pieces of both halves of a head.
template <typename A, typename C>
__global__ __launch_bounds__(256) void pages_append_kernel(PagesAppendArgs a) {
  const PagesArgs& p = a.p;
  __shared__ float cs[2][128];
  const int tid = threadIdx.x, hd = p.head_dim, half = hd / 2;
  const int64_t row = blockIdx.x;
  // the last sequence that starts at or before the row
  int n = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int b = b0 + (tid & 63);
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(b < p.batch && a.cu[b] <= row));
    n += c;
    if (c < 64) break;
  }
  if (n == 0 || row >= a.cu[n]) return;  // a row of no sequence: left as it is
  const int b = n - 1, past = a.past[b];
  if (past < 0) return;
  const int64_t pos = past + row - a.cu[b];
  const bool inside = pos < p.table_stride << p.page_bits;
  const int page = inside ? p.table[(int64_t)b * p.table_stride + (pos >> p.page_bits)] : -1;
  const bool ok = (uint32_t)page < (uint64_t)p.pages;
  const int64_t at = ok ? ((int64_t)page << p.page_bits) + (pos & ((1 << p.page_bits) - 1)) : 0;
  if (p.rope) {
    for (int i = tid; i < half; i += 256) rope_angle(pos, i, hd, p.log2_theta, &cs[0][i], &cs[1][i]);
    __syncthreads();
  }
  typedef A A4 __attribute__((ext_vector_type(4)));
  typedef C C4 __attribute__((ext_vector_type(4)));
  const int hp = half / 4, kvd = p.n_kv * hd;
  for (int i = tid; i < (p.n_q + p.n_kv) * hp; i += 256) {
    const int head = i / hp, e = 4 * (i - head * hp);
    const bool is_q = head < p.n_q;
    const int hh = is_q ? head : head - p.n_q;
    const A* x = is_q ? static_cast<const A*>(p.q) + row * p.q_stride : static_cast<const A*>(p.k) + row * p.k_stride;
    const A4 x0 = *reinterpret_cast<const A4*>(x + hh * hd + e), x1 = *reinterpret_cast<const A4*>(x + hh * hd + e + half);
    float y0[4], y1[4];
    A4 z0, z1;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float c = p.rope ? cs[0][e + j] : 1.0f, s = p.rope ? cs[1][e + j] : 0.0f;
      y0[j] = (float)x0[j] * c - (float)x1[j] * s;
      y1[j] = (float)x1[j] * c + (float)x0[j] * s;
      if (!ok) y0[j] = y1[j] = NAN;  // no page for the row: its outputs say so
      z0[j] = (A)y0[j];
      z1[j] = (A)y1[j];
    }
    A* o = is_q ? static_cast<A*>(a.q_out) + row * a.q_out_stride
                : a.k_out ? static_cast<A*>(a.k_out) + row * a.k_out_stride : nullptr;
    if (o) {
      *reinterpret_cast<A4*>(o + hh * hd + e) = z0;
      *reinterpret_cast<A4*>(o + hh * hd + e + half) = z1;
    }
    if (!is_q && ok) {
      C4 w0, w1;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        w0[j] = (C)y0[j];
        w1[j] = (C)y1[j];
      }
      C* kc = static_cast<C*>(p.kpages) + at * kvd + hh * hd + e;
      *reinterpret_cast<C4*>(kc) = w0;
      *reinterpret_cast<C4*>(kc + half) = w1;
    }
  }
  if (!ok) return;
  const A* vrow = static_cast<const A*>(p.v) + row * p.v_stride;
  for (int i = 4 * tid; i < kvd; i += 1024) {
    const A4 x = *reinterpret_cast<const A4*>(vrow + i);
    C4 y;
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = (C)(float)x[j];
    *reinterpret_cast<C4*>(static_cast<C*>(p.vpages) + at * kvd + i) = y;
  }
}

// Pages copied in every plane. The page numbers come as a kernel argument, so the
// caller's host arrays are free when the call returns.
constexpr int kCopyPairs = 240;  // 8 bytes each, within the argument space
constexpr int kCopyBytes = 16384;  // of a page and plane, by one workgroup: 4 x 16 bytes a thread
struct CopyPairs {
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
__global__ __launch_bounds__(256) void pages_copy_kernel(char* base, int64_t plane_bytes, int64_t page_bytes, int parts,
                                                         int n, CopyPairs pairs) {
  int id = blockIdx.x;
  const int part = id % parts;
  id /= parts;
  const int i = id % n, plane = id / n;
  const int64_t o = (int64_t)part * kCopyBytes;
  const char* s = base + plane * plane_bytes + pairs.src[i] * page_bytes + o;
  char* d = base + plane * plane_bytes + pairs.dst[i] * page_bytes + o;
  const int have = (int)(page_bytes - o < kCopyBytes ? page_bytes - o : kCopyBytes);
  constexpr int U = kCopyBytes / 4096;
  u32x4 x[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int e = 16 * ((int)threadIdx.x + 256 * u);
    if (e < have) x[u] = *reinterpret_cast<const u32x4*>(s + e);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int e = 16 * ((int)threadIdx.x + 256 * u);
    if (e < have) *reinterpret_cast<u32x4*>(d + e) = x[u];
  }
}

PagedPlan plan_paged_attention(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len,
                               int cu_count) {
  const int64_t group = n_q / n_kv, per_split = std::max<int64_t>(1, batch * n_kv * ((group + 15) / 16));
  const int64_t want = (max_len * per_split + 4 * cu_count - 1) / (4 * cu_count);
  const int64_t rows = std::min<int64_t>(std::max<int64_t>((want + 127) / 128 * 128, 128), 1024);
  PagedPlan p;
  p.split_rows = (int)rows;
  p.nsplit = (int)std::max<int64_t>(1, (max_len + rows - 1) / rows);
  p.work = p.nsplit > 1 ? (size_t)(batch * n_q * p.nsplit * (kRec + head_dim)) * sizeof(float) : 0;
  return p;
}

namespace {

template <typename A, typename C, int HD, bool PART>
hipError_t run_paged(const PagedAttnArgs& a, hipStream_t stream) {
  const PagesArgs& p = a.p;
  const int64_t htiles = (p.n_q / p.n_kv + 15) / 16;
  constexpr int lds = (16 * HD + 2 * HD + kPagedWaves * 16 * (HD + 2) + 16) * 4;
  const auto kernel = paged_attention_kernel<A, C, HD, PART>;
  if (lds > 65536) {
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds))
      return e;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.nsplit * p.batch * p.n_kv * htiles)), dim3(kPagedThreads), lds, stream,
                     a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.nsplit > 1) {
    hipLaunchKernelGGL(paged_merge_kernel<A>, dim3((unsigned)(p.batch * p.n_q)), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <typename A, typename C>
hipError_t run_paged_hd(const PagedAttnArgs& a, hipStream_t stream) {
  const int hd = a.p.head_dim;
  if (hd == 64) return run_paged<A, C, 64, false>(a, stream);
  if (hd == 128) return run_paged<A, C, 128, false>(a, stream);
  if (hd == 256) return run_paged<A, C, 256, false>(a, stream);
  if (hd < 64) return run_paged<A, C, 64, true>(a, stream);
  if (hd < 128) return run_paged<A, C, 128, true>(a, stream);
  return run_paged<A, C, 256, true>(a, stream);
}

template <typename A, typename C>
hipError_t run_append(const PagesAppendArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((pages_append_kernel<A, C>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(int dtype, int cache_dtype, const PagedAttnArgs& a, hipStream_t stream) {
  if (dtype == RQ_F32)
    return cache_dtype == RQ_F32 ? run_paged_hd<float, float>(a, stream) : run_paged_hd<float, __bf16>(a, stream);
  return run_paged_hd<__bf16, __bf16>(a, stream);
}

hipError_t launch_pages_append(int dtype, int cache_dtype, const PagesAppendArgs& a, hipStream_t stream) {
  if (dtype == RQ_F32)
    return cache_dtype == RQ_F32 ? run_append<float, float>(a, stream) : run_append<float, __bf16>(a, stream);
  return run_append<__bf16, __bf16>(a, stream);
}

int64_t pages_copy_groups(int64_t page_bytes) { return (page_bytes + kCopyBytes - 1) / kCopyBytes; }

hipError_t launch_pages_copy(void* base, int64_t planes, int64_t plane_bytes, int64_t page_bytes, const int32_t* src,
                             const int32_t* dst, int64_t n, hipStream_t stream) {
  const int64_t parts = pages_copy_groups(page_bytes);
  for (int64_t i = 0; i < n; i += kCopyPairs) {
    CopyPairs pairs;
    const int m = (int)std::min<int64_t>(kCopyPairs, n - i);
    std::copy(src + i, src + i + m, pairs.src);
    std::copy(dst + i, dst + i + m, pairs.dst);
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)(parts * m * planes)), dim3(256), 0, stream,
                       static_cast<char*>(base), plane_bytes, page_bytes, (int)parts, m, pairs);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace rq
