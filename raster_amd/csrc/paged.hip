// paged.hip — a key-value cache in pages: one new token of every sequence (RoPE,
// append, attention), a packed prompt's RoPE and append, pages copied.
//
// The batched form of attention.hip's decode step. A sequence's rows lie in pages
// of 2^b rows, found through its row of the page table. Pages hold at least 16 rows, so 16
// rows that start at a multiple of 16 lie in one page: a page number is looked up once
// for them, by the whole wave.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "attn_tile.h"
#include "paged_tile.h"

namespace rq {

namespace {

constexpr int kPagedThreads = 256, kPagedWaves = 4;

// LDS of 16 heads' queries as fragments: f32, or two or three bf16 terms
template <typename A, typename C>
constexpr int paged_query_bytes(int hd) {
  return 16 * hd * (sizeof(C) == 4 || sizeof(A) == 2 ? 4 : 6);
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
// Bound by the cache rows' way from memory: 8 sequences of 33 to 65 Ki rows, 64/8 heads x 128, bf16, pages of
// 64: 346 + 6 us (join) for 1.77 GB, 5.1 TB/s (a plain read 6.2; the workgroups' last round leaves CUs idle:
// busy 0.79); 32 of 0 to 8191 rows, 32/8 heads, f32 over bf16: 45 + 5 us for 233 MB, 5.1 TB/s. One sequence of
// 128 rows (f32, 16 heads): 9.7 us, the chain length - page number - row - scores - values of one workgroup a head.
//
// With a window (WIN) the ranges are of the rows that are walked, the sinks' blocks and from the window's first block
// on (paged_tile.h): 16 sequences of 1 to 65535 rows, window 4096 and 4 sinks, 32/8 heads, bf16, 197 MB: 35 + 4.5 us,
// 5.0 TB/s; without the window the same sequences have 1.25 GB.
//
// Over a bf16 cache the rotated queries and the weights P go in as NT bf16 terms: 3 for f32 activations (to
// 2^-24), 2 for bf16 ones (to 2^-17): the result's own rounding is what is left. Error of 8 sequences of 33 to 65 Ki
// rows, of its norm: 0.0017; with one term of the weights 0.0022, of the queries too 0.0028, all in the same time
// (372, 370 us of cold caches; 8 of 4000 rows, 32/8 heads, 34.3, 34.1; one of 128, 16 heads, 7.0, 6.9). An f32 cache
// is multiplied in f32.
template <typename A, typename C, int HD, bool PART, bool WIN>
__global__ __launch_bounds__(kPagedThreads) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr bool F32 = sizeof(C) == 4;
  constexpr int NT = F32 ? 1 : sizeof(A) == 2 ? 2 : 3;
  constexpr int kQueryBytes = paged_query_bytes<A, C>(HD);
  constexpr int E = HD / 16, KS = F32 ? HD / 16 : HD / 32, PE = 16 / (int)sizeof(C);
  constexpr int VP = E > PE ? E / PE : 1;     // 16-byte pieces of a lane's V elements
  constexpr int VW = E * (int)sizeof(C) / 4 / VP;  // words of a piece: 2 or 4
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const PagesArgs& p = a.p;
  const int hd = p.head_dim, half = hd / 2, group = p.n_q / p.n_kv, htiles = (group + 15) / 16, nh = min(group, 16);
  float* kr = sm + kQueryBytes / 4;  // [HD]; before it the queries as fragments, [term][step][lane] 16 bytes
  float* vn = kr + HD;               // [HD]
  float* wacc = vn + HD;       // [waves][heads][HD]; before that cos and sin [2][HD / 2]
  float* wm = wacc + kPagedWaves * nh * HD;  // [waves][16]
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
  constexpr int KT = 32, STEP = KT * kPagedWaves;
  // the query rows and the new row, and the wave's first page numbers: asked for with the
  // length, not after it
  constexpr int NE = HD / 32;  // pairs of query elements a thread
  const A* qrow = static_cast<const A*>(p.q) + (int64_t)b * p.q_stride + hq0 * hd;
  A q0[NE], q1[NE], n0[2], n1[2];  // n: of the new k and v
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = min(tid + n * kPagedThreads, heads * half - 1), hh = i / half, e = i - hh * half;
    q0[n] = qrow[hh * hd + e];
    q1[n] = qrow[hh * hd + e + half];
  }
  if (p.k != nullptr) {
    const A* krow = static_cast<const A*>(p.k) + (int64_t)b * p.k_stride + hkv * hd;
    const A* vrow = static_cast<const A*>(p.v) + (int64_t)b * p.v_stride + hkv * hd;
    const int e = min(tid, half - 1);
    n0[0] = krow[e], n0[1] = krow[e + half];
    n1[0] = vrow[e], n1[1] = vrow[e + half];
  }
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  const int r0 = split * a.split_rows, first = r0 + wave * KT;
  const int last_entry = max((int)p.table_stride - 1, 0);
  int page0 = -1, page1 = -1;
  if (!WIN && p.table_stride > 0) {
    page0 = trow[min(first >> p.page_bits, last_entry)];
    page1 = trow[min((first + 16) >> p.page_bits, last_entry)];
  }
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
  // one row past a whole number of ranges goes to the last range
  CachedRows<WIN> cr;
  cr.init(a, len, rows);
  const int nsplit = ranges_of(cr.walk, a.split_rows);
  if (split >= nsplit) return;
  const int r1 = split == nsplit - 1 ? cr.walk : r0 + a.split_rows;
  const int kvd = p.n_kv * hd;
  bool lost = false;  // a page number out of range

  // the page rows of 16 rows from r (a multiple of 16; past the end: of the range's first)
  auto row_base = [&](int page, int r) -> int64_t {
    const bool ok = (uint32_t)page < (uint64_t)p.pages;
    lost |= !ok;
    return ((int64_t)(ok ? page : 0) << p.page_bits) + (r & ((1 << p.page_bits) - 1));
  };
  auto base_of = [&](int r) -> int64_t {
    r = cr.row(r < r1 ? r : r0);
    return row_base(trow[r >> p.page_bits], r);
  };
  const C* kb = static_cast<const C*>(p.kpages) + hkv * hd;
  const C* vb = static_cast<const C*>(p.vpages) + hkv * hd;
  typedef uint32_t VPiece __attribute__((ext_vector_type(VW)));
  u32x4 xk[2][KS];
  VPiece xv[8][VP];
  auto load_k = [&](int64_t (&base)[2]) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const C* kp = kb + (base[t] + col) * kvd;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const int d = (F32 ? 16 * s : 32 * s) + PE * g;
        xk[t][s] = *reinterpret_cast<const u32x4*>(kp + (PART ? min(d, hd - PE) : d));
      }
    }
  };
  constexpr int VE = E / VP;  // elements of a piece; past the head's end it forms rows that nobody stores
  auto load_v = [&](int64_t (&base)[2]) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int q = 0; q < VP; q++)
          xv[4 * t + j][q] = *reinterpret_cast<const VPiece*>(
              vb + (base[t] + 4 * g + j) * kvd + (PART ? min(E * col + VE * q, hd - VE) : E * col + VE * q));
  };
  int64_t base[2] = {0, 0};
  if (first < r1) {
    if constexpr (WIN) {
      base[0] = base_of(first);
      base[1] = first + 16 < r1 ? base_of(first + 16) : base[0];
    } else {
      base[0] = row_base(page0, first);
      base[1] = first + 16 < r1 ? row_base(page1, first + 16) : base[0];
    }
    load_k(base);
    load_v(base);
  }

  // the rotated queries as the products' operands (zeros for heads and elements past the
  // end), and the new row as it is stored
  float* cs = wacc;
  if (p.rope && tid < half) rope_angle(len, tid, hd, p.log2_theta, cs + tid, cs + HD / 2 + tid);
  for (int i = tid; i < kQueryBytes / 16; i += kPagedThreads) reinterpret_cast<u32x4*>(sm)[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
  // element e of head hh: lane 16 g + hh of a step holds 32 s + 8 g .. + 7 (f32: 16 s + 4 g .. + 3)
  auto put_query = [&](int hh, int e, float x) {
    if constexpr (F32) {
      sm[((e >> 4) * 64 + ((e >> 2) & 3) * 16 + hh) * 4 + (e & 3)] = x;
    } else {
      __bf16 t[NT];
      split_terms<NT>(x, t);
      __bf16* at = reinterpret_cast<__bf16*>(sm) + ((e >> 5) * 64 + ((e >> 3) & 3) * 16 + hh) * 8 + (e & 7);
#pragma unroll
      for (int n = 0; n < NT; n++) at[n * 16 * HD] = t[n];
    }
  };
  auto get_query = [&](int hh, int e) {
    if constexpr (F32) {
      return sm[((e >> 4) * 64 + ((e >> 2) & 3) * 16 + hh) * 4 + (e & 3)];
    } else {
      const __bf16* at = reinterpret_cast<const __bf16*>(sm) + ((e >> 5) * 64 + ((e >> 3) & 3) * 16 + hh) * 8 + (e & 7);
      float x = 0.0f;
#pragma unroll
      for (int n = NT - 1; n >= 0; n--) x += (float)at[n * 16 * HD];
      return x;
    }
  };
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = tid + n * kPagedThreads, hh = i / half, e = i - hh * half;
    if (i < heads * half) {
      const float c = p.rope ? cs[e] : 1.0f, s = p.rope ? cs[HD / 2 + e] : 0.0f;
      const float x0 = (float)q0[n], x1 = (float)q1[n];
      put_query(hh, e, x0 * c - x1 * s);
      put_query(hh, e + half, x1 * c + x0 * s);
    }
  }
  const bool last = split == nsplit - 1;
  if (add && (last || split == 0)) {
    const int page = trow[len >> p.page_bits];
    const bool ok = (uint32_t)page < (uint64_t)p.pages;
    lost |= !ok;
    const int64_t at = (((int64_t)(ok ? page : 0) << p.page_bits) + (len & ((1 << p.page_bits) - 1))) * kvd + hkv * hd;
    if (tid < half) {
      const float c = p.rope ? cs[tid] : 1.0f, s = p.rope ? cs[HD / 2 + tid] : 0.0f;
      const float x0 = (float)n0[0], x1 = (float)n0[1];
      const C k0 = (C)(x0 * c - x1 * s), k1 = (C)(x1 * c + x0 * s), v0 = (C)(float)n1[0], v1 = (C)(float)n1[1];
      kr[tid] = (float)k0;
      kr[tid + half] = (float)k1;
      vn[tid] = (float)v0;
      vn[tid + half] = (float)v1;
      if (ok && split == 0 && ht == 0) {
        C *ko = static_cast<C*>(p.kpages) + at + tid, *vo = static_cast<C*>(p.vpages) + at + tid;
        ko[0] = k0;
        ko[half] = k1;
        vo[0] = v0;
        vo[half] = v1;
      }
    }
  }
  __syncthreads();

  f32x4 acc[E];
#pragma unroll
  for (int t = 0; t < E; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  for (int r = first; r < r1; r += STEP) {
    const bool more = r + STEP < r1;
    if (more) {  // (the last tile's rows are in flight or used: their addresses are no more needed)
      base[0] = base_of(r + STEP);
      base[1] = base_of(r + STEP + 16);
    }
    float s[8];
    f32x4 d[2] = {};
    int ql = lane;  // read anew for every tile: kept in registers they would cost a wave a SIMD
    asm volatile("" : "+v"(ql));
    const u32x4* qp = reinterpret_cast<const u32x4*>(sm) + ql;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      u32x4 qw[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) qw[n] = qp[(n * KS + ks) * 64];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        u32x4 kw = xk[t][ks];
        if (PART && (F32 ? 16 * ks : 32 * ks) + PE * g >= hd) kw = u32x4{0, 0, 0, 0};
        if constexpr (F32) {
          const f32x4 kf = __builtin_bit_cast(f32x4, kw), qf = __builtin_bit_cast(f32x4, qw[0]);
#pragma unroll
          for (int j = 0; j < 4; j++) d[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[j], d[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int n = 0; n < NT; n++)
            d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kw),
                                                           __builtin_bit_cast(bf16x8, qw[n]), d[t], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[4 * t + i] = r + 16 * t + 4 * g + i < r1 ? d[t][i] : -INFINITY;
    // a block that the window or the sinks end in
    const bool cut[2] = {!cr.sees_block(cr.row(r)), !cr.sees_block(cr.row(r + 16))};
    if constexpr (WIN) {
#pragma unroll
      for (int t = 0; t < 2; t++)
        if (cut[t])
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!cr.sees(cr.row(r + 16 * t) + 4 * g + i)) s[4 * t + i] = -INFINITY;
    }
    if (more) load_k(base);
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
    if (r + KT > r1 || cut[0] || cut[1]) {  // rows not seen hold anything: 0 times it must stay 0
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (r + 16 * (j >> 2) + 4 * g + (j & 3) >= r1 || !cr.sees(cr.row(r + 16 * (j >> 2)) + 4 * g + (j & 3)))
#pragma unroll
          for (int q = 0; q < VP; q++)
#pragma unroll
            for (int w = 0; w < VW; w++) xv[j][q][w] = 0;
    }
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < E; t++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(xv[j][t / PE][t % PE]), s[j], acc[t], 0, 0, 0);
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
          const uint32_t e0 = xv[2 * j][w / VW][w % VW], e1 = xv[2 * j + 1][w / VW][w % VW];
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
    if (more) load_v(base);
  }

  // the waves' states, then the new row (last range)
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (col < nh)
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int t = 0; t < E; t++) wacc[(wave * nh + col) * HD + E * (4 * g + i) + t] = acc[t][i];
  if (g == 0) {
    wm[wave * 16 + col] = m;
    wl[wave * 16 + col] = l;
  }
  if (add && last)
    for (int hh = wave; hh < heads; hh += kPagedWaves) {
      float dot = 0.0f;
      for (int d = lane; d < hd; d += 64) dot += get_query(hh, d) * kr[d];
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
      o += f * wacc[(w * nh + hh) * HD + d];
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
template <typename A, bool WIN>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
  const PagesArgs& p = a.p;
  const int hq = blockIdx.x % p.n_q, b = blockIdx.x / p.n_q, hd = p.head_dim, len = a.lens[b];
  const int64_t rows = (int64_t)len + (p.k != nullptr);
  if (len < 0 || rows > a.max_len || rows > p.table_stride << p.page_bits) return;
  CachedRows<WIN> cr;
  cr.init(a, len, rows);
  const int n = ranges_of(cr.walk, a.split_rows);
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
// for all heads; a thread takes 4 elements of both halves of a head at a time. Bound by memory: 8192 rows of bf16,
// 32/8 heads x 128, 33 us for 218 MB, 6.5 TB/s (a part of it still in the caches).
template <typename A, typename C>
__global__ __launch_bounds__(256) void pages_append_kernel(PagesAppendArgs a) {
  const PagesArgs& p = a.p;
  __shared__ float cs[2][128];
  const int tid = threadIdx.x, hd = p.head_dim, half = hd / 2;
  const int64_t row = blockIdx.x;
  // the last sequence that starts at or before the row
  const int n = count_first(p.batch, [&](int b) { return a.cu[b] <= row; });
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
// caller's host arrays are free when the call returns. A workgroup holds four loads a thread in flight and
// stores them: 1300 pages of 32 KB in 32 planes 566 us, 4.8 TB/s of reads and writes (a large copy 4.75).
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
  // About one workgroup a CU at max_len, of 128 to 512 rows, up to 1024 where a CU has more of them (2048: 16 Ki):
  // fewer leave CUs idle, more pay for records and the start of a workgroup. us, rows a range
  // (bf16 pages): 32/8 heads x 128, one sequence of 4096 rows 128: 12.5, 256: 13.1, 1024: 19.2; of
  // 32768 256: 34.7, 1024: 30.3; 32 of 0 to 8191 256: 55.0, 1024: 47.0, 2048: 68.6; 64/8 heads, 8 of
  // 33 to 65 Ki 1024: 363, 2048: 352; 8/4 x 256, 16 of 2000 128: 49.1, 512: 30.9.
  // Caches cold, 512 / 1024: 8 of 4000 (1000 rows a CU) 28.5 / 29.8, of 1 to 4000 25.5 / 27.6; 16/16 heads, 8 of 4000
  // (2000 a CU) 57.0 / 55.4, 4 of 16000 100.6 / 99.9.
  // With a group a CU and no more than 2048 rows before the new one, one range and no join: 32 of 1200
  // 38.7 -> 32.9, 64 of 2000 107 -> 99, 32 of 1 to 1200 26.2 -> 23.9, 64 of 1 to 2000 64.3 -> 65.4.
  const int64_t groups = std::max<int64_t>(1, batch * n_kv * ((n_q / n_kv + 15) / 16));
  const int64_t share = (max_len * groups + cu_count - 1) / std::max(cu_count, 1);
  const int64_t most = share >= 16384 || (max_len <= 2049 && groups >= cu_count) ? 2048 : share > 1024 ? 1024 : 512;
  const int64_t rows = std::min<int64_t>(std::max<int64_t>((share + 127) / 128 * 128, 128), most);
  PagedPlan p;
  p.split_rows = (int)rows;
  p.nsplit = (int)ranges_of(max_len, rows);
  p.work = p.nsplit > 1 ? (size_t)(batch * n_q * p.nsplit * (kRec + head_dim)) * sizeof(float) : 0;
  return p;
}

namespace {

template <typename A, typename C, int HD, bool PART, bool WIN>
hipError_t run_paged(const PagedAttnArgs& a, hipStream_t stream) {
  const PagesArgs& p = a.p;
  const int64_t htiles = (p.n_q / p.n_kv + 15) / 16;
  constexpr int kFixed = paged_query_bytes<A, C>(HD) + (2 * HD + kPagedWaves * 32 + 16) * 4;
  constexpr int kMaxLds = kFixed + kPagedWaves * 16 * HD * 4;
  const int lds = kFixed + kPagedWaves * std::min(p.n_q / p.n_kv, 16) * HD * 4;
  const auto kernel = paged_attention_kernel<A, C, HD, PART, WIN>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), kMaxLds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.nsplit * p.batch * p.n_kv * htiles)), dim3(kPagedThreads), lds, stream,
                     a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.nsplit > 1) {
    hipLaunchKernelGGL((paged_merge_kernel<A, WIN>), dim3((unsigned)(p.batch * p.n_q)), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <typename A, typename C, bool WIN>
hipError_t run_paged_hd(const PagedAttnArgs& a, hipStream_t stream) {
  const int hd = a.p.head_dim;
  if (hd == 64) return run_paged<A, C, 64, false, WIN>(a, stream);
  if (hd == 128) return run_paged<A, C, 128, false, WIN>(a, stream);
  if (hd == 256) return run_paged<A, C, 256, false, WIN>(a, stream);
  if (hd < 64) return run_paged<A, C, 64, true, WIN>(a, stream);
  if (hd < 128) return run_paged<A, C, 128, true, WIN>(a, stream);
  return run_paged<A, C, 256, true, WIN>(a, stream);
}

template <typename A, typename C>
hipError_t run_append(const PagesAppendArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((pages_append_kernel<A, C>), dim3((unsigned)a.rows), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

template <bool WIN>
static hipError_t launch_paged(int dtype, int cache_dtype, const PagedAttnArgs& a, hipStream_t stream) {
  if (dtype == RQ_F32)
    return cache_dtype == RQ_F32 ? run_paged_hd<float, float, WIN>(a, stream)
                                 : run_paged_hd<float, __bf16, WIN>(a, stream);
  return run_paged_hd<__bf16, __bf16, WIN>(a, stream);
}

hipError_t launch_paged_attention(int dtype, int cache_dtype, const PagedAttnArgs& a, hipStream_t stream) {
  return a.window > 0 ? launch_paged<true>(dtype, cache_dtype, a, stream)
                      : launch_paged<false>(dtype, cache_dtype, a, stream);
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
  const int64_t most = std::min<int64_t>(kCopyPairs, kMaxGroups / (parts * planes));
  for (int64_t i = 0; i < n; i += most) {
    CopyPairs pairs;
    const int m = (int)std::min<int64_t>(most, n - i);
    std::copy(src + i, src + i + m, pairs.src);
    std::copy(dst + i, dst + i + m, pairs.dst);
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)(parts * m * planes)), dim3(256), 0, stream,
                       static_cast<char*>(base), plane_bytes, page_bytes, (int)parts, m, pairs);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace rq
