// paged_q8.hip — a paged key-value cache in 8 bits: one new token of every sequence, a packed prompt's
// append, the stored rows as values.
//
// A block is 16 rows that start at a multiple of 16, of one KV head, keys and values apart: int8 codes c in
// -127 .. 127 and one f32 scale s, its values c s. Rows x that are appended to a block with scale s0 (0 where its
// first row is among them) give it the scale
//   s = max(s0, max |x| * f32(1 / 127)),   their codes round(x / s), those before them round(c (s0 / s)),
// in f32, each operation rounded by itself, ties to even: the same bits however the work is spread. A scale only
// rises while its block fills, so a code is rounded anew a few times at most (ln 16 of 16 rows in any
// order set a new maximum, on average) and each time by half a step. Where an x or s0 is not finite the scale is
// NaN: whoever attends the block gets NaN, as from an f32 cache, until its first row is written again.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "attn_tile.h"
#include "paged_tile.h"

namespace rq {

namespace {

constexpr int kBlock = 16;
constexpr int kThreads = 256, kWaves = 4;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

// max |x| of the new rows and the old scale (0: none) to the new scale
__device__ __forceinline__ float raised(float amax, bool all_finite, float s0) {
  const float s = fmaxf(s0, amax * (1.0f / 127.0f));
  return all_finite && finite(s0) ? s : NAN;
}
__device__ __forceinline__ int code_of(float x, float s) {
  return s > 0.0f ? (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.0f), 127.0f) : 0;
}
// four codes of a block whose scale rises from s0 to s
__device__ __forceinline__ uint32_t recoded(uint32_t w, float ratio) {
  uint32_t y = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int c = (int)rintf((float)(int8_t)(w >> (8 * j)) * ratio);
    y |= (uint32_t)(c & 255) << (8 * j);
  }
  return y;
}
__device__ __forceinline__ uint32_t pack4(const int (&c)[4]) {
  return (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 | (uint32_t)(c[3] & 255) << 24;
}
// x0, x1 rotated: every operation rounded by itself
__device__ __forceinline__ void rotate(float x0, float x1, float c, float s, float* y0, float* y1) {
#pragma clang fp contract(off)
  const float a0 = x0 * c, b0 = x1 * s, a1 = x1 * c, b1 = x0 * s;
  *y0 = a0 - b0;
  *y1 = a1 + b1;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

// The codes of a tile in registers, as of here: otherwise the compiler takes them apart where they are loaded, where that
// waits for the loads and needs four registers for one.
template <typename V, int N>
__device__ __forceinline__ void keep_whole(V (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    if constexpr (sizeof(V) == 4) {
      uint32_t w = x[i][0];
      asm volatile("" : "+v"(w));
      x[i][0] = w;
    } else {
      asm volatile("" : "+v"(x[i]));
    }
  }
}

// the bf16 values of 8 codes
__device__ __forceinline__ bf16x8 bf16_of_codes(uint32_t lo, uint32_t hi) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    f[j] = (float)(int8_t)(lo >> (8 * j));
    f[4 + j] = (float)(int8_t)(hi >> (8 * j));
  }
  u32x4 y;
#pragma unroll
  for (int j = 0; j < 4; j++) y[j] = high16_pair(__float_as_uint(f[2 * j]), __float_as_uint(f[2 * j + 1]));
  return __builtin_bit_cast(bf16x8, y);
}

// LDS: queries as fragments of NT bf16 terms, the block that the new row goes into (keys, values), its scales
template <typename A>
constexpr int q8_fixed_bytes(int hd) {
  return 16 * hd * 2 * (sizeof(A) == 2 ? 2 : 3) + 2 * kBlock * hd + (kWaves * 32 + 4) * 4;
}

// One workgroup: up to 16 query heads of a KV head, one range of a sequence's cached rows; its waves take tiles
// of KT rows in turn. As in the kernel over f32 and bf16 pages: S^T = K Q^T with keys in the rows of a 16x16 MFMA and heads in its
// columns, the weights the B operand of O^T += V^T P^T as they lie. Codes are exact in bf16 and are made bf16 in
// registers; a block's scale is one factor of its 16 scores and of its 16 weights, so the queries (NT
// bf16 terms) and the weights (NT terms) carry all the rounding that there is.
// Of K a lane reads 16 codes of its row, which are the operands of two MFMAs: slots 8 g .. 8 g + 7 of step
// 2 u + p hold the elements 64 u + 16 g + 8 p and on, in the queries too. Of V it reads E = HD / 16 neighbouring
// codes of the rows of its group.
//
// The block that the new row goes into is not walked over: the workgroup of the last range forms it anew in LDS
// (one wave the keys, one the values), writes it back, and one wave attends it from there. No other
// workgroup reads it, so none can see it half written.
template <typename A, int HD, bool PART>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_q8_kernel(PagedAttnArgs a) {
  constexpr int NT = sizeof(A) == 2 ? 2 : 3;
  constexpr int KT = HD == 256 ? 32 : 64, NB = KT / kBlock, STEP = KT * kWaves;
  constexpr int KP = HD / 64, E = HD / 16, VW = E / 4;  // 16-byte pieces of a K row a lane; codes and words of a V row
  constexpr int QS = HD / 32;                           // steps of 32 elements
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const PagesArgs& p = a.p;
  const int hd = p.head_dim, half = hd / 2, group = p.n_q / p.n_kv, htiles = (group + 15) / 16, nh = min(group, 16);
  uint32_t* tail_k = reinterpret_cast<uint32_t*>(sm + 16 * HD * 2 * NT / 4);  // [16][HD] codes
  uint32_t* tail_v = tail_k + kBlock * HD / 4;
  float* wm = reinterpret_cast<float*>(tail_v + kBlock * HD / 4);  // [waves][16]
  float* wl = wm + kWaves * 16;
  float* tail_s = wl + kWaves * 16;  // its scales
  float* wacc = tail_s + 4;          // [waves][heads][HD]; before that cos and sin [2][HD / 2]
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x;
  const int ht = id % htiles;
  id /= htiles;
  const int hkv = id % p.n_kv;
  id /= p.n_kv;
  const int b = id % p.batch, split = id / p.batch;
  const int hq0 = hkv * group + ht * 16, heads = min(group - ht * 16, 16);
  // the query rows, asked for with the length
  constexpr int NE = HD / 32;
  const A* qrow = static_cast<const A*>(p.q) + (int64_t)b * p.q_stride + hq0 * hd;
  A q0[NE], q1[NE];
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = min(tid + n * kThreads, heads * half - 1), hh = i / half, e = i - hh * half;
    q0[n] = qrow[hh * hd + e];
    q1[n] = qrow[hh * hd + e + half];
  }
  // the new row: its keys by wave 0, its values by wave 1
  const bool add = p.k != nullptr;
  constexpr int NP = HD > 128 ? 2 : 1;  // pairs a lane
  A n0[NP], n1[NP];
  if (add && wave < 2) {
    const A* row = wave == 0 ? static_cast<const A*>(p.k) + (int64_t)b * p.k_stride
                             : static_cast<const A*>(p.v) + (int64_t)b * p.v_stride;
#pragma unroll
    for (int n = 0; n < NP; n++) {
      const int e = hkv * hd + min(lane + 64 * n, half - 1);
      n0[n] = row[e];
      n1[n] = row[e + half];
    }
  }
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  // Page numbers: lane t holds that of block t of a tile, so one load brings them all. Those of the wave's first
  // tile are asked for with the length where no window moves it.
  const int r0 = split * a.split_rows, first = r0 + wave * KT, lane_t = min(lane & 7, NB - 1);
  const int last_entry = max((int)p.table_stride - 1, 0);
  const bool moved = a.window != INT32_MAX;
  int pages = -1;
  if (!moved && p.table_stride > 0) pages = trow[min((first + kBlock * lane_t) >> p.page_bits, last_entry)];
  const int len = a.lens[b];
  A* orow = static_cast<A*>(a.out) + (int64_t)b * a.out_stride + hq0 * hd;
  const int64_t rows = (int64_t)len + (add || a.ahead);
  const bool bad = rows > a.max_len || rows > p.table_stride << p.page_bits;
  if (len < 0 || bad || rows == 0) {  // idle slot or nothing to see: zeros; more rows than the call allows: NaN
    if (split == 0)
      for (int i = tid; i < heads * hd; i += kThreads) orow[i] = (A)(bad && len >= 0 ? NAN : 0.0f);
    return;
  }
  const int tail_row = len & ~(kBlock - 1), before = len & (kBlock - 1);  // of the block that the new row goes into
  CachedRows<true> cr;
  cr.init(a, add ? tail_row : (int)rows, rows);
  const int nsplit = ranges_of(cr.walk, a.split_rows);
  if (split >= nsplit) return;
  const bool last = split == nsplit - 1;
  const int r1 = last ? cr.walk : r0 + a.split_rows;
  const int kvd = p.n_kv * hd;
  bool lost = false;  // a page number out of range

  const int in_page = (1 << p.page_bits) - 1;
  auto ask_pages = [&](int r) { pages = trow[min(cr.row(r + kBlock * lane_t) >> p.page_bits, last_entry)]; };
  auto scale_at = [&](int64_t page, int row) -> int64_t {
    return page * a.scale_stride + ((row & in_page) >> 4) * p.n_kv + hkv;
  };
  const int8_t* kb = static_cast<const int8_t*>(p.kpages) + hkv * hd;
  const int8_t* vb = static_cast<const int8_t*>(p.vpages) + hkv * hd;
  typedef uint32_t VRow __attribute__((ext_vector_type(VW)));
  u32x4 xk[NB][KP];
  VRow xv[NB * 4];
  float sc = 0.0f;  // lane t < NB: scale of the keys of block t, lane 8 + t: of its values
  int64_t base[NB];  // rows in the pages, in scalar registers: an address is a scalar and one offset of the lane
  auto set_base = [&](int r) {  // of the tile whose pages are there; blocks past the range's end: the first again
    const int n = min((r1 - r + kBlock - 1) / kBlock, NB);  // blocks of the tile
    lost |= lane_t < n && (uint32_t)pages >= (uint64_t)p.pages;
    if ((uint32_t)pages >= (uint64_t)p.pages) pages = 0;
#pragma unroll
    for (int t = 0; t < NB; t++) {
      const int u = t < n ? t : 0;
      base[t] = ((int64_t)__builtin_amdgcn_readlane(pages, u) << p.page_bits) + (cr.row(r + kBlock * u) & in_page);
    }
  };
  auto load_scales = [&](int r) {
    const int n = min((r1 - r + kBlock - 1) / kBlock, NB);
    const int row = cr.row(r + (lane_t < n ? kBlock * lane_t : 0));
    const int first_page = __builtin_amdgcn_readlane(pages, 0);
    return (lane & 8 ? a.vscales : a.kscales)[scale_at(lane_t < n ? pages : first_page, row)];
  };
  const uint32_t k_off = col * kvd + (PART ? 0 : 16 * g), v_off = 4 * g * kvd;
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < NB; t++) {
      const int8_t* kp = kb + base[t] * kvd;
#pragma unroll
      for (int u = 0; u < KP; u++) {
        if constexpr (PART) {  // (a row's elements end at a multiple of 8; those past it meet zeros of the queries)
          const int d = 64 * u + 16 * g;
          const u32x2 lo = *reinterpret_cast<const u32x2*>(kp + (k_off + min(d, hd - 8)));
          const u32x2 hi = *reinterpret_cast<const u32x2*>(kp + (k_off + min(d + 8, hd - 8)));
          xk[t][u] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
          xk[t][u] = *reinterpret_cast<const u32x4*>(kp + 64 * u + k_off);
        }
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int t = 0; t < NB; t++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int8_t* vp = vb + (base[t] + j) * kvd;
        if constexpr (PART && E > 8) {
          const u32x2 lo = *reinterpret_cast<const u32x2*>(vp + (v_off + min(E * col, hd - 8)));
          const u32x2 hi = *reinterpret_cast<const u32x2*>(vp + (v_off + min(E * col + 8, hd - 8)));
          xv[4 * t + j][0] = lo[0], xv[4 * t + j][1] = lo[1];
          xv[4 * t + j][VW - 2] = hi[0], xv[4 * t + j][VW - 1] = hi[1];
        } else {  // (elements past the head's end form rows that nobody stores)
          xv[4 * t + j] = *reinterpret_cast<const VRow*>(vp + (v_off + (PART ? min(E * col, hd - E) : E * col)));
        }
      }
  };
  // the new row's block, from LDS, as block 0 of a tile
  auto take_tail_k = [&]() {
#pragma unroll
    for (int u = 0; u < KP; u++)
      xk[0][u] = *reinterpret_cast<const u32x4*>(tail_k + (col * HD + 64 * u + 16 * g) / 4);
    sc = tail_s[lane & 8 ? 1 : 0];
  };
  auto take_tail_v = [&]() {
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int w = 0; w < VW; w++) xv[j][w] = tail_v[((4 * g + j) * HD + E * col) / 4 + w];
  };
  if (first < r1) {
    if (moved) ask_pages(first);
    set_base(first);
    load_k();
    sc = load_scales(first);
    load_v();
    ask_pages(first + STEP);
  }

  // the rotated queries as operands (zeros for heads and elements past the end)
  float* cs = wacc;
  if (p.rope && tid < half) rope_angle(len, tid, hd, p.log2_theta, cs + tid, cs + HD / 2 + tid);
  for (int i = tid; i < 16 * HD * 2 * NT / 16; i += kThreads) reinterpret_cast<u32x4*>(sm)[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
  auto put_query = [&](int hh, int e, float x) {
    __bf16 t[NT];
    split_terms<NT>(x, t);
    __bf16* at = reinterpret_cast<__bf16*>(sm) +
                 ((2 * (e >> 6) + ((e >> 3) & 1)) * 64 + ((e >> 4) & 3) * 16 + hh) * 8 + (e & 7);
#pragma unroll
    for (int n = 0; n < NT; n++) at[n * 16 * HD] = t[n];
  };
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = tid + n * kThreads, hh = i / half, e = i - hh * half;
    if (i < heads * half) {
      float y0 = (float)q0[n], y1 = (float)q1[n];
      if (p.rope) rotate(y0, y1, cs[e], cs[HD / 2 + e], &y0, &y1);
      put_query(hh, e, y0);
      put_query(hh, e + half, y1);
    }
  }
  if (add && last && wave < 2) {  // the new row's block
    const int page = trow[tail_row >> p.page_bits];
    const bool store = (uint32_t)page < (uint64_t)p.pages;
    lost |= !store;
    const int64_t at = ((int64_t)(store ? page : 0) << p.page_bits) + (tail_row & in_page);
    int8_t* codes = static_cast<int8_t*>(wave == 0 ? p.kpages : p.vpages) + at * kvd + hkv * hd;
    float* scale = (wave == 0 ? a.kscales : a.vscales) + scale_at(store ? page : 0, tail_row);
    uint32_t* tail = wave == 0 ? tail_k : tail_v;
    const int words = hd / 4;
    uint32_t w[HD / 16];
#pragma unroll
    for (int n = 0; n < HD / 16; n++) {
      const int i = lane + 64 * n, r = i / words, c = i - r * words;
      w[n] = r < before ? *reinterpret_cast<const uint32_t*>(codes + (int64_t)r * kvd + 4 * c) : 0;
    }
    const float s0 = before > 0 ? *scale : 0.0f;
    float y0[NP], y1[NP], amax = 0.0f;
    bool good = true;
#pragma unroll
    for (int n = 0; n < NP; n++) {
      const int e = min(lane + 64 * n, half - 1);
      y0[n] = (float)n0[n], y1[n] = (float)n1[n];
      if (wave == 0 && p.rope) rotate(y0[n], y1[n], cs[e], cs[HD / 2 + e], &y0[n], &y1[n]);
      amax = fmaxf(amax, fmaxf(fabsf(y0[n]), fabsf(y1[n])));
      good = good && finite(y0[n]) && finite(y1[n]);
    }
    const float s = raised(wave_max(amax), __all(good), s0);
    const bool anew = s > s0;
    const float ratio = anew ? __fdiv_rn(s0, s) : 1.0f;
#pragma unroll
    for (int n = 0; n < HD / 16; n++) {
      const int i = lane + 64 * n, r = i / words, c = i - r * words;
      if (r < before) {
        const uint32_t y = anew ? recoded(w[n], ratio) : w[n];
        tail[(r * HD >> 2) + c] = y;
        if (anew && store) *reinterpret_cast<uint32_t*>(codes + (int64_t)r * kvd + 4 * c) = y;
      }
    }
#pragma unroll
    for (int n = 0; n < NP; n++) {
      const int e = lane + 64 * n;
      if (e < half) {
        const int8_t c0 = (int8_t)code_of(y0[n], s), c1 = (int8_t)code_of(y1[n], s);
        int8_t* t = reinterpret_cast<int8_t*>(tail) + before * HD + e;
        t[0] = c0;
        t[half] = c1;
        if (store) {
          codes[(int64_t)before * kvd + e] = c0;
          codes[(int64_t)before * kvd + e + half] = c1;
        }
      }
    }
    if (lane == 0) {
      tail_s[wave] = s;
      if (store) *scale = s;
    }
  }
  __syncthreads();

  f32x4 acc[E];
#pragma unroll
  for (int t = 0; t < E; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  // the wave's tiles, at the end the new row's block by the wave whose turn it is
  int r = first;
  const bool has_tail = add && last && wave == ((r1 - r0 + KT - 1) / KT) % kWaves;
  bool tail = first >= r1;
  if (tail && has_tail) {
    take_tail_k();
    take_tail_v();
  }
  for (bool go = !tail || has_tail; go;) {
    const bool more = !tail && r + STEP < r1, then_tail = !tail && !more && has_tail;
    // rows of block t count that are row at[t] of the sequence and on, before `end`, and seen
    const int end = tail ? len + 1 : cr.row(r1 - 1) + 1;
    int at[NB];
    float ks[NB], vs[NB];
#pragma unroll
    for (int t = 0; t < NB; t++) {
      at[t] = tail ? (t == 0 ? tail_row : INT32_MAX - kBlock)
                   : r + kBlock * t < r1 ? cr.row(r + kBlock * t) : INT32_MAX - kBlock;
      ks[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc), t));
      vs[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc), 8 + t));
    }
    if (more) set_base(r + STEP);
#pragma unroll
    for (int t = 0; t < NB; t++) keep_whole(xk[t]);
    f32x4 d[NB] = {};
    int ql = lane;  // read anew for every tile: kept in registers they would cost a wave a SIMD
    asm volatile("" : "+v"(ql));
    const u32x4* qp = reinterpret_cast<const u32x4*>(sm) + ql;
#pragma unroll
    for (int u = 0; u < KP; u++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        u32x4 qw[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) qw[n] = qp[(n * QS + 2 * u + h) * 64];
        bf16x8 kf[NB];
#pragma unroll
        for (int t = 0; t < NB; t++) kf[t] = bf16_of_codes(xk[t][u][2 * h], xk[t][u][2 * h + 1]);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int t = 0; t < NB; t++)
            d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t], __builtin_bit_cast(bf16x8, qw[n]), d[t], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);  // (left alone, the conversions of all steps come first and do not fit)
      }
    if (more) {
      load_k();
      sc = load_scales(r + STEP);
      ask_pages(r + 2 * STEP);
    } else if (then_tail) {
      take_tail_k();
    }
    float s[NB][4];
    uint32_t hidden[NB];  // bit i: row 4 g + i of the block
    bool cut = false;
#pragma unroll
    for (int t = 0; t < NB; t++) {
      const float f = ks[t] * a.scale2;
      const bool c = at[t] + kBlock > end || !cr.sees_block(at[t]);
      cut = cut || c;
#pragma unroll
      for (int i = 0; i < 4; i++) s[t][i] = d[t][i] * f;
      hidden[t] = 0;
      if (c)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int row = at[t] + 4 * g + i;
          if (row >= end || !cr.sees(row)) {
            s[t][i] = -INFINITY;
            hidden[t] |= 1u << i;
          }
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < NB; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < NB; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
        l += s[t][i];
      }
#pragma unroll
    for (int t = 0; t < E; t++) acc[t] *= alpha;
    keep_whole(xv);
#pragma unroll
    for (int t = 0; t < NB; t += 2) {  // 32 rows a product
      bf16x8 pb[NT];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int u = t + (j >> 2);
        float w = s[u][j & 3] * vs[u];
        if (cut && (hidden[u] >> (j & 3) & 1)) w = 0.0f;  // what is not seen may have any scale
        __bf16 x[NT];
        split_terms<NT>(w, x);
#pragma unroll
        for (int n = 0; n < NT; n++) pb[n][j] = x[n];
      }
#pragma unroll
      for (int e = 0; e < E; e += 4) {  // four elements, one word of the rows
        bf16x8 vf[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; j++) f[j] = (float)(int8_t)(xv[4 * t + j][e >> 2] >> (8 * i));
          u32x4 y;
#pragma unroll
          for (int j = 0; j < 4; j++) y[j] = high16_pair(__float_as_uint(f[2 * j]), __float_as_uint(f[2 * j + 1]));
          vf[i] = __builtin_bit_cast(bf16x8, y);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            acc[e + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], pb[n], acc[e + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more)
      load_v();
    else if (then_tail)
      take_tail_v();
    go = more || then_tail;
    tail = then_tail;
    r += STEP;
  }

  // the waves' states
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
  const bool any_lost = __syncthreads_or(lost);
  for (int i = tid; i < heads * hd; i += kThreads) {
    const int hh = i / hd, d = i - hh * hd;
    float mx = wm[hh];
#pragma unroll
    for (int w = 1; w < kWaves; w++) mx = fmaxf(mx, wm[w * 16 + hh]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float o = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float f = __builtin_amdgcn_exp2f(wm[w * 16 + hh] - ref);
      sum += f * wl[w * 16 + hh];
      o += f * wacc[(w * nh + hh) * HD + d];
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

// RoPE and append of packed rows, a workgroup the rows of one block and some of the heads, a wave a head at a time:
// its rows stay in registers between their maximum and their codes.
// Without cu row b is the one row of sequence b, at position past[b].
template <typename A, int HD>
__global__ __launch_bounds__(kThreads) void pages_append_q8_kernel(PagesAppendArgs a, int chunks) {
  const PagesArgs& p = a.p;
  __shared__ float cs[2][kBlock][HD / 2];
  const int tid = threadIdx.x, lane = tid & 63, hd = p.head_dim, half = hd / 2;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunk = blockIdx.x % chunks;
  const int64_t slot = blockIdx.x / chunks;
  // Sequence b takes the slots floor(cu[b] / 16) + 2 b and on, at least as many as it has blocks
  int b = (int)slot;
  int64_t c0 = slot, n = 1, nth = 0;
  if (a.cu != nullptr) {
    b = count_first(p.batch, [&](int i) { return clamp_cu(a.cu, i, a.rows) / kBlock + 2 * (int64_t)i <= slot; }) - 1;
    if (b < 0) return;
    c0 = clamp_cu(a.cu, b, a.rows);
    n = clamp_cu(a.cu, b + 1, a.rows) - c0;
    nth = slot - (c0 / kBlock + 2 * (int64_t)b);
  }
  const int64_t past = a.past[b];
  if (past < 0 || nth < 0) return;
  const int64_t block = past / kBlock + nth, pos0 = max(past, block * kBlock), pos1 = min(past + n, (block + 1) * kBlock);
  if (pos0 >= pos1) return;
  const int rows = (int)(pos1 - pos0), before = (int)(pos0 - block * kBlock);
  const int64_t row0 = c0 + pos0 - past;  // packed row of the first
  const bool inside = pos0 < p.table_stride << p.page_bits && (a.max_len == 0 || pos1 <= a.max_len);
  const int page = inside ? p.table[(int64_t)b * p.table_stride + (pos0 >> p.page_bits)] : -1;
  const bool ok = (uint32_t)page < (uint64_t)p.pages;
  const int in_page = (int)(block * kBlock & ((1 << p.page_bits) - 1));
  const int64_t at = ok ? ((int64_t)page << p.page_bits) + in_page : 0;  // of the block's first row
  if (p.rope) {
    for (int i = tid; i < rows * half; i += kThreads) {
      const int r = i / half, e = i - r * half;
      rope_angle(pos0 + r, e, hd, p.log2_theta, &cs[0][r][e], &cs[1][r][e]);
    }
    __syncthreads();
  }
  typedef A A4 __attribute__((ext_vector_type(4)));
  constexpr int N = kBlock * HD / 8 / 64;  // groups of 4 pairs a lane
  const int hp = half / 4, kvd = p.n_kv * hd, tasks = p.n_q + 2 * p.n_kv;
  for (int task = chunk * kWaves + wave; task < tasks; task += chunks * kWaves) {
    const int what = task < p.n_q ? 0 : task < p.n_q + p.n_kv ? 1 : 2;  // q, k, v
    const int head = what == 0 ? task : what == 1 ? task - p.n_q : task - p.n_q - p.n_kv;
    if (what == 0 && a.q_out == nullptr) continue;
    const A* x = static_cast<const A*>(what == 0 ? p.q : what == 1 ? p.k : p.v) + head * hd;
    const int64_t xs = what == 0 ? p.q_stride : what == 1 ? p.k_stride : p.v_stride;
    A* out = what == 2 ? nullptr : static_cast<A*>(what == 0 ? a.q_out : a.k_out);
    const int64_t os = what == 0 ? a.q_out_stride : a.k_out_stride;
    A4 x0[N], x1[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = 4 * (i - r * hp);
      if (r < rows) {
        x0[k] = *reinterpret_cast<const A4*>(x + (row0 + r) * xs + e);
        x1[k] = *reinterpret_cast<const A4*>(x + (row0 + r) * xs + e + half);
      }
    }
    float y0[N][4], y1[N][4], amax = 0.0f;
    bool good = true;
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = 4 * (i - r * hp);
      if (r >= rows) continue;
      A4 z0, z1;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        y0[k][j] = (float)x0[k][j], y1[k][j] = (float)x1[k][j];
        if (what < 2 && p.rope) rotate(y0[k][j], y1[k][j], cs[0][r][e + j], cs[1][r][e + j], &y0[k][j], &y1[k][j]);
        amax = fmaxf(amax, fmaxf(fabsf(y0[k][j]), fabsf(y1[k][j])));
        good = good && finite(y0[k][j]) && finite(y1[k][j]);
        z0[j] = (A)(ok ? y0[k][j] : NAN);  // no page for the row: its outputs say so
        z1[j] = (A)(ok ? y1[k][j] : NAN);
      }
      if (out != nullptr) {
        A* o = out + (row0 + r) * os + head * hd + e;
        *reinterpret_cast<A4*>(o) = z0;
        *reinterpret_cast<A4*>(o + half) = z1;
      }
    }
    if (what == 0 || !ok) continue;
    int8_t* codes = static_cast<int8_t*>(what == 1 ? p.kpages : p.vpages) + at * kvd + head * hd;
    float* scale = (what == 1 ? a.kscales : a.vscales) + page * a.scale_stride + (in_page >> 4) * p.n_kv + head;
    const float s0 = before > 0 ? *scale : 0.0f;
    const float s = raised(wave_max(amax), __all(good), s0);
    if (s > s0 && before > 0) {
      const float ratio = __fdiv_rn(s0, s);
      for (int i = lane; i < before * (hd / 4); i += 64) {
        const int r = i / (hd / 4);
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + (int64_t)r * kvd + 4 * (i - r * (hd / 4)));
        *w = recoded(*w, ratio);
      }
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = 4 * (i - r * hp);
      if (r >= rows) continue;
      int d0[4], d1[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        d0[j] = code_of(y0[k][j], s);
        d1[j] = code_of(y1[k][j], s);
      }
      int8_t* o = codes + (int64_t)(before + r) * kvd + e;
      *reinterpret_cast<uint32_t*>(o) = pack4(d0);
      *reinterpret_cast<uint32_t*>(o + half) = pack4(d1);
    }
    if (lane == 0) *scale = s;
  }
}

}  // namespace

namespace {

template <typename A, int HD, bool PART>
hipError_t run_paged_q8(const PagedAttnArgs& a, hipStream_t stream) {
  const PagesArgs& p = a.p;
  const int64_t htiles = (p.n_q / p.n_kv + 15) / 16;
  constexpr int kMaxLds = q8_fixed_bytes<A>(HD) + kWaves * 16 * HD * 4;
  const int lds = q8_fixed_bytes<A>(HD) + kWaves * std::min(p.n_q / p.n_kv, 16) * HD * 4;
  const auto kernel = paged_attention_q8_kernel<A, HD, PART>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), kMaxLds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.nsplit * p.batch * p.n_kv * htiles)), dim3(kThreads), lds, stream, a);
  return hipGetLastError();
}

template <typename A>
hipError_t run_paged_q8_hd(const PagedAttnArgs& a, hipStream_t stream) {
  const int hd = a.p.head_dim;
  if (hd == 64) return run_paged_q8<A, 64, false>(a, stream);
  if (hd == 128) return run_paged_q8<A, 128, false>(a, stream);
  if (hd == 256) return run_paged_q8<A, 256, false>(a, stream);
  if (hd < 64) return run_paged_q8<A, 64, true>(a, stream);
  if (hd < 128) return run_paged_q8<A, 128, true>(a, stream);
  return run_paged_q8<A, 256, true>(a, stream);
}

template <typename A, int HD>
hipError_t run_append_q8(const PagesAppendArgs& a, hipStream_t stream) {
  // A wave takes one head of a small call, more of a large one, so that the angles are formed less often
  const int64_t slots = append_q8_slots(a), tasks = a.p.n_q + 2 * a.p.n_kv;
  const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((tasks + kWaves - 1) / kWaves, (2048 + slots - 1) / slots));
  hipLaunchKernelGGL((pages_append_q8_kernel<A, HD>), dim3((unsigned)(slots * chunks)), dim3(kThreads), 0, stream, a,
                     (int)chunks);
  return hipGetLastError();
}

template <typename A>
hipError_t run_append_q8_hd(const PagesAppendArgs& a, hipStream_t stream) {
  if (a.p.head_dim <= 64) return run_append_q8<A, 64>(a, stream);
  if (a.p.head_dim <= 128) return run_append_q8<A, 128>(a, stream);
  return run_append_q8<A, 256>(a, stream);
}

// The stored rows of sequences, packed: a workgroup ROWS of them, whose places in the pages are looked up first.
// C: the pages' type (int8: codes times the block's scale), T: the rows'.
template <typename C, typename T, int ROWS>
__global__ __launch_bounds__(256) void pages_rows_kernel(PagesRowsArgs a) {
  const PagesArgs& p = a.p;
  __shared__ int64_t src[ROWS];  // row in the pages, -1: its page is missing, -2: a row of no sequence
  const int tid = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  if (tid < ROWS) {
    const int64_t row = row0 + tid;
    int64_t at = -2;
    if (row < a.rows && row >= a.cu[0] && row < a.cu[p.batch]) {
      int lo = 0, hi = p.batch;  // the last sequence that starts at or before the row
      while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (a.cu[mid] <= row)
          lo = mid;
        else
          hi = mid;
      }
      const int64_t pos = row - a.cu[lo];
      const bool inside = pos < p.table_stride << p.page_bits;
      const int page = inside ? p.table[(int64_t)lo * p.table_stride + (pos >> p.page_bits)] : -1;
      at = (uint32_t)page < (uint64_t)p.pages ? ((int64_t)page << p.page_bits) + (pos & ((1 << p.page_bits) - 1)) : -1;
    }
    src[tid] = at;
  }
  __syncthreads();
  typedef C C8 __attribute__((ext_vector_type(8)));
  typedef T T8 __attribute__((ext_vector_type(8)));
  const int hd = p.head_dim, kvd = p.n_kv * hd, per = kvd / 8;
  for (int i = tid; i < 2 * ROWS * per; i += 256) {
    const int r = i / (2 * per), j = i - r * 2 * per, e = 8 * (j >= per ? j - per : j);
    const bool is_v = j >= per;
    const int64_t at = src[r];
    if (at == -2) continue;
    T8 y;
    if (at < 0) {
#pragma unroll
      for (int n = 0; n < 8; n++) y[n] = (T)NAN;
    } else {
      const C8 x = *reinterpret_cast<const C8*>(static_cast<const C*>(is_v ? p.vpages : p.kpages) + at * kvd + e);
      float s = 1.0f;
      if constexpr (sizeof(C) == 1)
        s = (is_v ? a.vscales : a.kscales)[(at >> p.page_bits) * a.scale_stride +
                                           ((at & ((1 << p.page_bits) - 1)) >> 4) * p.n_kv + e / hd];
#pragma unroll
      for (int n = 0; n < 8; n++) {
        if constexpr (sizeof(C) == 1)
          y[n] = (T)((float)x[n] * s);
        else
          y[n] = (T)(float)x[n];
      }
    }
    T* out = static_cast<T*>(is_v ? a.v_out : a.k_out) + (row0 + r) * (is_v ? a.v_out_stride : a.k_out_stride) + e;
    *reinterpret_cast<T8*>(out) = y;
  }
}

template <typename C, typename T>
hipError_t run_rows(const PagesRowsArgs& a, hipStream_t stream) {
  constexpr int kRows = 4;
  hipLaunchKernelGGL((pages_rows_kernel<C, T, kRows>), dim3((unsigned)((a.rows + kRows - 1) / kRows)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t append_q8_slots(const PagesAppendArgs& a) {
  return a.cu ? a.rows / kBlock + 2 * (int64_t)a.p.batch : a.p.batch;
}

hipError_t launch_paged_attention_q8(int dtype, const PagedAttnArgs& a, hipStream_t stream) {
  const PagesArgs& p = a.p;
  PagedAttnArgs r = a;
  if (p.k != nullptr && p.n_q / p.n_kv > 16) {
    // Several workgroups a KV head would read the block that one of them rewrites: the row is appended first
    PagesAppendArgs n = {};
    n.p = p;
    n.past = a.lens;
    n.rows = p.batch;
    n.max_len = a.max_len;
    n.kscales = a.kscales, n.vscales = a.vscales, n.scale_stride = a.scale_stride;
    if (hipError_t e = launch_pages_append_q8(dtype, n, stream)) return e;
    r.p.k = r.p.v = nullptr;
    r.ahead = 1;
  }
  if (r.window == 0) r.window = INT32_MAX;
  if (hipError_t e = dtype == RQ_F32 ? run_paged_q8_hd<float>(r, stream) : run_paged_q8_hd<__bf16>(r, stream)) return e;
  return r.nsplit > 1 ? launch_paged_merge(dtype, r, stream) : hipSuccess;
}

hipError_t launch_pages_append_q8(int dtype, const PagesAppendArgs& a, hipStream_t stream) {
  return dtype == RQ_F32 ? run_append_q8_hd<float>(a, stream) : run_append_q8_hd<__bf16>(a, stream);
}

hipError_t launch_pages_rows(int dtype, int cache_dtype, const PagesRowsArgs& a, hipStream_t stream) {
  if (cache_dtype == RQ_I8)
    return dtype == RQ_F32 ? run_rows<int8_t, float>(a, stream) : run_rows<int8_t, __bf16>(a, stream);
  if (cache_dtype == RQ_BF16)
    return dtype == RQ_F32 ? run_rows<__bf16, float>(a, stream) : run_rows<__bf16, __bf16>(a, stream);
  return dtype == RQ_F32 ? run_rows<float, float>(a, stream) : run_rows<float, __bf16>(a, stream);
}

}  // namespace rq
