// paged_tile.h — device code that the kernels on a paged cache share (paged.hip, paged_q8.hip).
#pragma once

#include "paged.h"

namespace rq {

constexpr int kRec = 4;  // floats before the values of a range's record: maximum, sum

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

// Ranges of a sequence of len cached rows: the last may hold one row more, which is the
// new row's place in a cache that is full with it
__host__ __device__ __forceinline__ int64_t ranges_of(int64_t len, int64_t rows) {
  return len > rows + 1 ? (len - 1 + rows - 1) / rows : 1;
}

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

// The cached rows that a sequence's query walks over: those that it sees, by whole blocks of 16. In their order
// they are `walk` rows, of which row r is row(r) of the sequence. WIN: with a window, in which rows before `lo` are
// seen only as sinks.
template <bool WIN>
struct CachedRows {
  int walk, lo, sinks, sink_end, skip;
  // cached: rows to walk over in all, rows: those that there are, the new one included (the query's is the last)
  __device__ __forceinline__ void init(const PagedAttnArgs& a, int cached, int64_t rows) {
    walk = cached;
    if constexpr (WIN) {
      sinks = a.sinks;
      lo = (int)(rows > a.window ? rows - a.window : 0);
      sink_end = (sinks + 15) & ~15;
      skip = max(min(lo & ~15, cached) - sink_end, 0);
      walk -= skip;
    }
  }
  __device__ __forceinline__ int row(int r) const { return WIN && r >= sink_end ? r + skip : r; }
  // whether the query sees row `row` of the sequence; whether it sees all of the 16 from `row` on
  __device__ __forceinline__ bool sees(int row) const { return !WIN || row >= lo || row < sinks; }
  __device__ __forceinline__ bool sees_block(int row) const { return !WIN || row >= lo || row + 16 <= sinks; }
};

}  // namespace rq
