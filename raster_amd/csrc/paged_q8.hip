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
#include <type_traits>

#include "attn_tile.h"
#include "paged_tile.h"

namespace rq {

namespace {

constexpr int kBlock = 16;
constexpr int kThreads = 256, kWaves = 4, kTileRows = 64;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

// max |x| of the new rows and the old scale (0: none) to the new scale
__device__ __forceinline__ float raised(float amax, bool all_finite, float s0) {
  const float s = fmaxf(s0, amax * (1.0f / 127.0f));
  return all_finite && finite(s0) ? s : NAN;
}
__device__ __forceinline__ int code_of(float x, float s) {
  return s > 0.0f ? (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.0f), 127.0f) : 0;
}
__device__ __forceinline__ uint32_t pack4(const int (&c)[4]) {
  return (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 | (uint32_t)(c[3] & 255) << 24;
}
// four of them; inv: 1 / s. x inv is off by at most 2.3e-5 from the rounded x / s (127 times 3 roundings), so where
// it is further from a half than that it rounds alike: a third of the instructions of the divisions. (Not for tiny s,
// whose inverse and quotients have fewer bits.)
__device__ __forceinline__ uint32_t codes_of(const float* x, float s, float inv) {
  int c[4];
  float q[4], far = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    q[j] = x[j] * inv;
    const float r = rintf(q[j]);
    far = fmaxf(far, fabsf(q[j] - r));
    c[j] = (int)r;
  }
  if (!(s >= 1e-30f && far <= 0.49997f))
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = code_of(x[j], s);
  return pack4(c);
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
// x0, x1 rotated: every operation rounded by itself
__device__ __forceinline__ void rotate(float x0, float x1, float c, float s, float* y0, float* y1) {
#pragma clang fp contract(off)
  const float a0 = x0 * c, b0 = x1 * s, a1 = x1 * c, b1 = x0 * s;
  *y0 = a0 - b0;
  *y1 = a1 + b1;
}

// The angle of pair i in turns for one position; cos and sin of `turns`. Whole turns are taken off in 64 bits, then
// quarters, and |x| <= pi / 4 is left for Taylor's series to x^15 and x^16 (2^-54): a fifth of the instructions of a
// general sincospi.
__device__ __forceinline__ double turns_of(int i, int head_dim, double log2_theta) {
  return exp2(-2.0 * (double)i / (double)head_dim * log2_theta) * 0.15915494309189535;
}
__device__ __forceinline__ void cos_sin_turns(double turns, float* c, float* s) {
  turns -= rint(turns);
  const double quarter = rint(4.0 * turns), x = (turns - 0.25 * quarter) * 6.283185307179586, z = x * x;
  double sn = -1.0 / 1307674368000.0, cn = 1.0 / 20922789888000.0;
  sn = fma(sn, z, 1.0 / 6227020800.0);
  cn = fma(cn, z, -1.0 / 87178291200.0);
  sn = fma(sn, z, -1.0 / 39916800.0);
  cn = fma(cn, z, 1.0 / 479001600.0);
  sn = fma(sn, z, 1.0 / 362880.0);
  cn = fma(cn, z, -1.0 / 3628800.0);
  sn = fma(sn, z, -1.0 / 5040.0);
  cn = fma(cn, z, 1.0 / 40320.0);
  sn = fma(sn, z, 1.0 / 120.0);
  cn = fma(cn, z, -1.0 / 720.0);
  sn = fma(sn, z, -1.0 / 6.0);
  cn = fma(cn, z, 1.0 / 24.0);
  sn = fma(sn * z, x, x);
  cn = fma(fma(cn, z, -0.5), z, 1.0);
  const int q = (int)quarter;
  const double sv = q & 1 ? cn : sn, cv = q & 1 ? sn : cn;
  *s = (float)(q & 2 ? -sv : sv);
  *c = (float)((q + 1) & 2 ? -cv : cv);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The codes of a tile in registers, as of here: otherwise the compiler takes them apart where they are loaded, where
// that waits for the loads and needs several registers for one.
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

// A number in NT signed digits of 8 bits, as an operand of the int8 products beside the codes: x = sum_n digit n *
// 256^n, for |x| up to kDigitsMax<NT>. Queries are written so relative to a head's largest element, weights relative
// to their tile's largest, so f32 calls lose 2^-24 of that (NT = 3), bf16 ones 2^-16 (NT = 2); sums over products are
// exact.
template <typename A>
constexpr int kDigits = sizeof(A) == 2 ? 2 : 3;
template <int NT>
constexpr int kDigitsMax = NT == 2 ? 0x7F7E : 0x7F7F7C;
// the digits in the bytes of a word, from byte 0 on
template <int NT>
__device__ __forceinline__ uint32_t digits_of(int x) {
  constexpr uint32_t kBias = NT == 2 ? 0x8080u : 0x808080u;
  return ((uint32_t)x + kBias) ^ kBias;
}
// Digit n of four such words to word n
template <int NT>
__device__ __forceinline__ void pack_digits(const uint32_t (&x)[4], uint32_t (&d)[NT]) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400);
  d[0] = low16_pair(a, b);
  d[1] = high16_pair(a, b);
  if constexpr (NT == 3)
    d[2] = low16_pair(__builtin_amdgcn_perm(x[1], x[0], 0x07030602), __builtin_amdgcn_perm(x[3], x[2], 0x07030602));
}
// Byte n of four such words as a word, n the lane's: pick = n | (n + 4) << 8
__device__ __forceinline__ uint32_t pack_digit(const uint32_t (&x)[4], uint32_t pick) {
  return low16_pair(__builtin_amdgcn_perm(x[1], x[0], pick), __builtin_amdgcn_perm(x[3], x[2], pick));
}
// Sums over the columns that hold the digits of one number (8 or 4 apart), in each of them, the same bits in all:
// column c takes column c + 8 first, and of the two sums that there are then each column adds one to the other. (They
// have to be the same: a weight's digits are taken in different columns, each from its own copy.)
template <int APART>
__device__ __forceinline__ float sum_digits(float x) {
#pragma clang fp contract(off)  // (x is a product; fused into the sum it would differ from column to column)
  auto turned = [](float y, auto by) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x120 + decltype(by)::value, 0xf, 0xf, true));
  };
  x += turned(x, std::integral_constant<int, 8>{});
  if constexpr (APART == 4) x += turned(x, std::integral_constant<int, 4>{});
  return x;
}
// Sum of digit products to their value
__device__ __forceinline__ float value_of(int d0, int d1) { return (float)((d1 << 8) + d0); }
__device__ __forceinline__ float value_of(int d0, int d1, int d2) {
  return fmaf((float)((d2 << 8) + d1), 256.0f, (float)d0);
}
// The factor that takes numbers up to `most` to digits. (By the hardware's reciprocal, to one unit in the last place: an
// inverse of the same kind takes them back. The largest digit has room for it.) Up to 2^126, whose inverse is the
// smallest that the hardware forms: numbers below 1e-31 get fewer digits. Of numbers past 2^126 it forms none, so of a
// sixteenth of them; those powers of two change no other bit.
template <int NT>
__device__ __forceinline__ float digit_factor(float most) {
  return most > 0.0f ? fminf((float)kDigitsMax<NT> * 0.0625f * __builtin_amdgcn_rcpf(most * 0.0625f), 0x1p126f) : 0.0f;
}

// Ranges of rows, by the real lengths. Sequence b's walked rows are cut into ranges of R rows, one at least, and the
// ranges of all sequences numbered in order: R so that there are no more than a sequence each and `spare` more. So the
// grid needs no lengths, few of its workgroups find nothing to do, and those of a batch have about equally much. A
// single sequence's R is the call's, so that nothing waits for its length.
struct Range {
  // sequence, which of its ranges, how many (0: not known yet) and the number of the first; R
  int b, at, count, first, rows;
};
__device__ __forceinline__ int ranges_of_walk(int walk, int rows) {
  return max(1, (int)((uint32_t)(walk + rows - 1) / (uint32_t)rows));
}
// walked rows of a sequence: those of the new row's block are not among them
__device__ __forceinline__ int walked_of(const PagedAttnArgs& a, int len) {
  const bool add = a.p.k != nullptr;
  const int64_t rows = (int64_t)len + (add || a.ahead);
  if (len < 0 || rows > a.max_len || rows > a.p.table_stride << a.p.page_bits) return 0;
  CachedRows<true> cr;
  cr.init(a, add ? len & ~(kBlock - 1) : (int)rows, rows);
  return cr.walk;
}
// sums over the lanes up to each one
__device__ __forceinline__ uint32_t scan_lanes(uint32_t x) {
#define RQ_SCAN_STEP(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
  RQ_SCAN_STEP(0x111, 0xf);  // within 16 lanes: 1, 2, 4 and 8 before
  RQ_SCAN_STEP(0x112, 0xf);
  RQ_SCAN_STEP(0x114, 0xf);
  RQ_SCAN_STEP(0x118, 0xf);
  RQ_SCAN_STEP(0x142, 0xa);  // the last lane of the 16 before
  RQ_SCAN_STEP(0x143, 0xc);  // and of the 32 before
#undef RQ_SCAN_STEP
  return x;
}
// R of a call with `blocks` blocks of walked rows (at most 2^26 a sequence): R spare >= all rows, a multiple of
// split_rows
__device__ __forceinline__ int rows_a_range(const PagedAttnArgs& a, uint64_t blocks) {
  const int shift = blocks >> 32 ? 8 : 0;
  const uint64_t least = ((uint64_t)((uint32_t)(blocks >> shift) / (uint32_t)a.spare) + 1) << shift;
  const uint32_t unit = a.split_rows / kBlock;
  // (a scalar: the compiler divides in vector registers, and everything that follows from it would stay there)
  return __builtin_amdgcn_readfirstlane((int)(((uint32_t)min(least, (uint64_t)1 << 26) + unit - 1) / unit * unit * kBlock));
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }

// By a whole workgroup: the range of number `number`, or the first of sequence -1 - number. b = -1: there is none. Up
// to 64 sequences each wave looks by itself, a lane a sequence; more are planned by all threads (300 sequences of 1
// to 1000 rows in ranges by waves alone 150 us, so 125).
constexpr int kEach = 4, kPlanned = kThreads * kEach;  // sequences of a thread, of a launch
__device__ __forceinline__ Range range_of(const PagedAttnArgs& a, int number) {
  if (a.spare == 0) return {number < 0 ? -1 - number : number, 0, 1, number < 0 ? -1 - number : number, INT32_MAX};
  if (a.range_rows > 0) return {0, max(number, 0), 0, 0, a.range_rows};
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, batch = a.p.batch;
  if (batch <= 64) {
    const int walk = lane < batch ? walked_of(a, a.lens[lane]) : 0;
    const uint32_t sum = (uint32_t)(walk + kBlock - 1) / kBlock;
    const uint64_t blocks = ((uint64_t)last_lane(scan_lanes(sum >> 16)) << 16) + last_lane(scan_lanes(sum & 0xffff));
    const int rows = rows_a_range(a, blocks), n = lane < batch ? ranges_of_walk(walk, rows) : 0;
    const int first = (int)scan_lanes(n) - n;
    const bool mine = number < 0 ? lane == -1 - number : number >= first && number < first + n;
    const uint64_t found = __builtin_amdgcn_ballot_w64(mine);
    if (found == 0) return {-1, 0, 0, 0, rows};
    const int b = __builtin_ctzll(found), f = __builtin_amdgcn_readlane(first, b);
    return {b, number < 0 ? 0 : number - f, __builtin_amdgcn_readlane(n, b), f, rows};
  }
  __shared__ uint32_t high[kWaves], low[kWaves], count[kWaves];
  __shared__ int found[3];
  int walk[kEach], n[kEach], mine = 0;
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; i++) walk[i] = a.lens[min(tid * kEach + i, batch - 1)];
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    walk[i] = tid * kEach + i < batch ? walked_of(a, walk[i]) : 0;
    sum += (uint32_t)(walk[i] + kBlock - 1) / kBlock;
  }
  const uint32_t h = scan_lanes(sum >> 16), l = scan_lanes(sum & 0xffff);
  if (lane == 63) high[wave] = h, low[wave] = l;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  uint64_t blocks = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) blocks += ((uint64_t)high[w] << 16) + low[w];
  const int rows = rows_a_range(a, blocks);
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    n[i] = tid * kEach + i < batch ? ranges_of_walk(walk[i], rows) : 0;
    mine += n[i];
  }
  const uint32_t upto = scan_lanes(mine);
  if (lane == 63) count[wave] = upto;
  __syncthreads();
  int first = (int)upto - mine;
  for (int w = 0; w < wave; w++) first += count[w];
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const int b = tid * kEach + i;
    if (b < batch && (number < 0 ? b == -1 - number : number >= first && number < first + n[i]))
      found[0] = b, found[1] = first, found[2] = n[i];
    first += n[i];
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(found[0]);
  if (b < 0) return {-1, 0, 0, 0, rows};
  const int f = __builtin_amdgcn_readfirstlane(found[1]);
  return {b, number < 0 ? 0 : number - f, __builtin_amdgcn_readfirstlane(found[2]), f, rows};
}

// columns from one digit of a head to the next, where all digits of a group's heads fit into 16 of them
template <typename A>
constexpr int kApart = kDigits<A> == 2 ? 8 : 4;

// LDS: the digits of HW KV heads' queries, the blocks that the new row goes into (keys, values), the waves' maxima and
// sums, the queries' maxima and factors, the blocks' scales
template <typename A, int HD, int HW, bool SPREAD>
constexpr int q8_fixed_bytes() {
  return HW * (16 * HD * (SPREAD ? 1 : kDigits<A>) + 2 * kBlock * HD + 2 * 16 * 4) + (kWaves * 32 + 8) * 4;
}

// One workgroup: up to 16 query heads of each of HW KV heads, one range of a sequence's cached rows. kWaves / HW waves
// share a KV head and take tiles of 64 of its rows in turn (32 past 128 elements, for the registers).
//
// S^T = K Q^T with keys in the rows of a 16x16x64 int8 MFMA and heads in its columns: the 16 codes that a lane reads of
// its row are an operand as they lie, the queries' digits the other. A lane's 16 scores of a column, 4 g + i of block
// t, are its weights, whose digits in slot 4 t + i are an operand of O^T += V^T P^T as they lie; of V a lane reads E
// = HD / 16 neighbouring codes of the rows 4 g + i and turns 4 rows x 4 codes in registers (8 byte permutations). A
// block's scale is one factor of its scores and of its weights. Row i of result tile e is element E i + e. Each
// tile's weighted values are whole numbers, added to the f32 sums with the factor of their weights. (Codes made bf16
// for bf16 products: twice the instructions, 32 sequences of 0 to 8191 rows, 117 MB, 56 us, this way 45.)
//
// SPREAD: the digits of a group's heads fit into the 16 columns together (up to 8 heads in bf16, 4 in f32): column
// c + kApart n holds digit n of head c, one product does for all digits, and no column is idle. A score is the sum over
// its columns; weights are the same in each and give their own digit; the results' columns are summed at the end.
// The 117 MB 44.4 -> 39.5 us (f32, 3 digits), of it 2 us by keeping the rows' places in scalar registers.
//
// With many rows, HW = 4: the workgroup reads whole pieces of 512 bytes and more of a row at a time, where with HW = 1
// each KV head's 128 bytes are read by other compute units at other times: 8 sequences of 33 to 65 Ki rows 4.1 against
// 5.3 TB/s with the loads alone. With few, HW = 1: more waves at a sequence, each with less to walk.
//
// Bound: those 8 sequences, 888 MB, 165 to 175 us by card with 6 us for the join, 5.1 to 5.4 TB/s over both: by the
// memory (a plain read of a large array 6.1; these loads alone, on a card where the call took 175, 5.3). The 117 MB, about 230 rows a workgroup, 34 us: 11 of them until the first rows are
// there (lengths, plan, table, rows one after the other), then four tiles a wave of 630 vector instructions each,
// half of the time that is left. One sequence of 128 rows 9 us: those loads one after the other. A third workgroup a
// CU (the registers of SPREAD allow it) 42.6, and 888 MB 211: the ranges are shorter and the join is longer.
//
// The block that the new row goes into is not walked over: the workgroup of the last range forms it anew in LDS,
// writes it back, and one wave attends it from there. No other workgroup reads it, so none can see it half written.
template <typename A, int HD, bool PART, int HW, bool SPREAD>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_q8_kernel(PagedAttnArgs a) {
  constexpr int NT = kDigits<A>, APART = kApart<A>;
  constexpr int NM = SPREAD ? 1 : NT;  // operands for the digits
  constexpr int NB = HD == 256 ? 2 : 4, KT = NB * kBlock, RW = kWaves / HW, STEP = KT * RW;
  constexpr int KP = HD / 64, E = HD / 16, VW = E / 4;  // 16-byte pieces of a K row a lane; codes and words of a V row
  constexpr int kQuery = 16 * HD * NM;                  // bytes of a KV head's queries
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const PagesArgs& p = a.p;
  const int hd = p.head_dim, half = hd / 2, group = p.n_q / p.n_kv, htiles = (group + 15) / 16, nh = min(group, 16);
  uint32_t* tails = reinterpret_cast<uint32_t*>(sm + HW * kQuery / 4);  // [HW][keys, values][16][HD] codes
  float* wm = reinterpret_cast<float*>(tails + HW * 2 * kBlock * HD / 4);  // [waves][16]
  float* wl = wm + kWaves * 16;
  uint32_t* qmax = reinterpret_cast<uint32_t*>(wl + kWaves * 16);  // [HW][16] bits of the queries' largest |x|
  float* qinv = reinterpret_cast<float*>(qmax + HW * 16);          // [HW][16] what a digits' unit stands for
  float* tail_s = qinv + HW * 16;                                   // [HW][2] the blocks' scales
  float* wacc = tail_s + 8;  // [waves][heads][HD]; before that cos and sin [2][HD / 2]
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), hw = wave / RW, rw = wave % RW;
  int id = blockIdx.x;
  const int ht = id % htiles;
  id /= htiles;
  const int hkv0 = id % (p.n_kv / HW) * HW, hkv = hkv0 + hw;
  id /= p.n_kv / HW;
  const Range range = range_of(a, id);
  if (range.b < 0) return;
  const int b = range.b, split = range.at;
  const int heads = min(group - ht * 16, 16);
  const int per_head = heads * half;  // pairs of query elements of a KV head
  // the query rows, asked for with the length
  constexpr int kPairs = HW * (SPREAD ? APART : 16) * HD / 2, NE = (kPairs + kThreads - 1) / kThreads;
  const A* qrow = static_cast<const A*>(p.q) + (int64_t)b * p.q_stride + (hkv0 * group + ht * 16) * hd;
  A q0[NE], q1[NE];
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = min(tid + n * kThreads, HW * per_head - 1), k = HW > 1 ? i / per_head : 0, j = i - k * per_head;
    const int hh = j / half, e = j - hh * half;
    q0[n] = qrow[(k * group + hh) * hd + e];
    q1[n] = qrow[(k * group + hh) * hd + e + half];
  }
  // the new row: task t is the keys (t even) or the values of KV head t / 2, by wave t % kWaves
  const bool add = p.k != nullptr;
  constexpr int NP = HD > 128 ? 2 : 1, TASKS = (2 * HW + kWaves - 1) / kWaves;  // pairs a lane, tasks a wave
  A n0[TASKS][NP], n1[TASKS][NP];
  if (add)
#pragma unroll
    for (int k = 0; k < TASKS; k++) {
      const int task = min(wave + k * kWaves, 2 * HW - 1);
      const A* row = task & 1 ? static_cast<const A*>(p.v) + (int64_t)b * p.v_stride
                              : static_cast<const A*>(p.k) + (int64_t)b * p.k_stride;
#pragma unroll
      for (int n = 0; n < NP; n++) {
        const int e = (hkv0 + task / 2) * hd + min(lane + 64 * n, half - 1);
        n0[k][n] = row[e];
        n1[k][n] = row[e + half];
      }
    }
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  // Page numbers: lane t holds that of block t of a tile, so one load brings them all. Those of the wave's first
  // tile are asked for with the length where no window moves it.
  const int r0 = split == 0 ? 0 : split * range.rows, first = r0 + rw * KT, lane_t = min(lane & 7, NB - 1);
  const int last_entry = max((int)p.table_stride - 1, 0);
  const bool moved = a.window != INT32_MAX;
  int pages = -1;
  if (!moved && p.table_stride > 0) pages = trow[min((first + kBlock * lane_t) >> p.page_bits, last_entry)];
  // (as loaded it would stay in vector registers, with all that follows)
  const int len = __builtin_amdgcn_readfirstlane(a.lens[b]);
  A* orow = static_cast<A*>(a.out) + (int64_t)b * a.out_stride + (hkv0 * group + ht * 16) * hd;
  // element i of the workgroup's results: KV head k, query head hh, element d
  auto place = [&](int i, int* k, int* hh, int* d) {
    *k = HW > 1 ? i / (heads * hd) : 0;
    const int j = i - *k * heads * hd;
    *hh = j / hd;
    *d = j - *hh * hd;
  };
  const int64_t rows = (int64_t)len + (add || a.ahead);
  const bool bad = rows > a.max_len || rows > p.table_stride << p.page_bits;
  if (len < 0 || bad || rows == 0) {  // idle slot or nothing to see: zeros; more rows than the call allows: NaN
    if (split == 0)
      for (int i = tid; i < HW * heads * hd; i += kThreads) {
        int k, hh, d;
        place(i, &k, &hh, &d);
        orow[(k * group + hh) * hd + d] = (A)(bad && len >= 0 ? NAN : 0.0f);
      }
    return;
  }
  const int tail_row = len & ~(kBlock - 1), before = len & (kBlock - 1);  // of the block that the new row goes into
  CachedRows<true> cr;
  cr.init(a, add ? tail_row : (int)rows, rows);
  const int nsplit = range.count ? range.count : ranges_of_walk(cr.walk, range.rows);
  if (split >= nsplit) return;
  const bool last = split == nsplit - 1;
  const int r1 = last ? cr.walk : r0 + range.rows;
  const int kvd = p.n_kv * hd;
  bool lost = false;  // a page number out of range

  const int in_page = (1 << p.page_bits) - 1;
  auto ask_pages = [&](int r) { pages = trow[min(cr.row(r + kBlock * lane_t) >> p.page_bits, last_entry)]; };
  auto scale_at = [&](int64_t page, int row, int head) -> int64_t {
    return page * a.scale_stride + ((row & in_page) >> 4) * p.n_kv + head;
  };
  const int8_t* kb = static_cast<const int8_t*>(p.kpages) + hkv * hd;
  const int8_t* vb = static_cast<const int8_t*>(p.vpages) + hkv * hd;
  typedef uint32_t VRow __attribute__((ext_vector_type(VW)));
  i32x4 xk[NB][KP];
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
    return (lane & 8 ? a.vscales : a.kscales)[scale_at(lane_t < n ? pages : first_page, row, hkv)];
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
          xk[t][u] = __builtin_bit_cast(i32x4, u32x4{lo[0], lo[1], hi[0], hi[1]});
        } else {
          xk[t][u] = *reinterpret_cast<const i32x4*>(kp + 64 * u + k_off);
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
  const uint32_t* tail_k = tails + hw * (2 * kBlock * HD / 4);
  const uint32_t* tail_v = tail_k + kBlock * HD / 4;
  auto take_tail_k = [&]() {
#pragma unroll
    for (int u = 0; u < KP; u++)
      xk[0][u] = *reinterpret_cast<const i32x4*>(tail_k + (col * HD + 64 * u + 16 * g) / 4);
    sc = tail_s[2 * hw + (lane & 8 ? 1 : 0)];
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

  // the rotated queries' digits as operands (zeros for heads and elements past the end)
  float* cs = wacc;
  if (p.rope && tid < half) cos_sin_turns(len * turns_of(tid, hd, p.log2_theta), cs + tid, cs + HD / 2 + tid);
  for (int i = tid; i < HW * kQuery / 16; i += kThreads) reinterpret_cast<u32x4*>(sm)[i] = u32x4{0, 0, 0, 0};
  if (tid < HW * 16) qmax[tid] = 0;
  __syncthreads();
  float y0[NE], y1[NE];
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = tid + n * kThreads, k = HW > 1 ? i / per_head : 0, j = i - k * per_head, hh = j / half, e = j - hh * half;
    if (i < HW * per_head) {
      y0[n] = (float)q0[n], y1[n] = (float)q1[n];
      if (p.rope) rotate(y0[n], y1[n], cs[e], cs[HD / 2 + e], &y0[n], &y1[n]);
      // (bits of absolute values are in their order, NaN last)
      atomicMax(&qmax[k * 16 + hh], max(__float_as_uint(fabsf(y0[n])), __float_as_uint(fabsf(y1[n]))));
    }
  }
  if (add && last) {  // the new row's block
#pragma unroll
    for (int k = 0; k < TASKS; k++) {
      const int task = wave + k * kWaves, head = hkv0 + task / 2;
      if (task >= 2 * HW) break;
      const bool is_v = task & 1;
      const int page = trow[tail_row >> p.page_bits];
      const bool store = (uint32_t)page < (uint64_t)p.pages;
      lost |= !store;
      const int64_t at = ((int64_t)(store ? page : 0) << p.page_bits) + (tail_row & in_page);
      int8_t* codes = static_cast<int8_t*>(is_v ? p.vpages : p.kpages) + at * kvd + head * hd;
      float* scale = (is_v ? a.vscales : a.kscales) + scale_at(store ? page : 0, tail_row, head);
      uint32_t* tail = tails + task * (kBlock * HD / 4);
      const int words = hd / 4;
      uint32_t w[HD / 16];
#pragma unroll
      for (int n = 0; n < HD / 16; n++) {
        const int i = lane + 64 * n, r = i / words, c = i - r * words;
        w[n] = r < before ? *reinterpret_cast<const uint32_t*>(codes + (int64_t)r * kvd + 4 * c) : 0;
      }
      const float s0 = before > 0 ? *scale : 0.0f;
      float z0[NP], z1[NP], amax = 0.0f;
      bool good = true;
#pragma unroll
      for (int n = 0; n < NP; n++) {
        const int e = min(lane + 64 * n, half - 1);
        z0[n] = (float)n0[k][n], z1[n] = (float)n1[k][n];
        if (!is_v && p.rope) rotate(z0[n], z1[n], cs[e], cs[HD / 2 + e], &z0[n], &z1[n]);
        amax = fmaxf(amax, fmaxf(fabsf(z0[n]), fabsf(z1[n])));
        good = good && finite(z0[n]) && finite(z1[n]);
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
          const int8_t c0 = (int8_t)code_of(z0[n], s), c1 = (int8_t)code_of(z1[n], s);
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
        tail_s[task] = s;
        if (store) *scale = s;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NE; n++) {
    const int i = tid + n * kThreads, k = HW > 1 ? i / per_head : 0, j = i - k * per_head, hh = j / half, e = j - hh * half;
    if (i < HW * per_head) {
      const float f = digit_factor<NT>(__uint_as_float(qmax[k * 16 + hh]));
      // (a head of zeros: 0, of NaN: NaN)
      if (e == 0) qinv[k * 16 + hh] = f > 0.0f ? __builtin_amdgcn_rcpf(f) : __uint_as_float(qmax[k * 16 + hh]);
      char* at = reinterpret_cast<char*>(sm) + k * kQuery;
#pragma unroll
      for (int z = 0; z < 2; z++) {
        const int d = e + z * half;
        const uint32_t x = digits_of<NT>((int)rintf((z ? y1[n] : y0[n]) * f));
#pragma unroll
        for (int m = 0; m < NT; m++)
          at[(((SPREAD ? 0 : m * KP) + (d >> 6)) * 64 + 16 * ((d >> 4) & 3) + (SPREAD ? m * APART : 0) + hh) * 16 +
             (d & 15)] = (char)(x >> (8 * m));
      }
    }
  }
  __syncthreads();
  // the column's head, its digit and that one's weight
  const int hcol = SPREAD ? col & (APART - 1) : col, digit = SPREAD ? col / APART : 0;
  const float unit = digit == 0 ? 1.0f : digit == 1 ? 256.0f : digit == 2 ? 65536.0f : 0.0f;
  const uint32_t pick = digit | (digit + 4) << 8;
  const float qs = hcol < heads ? qinv[hw * 16 + hcol] * a.scale2 * unit : 0.0f;

  f32x4 acc[E];
#pragma unroll
  for (int t = 0; t < E; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  // the wave's tiles, at the end the new row's block by the wave of its head whose turn it is
  int r = first;
  const bool has_tail = add && last && rw == ((r1 - r0 + KT - 1) / KT) % RW;
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
      const bool there = tail ? t == 0 : r + kBlock * t < r1;
      at[t] = !there ? INT32_MAX - kBlock : tail ? tail_row : cr.row(r + kBlock * t);
      ks[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc), t));
      vs[t] = there ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc), 8 + t)) : 0.0f;
    }
    if (more) set_base(r + STEP);
    int ql = lane;  // read anew for every tile: kept in registers they would cost a wave a SIMD
    asm volatile("" : "+v"(ql));
    const i32x4* qp = reinterpret_cast<const i32x4*>(reinterpret_cast<const char*>(sm) + hw * kQuery) + ql;
    float s[NB][4];
#pragma unroll
    for (int t0 = 0; t0 < NB; t0 += 2) {  // two blocks at a time, for the registers
      i32x4 d[NM][2] = {};
#pragma unroll
      for (int u = 0; u < KP; u++) {
        i32x4 qw[NM];
#pragma unroll
        for (int n = 0; n < NM; n++) qw[n] = qp[(n * KP + u) * 64];
#pragma unroll
        for (int n = 0; n < NM; n++)
#pragma unroll
          for (int t = 0; t < 2; t++)
            d[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xk[t0 + t][u], qw[n], d[n][t], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const float f = ks[t0 + t] * qs;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (SPREAD)
            s[t0 + t][i] = sum_digits<APART>((float)d[0][t][i] * f);
          else if constexpr (NT == 2)
            s[t0 + t][i] = value_of(d[0][t][i], d[1][t][i]) * f;
          else
            s[t0 + t][i] = value_of(d[0][t][i], d[1][t][i], d[2][t][i]) * f;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more) {
      load_k();
      sc = load_scales(r + STEP);
      ask_pages(r + 2 * STEP);
    } else if (then_tail) {
      take_tail_k();
    }
#pragma unroll
    for (int t = 0; t < NB; t++) {
      if (at[t] + kBlock > end || !cr.sees_block(at[t]))
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int row = at[t] + 4 * g + i;
          if (row >= end || !cr.sees(row)) s[t][i] = -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < NB; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // Weights (with the scale of their block) are digits relative to the tile's largest: the tile's own maximum
    // first, so that none of a tile is lost beside another tile's
    const float top = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, vsum = 0.0f, wmax = 0.0f;
#pragma unroll
    for (int t = 0; t < NB; t++) {
      vsum += vs[t];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - top);
        sum += s[t][i];
        s[t][i] *= vs[t];
        wmax = fmaxf(wmax, s[t][i]);
      }
    }
    wmax = fmaxf(wmax, __shfl_xor(wmax, 16, 64));
    wmax = fmaxf(wmax, __shfl_xor(wmax, 32, 64));
    const float to_digits = digit_factor<NT>(wmax);
    i32x4 pd[NM] = {};
#pragma unroll
    for (int t = 0; t < NB; t++) {
      uint32_t x[4], y[NM];
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (uint32_t)(int)fmaf(s[t][i], to_digits, 0.5f) + (NT == 2 ? 0x8080u : 0x808080u);
      if constexpr (SPREAD)
        y[0] = pack_digit(x, pick);
      else
        pack_digits<NT>(x, y);
#pragma unroll
      for (int n = 0; n < NM; n++) pd[n][t] = (int)(y[n] ^ 0x80808080u);
    }
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ref), beta = __builtin_amdgcn_exp2f(mx - ref);
    m = mn;
    l = fmaf(l, alpha, sum * beta);
    // (a scale that is not finite makes the factor NaN)
    const float from_digits = (to_digits > 0.0f ? __builtin_amdgcn_rcpf(to_digits) : 0.0f) + 0.0f * vsum;
    const float wf = SPREAD ? from_digits * beta * unit : from_digits * beta;
    keep_whole(xv);
#pragma unroll
    for (int w = 0; w < VW; w++)  // four elements, one word of the rows
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        i32x4 vf[2] = {};
#pragma unroll
        for (int t = 0; t < NB; t++) {
          const uint32_t pick = e == 0 ? 0x05010400 : 0x07030602;
          const uint32_t x = __builtin_amdgcn_perm(xv[4 * t + 1][w], xv[4 * t][w], pick);
          const uint32_t y = __builtin_amdgcn_perm(xv[4 * t + 3][w], xv[4 * t + 2][w], pick);
          vf[0][t] = (int)low16_pair(x, y);
          vf[1][t] = (int)high16_pair(x, y);
        }
        i32x4 o[NM][2];
#pragma unroll
        for (int n = 0; n < NM; n++)
#pragma unroll
          for (int i = 0; i < 2; i++)
            o[n][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[i], pd[n], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          f32x4& sum_e = acc[4 * w + e + i];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float x;
            if constexpr (SPREAD)
              x = (float)o[0][i][j];
            else if constexpr (NT == 2)
              x = value_of(o[0][i][j], o[1][i][j]);
            else
              x = value_of(o[0][i][j], o[1][i][j], o[2][i][j]);
            sum_e[j] = fmaf(x, wf, sum_e[j] * alpha);
          }
          asm volatile("" : "+v"(sum_e));  // (else the sums sink past the next loads)
        }
        __builtin_amdgcn_sched_barrier(0);  // (left alone, all products come first and do not fit)
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
  if constexpr (SPREAD)
#pragma unroll
    for (int t = 0; t < E; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[t][i] = sum_digits<APART>(acc[t][i]);
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
  for (int i = tid; i < HW * heads * hd; i += kThreads) {
    int k, hh, d;
    place(i, &k, &hh, &d);
    const int w0 = k * RW;
    float mx = wm[w0 * 16 + hh];
#pragma unroll
    for (int w = 1; w < RW; w++) mx = fmaxf(mx, wm[(w0 + w) * 16 + hh]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float o = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < RW; w++) {
      const float f = __builtin_amdgcn_exp2f(wm[(w0 + w) * 16 + hh] - ref);
      sum += f * wl[(w0 + w) * 16 + hh];
      o += f * wacc[((w0 + w) * nh + hh) * HD + d];
    }
    if (any_lost) sum = NAN;
    if (nsplit == 1) {
      orow[(k * group + hh) * hd + d] = (A)(sum == 0.0f ? 0.0f : o / sum);
    } else {
      const int hq = (hkv0 + k) * group + ht * 16 + hh;
      float* rec = a.part + ((int64_t)id * p.n_q + hq) * (kRec + hd);
      rec[kRec + d] = o;
      if (d == 0) {
        rec[0] = mx;
        rec[1] = sum;
      }
    }
  }
}

// Joins the ranges' records of a (sequence, head), one workgroup each: head_dim / 4 lanes
// a record, the lane groups' sums added in order. 6 us of which 4 are the launch and the plan, done again here: with
// all records asked for at once 0.3 less.
template <typename A>
__global__ __launch_bounds__(256) void paged_q8_merge_kernel(PagedAttnArgs a) {
  const PagesArgs& p = a.p;
  const int hq = blockIdx.x % p.n_q, b = blockIdx.x / p.n_q, hd = p.head_dim;
  const Range range = range_of(a, -1 - b);
  const int n = range.count ? range.count : ranges_of_walk(walked_of(a, a.lens[b]), range.rows);
  if (n <= 1) return;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float sums[256 * 4];
  __shared__ float lsum[128];
  const int tid = threadIdx.x, dl = hd / 4, groups = 256 / dl, grp = tid / dl, d = tid % dl;
  const int64_t rs = (int64_t)p.n_q * (kRec + hd);
  const float* rec = a.part + ((int64_t)range.first * p.n_q + hq) * (kRec + hd);
  float mx = -INFINITY;
  for (int r = tid; r < n; r += 256) mx = fmaxf(mx, rec[r * rs]);
  mx = wave_max(mx);
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

// RoPE and append of packed rows, a workgroup the rows of one block and some of the heads, a wave a head at a time:
// its rows stay in registers between their maximum and their codes: each value is read once and each code written once.
// Bound by the memory: 8192 rows of 32/8 heads x 128 in bf16, 201 MB, 44 us, 4.6 TB/s (a copy reaches 4.9). 72 with
// an angle's sine and cosine by the general functions, 56 with 8 bytes a load, 50 with divisions and no load ahead of
// the angles. Without cu row b is the one row of sequence b, at position past[b].
template <typename A, int HD, int V>
__global__ __launch_bounds__(kThreads) void pages_append_q8_kernel(PagesAppendArgs a, int chunks) {
  const PagesArgs& p = a.p;
  // (rows 16 bytes apart more than they are long: 8 lanes read 16 of every 32 bytes of a row, the next 8 of the next row)
  __shared__ __attribute__((aligned(16))) float cs[2][kBlock][HD / 2 + 4];
  __shared__ double turns[HD / 2];
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
  const bool inside = pos0 < p.table_stride << p.page_bits && pos1 <= a.max_len;
  const int page = inside ? p.table[(int64_t)b * p.table_stride + (pos0 >> p.page_bits)] : -1;
  const bool ok = (uint32_t)page < (uint64_t)p.pages;
  const int in_page = (int)(block * kBlock & ((1 << p.page_bits) - 1));
  const int64_t at = ok ? ((int64_t)page << p.page_bits) + in_page : 0;  // of the block's first row
  typedef A AV __attribute__((ext_vector_type(V)));
  constexpr int N = (kBlock * HD / 2 / V + 63) / 64;  // groups of V pairs a lane
  const int hp = half / V, kvd = p.n_kv * hd, tasks = p.n_q + 2 * p.n_kv;
  const int task0 = (a.q_out == nullptr ? p.n_q : 0) + chunk * kWaves + wave;
  // a task's rows, asked for before the angles are formed, or before the rows of the one before are rounded
  AV x0[N], x1[N];
  auto ask = [&](int task) {
    if (task >= tasks) return;
    const int what = task < p.n_q ? 0 : task < p.n_q + p.n_kv ? 1 : 2;  // q, k, v
    const int head = what == 0 ? task : what == 1 ? task - p.n_q : task - p.n_q - p.n_kv;
    const A* x = static_cast<const A*>(what == 0 ? p.q : what == 1 ? p.k : p.v) + head * hd;
    const int64_t xs = what == 0 ? p.q_stride : what == 1 ? p.k_stride : p.v_stride;
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = V * (i - r * hp);
      if (r < rows) {
        x0[k] = *reinterpret_cast<const AV*>(x + (row0 + r) * xs + e);
        x1[k] = *reinterpret_cast<const AV*>(x + (row0 + r) * xs + e + half);
      }
    }
  };
  ask(task0);
  if (p.rope) {
    if (tid < half) turns[tid] = turns_of(tid, hd, p.log2_theta);
    __syncthreads();
    for (int i = tid; i < rows * half; i += kThreads) {
      const int r = i / half, e = i - r * half;
      cos_sin_turns((double)(pos0 + r) * turns[e], &cs[0][r][e], &cs[1][r][e]);
    }
    __syncthreads();
  }
  for (int task = task0; task < tasks; task += chunks * kWaves) {
    const int what = task < p.n_q ? 0 : task < p.n_q + p.n_kv ? 1 : 2;
    const int head = what == 0 ? task : what == 1 ? task - p.n_q : task - p.n_q - p.n_kv;
    A* out = what == 2 ? nullptr : static_cast<A*>(what == 0 ? a.q_out : a.k_out);
    const int64_t os = what == 0 ? a.q_out_stride : a.k_out_stride;
    float y0[N][V], y1[N][V];
    uint32_t most = 0;  // bits of the largest |y|: they are in the order of the numbers, infinities and NaN last
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = V * (i - r * hp);
      if (r >= rows) continue;
#pragma unroll
      for (int j = 0; j < V; j++) {
        y0[k][j] = (float)x0[k][j], y1[k][j] = (float)x1[k][j];
        if (what < 2 && p.rope) rotate(y0[k][j], y1[k][j], cs[0][r][e + j], cs[1][r][e + j], &y0[k][j], &y1[k][j]);
      }
      if (out != nullptr) {
        AV z0, z1;
#pragma unroll
        for (int j = 0; j < V; j++) z0[j] = (A)y0[k][j], z1[j] = (A)y1[k][j];
        if (!ok)  // no page for the row: its outputs say so
#pragma unroll
          for (int j = 0; j < V; j++) z0[j] = z1[j] = (A)NAN;
        A* o = out + (row0 + r) * os + head * hd + e;
        *reinterpret_cast<AV*>(o) = z0;
        *reinterpret_cast<AV*>(o + half) = z1;
      }
      if (what > 0)
#pragma unroll
        for (int j = 0; j < V; j++)
          most = max(most, max(__float_as_uint(y0[k][j]) & 0x7fffffff, __float_as_uint(y1[k][j]) & 0x7fffffff));
    }
    ask(task + chunks * kWaves);
    if (what == 0 || !ok) continue;
    int8_t* codes = static_cast<int8_t*>(what == 1 ? p.kpages : p.vpages) + at * kvd + head * hd;
    float* scale = (what == 1 ? a.kscales : a.vscales) + page * a.scale_stride + (in_page >> 4) * p.n_kv + head;
    const float s0 = before > 0 ? *scale : 0.0f;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, 64));
    const float s = raised(__uint_as_float(most), most < 0x7f800000, s0), inv = __fdiv_rn(1.0f, s);
    if (s > s0 && before > 0) {
      const float ratio = __fdiv_rn(s0, s);
      for (int i = lane; i < before * (hd / 4); i += 64) {
        const int r = i / (hd / 4);
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + (int64_t)r * kvd + 4 * (i - r * (hd / 4)));
        *w = recoded(*w, ratio);
      }
    }
    typedef uint32_t CV __attribute__((ext_vector_type(V / 4)));
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = lane + 64 * k, r = i / hp, e = V * (i - r * hp);
      if (r >= rows) continue;
      CV w0, w1;
#pragma unroll
      for (int n = 0; n < V / 4; n++) {
        w0[n] = codes_of(&y0[k][4 * n], s, inv);
        w1[n] = codes_of(&y1[k][4 * n], s, inv);
      }
      int8_t* o = codes + (int64_t)(before + r) * kvd + e;
      *reinterpret_cast<CV*>(o) = w0;
      *reinterpret_cast<CV*>(o + half) = w1;
    }
    if (lane == 0) *scale = s;
  }
}

}  // namespace

namespace {

template <typename A, int HD, bool PART, int HW, bool SPREAD>
hipError_t run_paged_q8(const PagedAttnArgs& a, hipStream_t stream) {
  const PagesArgs& p = a.p;
  const int64_t htiles = (p.n_q / p.n_kv + 15) / 16;
  constexpr int kFixed = q8_fixed_bytes<A, HD, HW, SPREAD>(), kMaxLds = kFixed + kWaves * 16 * HD * 4;
  const int lds = kFixed + kWaves * std::min(p.n_q / p.n_kv, 16) * HD * 4;
  const auto kernel = paged_attention_q8_kernel<A, HD, PART, HW, SPREAD>;
  static std::atomic<uint64_t> allowed{0};
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), kMaxLds, &allowed)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.batch + a.spare) * (p.n_kv / HW) * htiles)), dim3(kThreads), lds,
                     stream, a);
  return hipGetLastError();
}

template <typename A, int HD, bool PART>
hipError_t run_paged_q8_heads(const PagedAttnArgs& a, hipStream_t stream) {
  const bool spread = a.p.n_q / a.p.n_kv <= kApart<A>;
  if constexpr (HD <= 128)
    if (a.kv_heads == 4)
      return spread ? run_paged_q8<A, HD, PART, 4, true>(a, stream) : run_paged_q8<A, HD, PART, 4, false>(a, stream);
  return spread ? run_paged_q8<A, HD, PART, 1, true>(a, stream) : run_paged_q8<A, HD, PART, 1, false>(a, stream);
}

template <typename A>
hipError_t run_paged_q8_hd(const PagedAttnArgs& a, hipStream_t stream) {
  const int hd = a.p.head_dim;
  if (hd == 64) return run_paged_q8_heads<A, 64, false>(a, stream);
  if (hd == 128) return run_paged_q8_heads<A, 128, false>(a, stream);
  if (hd == 256) return run_paged_q8_heads<A, 256, false>(a, stream);
  if (hd < 64) return run_paged_q8_heads<A, 64, true>(a, stream);
  if (hd < 128) return run_paged_q8_heads<A, 128, true>(a, stream);
  return run_paged_q8_heads<A, 256, true>(a, stream);
}

template <typename A, int HD, int V>
hipError_t run_append_q8(const PagesAppendArgs& a, hipStream_t stream) {
  // A wave takes one head, though every workgroup forms its rows' angles; more only where the grid has no room. us, by
  // about 2048 workgroups / so: 8192 rows (32/8 x 128, bf16) 45.8 / 46.0, in f32 94 / 78, 16000 (64/8) 150 / 129
  const int64_t slots = append_q8_slots(a), tasks = a.p.n_q + 2 * a.p.n_kv;
  const int64_t chunks =
      std::max<int64_t>(1, std::min((tasks + kWaves - 1) / kWaves, kMaxGroups / std::max<int64_t>(slots, 1)));
  hipLaunchKernelGGL((pages_append_q8_kernel<A, HD, V>), dim3((unsigned)(slots * chunks)), dim3(kThreads), 0, stream, a,
                     (int)chunks);
  return hipGetLastError();
}

template <typename A, int V>
hipError_t run_append_q8_hd(const PagesAppendArgs& a, hipStream_t stream) {
  if (a.p.head_dim <= 64) return run_append_q8<A, 64, V>(a, stream);
  if (a.p.head_dim <= 128) return run_append_q8<A, 128, V>(a, stream);
  return run_append_q8<A, 256, V>(a, stream);
}

// The stored rows of sequences, packed: a workgroup ROWS of them, whose places in the pages are looked up first.
// C: the pages' type (int8: codes times the block's scale), T: the rows'.
// Bound by the memory, 16 or 32 bytes a store: 63 MB 14 us, 4.5 TB/s. Four rows a workgroup, so that a few hundred
// rows fill the card.
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

PagedQ8Plan plan_paged_attention_q8(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len,
                                    int cu_count) {
  batch = std::min<int64_t>(batch, kPlanned);
  const int64_t htiles = (n_q / n_kv + 15) / 16;
  PagedQ8Plan p;
  // Four KV heads a workgroup where a CU can have many rows times KV heads; us, one head / four, and rows at max_len
  // (caches cold, bf16, 32/8 heads x 128 unless said): 64 of 1000 45 / 48, 2000 | 32 of 2000 44 / 45, 2000 | 8 of
  // 4000 27 / 31, 1000 | 4 of 16000, 16/16 heads 71 / 65, 4000 | 64 of 1 to 4000 93 / 81, 8000 | 32 of 8000 133 /
  // 123, 8000 | 32 of 1 to 8191 (f32) 120 / 80, 8191 | 16 of 16000, 64/8 x 64 103 / 74, 8000 | 16 of 1 to 32000 157 /
  // 120, 16000 | 8 of 33 to 65 Ki, 64/8 heads 270 / 189, 16384
  const bool wide = n_kv % 4 == 0 && head_dim <= 128 && htiles == 1;
  p.kv_heads = wide && max_len * batch * n_kv > 3500 * (int64_t)cu_count ? 4 : 1;
  // Many short sequences fill the card unbroken, and no lengths have to be looked at nor results joined: one head /
  // four in ranges, one / four unbroken: 300 of 1 to 1000 116 / 125, 94 / 104 | 128 of 1 to 2000 91 / 99, 81 / 113 |
  // 128 of 2000 135 / 139, 126 / 132 | 1000 of 1 to 500, 16/8 x 64 107 / 117, 106 / 84. Not where one long one may
  // have to wait for a workgroup (3 of 4000 and 97 of 1 to 200 33, unbroken 56).
  const int64_t most_groups = batch * n_kv * htiles, enough = 3 * (int64_t)cu_count;
  const bool whole = max_len <= 2048 && most_groups >= enough;
  if (whole) p.kv_heads = wide && most_groups / 4 >= enough ? 4 : 1;
  const int64_t heads = n_kv / p.kv_heads * htiles;
  p.split_rows = kTileRows * kWaves / p.kv_heads;
  // As many ranges more than sequences as give every CU two workgroups; where there are many sequences, whose short
  // ends add up, no more than that in all (64 of 1 to 4000 96 -> 83, but 8 of 33 to 65 Ki 178 -> 190), and half as
  // many at least. A sequence of one or two rounds of tiles stays whole: the join would cost more.
  const int64_t most = whole || max_len <= 2 * p.split_rows ? 0 : batch * (max_len / p.split_rows), two = 2 * cu_count / heads;
  p.spare = (int)std::min<int64_t>(std::max<int64_t>({4 * batch >= two ? two - batch : two, two / 2, 1}), most);
  p.range_rows = 0;
  if (batch == 1 && p.spare > 0)
    p.range_rows = (int)((max_len / (p.spare + 1) + p.split_rows) / p.split_rows * p.split_rows);
  p.groups = (batch + p.spare) * heads;
  p.work = p.spare > 0 ? (size_t)((batch + p.spare) * n_q * (kRec + head_dim)) * sizeof(float) : 0;
  return p;
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
  const int64_t e = dtype == RQ_F32 ? 4 : 2;
  // (a launch's records are joined before the next one's are written)
  for (int64_t b = 0; b < p.batch; b += kPlanned) {
    PagedAttnArgs n = r;
    n.p.batch = (int)std::min<int64_t>(kPlanned, p.batch - b);
    n.p.table += b * p.table_stride;
    n.lens += b;
    auto from = [&](const void* x, int64_t stride) { return x ? static_cast<const char*>(x) + b * stride * e : nullptr; };
    n.p.q = from(r.p.q, p.q_stride);
    n.p.k = from(r.p.k, p.k_stride);
    n.p.v = from(r.p.v, p.v_stride);
    n.out = static_cast<char*>(r.out) + b * r.out_stride * e;
    if (hipError_t s = dtype == RQ_F32 ? run_paged_q8_hd<float>(n, stream) : run_paged_q8_hd<__bf16>(n, stream)) return s;
    if (n.spare > 0) {
      const dim3 grid((unsigned)(n.p.batch * p.n_q));
      if (dtype == RQ_F32)
        hipLaunchKernelGGL(paged_q8_merge_kernel<float>, grid, dim3(256), 0, stream, n);
      else
        hipLaunchKernelGGL(paged_q8_merge_kernel<__bf16>, grid, dim3(256), 0, stream, n);
      if (hipError_t s = hipGetLastError()) return s;
    }
  }
  return hipSuccess;
}

hipError_t launch_pages_append_q8(int dtype, const PagesAppendArgs& a, hipStream_t stream) {
  // 16 bytes a load where a half of a head is whole ones of them
  if (dtype == RQ_F32) return run_append_q8_hd<float, 4>(a, stream);
  return a.p.head_dim % 16 == 0 ? run_append_q8_hd<__bf16, 8>(a, stream) : run_append_q8_hd<__bf16, 4>(a, stream);
}

hipError_t launch_pages_rows(int dtype, int cache_dtype, const PagesRowsArgs& a, hipStream_t stream) {
  if (cache_dtype == RQ_I8)
    return dtype == RQ_F32 ? run_rows<int8_t, float>(a, stream) : run_rows<int8_t, __bf16>(a, stream);
  if (cache_dtype == RQ_BF16)
    return dtype == RQ_F32 ? run_rows<__bf16, float>(a, stream) : run_rows<__bf16, __bf16>(a, stream);
  return dtype == RQ_F32 ? run_rows<float, float>(a, stream) : run_rows<float, __bf16>(a, stream);
}

}  // namespace rq
