// attn_tile.h — tiles of the attention kernels over whole sequences
// (prompt.hip, prompt_bwd.hip): staging into LDS, MFMA fragments from it.
//
// A tile is ROWS rows of HD elements of T (bf16 or f32), one row a key, a query
// or a gradient row of one head. Every product of these kernels is a 32x32 MFMA
// whose operands hold 8 elements a lane (lane l: row l % 32, k slots 8 (l / 32) ..
// + 7): one v_mfma_f32_32x32x16_bf16, or for f32 eight v_mfma_f32_32x32x2_f32, one
// an element, so that both types share every layout below. An accumulator holds
// 16 values a lane: column l % 32, row 8 (i / 4) + 4 (l / 32) + i % 4.
//
// The rows of one product's result are the k slots of the next one (scores to
// weighted values). A lane's values i = 8 t .. 8 t + 7 are rows 16 t + 4 (l / 32) +
// {0 .. 3, 8 .. 11}, so they are a B fragment as they are when slot j of half h
// stands for row 16 t + 8 (j / 4) + 4 h + j % 4 on both sides; tile_frag_t reads the
// other side in that order. No value crosses lanes.
//
// In LDS a row's 16-byte pieces are permuted by the row (XOR), so that 16 rows at one
// column, and the 4 rows x 64 bytes of half a wave's transposing read, fall on
// different ones of the 64 banks (256 bytes).
#pragma once

#include <atomic>

#include "rq_internal.h"

namespace rq {

// Lets a kernel take `bytes` of dynamic LDS on the current device; `allowed` has a bit for
// each device that knows.
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>* allowed) {
  if (bytes <= 65536) return hipSuccess;
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev)) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (allowed->load(std::memory_order_acquire) & bit) return hipSuccess;
  if (hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  allowed->fetch_or(bit, std::memory_order_acq_rel);
  return hipSuccess;
}

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct TileType;
template <>
struct TileType<__bf16> {
  using Frag = bf16x8;
  static constexpr int kPiece = 8;  // elements of 16 bytes
};
template <>
struct TileType<float> {
  using Frag = f32x8;
  static constexpr int kPiece = 4;
};

__device__ __forceinline__ f32x16 tile_mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 tile_mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// the B fragment of accumulator values 8 t .. 8 t + 7 (bf16: rounded to nearest)
__device__ __forceinline__ void tile_pack(const float* v, bf16x8& f) {
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = (__bf16)v[j];
}
__device__ __forceinline__ void tile_pack(const float* v, f32x8& f) {
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = v[j];
}

template <typename T, int HD>
struct Tile {
  using Frag = typename TileType<T>::Frag;
  static constexpr int kPiece = TileType<T>::kPiece;
  static constexpr int kPieces = HD / kPiece;                  // of a row
  static constexpr int kPitch = (kPieces + 7) / 8 * 8 * 16;    // bytes from row to row
  static constexpr int bytes(int rows) { return rows * kPitch; }

  // 16 pieces and more: the row's low 4 bits, the lowest two on top; 8 pieces (two rows
  // side by side in the banks): bits 1 to 3
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (kPieces % 16 == 0) return ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
    return ((row & 2) << 1) | ((row >> 1) & 2) | ((row >> 3) & 1);
  }
  // byte offset of 16-byte piece c of a row
  static __device__ __forceinline__ int at(int row, int c) { return row * kPitch + ((c ^ swizzle(row)) << 4); }

  // A or B fragment: lane's row `row`, elements 16 s + 8 h .. + 7
  static __device__ __forceinline__ Frag frag(const char* lds, int row, int s, int h) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const bf16x8*>(lds + at(row, 2 * s + h));
    } else {
      const f32x4 x = *reinterpret_cast<const f32x4*>(lds + at(row, 4 * s + 2 * h));
      const f32x4 y = *reinterpret_cast<const f32x4*>(lds + at(row, 4 * s + 2 * h + 1));
      return f32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  }

  // Fragment of the transposed tile: lane's row is element 32 dt + l % 32, slot j of
  // half h is tile row r0 + 8 (j / 4) + 4 h + j % 4 (r0 a multiple of 16). bf16: two
  // transposing reads, in which lanes 4 r .. 4 r + 3 of a group of 16 give the
  // group's row r (16 elements) and lane i takes element i of the 4 rows.
  static __device__ __forceinline__ Frag frag_t(const char* lds, int r0, int dt, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int row = 4 * h + ((lane >> 2) & 3), d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char *p = lds + r0 * kPitch + at(row, d >> 3) + (d & 7) * 2, *p8 = lds + r0 * kPitch + at(row + 8, d >> 3) + (d & 7) * 2;
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p8);
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(bf16x8, s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
    } else {
      const int d = 32 * dt + (lane & 31);
      f32x8 f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int row = 8 * (j >> 2) + 4 * h + (j & 3);
        f[j] = *reinterpret_cast<const float*>(lds + r0 * kPitch + at(row, d >> 2) + (d & 3) * 4);
      }
      return f;
    }
  }

  // Fragment from memory: row pointer p (NULL: zeros) of hd elements.
  static __device__ __forceinline__ Frag frag_global(const T* p, int s, int h, int hd) {
    Frag f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (T)0.0f;
    if (p != nullptr && 16 * s + 8 * h < hd) f = *reinterpret_cast<const Frag*>(p + 16 * s + 8 * h);
    return f;
  }
};

// The fragments' loads are waited for here: otherwise the wait lands at their first use
// inside a loop, where it also waits for the loads in flight of the tile after next.
template <typename Frag, int N>
__device__ __forceinline__ void settle(Frag (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+v"(f[i]));
}

// Order of a block of N products, each with R reads from LDS, and N2 more with R2: the reads
// of kAhead products first, then a product and the reads of a later one in turn. Left to
// itself the scheduler puts a read, its wait and its product one after another, and every
// product waits out the latency.
template <int N, int R, int N2 = 0, int R2 = 0>
__device__ __forceinline__ void order_products() {
  constexpr int kMfma = 0x008, kRead = 0x100, kAhead = 6;
  __builtin_amdgcn_sched_group_barrier(kRead, kAhead * R, 0);
#pragma unroll
  for (int i = 0; i < N + N2; i++) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    if (i + kAhead < N)
      __builtin_amdgcn_sched_group_barrier(kRead, R, 0);
    else if (N2 > 0 && i + kAhead < N + N2)
      __builtin_amdgcn_sched_group_barrier(kRead, R2, 0);
  }
}

// A tile on its way from memory to LDS through registers: load() reads rows 0 ..
// nrows - 1 (the rest, and elements from hd on, are zeros: a buffer load past
// its range gives 0), store() writes them. `stride` is in elements and at most
// kMaxStride, so that a tile's byte offsets fit 32 bits.
constexpr int64_t kMaxTileStride = (int64_t)1 << 22;

template <typename T, int HD, int ROWS, int THREADS>
struct Stage {
  using TL = Tile<T, HD>;
  static constexpr int kTotal = ROWS * TL::kPieces;
  static constexpr int N = (kTotal + THREADS - 1) / THREADS;
  u32x4 x[N];

  __device__ __forceinline__ void load(const T* base, int64_t stride, int nrows, int hd, int tid) {
    const uint32_t sb = (uint32_t)(stride * (int64_t)sizeof(T));
    const int have = nrows > ROWS ? ROWS : nrows;
    const uint32_t range = have > 0 ? (uint32_t)(have - 1) * sb + (uint32_t)hd * sizeof(T) : 0u;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, (int)range, 0x00027000);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int id = tid + i * THREADS, row = id / TL::kPieces, c = id % TL::kPieces;
      const bool ok = c * TL::kPiece < hd && id < kTotal;
      const uint32_t off = ok ? (uint32_t)row * sb + (uint32_t)c * 16u : 0xFFFFFFF0u;
      x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
    }
  }
  __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int id = tid + i * THREADS, row = id / TL::kPieces, c = id % TL::kPieces;
      if (kTotal % THREADS == 0 || id < kTotal) *reinterpret_cast<u32x4*>(lds + TL::at(row, c)) = x[i];
    }
  }
};

// Workgroups of 256 threads in one launch: HIP takes fewer than 2^32 threads.
constexpr int64_t kMaxGroups = ((int64_t)1 << 24) - 1;

// The sequence and its tile that slot `slot` of a packed batch stands for. With
// tiles of `rows` rows, sequence b takes the slots floor(cu[b] / rows) + b up to
// floor(cu[b + 1] / rows) + b, at least as many as it has tiles: the grid is known
// without reading cu, and the slots left over end at once. cu is clamped to [0, total].
struct TileSpan {
  int64_t begin;  // first row of the sequence
  int len;        // its rows (0: the slot is empty)
  int row0;       // first row of the tile, in the sequence
  int seq;
};

__device__ __forceinline__ int64_t clamp_cu(const int32_t* cu, int64_t b, int64_t total) {
  const int64_t x = cu[b];
  return x < 0 ? 0 : x > total ? total : x;
}

// How many of the first n items, in order, `holds` is true for (true for a first part of them,
// false after it), by the whole wave: 64 items spread over what is left at a time.
template <typename F>
__device__ __forceinline__ int count_first(int n, F holds) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (;;) {
    const int step = (n + 63) / 64, at = lane * step;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < n && holds(lo + at)));
    if (step <= 1 || c == 0) return lo + c;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
}

__device__ __forceinline__ TileSpan tile_of_slot(const int32_t* cu, int batch, int64_t total, int rows, int64_t slot) {
  // the last sequence whose first slot is not past `slot`
  const int n = count_first(batch, [&](int b) { return clamp_cu(cu, b, total) / rows + b <= slot; });
  TileSpan t{0, 0, 0, 0};
  if (n == 0) return t;
  t.seq = n - 1;
  t.begin = clamp_cu(cu, t.seq, total);
  const int64_t end = clamp_cu(cu, n, total), row0 = (slot - (t.begin / rows + t.seq)) * rows;
  if (row0 < 0 || row0 >= end - t.begin) return t;  // (< 0: cu is not in order)
  t.len = (int)(end - t.begin);
  t.row0 = (int)row0;
  return t;
}

__host__ __device__ __forceinline__ int64_t tile_slots(int64_t total, int64_t batch, int rows) {
  return total / rows + batch;
}

}  // namespace rq
