// prompt.h — arguments of the attention over packed prompts (prompt.hip, prompt_bwd.hip).
#pragma once

#include "rq_internal.h"

namespace rq {

// Rows are q, k, v, out rows of the packed batch; strides in elements.
struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  int64_t rows_q, rows_k, slots, q_slots, k_slots;
  int batch, n_q, n_kv, head_dim, causal, cu_count;
  int window, sinks;  // keys that a query sees up to itself and, before those, of the first ones; 0, 0: all
  float scale, scale2;  // scale2 = scale log2 e
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  void* out;
  int64_t out_stride;
  float* lse;  // [n_q][rows_q], natural logarithm, or NULL
  // gradient only
  const void* dout;
  int64_t dout_stride;
  void *dq, *dk, *dv;
  int64_t dq_stride, dk_stride, dv_stride;
  float* delta;  // [n_q][rows_q]: dout . out
  float* part;   // [nsplit][dv, dk][rows_k][n_kv * head_dim] when nsplit > 1
  int nsplit;
  // With sink_tiles > 0 the gradients of the first sink_tiles tiles of 64 keys of every sequence (few_cut: of more than
  // sink_chunk queries) are summed by chunks of sink_chunk queries: sink_part [sink_slots][nsplit][sink_tiles][n_kv][dv, dk][64][head_dim]
  int sink_tiles, sink_chunk, few_cut;
  int64_t sink_slots;
  float* sink_part;
};

// With a window (WIN) the query at position i of its sequence sees the keys j <= i with i - j < window or
// j < sinks. Whole tiles of keys that no query of a workgroup sees, between the sinks and the first query's
// window, are walked past; what is left is masked where a tile is cut.
template <bool WIN>
struct Seen {  // by one query
  int last;
  __device__ __forceinline__ void init(const PromptArgs& a, int qi, int off, int lk) {
    last = a.causal ? min(lk - 1, qi + off) : lk - 1;
  }
  __device__ __forceinline__ bool sees(int key) const { return key <= last; }
};
template <>
struct Seen<true> {
  int last, first, sinks;
  __device__ __forceinline__ void init(const PromptArgs& a, int qi, int off, int lk) {
    last = min(lk - 1, qi + off);
    first = qi + off - a.window + 1;
    sinks = a.sinks;
  }
  __device__ __forceinline__ bool sees(int key) const { return key <= last && (key >= first || key < sinks); }
};

template <bool WIN>
struct Walk {  // the keys of a workgroup's steps
  __device__ __forceinline__ int leave_out(const PromptArgs&, int, int) { return 0; }
  __device__ __forceinline__ int key(int at) const { return at; }
  __device__ __forceinline__ int rows_from(int key, int lk) const { return lk - key; }  // that are read from `key` on
};
template <>
struct Walk<true> {
  int sink_end, sink_rows, skip;
  // pos: position of the first query, bk: keys of a step. Returns how many keys are left out.
  __device__ __forceinline__ int leave_out(const PromptArgs& a, int pos, int bk) {
    sink_end = (a.sinks + bk - 1) / bk * bk;
    const int begin = max(pos - a.window + 1, 0);
    skip = max(begin / bk * bk - sink_end, 0);
    // behind the sinks, where no query's window reaches, rows are taken as zeros: a NaN in their values must not
    // reach every later query
    sink_rows = begin >= sink_end ? a.sinks : sink_end;
    return skip;
  }
  __device__ __forceinline__ int key(int at) const { return at < sink_end ? at : at + skip; }
  __device__ __forceinline__ int rows_from(int key, int lk) const {
    return (key < sink_end ? min(lk, sink_rows) : lk) - key;
  }
};

// whether the query at `pos` sees by its window or the sinks any, or all, of the n keys from `key` on
template <bool WIN>
__device__ __forceinline__ bool window_any(const PromptArgs& a, int pos, int key, int n) {
  return !WIN || key + n - 1 > pos - a.window || key < a.sinks;
}
template <bool WIN>
__device__ __forceinline__ bool window_all(const PromptArgs& a, int pos, int key, int n) {
  return !WIN || key > pos - a.window || key + n <= a.sinks;
}

struct PromptBwdPlan {
  int nsplit, sink_tiles, sink_chunk, few_cut;
  int64_t groups, sink_slots;  // groups: of the largest launch
  size_t delta_bytes, part_bytes, work;
};
PromptBwdPlan plan_prompt_bwd(const PromptArgs& a);  // of its sizes

// queries of a workgroup of the kernel that launch_prompt_fwd takes: 32, 64 (both the split kernel), 128 or 256 (pair)
int prompt_fwd_tile(int dtype, const PromptArgs& a);
hipError_t launch_prompt_fwd(int dtype, const PromptArgs& a, hipStream_t stream);
hipError_t launch_prompt_bwd(int dtype, const PromptArgs& a, hipStream_t stream);

}  // namespace rq
