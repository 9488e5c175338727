// prompt.h — arguments of the attention over packed prompts (prompt.hip, prompt_bwd.hip).
#pragma once

#include "rq_internal.h"

namespace rq {

// Rows are q, k, v, out rows of the packed batch; strides in elements.
struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  int64_t rows_q, rows_k, slots, q_slots, k_slots;
  int batch, n_q, n_kv, head_dim, causal, cu_count;
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
};

struct PromptBwdPlan {
  int nsplit;
  int64_t groups;  // of the largest launch
  size_t delta_bytes, work;
};
PromptBwdPlan plan_prompt_bwd(int64_t batch, int64_t rows_q, int64_t rows_k, int64_t n_q, int64_t n_kv,
                              int64_t head_dim);

// queries of a workgroup of the kernel that launch_prompt_fwd takes: 32, 64 (both the split kernel), 128 or 256 (pair)
int prompt_fwd_tile(int dtype, const PromptArgs& a);
hipError_t launch_prompt_fwd(int dtype, const PromptArgs& a, hipStream_t stream);
hipError_t launch_prompt_bwd(int dtype, const PromptArgs& a, hipStream_t stream);

}  // namespace rq
