// paged.h — arguments of the kernels on a paged key-value cache (paged.hip).
#pragma once

#include "rq_internal.h"

namespace rq {

// Row r of a sequence lies in page table[r >> page_bits] at row r & (2^page_bits - 1);
// a page's rows are n_kv * head_dim values.
struct PagesArgs {
  void *kpages, *vpages;
  int64_t pages;
  const int32_t* table;  // [batch][table_stride]
  int64_t table_stride;  // table entries of a sequence
  int page_bits, n_q, n_kv, head_dim, batch;
  int rope;              // angles pos * 2^(-2 i / head_dim * log2_theta); 0: no rotation
  double log2_theta;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements
};

struct PagedAttnArgs {
  PagesArgs p;
  const int32_t* lens;  // [batch] cached rows, < 0: an idle slot
  int64_t max_len;      // rows that a sequence may have, the new one included
  float scale2;         // scale log2 e
  void* out;
  int64_t out_stride;
  int split_rows, nsplit;  // cached rows of a workgroup, and ranges at max_len
  float* part;             // records of the ranges when nsplit > 1
};

struct PagesAppendArgs {
  PagesArgs p;
  const int32_t *cu, *past;
  int64_t rows;
  void *q_out, *k_out;  // k_out may be NULL
  int64_t q_out_stride, k_out_stride;
};

// Rows of a range and their number for a call's shape; work: bytes of records.
struct PagedPlan {
  int split_rows, nsplit;
  size_t work;
};
PagedPlan plan_paged_attention(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len,
                               int cu_count);
// dtype: of q, k, v and out; cache_dtype: of the pages
hipError_t launch_paged_attention(int dtype, int cache_dtype, const PagedAttnArgs& a, hipStream_t stream);
hipError_t launch_pages_append(int dtype, int cache_dtype, const PagesAppendArgs& a, hipStream_t stream);
// workgroups of one page and plane
int64_t pages_copy_groups(int64_t page_bytes);
// src, dst: n page numbers in host memory, all dst different and none of them a src
hipError_t launch_pages_copy(void* base, int64_t planes, int64_t plane_bytes, int64_t page_bytes, const int32_t* src,
                             const int32_t* dst, int64_t n, hipStream_t stream);

}  // namespace rq
