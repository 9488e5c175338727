// paged.h — arguments of the kernels on a paged key-value cache (paged.hip).
#pragma once

#include <algorithm>

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
  int window, sinks;    // rows that the query sees up to its own and, before those, of the first ones; 0, 0: all
  float scale2;         // scale log2 e
  void* out;
  int64_t out_stride;
  int split_rows, nsplit;  // cached rows of a workgroup, and ranges at max_len
  float* part;             // records of the ranges when nsplit > 1
  // int8 pages: `spare` ranges more than there are sequences (0: a range a sequence), each of a multiple of
  // split_rows rows, or, of a single sequence, of range_rows. The scale of rows 16 i .. 16 i + 15 of a page and of a
  // KV head is scales[page * scale_stride + i * n_kv + head]
  // kv_heads: of a workgroup; ahead: the new row is in the pages already (and k is NULL)
  int spare, range_rows, kv_heads, ahead;
  float *kscales, *vscales;
  int64_t scale_stride;
};

struct PagesAppendArgs {
  PagesArgs p;
  const int32_t *cu, *past;
  int64_t rows;
  void *q_out, *k_out;  // k_out may be NULL
  int64_t q_out_stride, k_out_stride;
  // int8 pages only; cu NULL: row b is the one row of sequence b, and q_out may be NULL
  int64_t max_len;  // rows past it are not stored
  float *kscales, *vscales;
  int64_t scale_stride;
};

// Stored rows as values: sequence b's rows 0, 1, ... to rows cu[b] .. cu[b + 1] - 1 of k_out and v_out.
struct PagesRowsArgs {
  PagesArgs p;
  const int32_t* cu;
  int64_t rows;
  const float *kscales, *vscales;
  int64_t scale_stride;
  void *k_out, *v_out;
  int64_t k_out_stride, v_out_stride;
};

// Rows of a range and their number for a call's shape; work: bytes of records.
struct PagedPlan {
  int split_rows, nsplit;
  size_t work;
};
// max_len: rows that are walked over (walked_rows)
PagedPlan plan_paged_attention(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len,
                               int cu_count);
// The same for int8 pages, whose rows a range the kernel takes from the real lengths.
struct PagedQ8Plan {
  int split_rows, spare, range_rows, kv_heads;
  int64_t groups;  // workgroups of the largest launch
  size_t work;
};
PagedQ8Plan plan_paged_attention_q8(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len,
                                    int cu_count);
// of max_len rows those that a query with a window walks over, whole blocks of 16 at both ends
inline int64_t walked_rows(int64_t max_len, int64_t window, int64_t sinks) {
  return window > 0 ? std::min<int64_t>(max_len, (sinks + 15) / 16 * 16 + window + 16) : max_len;
}
// dtype: of q, k, v and out; cache_dtype: of the pages
hipError_t launch_paged_attention(int dtype, int cache_dtype, const PagedAttnArgs& a, hipStream_t stream);
hipError_t launch_pages_append(int dtype, int cache_dtype, const PagesAppendArgs& a, hipStream_t stream);
// over int8 pages
hipError_t launch_paged_attention_q8(int dtype, const PagedAttnArgs& a, hipStream_t stream);
hipError_t launch_pages_append_q8(int dtype, const PagesAppendArgs& a, hipStream_t stream);
// of blocks: the workgroups that its rows take at least
int64_t append_q8_slots(const PagesAppendArgs& a);
hipError_t launch_pages_rows(int dtype, int cache_dtype, const PagesRowsArgs& a, hipStream_t stream);
// workgroups of one page and plane
int64_t pages_copy_groups(int64_t page_bytes);
// src, dst: n page numbers in host memory, all dst different and none of them a src
hipError_t launch_pages_copy(void* base, int64_t planes, int64_t plane_bytes, int64_t page_bytes, const int32_t* src,
                             const int32_t* dst, int64_t n, hipStream_t stream);

}  // namespace rq
