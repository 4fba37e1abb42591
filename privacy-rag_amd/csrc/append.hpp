// New tokens of a step: norms and rotations of queries and keys, and the keys and values
// into the cache's pages (append.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace praghip {

struct AppendArgs {
  const void *q, *k, *v;  // [tokens][heads or kv_heads][dim]; strides in elements
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  void* out;  // [tokens][heads][dim]
  int64_t out_token, out_head;
  const void *q_norm, *k_norm;  // [dim] or null
  float eps;
  const float *cos, *sin;  // [positions][half]
  int64_t cos_row, sin_row;
  int positions, half;
  bool interleaved;
  void *k_pages, *v_pages;
  int64_t kp_page, kp_head, kp_token, vp_page, vp_head, vp_token;
  const int32_t *tables, *lengths, *starts;
  int64_t table_stride;
  int width, seqs, pages, page_shift, heads, kv_heads, dim, tokens;
};

hipError_t launch_page_append(const AppendArgs& a, int type, hipStream_t s);

}  // namespace praghip
