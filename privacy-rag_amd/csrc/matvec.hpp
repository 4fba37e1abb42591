// Few-row products with 4-bit weights (matvec.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace praghip {

struct MatvecArgs {
  const void* x;  // [m][k]
  int64_t x_stride;
  const uint8_t* w;  // [n][width bytes]
  int64_t w_stride;
  const void* scales;  // [n][groups]
  int64_t scale_stride;
  const uint8_t* zeros;  // [n][groups] or null
  int64_t zero_stride;
  void* y;  // [m][n]
  int64_t y_stride;
  int m, k, n, group, width;
  bool aligned;        // 16-byte loads of x and w stay within their rows
  bool vector_scales;  // eight scales, and eight zero points, are one aligned load
};

hipError_t launch_matvec_w4(const MatvecArgs& a, int type, hipStream_t s);

}  // namespace praghip
