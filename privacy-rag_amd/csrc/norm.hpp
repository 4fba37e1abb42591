// Root-mean-square norms with the residual's addition (norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace praghip {

struct NormArgs {
  const void *x, *residual, *weight;  // residual: or null
  void *out, *total;                  // total: or null
  int64_t x_row, residual_row, out_row, total_row;  // strides in elements
  int64_t rows;
  int n;
  float eps;
};

hipError_t launch_add_norm(const NormArgs& a, int type, hipStream_t s);

}  // namespace praghip
