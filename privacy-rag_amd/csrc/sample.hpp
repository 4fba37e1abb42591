// Tokens drawn from logits (sample.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace praghip {

// A row's arguments: its own where there is a list, else everybody's.
struct SampleArgs {
  const void* logits;  // [rows][vocab]
  int64_t row;         // stride in elements
  int rows, vocab, parts;
  const float *uniform, *temperature, *top_p, *min_p;  // uniform [rows]; the others [rows] or null
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* out;
  // the workspace: what parts hold, their bins, the rows' bins with sums up to each, the bins
  // that cuts fall in (three ranges, and whether top_k cuts), tokens of those bins
  struct SamplePart* part;       // [rows][parts]
  uint64_t *mass, *mass_to;      // [rows][parts][bins], [rows][bins]
  uint32_t *count, *count_to;
  int32_t* edges;                // [rows][8]
  uint32_t *listed, *list;       // [rows], [rows][vocab]
};

constexpr size_t kSampleVocab = size_t(1) << 20;
size_t sample_work_bytes(size_t rows, size_t vocab);
void sample_work(SampleArgs& a, void* work);
hipError_t launch_sample_tokens(const SampleArgs& a, int type, hipStream_t s);

}  // namespace praghip
