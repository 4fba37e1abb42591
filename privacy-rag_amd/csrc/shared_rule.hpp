// Which entry of a table a wave of the shared prefixes' attention looks up: arithmetic without
// HIP calls, so that it can be checked apart from the kernel (attention_shared.hip).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define SHARED_HD __host__ __device__ __forceinline__
#else
#define SHARED_HD inline
#endif

namespace praghip {

// The entry of either 16 keys of a block of 32, or the table's last one beyond it.  A wave looks
// up to eight blocks ahead, beyond a table of 2^31 positions too: its keys are numbers without
// a sign.
SHARED_HD uint32_t entry_at(uint32_t block, uint32_t half, int page_shift, uint32_t last) {
  const uint32_t entry = ((block << 5) + 16 * half) >> page_shift;
  return entry < last ? entry : last;
}

}  // namespace praghip
