// How many pages a sequence takes: arithmetic without HIP calls, so that it can be
// checked apart from the kernels (pages.hip).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define PAGES_HD __host__ __device__ __forceinline__
#else
#define PAGES_HD inline
#endif

namespace praghip {

PAGES_HD int pages_for(int64_t tokens, int shift) { return int((tokens + (1ll << shift) - 1) >> shift); }

// New pages of a sequence that grows by `more` from `old` tokens, -1 where a row of `width`
// pages, or a length's 32 bits, does not hold them.  64 bits, for a call's sum: 8192
// sequences of up to 2^31 - 1.
PAGES_HD int64_t new_pages(int64_t old, int64_t more, int64_t width, int shift) {
  const int64_t now = old + more;
  if (old < 0 || more < 0 || now > width << shift || now > INT32_MAX) return -1;
  return pages_for(now, shift) - pages_for(old, shift);
}

}  // namespace praghip
