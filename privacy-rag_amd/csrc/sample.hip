// Tokens drawn from rows of logits with given random numbers:
//   w_i = exp((x_i - max x) / T);  of the order by falling x, then rising i, the first k stay;
//   of those the shortest run whose sum reaches p times theirs;  of those the ones with w_i at
//   least min_p;  the token is the first, by i, up to which the sum of w is above u times
//   the sum of all that stay.
// Which token that is must not depend on the order of a sum, so weights are whole numbers: w
// in units of 2^-43 (of the power of two above the largest), from 64-bit products, added as
// integers of 64 bits.  A weight below 2^-45 of the largest counts as none.
//
// Reading the logits bounds it, and beside that the weights' 64-bit instructions, some 15 a
// token: a row is cut into parts of kPart tokens for a workgroup each.  Sorting nothing, the
// cuts are found in bins of 1/16 of a power of two:
// * the first kernel puts its part's counts and sums into bins (LDS, then the workspace),
//   relative to the part's own maximum, whose bin is a whole number of powers of two from any
//   other part's, so that parts are added by shifting;
// * in the second every part adds the row's bins, finds those in which a cut falls, and
//   appends its own tokens of those bins to the row's list.  The part that is done last cuts
//   the listed bins by value and index (digits of 10 bits), adds what stays of each part,
//   takes the part that the random number falls into and goes through that one by index.
// No part waits for another.  The order of the list changes nothing: sums are of integers,
// and cuts are by value and index.
#include "sample.hpp"

#include <climits>

#include "attention.hpp"

namespace praghip {

struct SamplePart {
  double anchor;  // the power of two at or above the part's largest weight
  uint64_t mass;  // of all its tokens
  float top;      // its largest logit
  uint32_t at;    // and the lowest index of it
};

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kEach = 16, kPart = kThreads * kEach;  // tokens of a thread, in pieces of 8, and of a part
constexpr int kRange = 46, kBins = kRange * 16;      // powers of two that weights span, and their bins
constexpr int kBits = 43;                            // of a weight's fraction
constexpr int kDigit = 10, kDigits = 1 << kDigit;
static_assert(kBins <= kThreads && kDigits == kThreads, "a thread has a bin, and a digit");

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef unsigned long long u64;

// ----------------------------------------------------------- logits, weights
__device__ __forceinline__ float plain(float x) {  // NaN counts as -infinity, +infinity as the largest number
  return fminf(fmaxf(x, kNegInf), 3.402823466e38f);
}
// eight logits from i on, -infinity beyond the row
template <typename T>
__device__ __forceinline__ void load8(const T* row, int i, int n, float (&x)[8]) {
  if (i + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = *reinterpret_cast<const f32x4_any*>(row + i), b = *reinterpret_cast<const f32x4_any*>(row + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4_any*>(row + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t v = a[j];
        x[2 * j] = low<T>(v), x[2 * j + 1] = high<T>(v);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < n ? float(row[i + j]) : kNegInf;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = plain(x[j]);
}

// What weights are relative to: a largest logit, the units of a logit, the anchor's distance.
struct Scale {
  double top, by, from;  // w = 2^((x - top) by + from), from in [-1, 0]
  double anchor;
};
__device__ __forceinline__ Scale scale_of(float top, float temperature) {
  Scale s;
  s.top = top;
  s.by = 1.4426950408889634074 / fmax(double(temperature), 1e-30);
  // (written out as one product and one addition: both kernels are to have the same bits.  Of
  // products beyond 2^52, whose fraction is lost, any distance is right: their tokens are
  // equal or too far apart to count)
  s.anchor = ceil(s.top * s.by);
  s.from = fmax(fmin(__builtin_fma(s.top, s.by, -s.anchor), 0.), -1.);
  return s;
}
// 2^y in units of 2^-kBits and its bin, of y in (-kRange, 0]: y in 1/256 by a table of their
// powers, the rest by the exponential series (z^4 / 24 is below 2^-42).
struct Weight {
  uint32_t bin;
  double units;
  __device__ __forceinline__ u64 whole() const {  // rounded to nearest
    return __builtin_bit_cast(u64, units + 4503599627370496.0) & ((u64(1) << 52) - 1);
  }
};
__device__ __forceinline__ double exponent(const Scale& s, float x) { return __builtin_fma(double(x) - s.top, s.by, s.from); }
__device__ __forceinline__ bool counts(double y) { return y > -kRange + 0.5; }  // (so that its bin exists)
__device__ __forceinline__ Weight weight(double y, const double* table) {
  constexpr double magic = 6755399441055744.0 / 256;  // 1.5 2^52 in units of 1/256
  const double moved = y + magic;
  const int n = int(uint32_t(__builtin_bit_cast(u64, moved)));
  const double z = (y - (moved - magic)) * 0.69314718055994530942;
  const double power = __builtin_fma(__builtin_fma(__builtin_fma(z, 1. / 6, 0.5), z, 1.), z, 1.) * table[n & 255];
  Weight w;
  w.bin = uint32_t(-n) >> 4;
  w.units = __builtin_bit_cast(double, __builtin_bit_cast(u64, power) + (u64(int64_t(n >> 8)) << 52));
  return w;
}
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 256) table[threadIdx.x] = ldexp(exp2(threadIdx.x / 256.), kBits);
}

struct Filters {
  float temperature, top_p, min_p;
  int top_k;
  __device__ __forceinline__ bool greedy() const { return !(temperature > 0); }
  __device__ __forceinline__ bool by_count() const { return top_k > 0; }
  __device__ __forceinline__ bool by_mass() const { return top_p < 1; }
  __device__ __forceinline__ bool by_weight() const { return min_p > 0; }
  __device__ __forceinline__ bool any() const { return by_count() || by_mass() || by_weight(); }
};
__device__ __forceinline__ Filters filters_of(const SampleArgs& a, int row) {
  Filters f;
  f.temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  f.top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  f.min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  f.top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  if (f.top_k >= a.vocab) f.top_k = 0;
  return f;
}

// --------------------------------------------------------- over the workgroup
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ u64 group_sum(u64 v, u64* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += lds[w];
  return v;
}
// the sum of the threads before, and with this one
template <typename V>
__device__ __forceinline__ V group_scan(V v, V* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const V up = __shfl_up(v, d, 64);
    if (int(threadIdx.x & 63) >= d) v += up;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < int(threadIdx.x >> 6); ++w) v += lds[w];
  return v;
}
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, uint32_t(__shfl_xor(int(v), d, 64)));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = max(v, lds[w]);
  return v;
}

// `share` (0 up to 1) times `of`, exactly, rounded down or up
__device__ __forceinline__ u64 times(float share, u64 of, bool up) {
  const uint32_t v = __builtin_bit_cast(uint32_t, share), e = v >> 23;
  const uint32_t digits = e ? (v & 0x7fffff) | 0x800000 : v & 0x7fffff;
  const unsigned __int128 product = (unsigned __int128)of * digits;
  const int shift = 150 - int(e ? e : 1);  // 23 and more
  if (shift > 100) return up && product ? 1 : 0;
  const u64 whole = u64(product >> shift);
  return whole + (up && (product & ((((unsigned __int128)1) << shift) - 1)) ? 1 : 0);
}

// larger for larger logits
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t v = __builtin_bit_cast(uint32_t, x + 0.f);  // (-0 as 0)
  return v >> 31 ? ~v : v | 0x80000000u;
}

// ------------------------------------------------------------ parts into bins
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_bins_kernel(SampleArgs a) {
  __shared__ u64 mass[kBins], sums[kWaves];
  __shared__ uint32_t count[kBins], tops[kWaves];
  __shared__ double table[256];
  const int part = blockIdx.x, row = blockIdx.y, first = part * kPart;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row;
  const Filters f = filters_of(a, row);
  float x[kEach / 8][8];
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) load8(logits, first + (i * kThreads + int(threadIdx.x)) * 8, a.vocab, x[i]);
  if (int(threadIdx.x) < kBins) mass[threadIdx.x] = 0, count[threadIdx.x] = 0;
  fill_table(table);
  if (part == 0 && threadIdx.x < 2) a.state[2 * row + threadIdx.x] = 0;
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[i][j]);
  const uint32_t key = group_max(key_of(top), tops);
  top = __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
  SamplePart* out = a.part + row * a.parts + part;
  if (f.greedy()) {
    uint32_t at = 0;  // the lowest index as the largest complement
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x[i][j] == top) at = max(at, ~uint32_t(first + (i * kThreads + int(threadIdx.x)) * 8 + j));
    at = group_max(at, tops);
    if (threadIdx.x == 0) *out = {0, 0, top, ~at};
    return;
  }
  const Scale s = scale_of(top, f.temperature);
  u64 total = 0;
  if (top > kNegInf) {
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double y = exponent(s, x[i][j]);
        if (counts(y)) {
          const Weight w = weight(y, table);
          const u64 units = w.whole();
          total += units;
          if (f.any()) {
            atomicAdd(&mass[w.bin], units);
            if (f.by_count()) atomicAdd(&count[w.bin], 1u);
          }
        }
      }
  }
  total = group_sum(total, sums);
  if (threadIdx.x == 0) *out = {s.anchor, total, top, 0};
  if (f.any() && int(threadIdx.x) < kBins) {
    const size_t at = (size_t(row) * a.parts + part) * kBins + threadIdx.x;
    a.mass[at] = mass[threadIdx.x];
    if (f.by_count()) a.count[at] = count[threadIdx.x];
  }
}

// ------------------------------------------------------------------- the cuts
// The order's part that stays: logits above `key`, and those of `key` up to index `last`.
struct Cut {
  uint32_t key;
  int last;
};
constexpr int kHeld = 4;  // listed tokens that a thread holds (beyond them they are read again)

template <typename T>
struct Row {
  const SampleArgs& a;
  const T* logits;
  const SamplePart* part;
  Filters f;
  Scale s;  // of the whole row
  const double* table;
  // a token's weight, and its bin as its own part has counted it
  __device__ __forceinline__ float logit(int i) const { return plain(float(logits[i])); }
  __device__ __forceinline__ int bin_of(int i, float x) const {
    const SamplePart& p = part[i / kPart];
    const double away = s.anchor - p.anchor;
    if (!(away < kRange)) return INT_MAX;
    const double y = exponent(scale_of(p.top, f.temperature), x);
    return counts(y) ? int(weight(y, table).bin) + 16 * int(away) : INT_MAX;
  }
};

// Scratch memory of the last part.
struct Scratch {
  u64 mass[kDigits];
  uint32_t count[kDigits];
  u64 sums[kWaves];
  uint32_t words[kWaves];
  uint32_t found, found_count;
  u64 found_mass;
};

// Counts and masses of the digits that `add` gives, of which the first up to which the count
// (the mass) is above `before`; where that is none, the last that has any, with `before` just
// below it.
struct Found {
  uint32_t digit, count, own_count;  // tokens of the digits before it, and its own
  u64 mass, own_mass;
};
template <typename F>
__device__ __forceinline__ Found find_digit(Scratch& lds, bool by_count, u64& before, F add) {
  lds.mass[threadIdx.x] = 0;
  lds.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) lds.found = kDigits - 1, lds.found_count = 0, lds.found_mass = 0;
  __syncthreads();
  add([&](uint32_t digit, u64 units) {
    atomicAdd(&lds.mass[digit], units);
    atomicAdd(&lds.count[digit], 1u);
  });
  __syncthreads();
  const u64 mass = lds.mass[threadIdx.x];
  const uint32_t count = lds.count[threadIdx.x];
  const u64 mass_to = group_scan<u64>(mass, lds.sums);
  const uint32_t count_to = group_scan<uint32_t>(count, lds.words);
  u64 all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += by_count ? u64(lds.words[w]) : lds.sums[w];
  if (all) before = min(before, all - 1);
  const bool here = by_count ? count && count_to > before && count_to - count <= before : mass && mass_to > before && mass_to - mass <= before;
  if (here) {
    lds.found = threadIdx.x;
    lds.found_count = count_to - count;
    lds.found_mass = mass_to - mass;
  }
  __syncthreads();
  const Found r = {lds.found, lds.found_count, lds.count[lds.found], lds.found_mass, lds.mass[lds.found]};
  __syncthreads();
  return r;
}

// The cut of one listed bin after the tokens whose sum reaches `target` (by_count: after
// `target` tokens), and the mass up to it.
template <typename T, typename E>
__device__ __forceinline__ Cut cut_bin(const Row<T>& row, Scratch& lds, int bin, bool by_count, u64 target, u64& mass_to, E each) {
  uint32_t most = 0, least = 0;  // (the least as the largest complement)
  each([&](int i, float x, int b) {
    if (b != bin) return;
    most = max(most, key_of(x));
    least = max(least, ~key_of(x));
  });
  most = group_max(most, lds.words);
  least = ~group_max(least, lds.words);
  // digits of how far a logit's key lies below the largest; `target` - 1 is before the cut
  uint32_t from = most;
  int shift = max(0, 32 - __clz(int(most - least)) - kDigit);
  u64 before = target - 1, mass = 0;
  Found d;
  for (;;) {
    d = find_digit(lds, by_count, before, [&](auto add) {
      each([&](int i, float x, int b) {
        if (b != bin) return;
        const uint32_t away = from - key_of(x);  // (wraps above `from`: no digit)
        if (away >> shift < kDigits) add(away >> shift, weight(exponent(row.s, x), row.table).whole());
      });
    });
    before -= by_count ? d.count : d.mass;
    mass += d.mass;
    from -= d.digit << shift;
    if (!shift) break;
    shift = max(0, shift - kDigit);
  }
  // tokens of one logit, and of one weight: how many of them, then up to which index
  const u64 own = d.own_count ? d.own_mass / d.own_count : 0;
  const u64 stay = by_count || !own ? before + 1 : before / own + 1;
  if (stay >= d.own_count) {
    mass_to = mass + d.own_mass;
    return {from, INT_MAX};
  }
  mass_to = mass + stay * own;
  uint32_t base = 0;
  u64 left = stay - 1;
  for (int s = kDigit; s >= 0; s -= kDigit) {
    d = find_digit(lds, true, left, [&](auto add) {
      each([&](int i, float x, int b) {
        if (b == bin && key_of(x) == from && (uint32_t(i) - base) >> s < kDigits) add((uint32_t(i) - base) >> s, 0);
      });
    });
    left -= d.count;
    base += d.digit << s;
  }
  return {from, int(base)};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_draw_kernel(SampleArgs a) {
  __shared__ Scratch lds;
  __shared__ u64 mass_to[kBins], part_mass[64];
  __shared__ uint32_t count_to[kBins];
  __shared__ double table[256];
  __shared__ int edges[6], last_one, token;
  const int part = blockIdx.x, row = blockIdx.y;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row;
  const SamplePart* parts = a.part + row * a.parts;
  const Filters f = filters_of(a, row);
  // the row's largest logit, the first part of those that have it
  float top = kNegInf;
  uint32_t at = 0;
  for (int p = 0; p < a.parts; ++p)
    if (parts[p].top > top) top = parts[p].top, at = parts[p].at;
  if (top == kNegInf || f.greedy()) {
    if (part == 0 && threadIdx.x == 0) a.out[row] = top == kNegInf ? -1 : int64_t(at);
    return;
  }
  if (!f.any() && part) return;
  fill_table(table);
  if (threadIdx.x < 64) part_mass[threadIdx.x] = 0;
  if (threadIdx.x < 6) edges[threadIdx.x] = threadIdx.x & 1 ? -1 : kBins;  // empty ranges
  __syncthreads();
  const Row<T> r = {a, logits, parts, f, scale_of(top, f.temperature), table};
  const double least = double(fminf(f.min_p, 1.f)) * weight(r.s.from, table).units;  // of min_p
  Cut cut = {0, INT_MAX};
  int whole = kBins;  // bins before it stay whole

  if (f.any()) {
    // the row's bins: this thread's, and sums up to it
    u64 mass = 0;
    uint32_t count = 0;
    for (int p = 0; p < a.parts; ++p) {
      const double away = r.s.anchor - parts[p].anchor;
      if (!(away < kRange)) continue;
      const int b = int(threadIdx.x) - 16 * int(away);
      if (b >= 0 && b < kBins) {
        const size_t i = (size_t(row) * a.parts + p) * kBins + b;
        mass += a.mass[i] >> int(away);
        if (f.by_count()) count += a.count[i];
      }
    }
    const u64 m = group_scan<u64>(mass, lds.sums);
    const uint32_t n = group_scan<uint32_t>(count, lds.words);
    if (int(threadIdx.x) < kBins) mass_to[threadIdx.x] = m, count_to[threadIdx.x] = n;
    __syncthreads();
    // the bins of the cuts: ranges of which one end may be open until a cut before is known
    const bool counted = f.by_count() && count_to[kBins - 1] > uint32_t(f.top_k);
    if (counted && int(threadIdx.x) < kBins && n >= uint32_t(f.top_k) && n - count < uint32_t(f.top_k)) edges[0] = edges[1] = threadIdx.x;
    __syncthreads();
    const int kbin = counted ? edges[0] : -1;
    const u64 most = counted ? mass_to[kbin] : mass_to[kBins - 1], fewest = counted ? (kbin ? mass_to[kbin - 1] : 0) : most;
    const auto share = [&](u64 of) { return max(u64(1), times(fmaxf(f.top_p, 0.f), of, true)); };  // what a run is to reach
    if (f.by_mass() && int(threadIdx.x) < kBins) {
      if (m >= share(fewest) && m - mass < share(fewest)) edges[2] = threadIdx.x;
      if (m >= share(most) && m - mass < share(most)) edges[3] = threadIdx.x;
    }
    if (f.by_weight() && threadIdx.x == 0) {  // (the logarithm is off by far less than 1/100 of a bin)
      const double y = r.s.from + log2(double(fminf(f.min_p, 1.f)));
      edges[4] = max(0, int(floor(-y * 16 - 0.51)));
      edges[5] = min(kBins - 1, int(floor(-y * 16 + 0.51)));
    }
    __syncthreads();
    // this part's tokens of those bins
    const int e0 = edges[0], e1 = edges[1], e2 = edges[2], e3 = edges[3], e4 = edges[4], e5 = edges[5];
    const double away = r.s.anchor - parts[part].anchor;
    if (away < kRange) {
      const Scale own = scale_of(parts[part].top, f.temperature);
      for (int i = 0; i < kEach / 8; ++i) {
        const int first = part * kPart + (i * kThreads + int(threadIdx.x)) * 8;
        float x[8];
        load8(logits, first, a.vocab, x);
        for (int j = 0; j < 8; ++j) {
          const double y = exponent(own, x[j]);
          if (!counts(y)) continue;
          const int b = int(weight(y, table).bin) + 16 * int(away);
          if ((b >= e0 && b <= e1) || (b >= e2 && b <= e3) || (b >= e4 && b <= e5)) {
            const uint32_t to = atomicAdd(a.state + 2 * row + 1, 1u);
            if (to < uint32_t(a.vocab)) a.list[int64_t(row) * a.vocab + to] = first + j;
          }
        }
      }
    }
    // the part that is done last goes on
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_one = atomicAdd(a.state + 2 * row, 1u) + 1 == uint32_t(a.parts);
    __syncthreads();
    if (!last_one) return;
    __threadfence();
    const int listed = int(min(__hip_atomic_load(a.state + 2 * row + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), uint32_t(a.vocab)));
    const uint32_t* list = a.list + int64_t(row) * a.vocab;
    int held[kHeld], held_bin[kHeld];
    float held_x[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int n = i * kThreads + threadIdx.x;
      held_bin[i] = -1;
      if (n < listed) {
        held[i] = int(list[n]);
        held_x[i] = r.logit(held[i]);
        held_bin[i] = r.bin_of(held[i], held_x[i]);
      }
    }
    const auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (held_bin[i] >= 0) f(held[i], held_x[i], held_bin[i]);
      for (int n = kHeld * kThreads + threadIdx.x; n < listed; n += kThreads) {
        const int i = int(list[n]);
        const float x = r.logit(i);
        f(i, x, r.bin_of(i, x));
      }
    };
    int bin = kBins;  // of the cut
    u64 stays = mass_to[kBins - 1];
    if (counted) {
      bin = kbin;
      cut = cut_bin(r, lds, kbin, true, u64(f.top_k) - (kbin ? count_to[kbin - 1] : 0), stays, each);
      stays += kbin ? mass_to[kbin - 1] : 0;
    }
    if (f.by_mass()) {
      const u64 target = share(stays);
      __syncthreads();
      if (int(threadIdx.x) < kBins && m >= target && m - mass < target) edges[0] = threadIdx.x;
      __syncthreads();
      // (a rounding that puts it outside the listed bins leaves the range's nearer end)
      bin = min(max(edges[0], e2), e3);
      const u64 before = bin ? mass_to[bin - 1] : 0;
      u64 unused;
      const Cut next = cut_bin(r, lds, bin, false, target > before ? target - before : 1, unused, each);
      if (!counted || bin < kbin || next.key > cut.key || (next.key == cut.key && next.last < cut.last)) cut = next;
    }
    whole = min(bin, f.by_weight() ? e4 : kBins);
    // what stays of each part: its whole bins, then the listed tokens one by one
    for (int p = 0; p < a.parts; ++p) {
      const double away = r.s.anchor - parts[p].anchor;
      if (!(away < kRange)) continue;
      const int b = int(threadIdx.x) - 16 * int(away);
      u64 v = 0;
      if (int(threadIdx.x) < whole && b >= 0 && b < kBins) v = a.mass[(size_t(row) * a.parts + p) * kBins + b] >> int(away);
      v = wave_sum(v);
      if ((threadIdx.x & 63) == 0 && v) atomicAdd(&part_mass[p], v);
    }
    each([&](int i, float x, int b) {
      if (b < whole || b >= kBins) return;
      const uint32_t key = key_of(x);
      const Weight w = weight(exponent(r.s, x), table);
      if ((key > cut.key || (key == cut.key && i <= cut.last)) && w.units >= least) atomicAdd(&part_mass[i / kPart], w.whole());
    });
  } else if (int(threadIdx.x) < a.parts) {
    const double away = r.s.anchor - parts[threadIdx.x].anchor;
    part_mass[threadIdx.x] = away < 64 ? parts[threadIdx.x].mass >> int(away) : 0;
  }
  __syncthreads();
  // the part that the random number falls into
  u64 all = 0;
  for (int p = 0; p < a.parts; ++p) all += part_mass[p];
  u64 left = min(times(fminf(fmaxf(a.uniform[row], 0.f), 1.f), all, false), all - 1);
  int mine = 0;
  while (mine < a.parts - 1 && left >= part_mass[mine]) left -= part_mass[mine++];
  // and its tokens by index: sums of each wave's 512, then within the one
  u64 sums[kEach / 8];
  float x[kEach / 8][8];
  const auto units = [&](int i, float v) -> u64 {
    const double y = exponent(r.s, v);
    const uint32_t key = key_of(v);
    if (!counts(y) || key < cut.key || (key == cut.key && i > cut.last)) return 0;
    const Weight w = weight(y, table);
    return f.by_weight() && w.units < least ? 0 : w.whole();
  };
  if (threadIdx.x == 0) token = -1;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) {
    const int first = mine * kPart + (i * kThreads + int(threadIdx.x)) * 8;
    load8(logits, first, a.vocab, x[i]);
    sums[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[i] += units(first + j, x[i][j]);
  }
  __syncthreads();
  u64 before = 0;  // of the pieces before
  bool done = false;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) {
    const u64 to = before + group_scan<u64>(sums[i], lds.sums), from = to - sums[i];
    if (!done && sums[i] && from <= left && left < to) {
      const int first = mine * kPart + (i * kThreads + int(threadIdx.x)) * 8;
      u64 at = from;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u64 w = units(first + j, x[i][j]);
        if (at <= left && left < at + w) token = first + j;
        at += w;
      }
    }
    for (int w = 0; w < kWaves; ++w) before += lds.sums[w];
    __syncthreads();
  }
  // (where roundings leave the number beyond the last token: that one)
  if (token < 0) {
    uint32_t latest = 0;
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = mine * kPart + (i * kThreads + int(threadIdx.x)) * 8 + j;
        if (units(n, x[i][j])) latest = max(latest, uint32_t(n) + 1);
      }
    latest = group_max(latest, lds.words);
    if (threadIdx.x == 0) token = latest ? int(latest) - 1 : -1;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.out[row] = token;
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(unsigned(a.parts), unsigned(a.rows));
  hipLaunchKernelGGL(sample_bins_kernel<T>, grid, dim3(kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_draw_kernel<T>, grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

size_t parts_of(size_t vocab) { return (vocab + kPart - 1) / kPart; }
size_t up(size_t bytes) { return (bytes + 15) / 16 * 16; }
static_assert(kSampleVocab <= size_t(kPart) * 64 && kSampleVocab <= size_t(1) << (2 * kDigit), "parts, and indices, of a row");

}  // namespace

size_t sample_work_bytes(size_t rows, size_t vocab) {
  const size_t parts = parts_of(vocab);
  return up(rows * parts * sizeof(SamplePart)) + rows * parts * kBins * (sizeof(uint64_t) + sizeof(uint32_t)) + rows * 2 * sizeof(uint32_t) +
         rows * vocab * sizeof(uint32_t);
}
void sample_work(SampleArgs& a, void* work) {
  a.parts = int(parts_of(size_t(a.vocab)));
  const size_t items = size_t(a.rows) * a.parts;
  char* at = static_cast<char*>(work);
  a.part = reinterpret_cast<SamplePart*>(at);
  at += up(items * sizeof(SamplePart));
  a.mass = reinterpret_cast<uint64_t*>(at);
  at += items * kBins * sizeof(uint64_t);
  a.count = reinterpret_cast<uint32_t*>(at);
  at += items * kBins * sizeof(uint32_t);
  a.state = reinterpret_cast<uint32_t*>(at);
  a.list = a.state + 2 * size_t(a.rows);
}

hipError_t launch_sample_tokens(const SampleArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F32 ? launch<float>(a, s) : type == PRAGHIP_F16 ? launch<_Float16>(a, s) : launch<__bf16>(a, s);
}

}  // namespace praghip
