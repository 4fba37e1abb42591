// Tokens drawn from rows of logits with given random numbers:
//   w_i = exp((x_i - max x) / T);  of the order by falling x, then rising i, the first k stay;
//   of those the shortest run whose sum reaches p times theirs;  of those the ones with w_i at
//   least min_p;  the token is the first, by i, up to which the sum of w is above u times
//   the sum of all that stay.
// Which token that is must not depend on the order of a sum, so weights are whole numbers: w
// in units of 2^-43 (of the power of two above the largest), from 64-bit products, added as
// integers of 64 bits.  A weight below 2^-44 of the largest counts as none.
//
// Reading the logits bounds it, and beside that the weights' 64-bit instructions, some 15 a
// token: a row is cut into parts of kPart tokens for a workgroup each.  Sorting nothing, the
// cuts are found in bins of 1/16 of a power of two, in three kernels:
// * bins: each part's counts and sums by bin (LDS, then the workspace), relative to the part's
//   own maximum, whose bin is a whole number of powers of two from any other part's, so that
//   parts are added by shifting;
// * list: workgroups of some parts add the row's bins, find those in which a cut falls, and
//   append their tokens of those bins to the row's list;
// * draw: a workgroup a row cuts the listed bins by value and index (few tokens by comparing each
//   with every other, more by digits of 10 bits of both together), adds what stays of each part,
//   takes the part that the random number falls into and goes through that one by index.
// The order of the list changes nothing: sums are of integers, and cuts are by value and index.
//
// Measured: 64 flat rows of 155,648 logits of 32 bits, cut by their sum, 54 us (16 + 19 + 20 by
// kernel; 16 bits without filters 22, where their bytes are 4); 8 rows of 16 bits with all
// filters 25 to 31; one of 32,768 21 (5 + 7 + 9).  Beside the launches, the chains of a row's cuts and its last part are
// what is left, on one workgroup a row.
#include "sample.hpp"

#include <algorithm>
#include <climits>

#include "attention.hpp"

namespace praghip {

struct SamplePart {
  double anchor;  // the power of two at or above the part's largest weight
  uint64_t mass;  // of all its tokens (of a row without filters)
  float top;      // its largest logit
  uint32_t at;    // and the lowest index of it
};

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kEach = 8, kPart = kThreads * kEach;  // tokens of a thread, in pieces of 8, and of a part
constexpr int kParts = kSampleVocab / kPart > 64 ? kSampleVocab / kPart : 64;  // of a row, at most
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
__device__ __forceinline__ Scale scale_by(float top, double by) {
  Scale s;
  s.top = top;
  s.by = by;
  // (written out as one product and one addition: both kernels are to have the same bits.  Of
  // products beyond 2^52, whose fraction is lost, any distance is right: their tokens are
  // equal or too far apart to count)
  s.anchor = ceil(s.top * s.by);
  s.from = fmax(fmin(__builtin_fma(s.top, s.by, -s.anchor), 0.), -1.);
  return s;
}
__device__ __forceinline__ double degrees(float temperature) { return fmax(double(temperature), 1e-30); }
__device__ __forceinline__ Scale scale_of(float top, float temperature) { return scale_by(top, 1.4426950408889634074 / degrees(temperature)); }
// 2^y in units of 2^-kBits and its bin, of y in (-kRange, 0]: y in 1/256 by a table of their
// powers, the rest by the exponential series (its fourth term is below 2^-42).
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
  const double z = y - (moved - magic);  // (the series' coefficients are ln 2, ln^2 2 / 2, ln^3 2 / 6)
  const double power =
      __builtin_fma(__builtin_fma(__builtin_fma(z, 0.055504108664821580, 0.24022650695910071), z, 0.69314718055994531), z, 1.) * table[n & 255];
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
// The lanes before and this one, by moves within rows of 16 lanes and from their last ones.
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CONTROL, ROWS, 0xf, false));
}
template <int CONTROL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
  return u64(moved<CONTROL, ROWS>(uint32_t(v))) | u64(moved<CONTROL, ROWS>(uint32_t(v >> 32))) << 32;
}
template <typename V, typename F>
__device__ __forceinline__ V wave_scan(V v, F with) {
  v = with(v, moved<0x111, 0xf>(v));
  v = with(v, moved<0x112, 0xf>(v));
  v = with(v, moved<0x114, 0xf>(v));
  v = with(v, moved<0x118, 0xf>(v));
  v = with(v, moved<0x142, 0xa>(v));
  return with(v, moved<0x143, 0xc>(v));
}
struct Sum {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Most {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return uint32_t(__builtin_amdgcn_readlane(int(v), 63)); }
__device__ __forceinline__ u64 last_lane(u64 v) { return u64(last_lane(uint32_t(v))) | u64(last_lane(uint32_t(v >> 32))) << 32; }

// The sum up to each of the waves' totals in LDS, for this wave's and of all (kWaves lanes have
// them).
template <typename V>
__device__ __forceinline__ V before_wave(const V* lds, V& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const V own = lane < kWaves ? lds[lane] : 0, to = wave_scan(own, Sum());
  all = last_lane(to);
  const V before = to - own;
  if constexpr (sizeof(V) == 8)
    return u64(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(before)), wave))) | u64(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(before >> 32)), wave))) << 32;
  else
    return uint32_t(__builtin_amdgcn_readlane(int(before), wave));
}
// Sums up to each thread, and of all; all threads call it.
template <typename V>
__device__ __forceinline__ V group_scan(V v, V* lds, V& all) {
  v = wave_scan(v, Sum());
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return v + before_wave(lds, all);
}
__device__ __forceinline__ u64 group_sum(u64 v, u64* lds) {
  u64 all;
  group_scan(v, lds, all);
  return all;
}
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* lds) {
  v = wave_scan(v, Most());
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return last_lane(wave_scan((threadIdx.x & 63) < kWaves ? lds[threadIdx.x & 63] : 0u, Most()));
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

__device__ __forceinline__ float logit_of(uint32_t key) { return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key); }

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
  if (part == 0 && threadIdx.x == 0) a.listed[row] = 0;
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[i][j]);
  top = logit_of(group_max(key_of(top), tops));
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
          if (f.any()) {
            atomicAdd(&mass[w.bin], units);
            if (f.by_count()) atomicAdd(&count[w.bin], 1u);
          } else {
            total += units;
          }
        }
      }
  }
  if (f.any())
    __syncthreads();
  else
    total = group_sum(total, sums);
  if (threadIdx.x == 0) *out = {s.anchor, total, top, 0};
  if (f.any() && int(threadIdx.x) < kBins) {
    const size_t at = (size_t(row) * a.parts + part) * kBins + threadIdx.x;
    a.mass[at] = mass[threadIdx.x];
    if (f.by_count()) a.count[at] = count[threadIdx.x];
  }
}

// --------------------------------------------------------------- what a row has
// The row's largest logit and the first part that has it, the same in all threads; every
// wave finds them for itself.
struct Largest {
  float top;
  int part;
};
__device__ __forceinline__ Largest largest_of(const SamplePart* parts, int count) {
  const int lane = threadIdx.x & 63;
  uint32_t key = 0;
  int part = 0;
  for (int p = lane; p < count; p += 64) {
    const uint32_t k = key_of(parts[p].top);
    if (k > key) key = k, part = p;
  }
  const uint32_t most = last_lane(wave_scan(key, Most()));
  const uint32_t first = ~last_lane(wave_scan(key == most ? ~uint32_t(part) : 0u, Most()));
  return {logit_of(most), int(first)};
}
__device__ __forceinline__ double least_of(const Filters& f, const Scale& s, const double* table) {  // of min_p
  return double(fminf(f.min_p, 1.f)) * weight(s.from, table).units;
}
// what a run of a mass `of` is to reach
__device__ __forceinline__ u64 share_of(const Filters& f, u64 of) { return max(u64(1), times(fmaxf(f.top_p, 0.f), of, true)); }
// a part's bins below the row's, in whole powers of two (kRange: too far to count)
__device__ __forceinline__ int away_of(const Scale& row, const SamplePart& part) {
  const double d = row.anchor - part.anchor;
  return d < kRange ? int(d) : kRange;
}
// A sum of weights in units of their part's largest, as one of the row's units, in which the tokens
// are drawn: nothing where the part's largest weight rounds to none of them (it is half a unit or
// less, and so is the rest), and one at least where it does not, so that a part that is drawn has
// a token with a unit, and one that has none is not drawn.
__device__ __forceinline__ u64 of_row(const Scale& row, u64 sum, float top, int away) {
  return sum && exponent(row, top) > -(kBits + 1) ? max(u64(1), sum >> away) : 0;
}
constexpr int kIndex = 20;  // bits of a token's index
constexpr uint32_t kIndexes = (1u << kIndex) - 1;

// ---------------------------------------------------------- tokens of the cuts' bins
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_list_kernel(SampleArgs a, int parts_each, int groups) {
  __shared__ u64 sums[kWaves], mass_to[kBins];
  __shared__ uint32_t words[kWaves], count_to[kBins], base;
  __shared__ int edges[6], aways[kParts];
  __shared__ float limits[3 * kParts][2];
  // Workgroups go to the eight XCDs in turn: eight rows at a time take turns too, so that a row's
  // are on one, whose L2 then reads the row's bins once (with rows one after the other 55 us for
  // 53).
  const int turn = int(blockIdx.x) / (8 * groups), within = int(blockIdx.x) - turn * 8 * groups;
  const int some = min(a.rows - turn * 8, 8), row = turn * 8 + within % some, group = within / some;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row;
  const SamplePart* parts = a.part + row * a.parts;
  const Filters f = filters_of(a, row);
  if (f.greedy() || !f.any()) return;
  const float top = largest_of(parts, a.parts).top;
  if (top == kNegInf) return;
  const Scale s = scale_of(top, f.temperature);
  if (int(threadIdx.x) < a.parts) aways[threadIdx.x] = away_of(s, parts[threadIdx.x]);
  if (threadIdx.x < 6) edges[threadIdx.x] = threadIdx.x & 1 ? -1 : kBins;  // empty ranges
  __syncthreads();
  // the row's bins: this thread's, and sums up to it
  u64 mass = 0;
  uint32_t count = 0;
  {
    const uint64_t* of = a.mass + size_t(row) * a.parts * kBins;
    const uint32_t* many = a.count + size_t(row) * a.parts * kBins;
    const int bin = min(int(threadIdx.x), kBins - 1);
    const bool has = int(threadIdx.x) < kBins;
    for (int p = 0; p < a.parts; p += 4) {  // (four parts' loads at once, and none behind a condition)
      u64 v[4];
      uint32_t n[4];
      int away[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = min(p + i, a.parts - 1);
        away[i] = p + i < a.parts ? aways[q] : kRange;
        b[i] = bin - 16 * away[i];
        v[i] = of[q * kBins + max(b[i], 0)];
        n[i] = f.by_count() ? many[q * kBins + max(b[i], 0)] : 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool here = has & (b[i] >= 0) & (away[i] < kRange);
        mass += here ? v[i] >> away[i] : 0;
        count += here ? n[i] : 0;
      }
    }
  }
  u64 mass_all;
  uint32_t count_all;
  const u64 m = group_scan(mass, sums, mass_all);
  const uint32_t n = group_scan(count, words, count_all);
  if (int(threadIdx.x) < kBins) mass_to[threadIdx.x] = m, count_to[threadIdx.x] = n;
  // the bins of the cuts; that of a sum lies between two, until the cut by count is known
  const bool counted = f.by_count() && count_all > uint32_t(f.top_k);
  if (counted && n >= uint32_t(f.top_k) && n - count < uint32_t(f.top_k)) edges[0] = edges[1] = threadIdx.x;
  if (f.by_weight() && threadIdx.x == 0) {  // (the logarithm is off by far less than 1/100 of a bin)
    const double y = s.from + log2(double(fminf(f.min_p, 1.f)));
    edges[4] = max(0, int(fmin(floor(-y * 16 - 0.51), double(kBins))));
    edges[5] = min(kBins - 1, int(fmin(floor(-y * 16 + 0.51), double(kBins))));
  }
  __syncthreads();
  if (f.by_mass()) {
    const int kbin = counted ? edges[0] : kBins;
    const u64 most = share_of(f, counted ? mass_to[kbin] : mass_all), fewest = share_of(f, !counted ? mass_all : kbin ? mass_to[kbin - 1] : 0);
    if (m >= fewest && m - mass < fewest) edges[2] = threadIdx.x;
    if (m >= most && m - mass < most) edges[3] = threadIdx.x;
    __syncthreads();
  }
  if (group == 0) {  // for the draw
    if (int(threadIdx.x) < kBins) {
      a.mass_to[size_t(row) * kBins + threadIdx.x] = m;
      a.count_to[size_t(row) * kBins + threadIdx.x] = n;
    }
    if (threadIdx.x < 8) a.edges[size_t(row) * 8 + threadIdx.x] = threadIdx.x < 6 ? edges[threadIdx.x] : int(counted);
  }
  // Tokens whose logit may be in one of those bins, by 32 bits and a little room on both sides
  // (where that is no number, all of them): the draw looks at the few by 64.  The limits of this
  // workgroup's parts are some threads' each (by all threads, 64-bit products took longer than
  // the tokens).
  const int begin = group * parts_each, end = min(begin + parts_each, a.parts);
  if (int(threadIdx.x) < 3 * (end - begin)) {
    const int part = begin + int(threadIdx.x) / 3, r = int(threadIdx.x) % 3;
    const int first = edges[2 * r], last = edges[2 * r + 1], away = aways[part];
    const Scale own = scale_by(parts[part].top, s.by);
    const double each = 0.69314718055994531 * degrees(f.temperature), room = 1e-6 * (fabs(own.top) + 50 * each);
    limits[threadIdx.x][0] = first > last ? kNegInf : float(own.top + ((-16. * (first - 16 * away) + 0.5) / 256 - own.from) * each + room);
    limits[threadIdx.x][1] = first > last ? -kNegInf : float(own.top + ((-16. * (last - 16 * away) - 15.5) / 256 - own.from) * each - room);
  }
  __syncthreads();
  for (int part = begin; part < end; ++part) {
    if (aways[part] == kRange) continue;
    float upper[3], lower[3];
#pragma unroll
    for (int r = 0; r < 3; ++r) upper[r] = limits[3 * (part - begin) + r][0], lower[r] = limits[3 * (part - begin) + r][1];
    uint32_t found = 0;  // a bit for each of the thread's tokens
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i) {
      float x[8];
      load8(logits, part * kPart + (i * kThreads + int(threadIdx.x)) * 8, a.vocab, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bool maybe = false;
#pragma unroll
        for (int r = 0; r < 3; ++r) maybe |= !(x[j] > upper[r]) & !(x[j] < lower[r]);
        if (maybe && x[j] > kNegInf) found |= 1u << (8 * i + j);
      }
    }
    uint32_t all;
    const uint32_t mine = __popc(found);
    uint32_t at = group_scan(mine, words, all) - mine;
    if (!all) continue;
    if (threadIdx.x == 0) base = atomicAdd(a.listed + row, all);
    __syncthreads();
    uint32_t* list = a.list + int64_t(row) * a.vocab;
    for (at += base; found; found &= found - 1) {
      const int bit = __ffs(found) - 1;
      list[at++] = uint32_t(part * kPart + ((bit >> 3) * kThreads + int(threadIdx.x)) * 8 + (bit & 7));
    }
  }
}

// -------------------------------------------------------------------------- draw
// Scratch memory of the cuts.
struct Scratch {
  u64 amount[kDigits];
  uint32_t count[kDigits];
  u64 sums[kWaves];
  uint32_t words[2 * kWaves];
  uint32_t digit;
  u64 before, value;
};
constexpr int kHeld = 4;   // listed tokens that a thread holds (beyond them they are read again)
// Up to so many listed tokens are compared each with every other, by all threads (8 rows of
// 155,648 25 us for 27 by one wave's lanes, 64 rows of 16,384 24 for 33 by digits; at 256, 8 rows
// of 16,384 cut by their sum take 27 for 24).
constexpr int kFew = 128;

// Listed tokens: an index, the logit's key, the bin, the units.
struct Token {
  int index, bin;
  uint32_t key;
  u64 units;
};

// The order within a bin, as one number: how far a logit's key lies below the bin's largest,
// then the index.
__device__ __forceinline__ u64 place_of(uint32_t most, const Token& t) { return u64(most - t.key) << kIndex | u64(t.index); }

// The last token that stays of a bin of `each` token: the first up to which the amounts (1, or
// units, of each) are above `before`, or the last of all.
template <typename E>
__device__ __forceinline__ u64 cut_bin(Scratch& lds, int bin, u64 before, bool by_count, uint32_t most, uint32_t least, E each) {
  u64 from = 0;
  int shift = max(0, 32 - (most > least ? __clz(int(most - least)) : 32) + kIndex - kDigit);
#pragma unroll 1
  for (;;) {
    lds.amount[threadIdx.x] = 0;
    lds.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) lds.digit = 0, lds.before = 0, lds.value = from;
    __syncthreads();
    each([&](const Token& t) {
      const u64 digit = (place_of(most, t) - from) >> shift;  // (wraps below `from`: no digit)
      if (t.bin == bin && digit < kDigits) {
        atomicAdd(&lds.amount[digit], by_count ? 1 : t.units);
        atomicAdd(&lds.count[digit], 1u);
      }
    });
    __syncthreads();
    const u64 mine = lds.amount[threadIdx.x];
    u64 all;
    const u64 to = group_scan(mine, lds.sums, all);
    before = min(before, max(u64(1), all) - 1);  // (changes it the first time alone)
    if (mine && to > before && to - mine <= before) {
      lds.digit = threadIdx.x;
      lds.before = to - mine;
    }
    __syncthreads();
    const uint32_t digit = lds.digit;
    before -= lds.before;
    const bool one = lds.count[digit] <= 1;
    from += u64(digit) << shift;
    if (one || !shift) break;
    __syncthreads();  // all have read them
    shift = max(0, shift - kDigit);
  }
  // the one token of the last digit
  each([&](const Token& t) {
    const u64 place = place_of(most, t);
    if (t.bin == bin && (place - from) >> shift == 0) lds.value = place;
  });
  __syncthreads();
  const u64 value = lds.value;
  __syncthreads();
  return value;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_draw_kernel(SampleArgs a) {
  __shared__ Scratch lds;
  __shared__ u64 part_mass[kParts];
  __shared__ double table[256], from[kParts];
  __shared__ float tops[kParts];
  __shared__ int token, aways[kParts];
  const int row = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row;
  const SamplePart* parts = a.part + row * a.parts;
  const Filters f = filters_of(a, row);
  const Largest largest = largest_of(parts, a.parts);
  if (largest.top == kNegInf || f.greedy()) {
    if (threadIdx.x == 0) a.out[row] = largest.top == kNegInf ? -1 : int64_t(parts[largest.part].at);
    return;
  }
  fill_table(table);
  const Scale s = scale_of(largest.top, f.temperature);
  if (int(threadIdx.x) < kParts) part_mass[threadIdx.x] = 0;
  if (int(threadIdx.x) < a.parts) {
    const SamplePart part = parts[threadIdx.x];
    const int away = away_of(s, part);
    aways[threadIdx.x] = away;
    tops[threadIdx.x] = part.top;
    from[threadIdx.x] = scale_of(part.top, f.temperature).from;
    if (!f.any()) part_mass[threadIdx.x] = of_row(s, part.mass, part.top, away);
  }
  if (threadIdx.x == 0) token = -1;
  __syncthreads();
  const double least = f.by_weight() ? least_of(f, s, table) : 0;
  // what stays: logits above `key`, and those of `key` up to index `last`
  uint32_t key = 0;
  int last = INT_MAX;
  const auto stays = [&](uint32_t k, int i) { return k > key || (k == key && i <= last); };

  if (f.any()) {
    const int* edges = a.edges + size_t(row) * 8;
    const uint64_t* mass_to = a.mass_to + size_t(row) * kBins;
    const int listed = int(min(a.listed[row], uint32_t(a.vocab)));
    const uint32_t* list = a.list + int64_t(row) * a.vocab;
    // a token, with the bin that its part counted it in
    const auto token_of = [&](int i) -> Token {
      const float x = plain(float(logits[i]));
      const int p = i / kPart;
      const double y = __builtin_fma(double(x) - double(tops[p]), s.by, from[p]);
      const bool has = counts(y) && aways[p] < kRange;
      return {i, has ? int(weight(y, table).bin) + 16 * aways[p] : INT_MAX, key_of(x), weight(exponent(s, x), table).whole()};
    };
    Token held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int n = i * kThreads + threadIdx.x;
      held[i] = {0, -1, 0, 0};
      if (i * kThreads < listed) {  // (all lanes load, as others read them)
        held[i] = token_of(int(list[min(n, listed - 1)]));
        if (n >= listed) held[i].bin = -1;
      }
    }
    const auto each = [&](auto with) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (i * kThreads < listed && held[i].bin >= 0) with(held[i]);
#pragma unroll 1
      for (int n = kHeld * kThreads + threadIdx.x; n < listed; n += kThreads) with(token_of(int(list[n])));
    };
    const bool counted = edges[6];
    const int kbin = counted ? edges[0] : kBins, e2 = edges[2], e3 = edges[3], e4 = edges[4];
    int bin = kBins;
    u64 all = mass_to[kBins - 1];
    // the cut by count, then the one by mass of what it leaves
    const auto count_before = [&] { return u64(f.top_k) - 1 - (kbin ? a.count_to[size_t(row) * kBins + kbin - 1] : 0); };
    const auto mass_bin = [&](u64 target) {  // (it is one of the listed range; that is one bin, nearly always)
      int b = e2;
      while (b < e3 && mass_to[b] < target) ++b;
      return b;
    };
    if (listed <= kFew) {
      // Sums up to each token in its bin: `width` threads have a token each, as have the next ones,
      // which look at others; the order is one number, the larger first.
      const int width = listed <= 64 ? 64 : kFew, mine = int(threadIdx.x) & (width - 1);
      if (int(threadIdx.x) < kFew) {
        lds.amount[threadIdx.x] = 0, lds.amount[kFew + threadIdx.x] = held[0].units;
        lds.amount[2 * kFew + threadIdx.x] = u64(held[0].key) << 32 | ~uint32_t(held[0].index);
        lds.count[threadIdx.x] = 0, lds.count[kFew + threadIdx.x] = uint32_t(held[0].bin);
      }
      __syncthreads();
      const u64 order = lds.amount[2 * kFew + mine], units = lds.amount[kFew + mine];
      const int own_bin = int(lds.count[kFew + mine]);
      if (mine < listed) {
        u64 part = 0;
        uint32_t some = 0;
#pragma unroll 4
        for (int n = int(threadIdx.x) / width; n < listed; n += kThreads / width) {
          const bool before = (int(lds.count[kFew + n]) == own_bin) & (lds.amount[2 * kFew + n] >= order);
          part += before ? lds.amount[kFew + n] : 0, some += before;
        }
        if (some) atomicAdd(&lds.amount[mine], part), atomicAdd(&lds.count[mine], some);
      }
      __syncthreads();
      const bool has = int(threadIdx.x) < listed;
      const u64 mass = has ? lds.amount[mine] : 0;  // up to it, in its bin
      const uint32_t count = has ? lds.count[mine] : 0;
      // cuts behind the token of the one thread whose it is; returns whether there is one
      u64 reached = 0;
      const auto take = [&](bool own) {
        if (threadIdx.x == 0) lds.digit = 0;
        __syncthreads();
        if (own) lds.digit = 1, lds.value = order, lds.before = mass;
        __syncthreads();
        const bool found = lds.digit != 0;
        if (found) {
          const uint32_t k = uint32_t(lds.value >> 32);
          const int i = int(~uint32_t(lds.value));
          reached = lds.before;
          if (stays(k, i)) key = k, last = i;
        }
        __syncthreads();
        return found;
      };
      if (counted) {
        bin = kbin;
        take(has && own_bin == bin && count == uint32_t(count_before()) + 1);
        all = (bin ? mass_to[bin - 1] : 0) + reached;
      }
      if (f.by_mass()) {
        const u64 target = share_of(f, all);
        bin = mass_bin(target);
        const u64 to = bin ? mass_to[bin - 1] : 0, need = target > to ? target - to : 1;
        const bool own = has && own_bin == bin;
        if (!take(own && mass >= need && mass - units < need)) {  // (the last of the bin, where roundings leave the sum below)
          const uint32_t most = group_max(own ? count : 0, lds.words);
          take(own && count == most);
        }
      }
    } else {
#pragma unroll 1
      for (int turn = counted ? 0 : 1; turn < (f.by_mass() ? 2 : 1); ++turn) {
        u64 before;  // amounts, in the cut's bin, before the last that stays
        if (turn == 0) {
          bin = kbin;
          before = count_before();
        } else {
          if (counted) {
            u64 mine = 0;
            each([&](const Token& t) {
              if (t.bin == bin && stays(t.key, t.index)) mine += t.units;
            });
            all = group_sum(mine, lds.sums) + (bin ? mass_to[bin - 1] : 0);
          }
          const u64 target = share_of(f, all);
          bin = mass_bin(target);
          const u64 to = bin ? mass_to[bin - 1] : 0;
          before = target > to ? target - to - 1 : 0;
        }
        uint32_t most = 0, complement = 0;  // of the bin's keys
        each([&](const Token& t) {
          if (t.bin == bin) most = max(most, t.key), complement = max(complement, ~t.key);
        });
        most = group_max(most, lds.words);
        complement = group_max(complement, lds.words + kWaves);
        const u64 place = cut_bin(lds, bin, before, turn == 0, most, ~complement, each);
        const uint32_t new_key = most - uint32_t(place >> kIndex);
        const int new_last = int(place & kIndexes);
        if (stays(new_key, new_last)) key = new_key, last = new_last;
      }
    }
    // what stays of each part: its whole bins, a wave for a part, then the listed tokens
    const int whole = min(bin, f.by_weight() ? e4 : kBins);
    for (int p = wave; p < a.parts; p += kWaves) {
      u64 v = 0;
      for (int b = lane; b < min(whole - 16 * aways[p], kBins); b += 64) v += a.mass[(size_t(row) * a.parts + p) * kBins + b];
      v = wave_scan(v, Sum());
      if (lane == 63 && v) atomicAdd(&part_mass[p], of_row(s, v, tops[p], aways[p]));
    }
    each([&](const Token& t) {
      if (t.bin < whole || t.bin >= kBins || !stays(t.key, t.index)) return;
      if (f.by_weight() && weight(exponent(s, plain(float(logits[t.index]))), table).units < least) return;
      atomicAdd(&part_mass[t.index / kPart], t.units);
    });
    __syncthreads();
  }
  // the part that the random number falls into: the parts' masses by lanes, some each
  u64 left;
  int mine = 0;
  {
    constexpr int kLane = kParts / 64;
    u64 own = 0;
#pragma unroll
    for (int i = 0; i < kLane; ++i) own += part_mass[lane * kLane + i];
    const u64 to = wave_scan(own, Sum()), all = last_lane(to);
    left = min(times(fminf(fmaxf(a.uniform[row], 0.f), 1.f), all, false), max(u64(1), all) - 1);
    const int from = max(0, __ffsll((long long)__ballot(to > left)) - 1);
    left -= __shfl(to - own, from, 64);
    mine = from * kLane;
    while (mine < (from + 1) * kLane - 1 && left >= part_mass[mine]) left -= part_mass[mine++];
  }
  // and its tokens by index, kEach neighbours a thread
  const int first = mine * kPart + int(threadIdx.x) * kEach;
  u64 units[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach / 8; ++i) {
    float x[8];
    load8(logits, first + 8 * i, a.vocab, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = 8 * i + j;
      units[n] = 0;
      const double y = exponent(s, x[j]);
      if (stays(key_of(x[j]), first + n) && counts(y)) {
        const Weight w = weight(y, table);
        if (w.units >= least) units[n] = w.whole();
      }
      sum += units[n];
    }
  }
  u64 all;
  u64 at = group_scan(sum, lds.sums, all) - sum;
  // (the part's sum and that of its tokens' rounded units differ a little: the number keeps its
  // distance from the nearer end, so that the first and the last token are drawn at theirs)
  const u64 behind = part_mass[mine] - left;
  left = left < behind ? min(left, all - 1) : all - min(all, behind);
  if (at <= left && left < at + sum) {
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      if (at <= left && left < at + units[n]) token = first + n;
      at += units[n];
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.out[row] = token;
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(unsigned(a.parts), unsigned(a.rows));
  hipLaunchKernelGGL(sample_bins_kernel<T>, grid, dim3(kThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.top_k || a.top_p || a.min_p || a.top_k_all > 0 || a.top_p_all < 1 || a.min_p_all > 0) {
    // as many parts for a workgroup, which adds the row's bins first, as leave one workgroup a CU
    // (64 rows of 155,648, all filters: 53 us for the call; with two a CU 56)
    const int each = std::min((a.parts * a.rows + 255) / 256, a.parts), groups = (a.parts + each - 1) / each;
    hipLaunchKernelGGL(sample_list_kernel<T>, dim3(unsigned(groups * a.rows)), dim3(kThreads), 0, s, a, each, groups);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(sample_draw_kernel<T>, dim3(unsigned(a.rows)), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

size_t parts_of(size_t vocab) { return (vocab + kPart - 1) / kPart; }
size_t up(size_t bytes) { return (bytes + 15) / 16 * 16; }
static_assert(kSampleVocab <= size_t(1) << kIndex && kParts <= kThreads && kParts % 64 == 0, "indexes, and parts, of a row");

}  // namespace

size_t sample_work_bytes(size_t rows, size_t vocab) {
  const size_t parts = parts_of(vocab);
  return up(rows * parts * sizeof(SamplePart)) + rows * (parts + 1) * kBins * (sizeof(uint64_t) + sizeof(uint32_t)) +
         rows * (8 + 1 + vocab) * sizeof(uint32_t);
}
void sample_work(SampleArgs& a, void* work) {
  a.parts = int(parts_of(size_t(a.vocab)));
  const size_t items = size_t(a.rows) * a.parts;
  char* at = static_cast<char*>(work);
  a.part = reinterpret_cast<SamplePart*>(at);
  at += up(items * sizeof(SamplePart));
  a.mass = reinterpret_cast<uint64_t*>(at);
  a.mass_to = a.mass + items * kBins;
  a.count = reinterpret_cast<uint32_t*>(a.mass_to + size_t(a.rows) * kBins);
  a.count_to = a.count + items * kBins;
  a.edges = reinterpret_cast<int32_t*>(a.count_to + size_t(a.rows) * kBins);
  a.listed = reinterpret_cast<uint32_t*>(a.edges + size_t(a.rows) * 8);
  a.list = a.listed + a.rows;
}

hipError_t launch_sample_tokens(const SampleArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F32 ? launch<float>(a, s) : type == PRAGHIP_F16 ? launch<_Float16>(a, s) : launch<__bf16>(a, s);
}

}  // namespace praghip
