// Rows of a root-mean-square norm, with the residual's addition before it:
//   s = x + r,   y = s w / sqrt(mean s^2 + eps)
// s is a 32-bit sum, rounded once where it is kept (total) and not at all where the norm
// reads it; the mean is a 32-bit sum too, of parts that are 64-bit ones in the widest rows.
//
// Bytes bound it: each of x, r, y and s moves once, so a row stays in registers between its
// sum and its output.  A row of up to 2048 values is a wave's, whose sum takes lane
// exchanges alone; longer ones are a workgroup's of 256 or 1024 threads, and rows that its
// registers do not hold (beyond 32768 values) are read twice.
//
// A thread takes 8 values at any address (rows of an odd width start anywhere).  A load
// behind a condition would be waited for where the condition ends, so all are made: those of
// the last values, and of threads beyond them, from the row's last eight.  What two threads
// then hold counts once, and both write the same to it.
//
// Measured: 8,192 rows of 1,024 with the addition 11 us for 67 MB (6.1 TB/s, from the caches in
// part; a large copy has 5.1), 1,003 rows of 4,099 without it 6.9 us for 16 MB, 8 rows of 1,024
// 2.8 us, one launch's latency.
#include "norm.hpp"

#include <algorithm>

#include "attention.hpp"

namespace praghip {
namespace {

// Workgroups of a grid's row: a launch has below 2^32 threads in one dimension.
constexpr int64_t kSlab = 1 << 18;
__device__ __forceinline__ int64_t group_index() { return int64_t(blockIdx.y) * kSlab + blockIdx.x; }

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of 16-bit data

// Eight values of a row from i on.  WHOLE: i + 8 <= n; else zeros beyond n.
template <bool WHOLE, typename T>
__device__ __forceinline__ u32x4 load8(const T* row, int i, int n) {
  if (WHOLE || i + 8 <= n) return *reinterpret_cast<const u32x4_any*>(row + i);
  u32x4 v = {0, 0, 0, 0};
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (i + j < n) v[j / 2] |= uint32_t(p[i + j]) << (16 * (j & 1));
  return v;
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store8(T* row, int i, int n, u32x4 v) {
  if (WHOLE || i + 8 <= n) {
    *reinterpret_cast<u32x4_any*>(row + i) = v;
    return;
  }
  uint16_t* p = reinterpret_cast<uint16_t*>(row);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (i + j < n) p[i + j] = uint16_t(v[j / 2] >> (16 * (j & 1)));
}

template <typename T>
__device__ __forceinline__ void widen8(u32x4 x, float (&s)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t v = x[j];
    s[2 * j] = low<T>(v), s[2 * j + 1] = high<T>(v);
  }
}
template <typename T>
__device__ __forceinline__ u32x4 packed8(const float (&s)[8]) {
  return u32x4{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3]), pack2<T>(s[4], s[5]), pack2<T>(s[6], s[7])};
}

// The sum over a row's threads, in an order that their number alone decides.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += lds[w];
  }
  return v;
}
__device__ __forceinline__ float factor(const NormArgs& a, float sum) { return 1.f / sqrtf(sum / float(a.n) + a.eps); }

// Rows of 8 values or more, held: THREADS x CHUNKS x 8 >= n.  A workgroup of 256 has 256 /
// THREADS rows.
template <typename T, int THREADS, int CHUNKS, bool ADD>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) add_norm_kernel(NormArgs a) {
  __shared__ float lds[16];
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  const int t = threadIdx.x % THREADS;
  const int64_t row = group_index() * kRows + threadIdx.x / THREADS;
  if (row >= a.rows) return;  // (a whole wave's, or the workgroup's)
  const T *x = static_cast<const T*>(a.x) + row * a.x_row, *r = static_cast<const T*>(a.residual) + row * a.residual_row;
  u32x4 xs[CHUNKS], rs[CHUNKS], w[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = min((c * THREADS + t) * 8, a.n - 8);
    xs[c] = load8<true>(x, i, a.n);
    if constexpr (ADD) rs[c] = load8<true>(r, i, a.n);
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) w[c] = load8<true>(static_cast<const T*>(a.weight), min((c * THREADS + t) * 8, a.n - 8), a.n);
  float s[CHUNKS][8];
  float sum = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * THREADS + t) * 8, before = i - min(i, a.n - 8);  // values that are a neighbour's
    widen8<T>(xs[c], s[c]);
    if constexpr (ADD) {
      float add[8];
      widen8<T>(rs[c], add);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[c][j] += add[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += j >= before ? s[c][j] * s[c][j] : 0.f;
  }
  const float by = factor(a, row_sum<THREADS>(sum, lds));
  T *out = static_cast<T*>(a.out) + row * a.out_row, *total = static_cast<T*>(a.total) + row * a.total_row;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * THREADS + t) * 8;
    if (i >= a.n) continue;
    float y[8];
    widen8<T>(w[c], y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= s[c][j] * by;
    store8<true>(out, min(i, a.n - 8), a.n, packed8<T>(y));
    if (ADD && a.total) store8<true>(total, min(i, a.n - 8), a.n, packed8<T>(s[c]));
  }
}

// Rows of any width, by 1024 threads that read them twice (a row's values are written by the
// thread that has read them, so that total may be the residual's memory here too).
template <typename T>
__global__ void __launch_bounds__(1024) add_norm_any_kernel(NormArgs a) {
  __shared__ float lds[16];
  const int64_t row = group_index();
  if (row >= a.rows) return;
  const T *x = static_cast<const T*>(a.x) + row * a.x_row, *r = static_cast<const T*>(a.residual) + row * a.residual_row;
  T *out = static_cast<T*>(a.out) + row * a.out_row, *total = static_cast<T*>(a.total) + row * a.total_row;
  const auto summed = [&](int i, float(&s)[8]) {
    widen8<T>(load8<false>(x, i, a.n), s);
    if (a.residual) {
      float add[8];
      widen8<T>(load8<false>(r, i, a.n), add);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += add[j];
    }
  };
  // (a thread has up to 2^20 squares of a row: 32 bits lost up to 2^-6 of their sum)
  float s[8];
  double sum = 0;
  for (int64_t i = threadIdx.x * 8; i < a.n; i += 1024 * 8) {
    summed(int(i), s);
    float some = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) some += s[j] * s[j];
    sum += some;
  }
  const float by = factor(a, row_sum<1024>(float(sum), lds));
  for (int64_t i = threadIdx.x * 8; i < a.n; i += 1024 * 8) {
    summed(int(i), s);
    float y[8];
    widen8<T>(load8<false>(static_cast<const T*>(a.weight), int(i), a.n), y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= s[j] * by;
    store8<false>(out, int(i), a.n, packed8<T>(y));
    if (a.total) store8<false>(total, int(i), a.n, packed8<T>(s));
  }
}

dim3 grid_of(int64_t groups) { return dim3(unsigned(std::min(groups, kSlab)), unsigned((groups + kSlab - 1) / kSlab)); }

template <typename T, int THREADS, int CHUNKS>
void launch_held(const NormArgs& a, hipStream_t s) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  hipLaunchKernelGGL((a.residual ? add_norm_kernel<T, THREADS, CHUNKS, true> : add_norm_kernel<T, THREADS, CHUNKS, false>),
                     grid_of((a.rows + kRows - 1) / kRows), dim3(THREADS < 256 ? 256 : THREADS), 0, s, a);
}

template <typename T>
hipError_t launch(const NormArgs& a, hipStream_t s) {
  if (a.n < 8 || a.n > 1024 * 32)
    hipLaunchKernelGGL((add_norm_any_kernel<T>), grid_of(a.rows), dim3(1024), 0, s, a);
  else if (a.n <= 512)
    launch_held<T, 64, 1>(a, s);
  else if (a.n <= 1024)
    launch_held<T, 64, 2>(a, s);
  else if (a.n <= 2048)
    launch_held<T, 64, 4>(a, s);
  else if (a.n <= 4096)
    launch_held<T, 256, 2>(a, s);
  else if (a.n <= 8192)
    launch_held<T, 256, 4>(a, s);
  else if (a.n <= 16384)
    launch_held<T, 1024, 2>(a, s);
  else
    launch_held<T, 1024, 4>(a, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_add_norm(const NormArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch<_Float16>(a, s) : launch<__bf16>(a, s);
}

}  // namespace praghip
