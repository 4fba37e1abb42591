// Products of a few rows with 4-bit weights and group scales:
//   y[m][n] = sum_k x[m][k] (w[n][k] - z[n][k / G]) s[n][k / G]
// with w in 0 .. 15, two to a byte in rows as they are stored (the lower four bits
// first), z 8 where there are no zero points.
//
// Reading the weights bounds it: N K / 2 bytes for 2 M N K operations.  What the
// kernel saves is everything beside that stream: the weights go from memory into the
// matrix cores' operand with two vector instructions per pair, for 16 rows of x at a
// time (a product of one row costs what one of 16 does).
//
// * A lane loads 16 bytes of its column n = lane % 16: 32 values of k, four lanes a
//   column.  Four lane swaps turn the 4 x 4 words of those lanes, after which word s
//   of lane quad g holds k = 32 s + 8 g .. + 7, the operand of step s: each step then
//   stays within a group of 32.
// * A pair is (w >> 4 i) & 0xF000F moved into the fraction of the value 16: 16 + w is
//   exact in both types with no conversion.  It pairs values i and i + 4 of a word, and
//   x is put into that order instead, once for all columns.
// * With a = sum x (16 + w) and X = sum x over a group (a product with ones, exact to
//   the accumulator's rounding), y += s (a - (16 + z) X).  16 is the smallest offset
//   that keeps all 16 values in one binade, so the difference loses at most two bits
//   of the 32-bit sum.
// Waves of a workgroup take K blocks of 128 in turn and add their sums through LDS in
// order.
#include "matvec.hpp"

#include <algorithm>

#include "attention.hpp"

namespace praghip {
namespace {

constexpr int kBlockK = 128;

template <typename T>
struct Nibble;  // where a nibble goes in 16's fraction
template <>
struct Nibble<__bf16> {
  static constexpr int shift = 3;
  static constexpr uint32_t sixteen = 0x41804180u, one = 0x3f803f80u;
};
template <>
struct Nibble<_Float16> {
  static constexpr int shift = 6;
  static constexpr uint32_t sixteen = 0x4c004c00u, one = 0x3c003c00u;
};

template <typename T>
__device__ __forceinline__ u32x4 widen(uint32_t w) {
  using P = Nibble<T>;
  constexpr uint32_t mask = 0x000f000fu << P::shift;
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int by = 4 * i - P::shift;
    r[i] = ((by >= 0 ? w >> by : w << -by) & mask) | P::sixteen;
  }
  return r;
}

// eight values from k on of a row of x, in the order 0 4 1 5 2 6 3 7
template <typename T, bool ALIGNED>
__device__ __forceinline__ u32x4 load_x(const T* row, bool has, int k, int K) {
  u32x4 x = {0, 0, 0, 0};
  if (has && k < K) {
    if (ALIGNED && k + 8 <= K) {
      x = *reinterpret_cast<const u32x4*>(row + k);
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) x[i / 2] |= uint32_t(p[k + i]) << (16 * (i & 1));
    }
  }
  return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}

template <bool ALIGNED>
__device__ __forceinline__ u32x4 load_w(const uint8_t* row, int at, int width) {
  u32x4 w = {0, 0, 0, 0};
  if (at >= width) return w;
  if (ALIGNED) return *reinterpret_cast<const u32x4*>(row + at);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (at + i < width) w[i / 4] |= uint32_t(row[at + i]) << (8 * (i & 3));
  return w;
}

// MT tiles of 16 rows of x, NT tiles of 16 columns a wave, KW waves along K
template <typename T, int MT, int NT, bool ALIGNED, bool ZEROS>
__global__ void __launch_bounds__(256) matvec_w4_kernel(MatvecArgs a, int kw) {
  extern __shared__ float sums[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int part = wave % kw, tile = (blockIdx.x * (4 / kw) + wave / kw) * NT;
  const int m0 = blockIdx.y * 16 * MT, groups = (a.k + a.group - 1) / a.group, steps = a.group / 32;

  f32x4 y[NT][MT];
  const uint8_t* row[NT];
  const T* scale[NT];
  const uint8_t* zero[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min((tile + t) * 16 + col, a.n - 1);
    row[t] = a.w + n * a.w_stride;
    scale[t] = static_cast<const T*>(a.scales) + n * a.scale_stride;
    zero[t] = ZEROS ? a.zeros + n * a.zero_stride : nullptr;
#pragma unroll
    for (int i = 0; i < MT; ++i) y[t][i] = f32x4{0, 0, 0, 0};
  }
  const T* x[MT];
  bool has[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + col;
    has[i] = m < a.m;
    x[i] = static_cast<const T*>(a.x) + (has[i] ? m : 0) * a.x_stride;
  }
  f32x4 acc[NT][MT], ones[MT];
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      ones[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][i] = f32x4{0, 0, 0, 0};
    }
  };
  const auto finish = [&](int g) {
    if (g >= groups) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float s = float(scale[t][g]), c = 16.f + (ZEROS ? float(zero[t][g]) : 8.f);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) y[t][i][r] += s * (acc[t][i][r] - c * ones[i][r]);
    }
    clear();
  };
  clear();
  const u32x4 one = {Nibble<T>::one, Nibble<T>::one, Nibble<T>::one, Nibble<T>::one};
  if (tile * 16 < a.n) {
    for (int kb = part * kBlockK; kb < a.k; kb += kw * kBlockK) {
      u32x4 w[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) w[t] = load_w<ALIGNED>(row[t], kb / 2 + 16 * quad, a.width);
#pragma unroll
      for (int t = 0; t < NT; ++t) {  // the words of four lanes of a column, turned
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto r = __builtin_amdgcn_permlane32_swap(w[t][i], w[t][i + 2], false, false);
          w[t][i] = r[0];
          w[t][i + 2] = r[1];
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const auto r = __builtin_amdgcn_permlane16_swap(w[t][i], w[t][i + 1], false, false);
          w[t][i] = r[0];
          w[t][i + 1] = r[1];
        }
      }
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const int k = kb + 32 * st;
        u32x4 xf[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          xf[i] = load_x<T, ALIGNED>(x[i], has[i], k + 8 * quad, a.k);
          ones[i] = Half<T>::mma16(xf[i], one, ones[i]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const u32x4 wf = widen<T>(w[t][st]);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[t][i] = Half<T>::mma16(xf[i], wf, acc[t][i]);
        }
        // a group ends here, or this wave's part of it does
        if ((k / 32 + 1) % steps == 0 || (st == 3 && kw > 1)) finish(k / a.group);
      }
    }
    if (kw == 1) finish((a.k - 1) / a.group);
  }
  if (kw > 1) {
    float* mine = sums + wave * NT * MT * 256 + lane * 4;
    if (part) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(mine + (t * MT + i) * 256) = y[t][i];
    }
    __syncthreads();
    if (part) return;
    for (int p = 1; p < kw; ++p)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) y[t][i] += *reinterpret_cast<const f32x4*>(mine + (p * NT * MT + t * MT + i) * 256);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = (tile + t) * 16 + col;
    if (n >= a.n) continue;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + 16 * i + 4 * quad + r;
        if (m < a.m) static_cast<T*>(a.y)[m * a.y_stride + n] = T(y[t][i][r]);
      }
  }
}

template <typename T, int MT, int NT>
hipError_t launch(const MatvecArgs& a, int kw, hipStream_t s) {
  const bool z = a.zeros != nullptr;
  const auto kernel = a.aligned ? (z ? matvec_w4_kernel<T, MT, NT, true, true> : matvec_w4_kernel<T, MT, NT, true, false>)
                                : (z ? matvec_w4_kernel<T, MT, NT, false, true> : matvec_w4_kernel<T, MT, NT, false, false>);
  const unsigned tiles = unsigned((a.n + 16 * NT - 1) / (16 * NT)), per = 4 / kw;
  hipLaunchKernelGGL(kernel, dim3((tiles + per - 1) / per, (a.m + 16 * MT - 1) / (16 * MT)), dim3(256),
                     kw > 1 ? 4 * NT * MT * 256 * sizeof(float) : 0, s, a, kw);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const MatvecArgs& a, hipStream_t s) {
  const int tiles = (a.n + 15) / 16, blocks = (a.k + kBlockK - 1) / kBlockK;
  if (tiles >= 4096) return a.m <= 16 ? launch<T, 1, 4>(a, 1, s) : launch<T, 2, 4>(a, 1, s);
  const int kw = blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
  return a.m <= 16 ? launch<T, 1, 1>(a, kw, s) : launch<T, 2, 1>(a, kw, s);
}

}  // namespace

hipError_t launch_matvec_w4(const MatvecArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_type<_Float16>(a, s) : launch_type<__bf16>(a, s);
}

}  // namespace praghip
