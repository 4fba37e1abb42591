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
//   that keeps all 16 values in one binade.  The two sums are 32-bit ones of up to G
//   terms: a group's part of y is off by at most G 2^-24 s sum |x| (32 + w + z), also
//   where w is near z and the part itself is small.
// Waves of a workgroup take K blocks of 128 in turn and add their sums through LDS in
// order.  1024 x 4096, one row: the kernel takes 5.5 us, the host's call 8.0 to 8.6.
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

// The sums of the waves along K, in order, and y's values.
template <typename T, int MT>
__device__ __forceinline__ void finish_rows(const MatvecArgs& a, f32x4 (&y)[MT], float* sums, int kw, int part, int wave,
                                            int lane, int tile, int m0) {
  const int col = lane & 15, quad = lane >> 4;
  if (kw > 1) {
    float* mine = sums + wave * MT * 256 + lane * 4;
    if (part) {
#pragma unroll
      for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(mine + i * 256) = y[i];
    }
    __syncthreads();
    if (part) return;
    for (int p = 1; p < kw; ++p)
#pragma unroll
      for (int i = 0; i < MT; ++i) y[i] += *reinterpret_cast<const f32x4*>(mine + (p * MT + i) * 256);
  }
  const int n = tile * 16 + col;
  if (n >= a.n) return;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + 16 * i + 4 * quad + r;
      if (m < a.m) static_cast<T*>(a.y)[m * a.y_stride + n] = T(y[i][r]);
    }
}

// the words of the four lanes of a column, turned: word s of quad g is word g of quad s
__device__ __forceinline__ u32x4 turned(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[i], w[i + 2], false, false);
    w[i] = r[0];
    w[i + 2] = r[1];
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[i], w[i + 1], false, false);
    w[i] = r[0];
    w[i + 1] = r[1];
  }
  return w;
}

// MT tiles of 16 rows of x, one of 16 columns a wave, kw waves along K: any group
template <typename T, int MT, bool ALIGNED, bool ZEROS>
__global__ void __launch_bounds__(256) matvec_w4_kernel(MatvecArgs a, int kw) {
  extern __shared__ float sums[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int part = wave % kw, tile = blockIdx.x * (4 / kw) + wave / kw;
  const int m0 = blockIdx.y * 16 * MT, groups = (a.k + a.group - 1) / a.group, steps = a.group / 32;

  const int n = min(tile * 16 + col, a.n - 1);
  const uint8_t* const row = a.w + n * a.w_stride;
  const T* const scale = static_cast<const T*>(a.scales) + n * a.scale_stride;
  const uint8_t* const zero = ZEROS ? a.zeros + n * a.zero_stride : nullptr;
  f32x4 y[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) y[i] = f32x4{0, 0, 0, 0};
  const T* x[MT];
  bool has[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + col;
    has[i] = m < a.m;
    x[i] = static_cast<const T*>(a.x) + (has[i] ? m : 0) * a.x_stride;
  }
  f32x4 acc[MT], ones[MT];
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = ones[i] = f32x4{0, 0, 0, 0};
  };
  const auto finish = [&](int g) {
    if (g >= groups) return;
    const float s = float(scale[g]), c = 16.f + (ZEROS ? float(zero[g]) : 8.f);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) y[i][r] += s * (acc[i][r] - c * ones[i][r]);
    clear();
  };
  clear();
  const u32x4 one = {Nibble<T>::one, Nibble<T>::one, Nibble<T>::one, Nibble<T>::one};
  if (tile * 16 < a.n) {
    for (int kb = part * kBlockK; kb < a.k; kb += kw * kBlockK) {
      const u32x4 w = turned(load_w<ALIGNED>(row, kb / 2 + 16 * quad, a.width));
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const int k = kb + 32 * st;
        u32x4 xf[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          xf[i] = load_x<T, ALIGNED>(x[i], has[i], k + 8 * quad, a.k);
          ones[i] = Half<T>::mma16(xf[i], one, ones[i]);
        }
        const u32x4 wf = widen<T>(w[st]);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = Half<T>::mma16(xf[i], wf, acc[i]);
        // a group ends here, or this wave's part of it does
        if ((k / 32 + 1) % steps == 0 || (st == 3 && kw > 1)) finish(k / a.group);
      }
    }
    if (kw == 1) finish((a.k - 1) / a.group);
  }
  finish_rows<T, MT>(a, y, sums, kw, part, wave, lane, tile, m0);
}

// For groups of 32 S, S = 1, 2 or 4, many columns and whole turns.  A turn is eight groups, 2 S blocks
// of 128: their weights are under way together (a row's bytes one after the other: with
// one block at a time all waves of the chip asked for the same 64 of every K / 2 bytes, and
// so of the same memory channels), and their scales and zero points come as one load of 16
// and of 8 bytes a column (a load for each of them took more of the memory path than the
// weights).  x stands in LDS, `part` values of k at a time, in the order that the weights pair
// up in.  A workgroup stays and takes tiles of columns in turn, and the next turn's weights
// are under way beside a turn's products (no load stands behind a condition: at the join the
// compiler would wait for it).  16 rows, K = 1024, 155,648 columns: 24.6 us, 3.7 TB/s of the
// 5.1 of a large copy.
template <int S>
struct Turn {
  u32x4 w[2 * S], sc;
  u32x2 zc;
};
template <typename T, int MT, int S, bool ZEROS>
__global__ void __launch_bounds__(256) matvec_w4_groups_kernel(MatvecArgs a, int part) {
  constexpr int kTurn = 256 * S;
  extern __shared__ float lds[];
  uint16_t* const xs = reinterpret_cast<uint16_t*>(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4, row_step = part + 8;  // a row in LDS: 16 bytes more than its data
  const int m0 = blockIdx.y * 16 * MT, turns = a.k / kTurn;
  const int sets = (a.n + 63) / 64;  // of a workgroup's tiles

  const auto load = [&](Turn<S>& u, int set, int turn) {
    const int k0 = turn * kTurn, g0 = 8 * turn, n = min((set * 4 + wave) * 16 + col, a.n - 1);
    const uint8_t* const row = a.w + n * a.w_stride + 16 * quad + k0 / 2;
#pragma unroll
    for (int b = 0; b < 2 * S; ++b) u.w[b] = *reinterpret_cast<const u32x4*>(row + 64 * b);
    u.sc = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.scales) + n * a.scale_stride + g0);
    if (ZEROS) u.zc = *reinterpret_cast<const u32x2*>(a.zeros + n * a.zero_stride + g0);
  };
  const auto stage = [&](int from) {
    const int chunks = part / 8;
    for (int c = threadIdx.x; c < 16 * MT * chunks; c += 256) {
      const int r = c / chunks, k = (c - r * chunks) * 8;
      const bool has = m0 + r < a.m;
      *reinterpret_cast<u32x4*>(xs + r * row_step + k) =
          load_x<T, true>(static_cast<const T*>(a.x) + (has ? m0 + r : 0) * a.x_stride, has, from + k, a.k);
    }
    __syncthreads();
  };
  f32x4 y[MT];
  const u32x4 one = {Nibble<T>::one, Nibble<T>::one, Nibble<T>::one, Nibble<T>::one};
  const auto multiply = [&](const Turn<S>& u, int at) {  // `at`: the turn's place in LDS
    f32x4 acc[MT], ones[MT];
#pragma unroll
    for (int b = 0; b < 2 * S; ++b) {
      const u32x4 v = turned(u.w[b]);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const bool first = (4 * b + st) % S == 0;
        const f32x4 none = {0, 0, 0, 0};
        u32x4 xf[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          xf[i] = *reinterpret_cast<const u32x4*>(xs + (16 * i + col) * row_step + at + kBlockK * b + 32 * st + 8 * quad);
          ones[i] = Half<T>::mma16(xf[i], one, first ? none : ones[i]);
        }
        const u32x4 wf = widen<T>(v[st]);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = Half<T>::mma16(xf[i], wf, first ? none : acc[i]);
        if ((4 * b + st + 1) % S == 0) {
          const int g = (4 * b + st) / S;
          const float s = g & 1 ? high<T>(u.sc[g / 2]) : low<T>(u.sc[g / 2]);
          const float c = 16.f + (ZEROS ? float(u.zc[g / 4] >> (8 * (g & 3)) & 255) : 8.f);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[i][r] += s * (acc[i][r] - c * ones[i][r]);
        }
      }
    }
  };
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < MT; ++i) y[i] = f32x4{0, 0, 0, 0};
  };

  Turn<S> u[2];
  clear();
  int set = blockIdx.x, turn = 0, staged = -1;
  load(u[0], set, 0);
  while (set < sets) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      int next = turn + 1, next_set = set;
      if (next == turns) next = 0, next_set += gridDim.x;
      load(u[b ^ 1], min(next_set, sets - 1), next);
      const int from = turn * kTurn / part * part;
      if (from != staged) {
        if (staged >= 0) __syncthreads();  // the part before has been read
        stage(from);
        staged = from;
      }
      multiply(u[b], turn * kTurn - from);
      if (next == 0) {
        finish_rows<T, MT>(a, y, nullptr, 1, 0, wave, lane, set * 4 + wave, m0);
        clear();
        if (next_set >= sets) return;
      }
      turn = next, set = next_set;
    }
  }
}

template <typename T, int MT, int S>
hipError_t launch_groups(const MatvecArgs& a, hipStream_t s) {
  const auto kernel = a.zeros ? matvec_w4_groups_kernel<T, MT, S, true> : matvec_w4_groups_kernel<T, MT, S, false>;
  // x in LDS as a whole up to 64 KiB, two workgroups of a CU; three where there is room for four
  // (155,648 columns of K = 1024 and one row: 20.9 us, four 22.8)
  const int whole = a.k, part = MT * whole <= 2048 ? whole : 2048 / MT;
  const unsigned sets = unsigned((a.n + 63) / 64), most = MT * whole <= 1024 ? 768 : 512;
  hipLaunchKernelGGL(kernel, dim3(std::min(sets, most), (a.m + 16 * MT - 1) / (16 * MT)), dim3(256),
                     size_t(16) * MT * (part + 8) * 2, s, a, part);
  return hipGetLastError();
}
template <typename T, int S>
hipError_t launch_groups(const MatvecArgs& a, hipStream_t s) {
  return a.m <= 16 ? launch_groups<T, 1, S>(a, s) : launch_groups<T, 2, S>(a, s);
}

template <typename T, int MT>
hipError_t launch(const MatvecArgs& a, int kw, hipStream_t s) {
  const bool z = a.zeros != nullptr;
  const auto kernel = a.aligned ? (z ? matvec_w4_kernel<T, MT, true, true> : matvec_w4_kernel<T, MT, true, false>)
                                : (z ? matvec_w4_kernel<T, MT, false, true> : matvec_w4_kernel<T, MT, false, false>);
  const unsigned tiles = unsigned((a.n + 15) / 16), per = 4 / kw;
  hipLaunchKernelGGL(kernel, dim3((tiles + per - 1) / per, (a.m + 16 * MT - 1) / (16 * MT)), dim3(256),
                     kw > 1 ? 4 * MT * 256 * sizeof(float) : 0, s, a, kw);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const MatvecArgs& a, hipStream_t s) {
  const int blocks = (a.k + kBlockK - 1) / kBlockK;
  // where there are columns enough for a wave of each SIMD: its turn of eight groups is a
  // long piece of K (K = 4096, one row: 16384 columns 17.6 us against 26.1, 8192 15.8 against
  // 16.2; K = 1024, 16 rows: 32768 columns 9.8 against 17.2)
  if (a.aligned && a.vector_scales && a.n >= 16384 && a.k % (8 * a.group) == 0) {
    if (a.group == 32) return launch_groups<T, 1>(a, s);
    if (a.group == 64) return launch_groups<T, 2>(a, s);
    if (a.group == 128) return launch_groups<T, 4>(a, s);
  }
  // else the waves of a workgroup share K (1024 x 4096, one row: 8.5 us, by one wave a tile 11.9)
  const int kw = blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
  return a.m <= 16 ? launch<T, 1>(a, kw, s) : launch<T, 2>(a, kw, s);
}

}  // namespace

hipError_t launch_matvec_w4(const MatvecArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_type<_Float16>(a, s) : launch_type<__bf16>(a, s);
}

}  // namespace praghip
