// New tokens of a step into a paged cache, with what stands between the projection and the
// attention: for queries and keys of the token at position p
//   x^ = x w / sqrt(mean x^2 + eps)                       (where there are norms)
//   a' = a cos[p] - b sin[p],  b' = b cos[p] + a sin[p]   (pairs of the first 2 half values)
// in 32 bits, rounded once; queries go to `out`, keys and values to the pages.
//
// Bytes bound it: each value is read and written once.  A wave takes one token (whose
// sequence and place are then the same for its lanes: scalar loads and a scalar search) and
// `heads_each` of its heads, 16 bytes a lane: 8, 16 or 32 lanes a head, whose squares are
// summed by lane exchanges.  The other value of a pair that is half a rotation away comes from
// its lane (read from memory a second time, 4 x 2048 tokens took 42 us instead of 34), or,
// where the half is no multiple of eight, value by value from memory; pairs of neighbours are
// in one lane.
//
// From 16 MiB of results on, half of what the L2s hold, stores pass the caches by: a kernel's
// end waits for the dirty lines (4 x 2048 tokens of 16 heads of 128 over 8: 26 us, 5.3 TB/s,
// where a large copy has 5.1, and 34 through the caches; with the attention after it, which then
// reads more from memory, both take 139 us).  3 sequences of some 500 tokens, 32 heads of 64 over 4, take
// 6 us, 8 single tokens 4.2, a launch and a chain of dependent reads.
#include "append.hpp"

#include <algorithm>

#include "attention.hpp"

namespace praghip {
namespace {

typedef f32x4 f32x4_any __attribute__((aligned(4)));

constexpr unsigned kSlab = 1 << 18;  // workgroups of a grid's row: a launch has below 2^32 threads in one dimension

template <typename T>
__device__ __forceinline__ void widen8(u32x4 x, float (&s)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t v = x[j];
    s[2 * j] = low<T>(v), s[2 * j + 1] = high<T>(v);
  }
}

// LANES of a head; HALVES: 0 for pairs of neighbours, 1 for pairs half a rotation apart in
// whole pieces of eight, 2 where the half is no multiple of eight.
template <typename T, int LANES, int HALVES, bool PAST>
__global__ void __launch_bounds__(256) page_append_kernel(AppendArgs a, int waves_each, int heads_each) {
  constexpr int kHeads = 64 / LANES;  // of a wave at a time
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane((blockIdx.y * kSlab + blockIdx.x) * 4 + (threadIdx.x >> 6));
  const int token = int(wave / uint32_t(waves_each)), part = int(wave) - token * waves_each;
  if (token >= a.tokens) return;
  int lo = 0, hi = a.seqs - 1;  // the last sequence that starts at or before the token
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.starts[mid] <= token)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int begin = a.starts[lo], end = a.starts[lo + 1];
  if (token < begin || token >= end) return;
  const int64_t at = int64_t(a.lengths[lo]) - end + token;
  int page = -1;
  if (at >= 0 && at >> a.page_shift < a.width) page = a.tables[lo * a.table_stride + (at >> a.page_shift)];
  if (page >= a.pages) page = -1;
  const int64_t row = at & ((1 << a.page_shift) - 1);
  const int64_t place = at < 0 ? 0 : at < a.positions ? at : a.positions - 1;

  const int d = lane % LANES * 8, all = a.heads + 2 * a.kv_heads;
  const bool has = d < a.dim;
  // cosines and sines of this lane's values, the sines with the sign of the pair's other
  // value; a value that is not turned takes 1 and 0
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = 1.f, sn[j] = 0.f;
  if (d < 2 * a.half) {
    const float *c = a.cos + place * a.cos_row, *s = a.sin + place * a.sin_row;
    if constexpr (HALVES == 1) {
      const int i = d < a.half ? d : d - a.half;
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const f32x4 c4 = *reinterpret_cast<const f32x4_any*>(c + i + j), s4 = *reinterpret_cast<const f32x4_any*>(s + i + j);
#pragma unroll
        for (int n = 0; n < 4; ++n) cs[j + n] = c4[n], sn[j + n] = d < a.half ? -s4[n] : s4[n];
      }
    } else if (HALVES == 0 && d + 8 <= 2 * a.half) {
      const f32x4 c4 = *reinterpret_cast<const f32x4_any*>(c + d / 2), s4 = *reinterpret_cast<const f32x4_any*>(s + d / 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j] = c4[j / 2], sn[j] = j & 1 ? s4[j / 2] : -s4[j / 2];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = d + j, i = HALVES == 0 ? e >> 1 : e < a.half ? e : e - a.half;
        if (e >= 2 * a.half) continue;
        cs[j] = c[i];
        sn[j] = (HALVES == 0 ? !(j & 1) : e < a.half) ? -s[i] : s[i];
      }
    }
  }
  for (int h = part * heads_each + lane / LANES; h < min((part + 1) * heads_each, all); h += kHeads) {
    const bool is_q = h < a.heads, is_v = h >= a.heads + a.kv_heads;
    const int kvh = h - a.heads - (is_v ? a.kv_heads : 0);
    const T* from = is_q   ? static_cast<const T*>(a.q) + token * a.q_token + h * a.q_head
                    : is_v ? static_cast<const T*>(a.v) + token * a.v_token + kvh * a.v_head
                           : static_cast<const T*>(a.k) + token * a.k_token + kvh * a.k_head;
    u32x4 got = {0, 0, 0, 0};
    if (has) got = *reinterpret_cast<const u32x4*>(from + d);
    T* to = is_q   ? static_cast<T*>(a.out) + token * a.out_token + h * a.out_head
            : is_v ? static_cast<T*>(a.v_pages) + page * a.vp_page + kvh * a.vp_head + row * a.vp_token
                   : static_cast<T*>(a.k_pages) + page * a.kp_page + kvh * a.kp_head + row * a.kp_token;
    if (!is_v) {
      float x[8], y[8];
      widen8<T>(got, x);
      const T* norm = static_cast<const T*>(is_q ? a.q_norm : a.k_norm);
      float w[8], by = 1.f;
      if (norm) {
        float sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
#pragma unroll
        for (int s = 1; s < LANES; s <<= 1) sum += __shfl_xor(sum, s, 64);
        by = 1.f / sqrtf(sum / float(a.dim) + a.eps);
        widen8<T>(*reinterpret_cast<const u32x4*>(norm + (has ? d : 0)), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= by * w[j];
      }
      if constexpr (HALVES == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = d + j < 2 * a.half ? x[j ^ 1] : 0.f;  // (infinite ones times 0 are NaN)
      } else if constexpr (HALVES == 1) {
        const int other = d < a.half ? d + a.half : d - a.half;
        const int at = (lane / LANES * LANES + (d < 2 * a.half ? other >> 3 : 0)) << 2;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(at, __builtin_bit_cast(int, x[j])));
          y[j] = d < 2 * a.half ? v : 0.f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = d + j, other = e < a.half ? e + a.half : e - a.half;
          y[j] = e < 2 * a.half ? float(from[other]) : 0.f;
          if (norm) y[j] *= e < 2 * a.half ? by * float(norm[other]) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        got[j] = pack2<T>(x[2 * j] * cs[2 * j] + y[2 * j] * sn[2 * j], x[2 * j + 1] * cs[2 * j + 1] + y[2 * j + 1] * sn[2 * j + 1]);
    }
    if (has && (is_q || page >= 0)) {
      if constexpr (PAST)
        __builtin_nontemporal_store(got, reinterpret_cast<u32x4*>(to + d));
      else
        *reinterpret_cast<u32x4*>(to + d) = got;
    }
  }
}

template <typename T, int LANES, bool PAST>
hipError_t launch_past(const AppendArgs& a, hipStream_t s) {
  const int all = a.heads + 2 * a.kv_heads, turn = 64 / LANES;
  // Four turns a wave where there are tokens enough (one: 47 us instead of 42; eight: 47), one
  // for short calls, whose latency counts.
  const int turns = (all + turn - 1) / turn;
  const int each = a.tokens >= 512 ? std::min(turns, 4) : 1, waves = (turns + each - 1) / each;
  const auto kernel = a.interleaved   ? page_append_kernel<T, LANES, 0, PAST>
                      : a.half % 8 ? page_append_kernel<T, LANES, 2, PAST>
                                   : page_append_kernel<T, LANES, 1, PAST>;
  const unsigned groups = unsigned((int64_t(a.tokens) * waves + 3) / 4);
  hipLaunchKernelGGL(kernel, dim3(std::min(groups, kSlab), (groups + kSlab - 1) / kSlab), dim3(256), 0, s, a, waves, each * turn);
  return hipGetLastError();
}
template <typename T, int LANES>
hipError_t launch(const AppendArgs& a, hipStream_t s) {
  const int64_t bytes = int64_t(a.tokens) * (a.heads + 2 * a.kv_heads) * a.dim * 2;
  return bytes >= (16 << 20) ? launch_past<T, LANES, true>(a, s) : launch_past<T, LANES, false>(a, s);
}
template <typename T>
hipError_t launch_dim(const AppendArgs& a, hipStream_t s) {
  return a.dim <= 64 ? launch<T, 8>(a, s) : a.dim <= 128 ? launch<T, 16>(a, s) : launch<T, 32>(a, s);
}

}  // namespace

hipError_t launch_page_append(const AppendArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_dim<_Float16>(a, s) : launch_dim<__bf16>(a, s);
}

}  // namespace praghip
