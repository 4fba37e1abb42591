// Attention of one new token per sequence over a paged key/value cache:
//   s_j = scale q.k_j over the visible keys j,  m = max s_j,  l = sum 2^(s_j - m),
//   o = sum 2^(s_j - m) v_j / l,   lse = (m + log2 l) ln 2
// in one pass over the cache with a running m and l (the scale holds log2 e).
//
// The work is read once: 4 dim bytes of K and V per key and key/value head, for
// 4 dim group operations, so the bytes bound it.  What decides is that every CU
// always has loads under way, whatever the lengths are: the blocks of 32 keys of
// all sequences and heads stand in one row, and every wave of the grid takes an
// equal stretch of it, across heads and sequences.
//
// A wave works by itself, with no LDS in its loop:
// * S^T = K Q^T by 16x16x32 products, 16 keys a tile: a lane's 8 values of a key
//   are contiguous in the page, so K goes from memory into the operand;
// * the products' layout leaves a lane with query column lane % 16 and the four
//   keys 4 (lane / 16) + 0..3 of both tiles.  Taking these eight as the lane's
//   slots of the second product's sum needs no exchange for P; V is loaded by
//   whole rows (dim / 16 values of each of the lane's eight keys), and byte
//   permutes turn 8 keys x dim / 16 values into the operand of O^T = V^T P^T;
// * 16 query columns are the heads of one key/value head (groups above 16 take
//   several turns), so m, l and the factor of O are one value per lane.
// P goes into the product as a sum of two 16-bit values: 8 more of 24 products per
// block, which the loads hide, and the rounding of P drops out of the error (in float16,
// whose P is up to 2^15, it is 2^-40 of the strongest key's).
//
// A stretch that holds a head's blocks from first to last writes the output.
// Else its m, l and o go to LDS, where the workgroup merges neighbours, and what a
// workgroup holds in part goes to the workspace, at most two pieces of it; the
// join kernel adds the pieces in order, so results do not depend on timing.
//
// 64 sequences of 0 to 8192 tokens, 16 heads of 128 over 8 (627 MB): 120 us, 5.2 TB/s where
// a large copy has 5.1.  Four through a window of 32768, 32 heads of 64 over 4 (134 MB): 35.5
// us of the copy's 26.  One of 2049 tokens (8 MB): 13.3 to 15 us by run, a chain of dependent
// reads (lengths, tables, keys) in 10 us and the join's launch in 4.
#include "attention.hpp"

namespace praghip {
namespace {

constexpr int kWaves = 4;

template <typename T, int D>
struct DecodeShape {
  static constexpr int steps = D / 32;       // of the first product
  static constexpr int per = D / 16;         // values of a key's row that a lane holds
  static constexpr int words = per / 2;
  static constexpr int tiles16 = (per + 7) / 8;
};

// Blocks of all heads over the grid's waves: each of the first `extra` has one more than
// the others, so a workgroup with a later neighbour that has blocks has blocks itself.
struct Range {
  uint32_t each, extra;
  __device__ __forceinline__ Range(uint32_t blocks, uint32_t waves) : each(blocks / waves), extra(blocks - each * waves) {}
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return each * w + min(w, extra); }
  // the wave whose stretch holds block u
  __device__ __forceinline__ uint32_t of(uint32_t u) const {
    const uint32_t longer = extra * (each + 1);
    return u < longer ? u / (each + 1) : extra + (u - longer) / each;
  }
};

// pieces of the workspace: [workgroup][2] of rows x (dim + 2)
// (a multiple of four floats, which the join loads together)
__host__ __device__ __forceinline__ size_t piece_floats(int rows, int D) { return size_t(rows) * D + (2 * rows + 3) / 4 * 4; }

// a load of the cache, past the caches or not
template <bool PAST, typename V>
__device__ __forceinline__ V fetch(const V* p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  return *p;
}

template <typename T, int D, bool EXACT, bool PAST>
__global__ void __launch_bounds__(kWaves * 64) paged_decode_kernel(DecodeArgs a) {
  using S = DecodeShape<T, D>;
  extern __shared__ float lds[];
  __shared__ int piece_id[2 * kWaves], piece_flags[2 * kWaves];
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int qtiles = (c.group + 15) >> 4, heads = c.kv_heads * qtiles, rows = min(c.group, 16);
  if (threadIdx.x < 2 * kWaves) piece_id[threadIdx.x] = -1;
  __syncthreads();

  // key blocks before each stretch of sequences, one stretch per lane; every wave counts
  // for itself, which takes no exchange with the others (for seqs / 64 reads one after the
  // other: meant for thousands of sequences, not for the 2^20 that are allowed)
  const int per = (c.seqs + 63) >> 6;
  uint32_t mine = 0;
  for (int i = 0; i < per; ++i) {
    const int s = lane * per + i;
    if (s < c.seqs) {
      const int n = length_of(c, s);
      mine += visible_blocks(c, n - 1, n - 1, 5).count();
    }
  }
  uint32_t sum = mine;  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  if (blockIdx.x == 0 && wave == 0) {  // for the join
    uint32_t at = sum - mine;
    for (int i = 0; i < per; ++i) {
      const int s = lane * per + i;
      if (s >= c.seqs) break;
      a.base[s] = at;
      const int n = length_of(c, s);
      at += visible_blocks(c, n - 1, n - 1, 5).count();
      if (s == c.seqs - 1) a.base[c.seqs] = at;
    }
  }
  const Range range(uint32_t(__builtin_amdgcn_readlane(int(sum), 63)) * heads, gridDim.x * kWaves);
  const uint32_t wg_begin = range.begin(blockIdx.x * kWaves), wg_end = range.begin(blockIdx.x * kWaves + kWaves);
  const uint32_t u_begin = range.begin(blockIdx.x * kWaves + wave), u_end = range.begin(blockIdx.x * kWaves + wave + 1);
  uint32_t u = u_begin;

  if (u < u_end) {
    // the sequence of block u: its lane's stretch (the stretches before it end at or before
    // u), then along the stretch
    const int from_lane = __popcll(__ballot(sum * heads <= u));
    int s = from_lane * per;
    uint32_t base = uint32_t(__builtin_amdgcn_readlane(int(sum - mine), from_lane)) * heads;
    while (u < u_end) {
      const int len = length_of(c, s);
      const Blocks blocks = visible_blocks(c, len - 1, len - 1, 5);
      const int nb = blocks.count();
      if (u >= base + uint32_t(nb) * heads) {
        base += uint32_t(nb) * heads;
        ++s;
        continue;
      }
      const int h = int((u - base) / uint32_t(nb)), first = int(u - base) - h * nb;
      const int count = min(nb - first, int(u_end - u));
      const int kvh = h / qtiles, head0 = kvh * c.group + (h - kvh * qtiles) * 16;
      const bool has = (h - kvh * qtiles) * 16 + col < c.group;

      u32x4 q[S::steps];
#pragma unroll
      for (int i = 0; i < S::steps; ++i) {
        q[i] = u32x4{0, 0, 0, 0};
        const int d = 32 * i + 8 * quad;
        if (has && (EXACT || d < c.dim))
          q[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + s * a.q_seq + (head0 + col) * a.q_head + d);
        q[i] ^= c.flip;
      }
      f32x4 o[S::per];
#pragma unroll
      for (int j = 0; j < S::per; ++j) o[j] = f32x4{0, 0, 0, 0};
      float m = kNegInf, l = 0;

      const int from = c.window > 0 ? len - c.window : 0;  // first position of the window
      for (int i = first; i < first + count; ++i) {
        const int kb = blocks.at(i) << 5;
        u32x4 kf[2][S::steps];
        uint32_t vr[8][S::words];
        bool page_ok[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int at = (kb + 16 * t) >> c.page_shift;
          int page = at < int((c.capacity) >> c.page_shift) ? c.tables[s * c.table_stride + at] : -1;
          page_ok[t] = page >= 0 && page < c.pages;
          page = page_ok[t] ? page : 0;
          const int row = (kb + 16 * t) & ((1 << c.page_shift) - 1);
          const T* kp = static_cast<const T*>(c.k) + uint64_t(page) * c.k_page + uint64_t(kvh) * c.k_head + uint64_t(row + col) * c.k_token + 8 * quad;
#pragma unroll
          for (int n = 0; n < S::steps; ++n) {
            kf[t][n] = u32x4{0, 0, 0, 0};
            if (EXACT || 32 * n + 8 * quad < c.dim) kf[t][n] = fetch<PAST>(reinterpret_cast<const u32x4*>(kp + 32 * n));
          }
          const T* vp = static_cast<const T*>(c.v) + uint64_t(page) * c.v_page + uint64_t(kvh) * c.v_head + uint64_t(row + 4 * quad) * c.v_token + S::per * col;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int w = 0; w < S::words; ++w) vr[4 * t + e][w] = 0;
            if (EXACT || S::per * col < c.dim) {
              if constexpr (S::words == 2) {
                const u32x2 x = fetch<PAST>(reinterpret_cast<const u32x2*>(vp + uint64_t(e) * c.v_token));
                vr[4 * t + e][0] = x[0];
                vr[4 * t + e][1] = x[1];
              } else {
#pragma unroll
                for (int w = 0; w < S::words; w += 4) {
                  if (!EXACT && S::per * col + 2 * w >= c.dim) continue;
                  const u32x4 x = fetch<PAST>(reinterpret_cast<const u32x4*>(vp + uint64_t(e) * c.v_token + 2 * w));
#pragma unroll
                  for (int b = 0; b < 4; ++b) vr[4 * t + e][w + b] = x[b];
                }
              }
            }
          }
        }
        f32x4 st[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int n = 0; n < S::steps; ++n) {
          st[0] = Half<T>::mma16(kf[0][n], q[n], st[0]);
          st[1] = Half<T>::mma16(kf[1][n], q[n], st[1]);
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = st[e >> 2][e & 3] * c.scale;
        const bool whole = page_ok[0] && page_ok[1] && kb + 32 <= len && (kb >= from || kb + 32 <= c.sinks);
        if (!whole) {  // keys that the query does not see count as nothing, whatever their page holds
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = kb + 16 * (e >> 2) + 4 * quad + (e & 3);
            const bool sees = bool(page_ok[e >> 2]) & (at < len) & ((at >= from) | (at < c.sinks));
            x[e] = sees ? x[e] : kNegInf;
#pragma unroll
            for (int w = 0; w < S::words; ++w) vr[e][w] = sees ? vr[e][w] : 0;
          }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        top = fmaxf(m, max32(max16(top)) - Half<T>::most);
        if (__any(top > m)) {
          const float f = __builtin_amdgcn_exp2f(m - origin(top));
          l *= f;
#pragma unroll
          for (int j = 0; j < S::per; ++j) o[j] *= f;
          m = top;
        }
        uint32_t hi[4], rest[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(x[e] - origin(m)), p1 = __builtin_amdgcn_exp2f(x[e + 1] - origin(m));
          l += p0 + p1;
          hi[e / 2] = pack2<T>(p0, p1);
          rest[e / 2] = pack2<T>(p0 - low<T>(hi[e / 2]), p1 - high<T>(hi[e / 2]));
        }
        const u32x4 ph = {hi[0], hi[1], hi[2], hi[3]}, pl = {rest[0], rest[1], rest[2], rest[3]};
#pragma unroll
        for (int j = 0; j < S::per; ++j) {
          u32x4 vt;
#pragma unroll
          for (int p = 0; p < 4; ++p)
            vt[p] = __builtin_amdgcn_perm(vr[2 * p + 1][j / 2], vr[2 * p][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
          o[j] = Half<T>::mma16(vt, ph, o[j]);
          o[j] = Half<T>::mma16(vt, pl, o[j]);
        }
      }
      l = sum32(sum16(l));

      if (first == 0 && count == nb) {
        if (has) {
          const float r = l > 0 || l != l ? 1.f / l : 0.f;
          T* out = static_cast<T*>(a.out) + s * a.out_seq + (head0 + col) * a.out_head;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = (4 * quad + e) * S::per;
#pragma unroll
            for (int j = 0; j < S::per; j += 2)
              if (EXACT || d + j < c.dim)
                *reinterpret_cast<uint32_t*>(out + d + j) = pack2<T>(o[j][e] * r, o[j + 1][e] * r);
          }
          if (a.lse && quad == 0)
            a.lse[int64_t(s) * c.kv_heads * c.group + head0 + col] = (m + __builtin_amdgcn_logf(l)) * kLn2;
        }
      } else {
        const int slot = 2 * wave + (u != u_begin);
        float* to = lds + slot * piece_floats(rows, D);
        if (col < rows) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < S::per; ++j) to[col * D + (4 * quad + e) * S::per + j] = o[j][e];
          if (quad == 0) {
            to[rows * D + col] = m;
            to[rows * D + rows + col] = l;
          }
        }
        if (lane == 0) {
          const uint32_t b = base + uint32_t(h) * nb;
          piece_id[slot] = s * heads + h;
          piece_flags[slot] = (b >= wg_begin && b + nb <= wg_end ? 1 : 0) | (b > wg_begin ? 2 : 0);
        }
      }
      u += count;
    }
  }
  __syncthreads();
  // neighbouring pieces of one head, merged in order
  for (int e = 0; e < 2 * kWaves; ++e) {
    const int id = piece_id[e];
    if (id < 0) continue;
    int last = e;
    for (int n = e + 1; n < 2 * kWaves; ++n)
      if (piece_id[n] == id)
        last = n;
      else if (piece_id[n] >= 0)
        break;
    const int s = id / heads, h = id - s * heads, kvh = h / qtiles, head0 = kvh * c.group + (h - kvh * qtiles) * 16;
    const bool complete = piece_flags[e] & 1;
    float* to = a.work + (size_t(blockIdx.x) * 2 + (piece_flags[e] >> 1)) * piece_floats(rows, D);
    const int have = min(16, c.group - (h - kvh * qtiles) * 16);
    for (int i = threadIdx.x; i < have * D; i += kWaves * 64) {
      const int r = i / D, d = i - r * D;
      float m = kNegInf;
      for (int n = e; n <= last; ++n)
        if (piece_id[n] >= 0) m = fmaxf(m, lds[n * piece_floats(rows, D) + rows * D + r]);
      float sum = 0, l = 0;
      for (int n = e; n <= last; ++n) {
        if (piece_id[n] < 0) continue;
        const float* p = lds + n * piece_floats(rows, D);
        const float f = __builtin_amdgcn_exp2f(p[rows * D + r] - origin(m));
        sum += f * p[i];
        l += f * p[rows * D + rows + r];
      }
      if (complete) {
        const float inv = l > 0 || l != l ? 1.f / l : 0.f;
        if (EXACT || d < c.dim) static_cast<T*>(a.out)[s * a.out_seq + (head0 + r) * a.out_head + d] = T(sum * inv);
        if (a.lse && d == 0)
          a.lse[int64_t(s) * c.kv_heads * c.group + head0 + r] = (m + __builtin_amdgcn_logf(l)) * kLn2;
      } else {
        to[i] = sum;
        if (d == 0) {
          to[rows * D + r] = m;
          to[rows * D + rows + r] = l;
        }
      }
    }
    e = last;
  }
}

// One workgroup per sequence and query head, for heads that workgroups share and rows that
// see nothing.  Each D / 4 threads merge every (1024 / D)-th piece, with the next pieces'
// loads under way, and LDS the results, all in a fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(DecodeArgs a, unsigned workgroups) {
  constexpr int per = D / 4, sets = 256 / per;
  __shared__ __attribute__((aligned(16))) float part[sets][D];
  __shared__ float tops[sets], sums[sets];
  const CacheArgs& c = a.c;
  const int all = c.kv_heads * c.group, s = blockIdx.x / all, head = blockIdx.x - s * all, kvh = head / c.group;
  const int qtiles = (c.group + 15) >> 4, heads = c.kv_heads * qtiles, rows = min(c.group, 16);
  const int g = head - kvh * c.group, h = kvh * qtiles + (g >> 4), r = g & 15;
  const uint32_t b0 = a.base[s], nb = a.base[s + 1] - b0, b = b0 * heads + h * nb, total = a.base[c.seqs] * heads;
  const int set = threadIdx.x / per, d = threadIdx.x % per * 4;
  T* const out = static_cast<T*>(a.out) + s * a.out_seq + head * a.out_head;
  float m = kNegInf, l = 0;
  f32x4 o = {0, 0, 0, 0};
  if (nb) {
    const Range range(total, workgroups * kWaves);
    const uint32_t w0 = range.of(b) / kWaves, w1 = range.of(b + nb - 1) / kWaves;
    if (w0 == w1) return;
    const size_t piece = piece_floats(rows, D);
    const uint32_t second = b > range.begin(w0 * kWaves);  // the first workgroup's other piece
    for (uint32_t w = w0 + set; w <= w1; w += sets) {
      const float* const p = a.work + (size_t(w) * 2 + (w == w0 ? second : 0)) * piece;
      const f32x4 po = *reinterpret_cast<const f32x4*>(p + r * D + d);
      const float pm = p[rows * D + r], pl = p[rows * D + rows + r], top = fmaxf(m, pm);
      const float f = __builtin_amdgcn_exp2f(m - origin(top)), pf = __builtin_amdgcn_exp2f(pm - origin(top));
      o = o * f + po * pf;
      l = l * f + pl * pf;
      m = top;
    }
  }
  *reinterpret_cast<f32x4*>(&part[set][d]) = o;
  if (d == 0) {
    tops[set] = m;
    sums[set] = l;
  }
  __syncthreads();
  if (int(threadIdx.x) >= D) return;
  m = kNegInf;
#pragma unroll
  for (int i = 0; i < sets; ++i) m = fmaxf(m, tops[i]);
  float sum = 0;
  l = 0;
#pragma unroll
  for (int i = 0; i < sets; ++i) {
    const float f = __builtin_amdgcn_exp2f(tops[i] - origin(m));
    sum += f * part[i][threadIdx.x];
    l += f * sums[i];
  }
  const float inv = l > 0 || l != l ? 1.f / l : 0.f;
  if (int(threadIdx.x) < c.dim) out[threadIdx.x] = T(sum * inv);
  if (a.lse && threadIdx.x == 0) a.lse[int64_t(s) * all + head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int D>
hipError_t launch(const DecodeArgs& a, unsigned workgroups, hipStream_t s) {
  const int rows = std::min(a.c.group, 16);
  const size_t lds = 2 * kWaves * piece_floats(rows, D) * sizeof(float);
  const bool exact = a.c.dim == D;
  const auto kernel = a.past ? (exact ? paged_decode_kernel<T, D, true, true> : paged_decode_kernel<T, D, false, true>)
                             : (exact ? paged_decode_kernel<T, D, true, false> : paged_decode_kernel<T, D, false, false>);
  hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(kWaves * 64), lds, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((decode_join_kernel<T, D>), dim3(unsigned(a.c.seqs) * a.c.kv_heads * a.c.group), dim3(256), 0, s, a, workgroups);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_dim(const DecodeArgs& a, unsigned workgroups, hipStream_t s) {
  return a.c.dim <= 64 ? launch<T, 64>(a, workgroups, s) : a.c.dim <= 128 ? launch<T, 128>(a, workgroups, s) : launch<T, 256>(a, workgroups, s);
}

}  // namespace

// As many workgroups as the chip holds at three a CU (two: 140 us where three took 131), and
// no more than there are blocks for their waves.
unsigned decode_workgroups(size_t seqs, size_t kv_heads, size_t group, size_t keys) {
  const size_t blocks = seqs * kv_heads * ((group + 15) / 16) * ((keys + 31) / 32 + 1);
  return unsigned(std::max<size_t>(1, std::min<size_t>((blocks + kWaves - 1) / kWaves, 256 * 3)));
}
size_t decode_work_floats(unsigned workgroups, size_t group, size_t dim) {
  const size_t D = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  return size_t(workgroups) * 2 * piece_floats(int(std::min<size_t>(group, 16)), int(D));
}

hipError_t launch_paged_decode(const DecodeArgs& a, int type, unsigned workgroups, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_dim<_Float16>(a, workgroups, s) : launch_dim<__bf16>(a, workgroups, s);
}

}  // namespace praghip
