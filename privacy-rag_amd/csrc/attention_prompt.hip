// Attention of a prompt's tokens over a paged key/value cache, causal, with a
// sliding window and a few first tokens that stay visible: the query at position p
// sees key j where j <= p and (j < sinks or j > p - window).  The cache holds the
// prompt's own keys already.
//
// One pass over the keys with a running maximum and sum.  4 dim operations per pair
// of query and key on 32x32x16 products bound it, and beside them one exponential
// per pair.  A workgroup takes 32 rows a wave; a row is one token's one head of the
// group that shares a key/value head, so K and V are read once for the group, and
// tiles of 64 keys go through LDS, two in turn.
//
// S^T = K Q^T puts a query into a lane's column with 16 of 32 keys in its registers:
// the maximum and the sum need one exchange (with lane ^ 32), and the factor of O^T
// = V^T P^T is one value per lane.  Taking the keys that a lane holds as its slots of
// the second product's sum (slot e of half h of step t: key 16 t + 8 (e / 4) + 4 h +
// e % 4), P goes from the first product's registers into the second's with no
// exchange; V's operand in that order is a transposed LDS read of 4 keys x 16 columns.
// P is rounded to the 16 bits that the product takes (its sum is kept in 32).
//
// LDS rows have 2 dim bytes; 16-byte chunk x of row r is at x ^ f(r), so that both
// kinds of reads spread over all banks.
//
// Where row tiles alone would leave CUs idle, each tile's keys are split over
// workgroups; their m, l and o go to the workspace and a second kernel joins them in
// order.
#include "attention.hpp"

namespace praghip {
namespace {

constexpr int kTile = 64;  // keys of a tile

template <typename T, int D, int NW, bool EXACT>
__global__ void __launch_bounds__(NW * 64, NW / 4) paged_prompt_kernel(PromptArgs a, int ntile) {
  constexpr int ROWS = 32 * NW, CPR = D / 8, PER = kTile * CPR / (NW * 64);  // chunks of a row, of a thread
  constexpr int steps = D / 16, blocks32 = D / 32;
  extern __shared__ uint32_t lds[];
  T* const kbuf = reinterpret_cast<T*>(lds);            // [2][64][D]
  T* const vbuf = kbuf + 2 * kTile * D;                 // [2][64][D]
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;

  // heads next to one another: with as many key/value heads as XCDs each L2 holds
  // one head's cache; later row tiles first, which see the most keys
  int index = blockIdx.x;
  const int kvh = index % c.kv_heads;
  index /= c.kv_heads;
  const int split = index % a.splits;
  index /= a.splits;
  const int s = index % c.seqs, tile = ntile - 1 - index / c.seqs;
  const int begin = min(max(a.starts[s], 0), a.total), count = min(max(a.starts[s + 1], begin), a.total) - begin;
  const int64_t nrow = int64_t(count) * c.group, row0 = int64_t(tile) * ROWS;
  if (row0 >= nrow) return;
  const int len = length_of(c, s), shift = len - count;  // position of token t: t + shift

  const int64_t row = row0 + wave * 32 + col;
  const bool has = row < nrow;
  const int token = has ? int(row / c.group) : 0, head = kvh * c.group + (has ? int(row - int64_t(token) * c.group) : 0);
  const int place = has ? token + shift : -1, from = c.window > 0 ? place - c.window : -1;  // keys above `from` are in the window
  const int64_t wlast = min(row0 + wave * 32 + 31, nrow - 1);
  const int wmin = row0 + wave * 32 < nrow ? int((row0 + wave * 32) / c.group) + shift : 0;
  const int wmax = row0 + wave * 32 < nrow ? int(wlast / c.group) + shift : -1;

  const Blocks blocks = visible_blocks(c, max(0, int(row0 / c.group) + shift), int((min(row0 + ROWS, nrow) - 1) / c.group) + shift, 6);
  const int nb = blocks.count(), i0 = int(int64_t(nb) * split / a.splits), i1 = int(int64_t(nb) * (split + 1) / a.splits);

  u32x4 q[steps];
#pragma unroll
  for (int n = 0; n < steps; ++n) {
    q[n] = u32x4{0, 0, 0, 0};
    const int d = 16 * n + 8 * half;
    if (has && (EXACT || d < c.dim))
      q[n] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + (begin + token) * a.q_token + head * a.q_head + d);
  }
  f32x16 o[blocks32];
#pragma unroll
  for (int b = 0; b < blocks32; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0;
  float m = kNegInf, l = 0;

  const auto fk = [](int r) { return D == 64 ? (r >> 1) & 7 : r & 15; };
  const auto fv = [](int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; };
  const int width = int(c.capacity >> c.page_shift);

  u32x4 kx[PER], vx[PER];
  uint32_t pages_ok = 0;  // groups of 16 keys of the tile in registers that have a page
  const auto load = [&](int kb) {
    uint32_t ok = 0;
    {
      const int at = (kb + 16 * (lane & 3)) >> c.page_shift;
      const int page = at < width ? c.tables[s * c.table_stride + at] : -1;
      ok = uint32_t(__ballot(page >= 0 && page < c.pages)) & 15;
    }
    pages_ok = ok;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int chunk = threadIdx.x + i * NW * 64, r = chunk / CPR, x = chunk % CPR, at = kb + r;
      kx[i] = vx[i] = u32x4{0, 0, 0, 0};
      if (at < len && (ok >> (r >> 4) & 1) && (EXACT || 8 * x < c.dim)) {
        const int64_t page = c.tables[s * c.table_stride + (at >> c.page_shift)];
        const int in = at & ((1 << c.page_shift) - 1);
        kx[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(c.k) + page * c.k_page + kvh * c.k_head + in * c.k_token + 8 * x);
        vx[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(c.v) + page * c.v_page + kvh * c.v_head + in * c.v_token + 8 * x);
      }
    }
  };
  const auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int chunk = threadIdx.x + i * NW * 64, r = chunk / CPR, x = chunk % CPR;
      *reinterpret_cast<u32x4*>(kbuf + buf * kTile * D + r * D + 8 * (x ^ fk(r))) = kx[i];
      *reinterpret_cast<u32x4*>(vbuf + buf * kTile * D + r * D + 8 * (x ^ fv(r))) = vx[i];
    }
  };

  if (i0 < i1) {
    load(blocks.at(i0) * kTile);
    store(0);
  }
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    const int kb = blocks.at(i) * kTile, buf = (i - i0) & 1;
    const uint32_t ok = pages_ok;
    if (i + 1 < i1) load(blocks.at(i + 1) * kTile);
    const bool any = kb <= wmax && (c.window == 0 || kb + kTile > wmin - c.window + 1 || kb < c.sinks);
    if (any) {
      f32x16 st[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[t][r] = 0;
#pragma unroll
        for (int n = 0; n < steps; ++n) {
          const int r = 32 * t + col;
          const u32x4 kf = *reinterpret_cast<const u32x4*>(kbuf + buf * kTile * D + r * D + 8 * ((2 * n + half) ^ fk(r)));
          st[t] = Half<T>::mma32(kf, q[n], st[t]);
        }
      }
      const bool whole = ok == 15 && kb + kTile - 1 <= wmin && (c.window == 0 || kb > wmax - c.window || kb + kTile <= c.sinks);
      float top = m, x[32];
#pragma unroll
      for (int r = 0; r < 32; ++r) x[r] = st[r >> 4][r & 15] * c.scale;
      if (!whole) {
#pragma unroll
        for (int r = 0; r < 32; ++r) {
          const int key = 8 * (r >> 2) + 4 * half + (r & 3), at = kb + key;
          const bool sees = (at <= place) & ((at > from) | (at < c.sinks)) & bool(ok >> (key >> 4) & 1);
          x[r] = sees ? x[r] : kNegInf;
        }
      }
#pragma unroll
      for (int r = 0; r < 32; ++r) top = fmaxf(top, x[r]);
      top = max32(top);
      if (__any(top > m)) {
        const float f = __builtin_amdgcn_exp2f(m - origin(top));
        l *= f;
#pragma unroll
        for (int b = 0; b < blocks32; ++b) o[b] *= f;
        m = top;
      }
      u32x4 p[4];
#pragma unroll
      for (int r = 0; r < 32; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(x[r] - origin(m)), p1 = __builtin_amdgcn_exp2f(x[r + 1] - origin(m));
        l += p0 + p1;
        p[r >> 3][(r & 7) >> 1] = pack2<T>(p0, p1);
      }
      const int trow = 4 * half + ((lane & 15) >> 2), tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int b = 0; b < blocks32; ++b) {
          u32x4 vt;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 16 * t + 8 * e + trow, d = 32 * b + tcol;
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            const auto x = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                           vbuf + buf * kTile * D + r * D + 8 * ((d >> 3) ^ fv(r)) + (d & 7))));
            vt[2 * e] = x[0];
            vt[2 * e + 1] = x[1];
          }
          o[b] = Half<T>::mma32(vt, p[t], o[b]);
        }
    }
    if (i + 1 < i1) store(buf ^ 1);
    __syncthreads();
  }
  l = sum32(l);

  if (a.splits == 1) {
    if (!has) return;
    const float r = l > 0 || l != l ? 1.f / l : 0.f;
    T* out = static_cast<T*>(a.out) + (begin + token) * a.out_token + head * a.out_head;
#pragma unroll
    for (int b = 0; b < blocks32; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * b + 8 * e + 4 * half;
        if (EXACT || d < c.dim)
          *reinterpret_cast<u32x2*>(out + d) = u32x2{pack2<T>(o[b][4 * e] * r, o[b][4 * e + 1] * r), pack2<T>(o[b][4 * e + 2] * r, o[b][4 * e + 3] * r)};
      }
    if (a.lse && half == 0)
      a.lse[int64_t(begin + token) * c.kv_heads * c.group + head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  } else if (has) {
    float* to = a.work + (((int64_t(s) * ntile + tile) * c.kv_heads + kvh) * a.splits + split) * ROWS * (D + 2);
    const int r = wave * 32 + col;
#pragma unroll
    for (int b = 0; b < blocks32; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(to + r * D + 32 * b + 8 * e + 4 * half) = f32x4{o[b][4 * e], o[b][4 * e + 1], o[b][4 * e + 2], o[b][4 * e + 3]};
    if (half == 0) {
      to[ROWS * D + r] = m;
      to[ROWS * D + ROWS + r] = l;
    }
  }
}

// One wave per row: the splits' m, l and o in order.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptArgs a, int ntile) {
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63;
  int64_t index = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int r = int(index % ROWS);
  index /= ROWS;
  const float* from = a.work + index * a.splits * ROWS * (D + 2);
  const int kvh = int(index % c.kv_heads);
  index /= c.kv_heads;
  const int tile = int(index % ntile), s = int(index / ntile);
  const int begin = min(max(a.starts[s], 0), a.total), count = min(max(a.starts[s + 1], begin), a.total) - begin;
  const int64_t row = int64_t(tile) * ROWS + r;
  if (row >= int64_t(count) * c.group) return;
  const int token = int(row / c.group), head = kvh * c.group + int(row - int64_t(token) * c.group);
  float m = kNegInf, l = 0, sum[D / 64] = {};
  for (int i = 0; i < a.splits; ++i) m = fmaxf(m, from[int64_t(i) * ROWS * (D + 2) + ROWS * D + r]);
  for (int i = 0; i < a.splits; ++i) {
    const float* p = from + int64_t(i) * ROWS * (D + 2);
    const float f = __builtin_amdgcn_exp2f(p[ROWS * D + r] - origin(m));
    l += f * p[ROWS * D + ROWS + r];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) sum[j] += f * p[r * D + lane + 64 * j];
  }
  const float inv = l > 0 || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const int d = lane + 64 * j;
    if (d < c.dim) static_cast<T*>(a.out)[(begin + token) * a.out_token + head * a.out_head + d] = T(sum[j] * inv);
  }
  if (a.lse && lane == 0) a.lse[int64_t(begin + token) * c.kv_heads * c.group + head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// rows of a workgroup: eight waves of 32, four where a row of 256 values takes the
// registers of two
int tile_rows(size_t dim) { return dim <= 128 ? 256 : 128; }
int tiles_of(size_t max_rows, size_t group, size_t dim) {
  return int((max_rows * group + tile_rows(dim) - 1) / tile_rows(dim));
}

template <typename T, int D, int NW>
hipError_t launch(const PromptArgs& a, hipStream_t s) {
  const int ntile = tiles_of(a.max_rows, a.c.group, a.c.dim);
  const size_t lds = size_t(4) * kTile * D * sizeof(T);
  const auto kernel = a.c.dim == D ? paged_prompt_kernel<T, D, NW, true> : paged_prompt_kernel<T, D, NW, false>;
  const unsigned groups = unsigned(ntile) * a.c.seqs * a.c.kv_heads;
  hipLaunchKernelGGL(kernel, dim3(groups * a.splits), dim3(NW * 64), lds, s, a, ntile);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL((prompt_join_kernel<T, D, 32 * NW>), dim3(groups * (32 * NW / 4)), dim3(256), 0, s, a, ntile);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_dim(const PromptArgs& a, hipStream_t s) {
  return a.c.dim <= 64 ? launch<T, 64, 8>(a, s) : a.c.dim <= 128 ? launch<T, 128, 8>(a, s) : launch<T, 256, 4>(a, s);
}

}  // namespace

int prompt_splits(size_t seqs, size_t kv_heads, size_t group, size_t dim, size_t max_rows, size_t keys) {
  const size_t tiles = size_t(tiles_of(max_rows, group, dim)) * seqs * kv_heads;
  if (!tiles || tiles > 128) return 1;
  return int(std::max<size_t>(1, std::min<size_t>(256 / tiles, keys / (4 * kTile))));
}
size_t prompt_work_floats(int splits, size_t seqs, size_t kv_heads, size_t group, size_t dim, size_t max_rows) {
  if (splits <= 1) return 0;
  const size_t D = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  return size_t(tiles_of(max_rows, group, dim)) * seqs * kv_heads * splits * tile_rows(dim) * (D + 2);
}

hipError_t launch_paged_prompt(const PromptArgs& a, int type, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_dim<_Float16>(a, s) : launch_dim<__bf16>(a, s);
}

}  // namespace praghip
