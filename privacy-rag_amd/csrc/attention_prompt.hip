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

// 16 bytes a lane from memory into LDS at M0 + 16 lane (global_load_lds_dwordx4).  The
// compiler adds no wait of its own for an asm, so the caller waits before it reads; the
// asm starts with the wait state that the DMA needs after the write of M0.
__device__ __forceinline__ void dma16(const void* src, void* lds_wave_base) {
  const unsigned at = unsigned(reinterpret_cast<uintptr_t>((void __attribute__((address_space(3)))*)(lds_wave_base)));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(__builtin_amdgcn_readfirstlane(at))
               : "memory");
}

// One tile's scores, 16 of 32 keys in st[t] for the lane's query, into P: the running
// maximum, the sum of P and O's factor.  Within 2^kSlack of it the old maximum stays in
// use: P may then be up to 2^kSlack, with the same relative rounding, and the dim / 2
// products with the factor are left out.
constexpr float kSlack = 8;
template <typename T, int B>
__device__ __forceinline__ void soften(const f32x16 (&st)[2], u32x4 (&p)[4], f32x16 (&o)[B], float& m, float& l, float scale) {
  float x[32], top = m;
#pragma unroll
  for (int r = 0; r < 32; ++r) x[r] = st[r >> 4][r & 15] * scale;
#pragma unroll
  for (int r = 0; r < 32; ++r) top = fmaxf(top, x[r]);
  top = max32(top);
  if (__any(top > m + kSlack)) {
    const float f = __builtin_amdgcn_exp2f(m - origin(top));
    l *= f;
#pragma unroll
    for (int b = 0; b < B; ++b) o[b] *= f;
    m = top;
  }
  const float base = origin(m);
#pragma unroll
  for (int r = 0; r < 32; r += 2) {
    const float p0 = __builtin_amdgcn_exp2f(x[r] - base), p1 = __builtin_amdgcn_exp2f(x[r + 1] - base);
    l += p0 + p1;
    p[r >> 3][(r & 7) >> 1] = pack2<T>(p0, p1);
  }
}

template <typename T, int D, int NW, bool EXACT>
__global__ void __launch_bounds__(NW * 64, NW / 4) paged_prompt_kernel(PromptArgs a, int ntile) {
  constexpr int ROWS = 32 * NW, CPR = D / 8;  // 16-byte chunks of a row
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
    q[n] ^= c.flip;
  }
  f32x16 o[blocks32];
#pragma unroll
  for (int b = 0; b < blocks32; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0;
  float m = kNegInf, l = 0;

  // tiles come by DMA, 1 KiB an instruction: RPI rows, whose page is one, and 16 bytes
  // a lane, which takes the chunk that belongs at its place
  constexpr int RPI = 64 / CPR, PER = kTile / RPI / NW;
  const auto fk = [](int r) { return D == 64 ? (r >> 1) & 7 : r & 15; };
  const auto fv = [](int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; };
  const int width = int(c.capacity >> c.page_shift), inrow = lane / CPR;
  const int32_t* const table = c.tables + s * c.table_stride;
  // lane x % 4 holds the page of the tile's keys 16 x .. 16 x + 15; -1: none
  const auto pages_of = [&](int kb) {
    const int at = (kb + 16 * (lane & 3)) >> c.page_shift;
    const int page = at < width ? table[at] : -1;
    return page < c.pages ? page : -1;
  };
  const auto load = [&](int kb, int pages, int buf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r0 = RPI * (wave + NW * i), r = r0 + inrow;
      const int page = max(0, __builtin_amdgcn_readlane(pages, r0 >> 4)), in = (kb + r0) & ((1 << c.page_shift) - 1);
      const T* const kp = static_cast<const T*>(c.k) + page * c.k_page + kvh * c.k_head + in * c.k_token;
      const T* const vp = static_cast<const T*>(c.v) + page * c.v_page + kvh * c.v_head + in * c.v_token;
      const int xk = (lane % CPR) ^ fk(r), xv = (lane % CPR) ^ fv(r);
      if (EXACT || 8 * xk < c.dim) dma16(kp + inrow * c.k_token + 8 * xk, kbuf + (buf * kTile + r0) * D);
      if (EXACT || 8 * xv < c.dim) dma16(vp + inrow * c.v_token + 8 * xv, vbuf + (buf * kTile + r0) * D);
    }
  };
  // the wave's own loads have arrived; rows of V that are no key of the sequence's hold
  // whatever their page does, and P's zeros would not silence a NaN there
  const auto arrived = [&](int kb, uint32_t ok, int buf) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (ok != 15 || kb + kTile > len) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r0 = RPI * (wave + NW * i), r = r0 + inrow;
        if (kb + r >= len || !(ok >> (r0 >> 4) & 1))
          *reinterpret_cast<u32x4*>(vbuf + (buf * kTile + r0) * D + 8 * lane) = u32x4{0, 0, 0, 0};
      }
    }
    __syncthreads();
  };
  if (!EXACT) {  // columns beyond dim are never loaded
    for (int i = threadIdx.x; i < 4 * kTile * CPR; i += NW * 64) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }

  int kb = 0, next = 0, pages = -1;
  uint32_t ok = 0, next_ok = 0;
  if (i0 < i1) {
    kb = blocks.at(i0) * kTile;
    const int mine = pages_of(kb);
    ok = uint32_t(__ballot(mine >= 0)) & 15;
    if (i0 + 1 < i1) pages = pages_of(blocks.at(i0 + 1) * kTile);
    load(kb, mine, 0);
    arrived(kb, ok, 0);
  }
  for (int i = i0; i < i1; ++i, kb = next, ok = next_ok) {
    const int buf = (i - i0) & 1;
    if (i + 1 < i1) {
      next = blocks.at(i + 1) * kTile;
      const int mine = pages;
      next_ok = uint32_t(__ballot(mine >= 0)) & 15;
      if (i + 2 < i1) pages = pages_of(blocks.at(i + 2) * kTile);
      load(next, mine, buf ^ 1);
    }
    const bool any = kb <= wmax && (c.window == 0 || kb + kTile > wmin - c.window + 1 || kb < c.sinks);
    if (any) {
      f32x16 st[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[t][r] = 0;
#pragma unroll
      for (int n = 0; n < steps; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int r = 32 * t + col;
          const u32x4 kf = *reinterpret_cast<const u32x4*>(kbuf + (buf * kTile + r) * D + 8 * ((2 * n + half) ^ fk(r)));
          st[t] = Half<T>::mma32(kf, q[n], st[t]);
        }
      const bool whole = ok == 15 && kb + kTile - 1 <= wmin && (c.window == 0 || kb > wmax - c.window || kb + kTile <= c.sinks);
      u32x4 p[4];
      if (!whole) {  // before the scale, which is positive: the compiler would canonicalise
                     // each of the values that pass a join of branches into a maximum
#pragma unroll
        for (int r = 0; r < 32; ++r) {
          const int key = 8 * (r >> 2) + 4 * half + (r & 3), at = kb + key;
          const bool sees = (at <= place) & ((at > from) | (at < c.sinks)) & bool(ok >> (key >> 4) & 1);
          st[r >> 4][r & 15] = sees ? st[r >> 4][r & 15] : kNegInf;
        }
      }
      soften<T, blocks32>(st, p, o, m, l, c.scale);
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
                           vbuf + (buf * kTile + r) * D + 8 * ((d >> 3) ^ fv(r)) + (d & 7))));
            vt[2 * e] = x[0];
            vt[2 * e + 1] = x[1];
          }
          o[b] = Half<T>::mma32(vt, p[t], o[b]);
        }
    }
    if (i + 1 < i1) arrived(next, next_ok, buf ^ 1);
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
