// Attention of a prompt's tokens over a paged key/value cache, causal, with a
// sliding window and a few first tokens that stay visible: the query at position p
// sees key j where j <= p and (j < sinks or j > p - window).  The cache holds the
// prompt's own keys already.
//
// One pass over the keys with a running maximum and sum.  4 dim operations per pair
// of query and key on 32x32x16 products bound it, and beside them one exponential
// per pair.  A workgroup takes 32 rows a wave; a row is one token's one head of the
// group that shares a key/value head, so K and V are read once for the group, and
// tiles of 64 keys (32 where a row has 256 values) go through LDS by DMA, four slots in
// turn.  A turn is software-pipelined by hand: 32 keys' exponentials stand beside the next
// 32 keys' scores, LDS reads and loads between the products.
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
//
// 8192 tokens, 16 heads of 128 over 8: 262 to 279 us by card, 1.0 PFLOP/s (a large bfloat16
// product of the library's reaches 1.2): matrix cores and vector units are busy 45% of the time each, hardly
// at once, with the two waves that a SIMD has registers for.  Four chunks of up to 512 tokens
// through a window of 2048, 32 heads of 64 over 4: 54 us, with CUs busy 57% of the time, as
// the chunks' lengths differ (equal stretches of all tiles' keys instead, which a workgroup
// takes across tiles: 71), and twice dim 128's share of exponentials in a busy one.  Three
// prompts of up to 77 tokens: 11 us, a chain of dependent reads.  Rows of 256 values have one
// wave a SIMD and all of its registers: 4096 tokens of 8 heads over 4 197 us, 350 TFLOP/s.
#include "attention.hpp"

#include <type_traits>

namespace praghip {
namespace {

constexpr int kRing = 4;      // tiles of K, and of V, in LDS
constexpr int kGroups = 512;  // groups of 16 keys whose addresses are in LDS, by halves
constexpr int kFlags = 64;    // bytes of LDS beside them
// keys of a tile
template <int D>
constexpr int tile_keys() {
  return D == 256 ? 32 : 64;
}

// LDS addresses as they are: through generic pointers every access would test for null
typedef __attribute__((address_space(3))) char* Lds;
template <typename V>
__device__ __forceinline__ __attribute__((address_space(3))) V* lds_at(Lds p) {
  return (__attribute__((address_space(3))) V*)p;
}

// 16 bytes a lane, from base + its offset, into LDS at M0 + 16 lane.  The
// compiler adds no wait of its own for an asm, so the caller waits before it reads; and
// the asm starts with the wait states that the DMA needs after the writes of M0 (one) and,
// by a VALU, of the base (five).
__device__ __forceinline__ void dma16(uint64_t base, uint32_t offset, Lds to) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(to))))
               : "memory");
}

// (a maximum that keeps NaN takes its operands as they are, with no instructions to
// canonicalise them)
__device__ __forceinline__ float top_of(const f32x16& st) {
  float top = kNegInf;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = __builtin_elementwise_maximum(top, st[r]);
  return top;
}
// The exponents' origin m, and with it l's and O's factor, where the lane's half of the keys
// has `top`.  A new m is the maximum, in float16 2^kLift below it (attention.hpp).  While P
// stays within 2^(kLift + kSlack) the old one stays in use, with the same relative rounding, and
// the products with the factor are left out.  What the slack takes of float16's range is lost for
// small P: with 4, P of 2^-26 of the strongest key's is rounded to 2^-10 of itself, and calls take up to
// 1% longer than with bfloat16's 8 (2000 tokens of 8 heads of 256: 72.9 us of 72.4; with 3, 74.7).
template <typename T>
constexpr float kSlack = Half<T>::most > 0 ? 4 : 8;
template <typename T>
constexpr float kLift = Half<T>::most > 0 ? Half<T>::most - kSlack<T> : 0;
template <typename T, int B>
__device__ __forceinline__ void raise(float top, f32x16 (&o)[B], float& m, float& l, float scale, float lower) {
  const Two both = swap32(top);
  top = __builtin_elementwise_maximum(both.a, both.b);
  if (__any((top - m) * scale > kSlack<T> + kLift<T>)) {
    top = __builtin_elementwise_maximum(kLift<T> > 0 ? top - lower : top, m);
    const float f = __builtin_amdgcn_exp2f((m - origin(top)) * scale);
    l *= f;
#pragma unroll
    for (int b = 0; b < B; ++b) o[b] *= f;
    m = top;
  }
}

template <typename T, int D, int NW, bool EXACT>
__global__ void __launch_bounds__(NW * 64, NW / 4) paged_prompt_kernel(PromptArgs a, int ntile) {
  constexpr int ROWS = 32 * NW, CPR = D / 8;  // 16-byte chunks of a row
  constexpr int steps = D / 16, blocks32 = D / 32;
  extern __shared__ uint32_t lds[];
  constexpr int TK = tile_keys<D>(), ROW = 2 * D, TILE = TK * ROW;  // bytes
  const Lds kbuf = (Lds)lds, vbuf = kbuf + kRing * TILE;  // [kRing][TK][D] each
  const Lds list = vbuf + kRing * TILE, flags = list + 16 * kGroups;
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

  const Blocks blocks = visible_blocks(c, max(0, int(row0 / c.group) + shift), int((min(row0 + ROWS, nrow) - 1) / c.group) + shift, TK == 32 ? 5 : 6);
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
  constexpr int RPI = 64 / CPR, PER = TK / RPI / NW, GROUPS = TK / 16, TURNS = 64 / GROUPS;
  constexpr int AHEAD = TK == 64 ? 3 : 4;  // tiles that K's loads go ahead (the keys of 64 after a turn's are read in it)
  const auto fk = [](int r) { return D == 64 ? (r >> 1) & 7 : r & 15; };
  const auto fv = [](int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; };
  const int width = int(c.capacity >> c.page_shift), inrow = lane / CPR;
  // Where 16 keys begin in memory, kGroups / 2 groups at a time in LDS: the addresses of K
  // and V; the top bit of V's says that they have no page (they read page 0's).
  const auto fill_list = [&](int i) {
    const int at = (i - i0) * GROUPS;
    for (int x = threadIdx.x; x < min(kGroups / 2, (i1 - i) * GROUPS); x += NW * 64) {
      const int key = blocks.at(i + x / GROUPS) * TK + 16 * (x % GROUPS), entry = key >> c.page_shift;
      int page = entry < width ? c.tables[s * c.table_stride + entry] : -1;
      const bool none = page < 0 || page >= c.pages;
      if (none & (key < len)) *lds_at<int>(flags) = 1;
      page = none ? 0 : page;
      const uint32_t in = key & ((1 << c.page_shift) - 1);
      const uint64_t ka = uint64_t(uintptr_t(static_cast<const T*>(c.k) + uint64_t(kvh) * c.k_head + uint64_t(uint32_t(page)) * c.k_page + uint64_t(in) * c.k_token));
      const uint64_t va = uint64_t(uintptr_t(static_cast<const T*>(c.v) + uint64_t(kvh) * c.v_head + uint64_t(uint32_t(page)) * c.v_page + uint64_t(in) * c.v_token));
      *lds_at<u32x4>(list + 16 * (at % kGroups + x)) = u32x4{uint32_t(ka), uint32_t(ka >> 32), uint32_t(va), uint32_t(va >> 32) | (none ? 1u << 31 : 0)};
    }
    __syncthreads();
  };
  // Of these a wave holds 64 in its lanes, one instruction away: an LDS read's latency and
  // a product for each address before each load cost more than the products of a tile.
  uint32_t klow = 0, khigh = 0, vlow = 0, vhigh = 0, koff[PER], voff[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {  // a wave's rows start at a multiple of RPI within 16 keys
    const int r0 = RPI * (wave + NW * n), r = r0 + inrow;
    koff[n] = 2 * ((r & 15) * c.k_token + 8 * ((lane % CPR) ^ fk(r)));
    voff[n] = 2 * ((r & 15) * c.v_token + 8 * ((lane % CPR) ^ fv(r)));
  }
  bool missing = false;  // some key has no page: no tile is taken as seen whole
  // (taken where all lanes are active: what moves klow elsewhere and back then moves all of it)
  const auto lane_of = [](uint32_t lo, uint32_t hi, int x) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(hi, x))) << 32 | uint32_t(__builtin_amdgcn_readlane(lo, x));
  };
  const auto load_k = [&](int at, int slot) {  // `at` counts the tiles from i0
    if (at % TURNS == 0) {
      const u32x2 x = *lds_at<u32x2>(list + 16 * (at * GROUPS % kGroups + lane));
      klow = x[0], khigh = x[1];
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int r0 = RPI * (wave + NW * n);
      const uint64_t base = lane_of(klow, khigh, at % TURNS * GROUPS + (r0 >> 4));
      if (EXACT || 8 * ((lane % CPR) ^ fk(r0 + inrow)) < c.dim) dma16(base, koff[n], kbuf + slot * TILE + r0 * ROW);
    }
  };
  const auto load_v = [&](int at, int slot) {
    if (at % TURNS == 0) {
      const u32x2 x = *lds_at<u32x2>(list + 16 * (at * GROUPS % kGroups + lane) + 8);
      vlow = x[0], vhigh = x[1] & 0x7fffffffu;
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int r0 = RPI * (wave + NW * n);
      const uint64_t base = lane_of(vlow, vhigh, at % TURNS * GROUPS + (r0 >> 4));
      if (EXACT || 8 * ((lane % CPR) ^ fv(r0 + inrow)) < c.dim) dma16(base, voff[n], vbuf + slot * TILE + r0 * ROW);
    }
  };
  // which groups of 16 keys of a tile have a page
  const auto groups_of = [&](int at) {
    uint32_t none = 0;
#pragma unroll
    for (int x = 0; x < GROUPS; ++x) none |= *lds_at<uint32_t>(list + 16 * ((at * GROUPS + x) % kGroups) + 12) >> 31 << x;
    return ~uint32_t(__builtin_amdgcn_readfirstlane(none));
  };
  // The wave's own loads of V's tile and K's after it have arrived, a turn's of later ones
  // are under way; rows of V that are no key of the sequence's hold whatever their page
  // does, and P's zeros would not silence a NaN there.
  const auto arrived = [&](int i, bool more) {
    if (more)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int kb = blocks.at(i) * TK;
    if (missing || kb + TK > len) {
      const uint32_t held = groups_of(i - i0);
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int r0 = RPI * (wave + NW * n);
        if (kb + r0 + inrow >= len || !(held >> (r0 >> 4) & 1))
          *lds_at<u32x4>(vbuf + (i - i0) % kRing * TILE + r0 * ROW + 16 * lane) = u32x4{0, 0, 0, 0};
      }
    }
    __syncthreads();
  };
  if (!EXACT) {  // columns beyond dim are never loaded
    for (int i = threadIdx.x; i < 2 * kRing * TK * CPR; i += NW * 64) *lds_at<u32x4>(kbuf + 16 * i) = u32x4{0, 0, 0, 0};
  }
  if (threadIdx.x == 0) *lds_at<int>(flags) = 0;
  __syncthreads();

  // Fragments of 32 keys: of K, rows for S^T = K Q^T, and of V, by transposed reads for
  // O^T = V^T P^T.  `slot` and t are constants, and so all but a few addresses.
  const auto read_k = [&](int slot, int t, int n) {
    return *lds_at<u32x4>(kbuf + slot * TILE + (32 * t + col) * ROW + 16 * ((2 * n + half) ^ fk(col)));
  };
  const int trow = 4 * half + ((lane & 15) >> 2), tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const auto read_v = [&](int slot, int t, int n, int b, int e) {
    const int r = 32 * t + 16 * n + 8 * e + trow, d = 32 * b + tcol;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(
                                         vbuf + slot * TILE + r * ROW + 16 * ((d >> 3) ^ fv(trow)) + 2 * (d & 7))));
  };

  // Turn i takes tile i through the softmax and into O, 32 keys at a time, each beside the
  // products of the next 32 keys' scores, which depend on nothing in it: the matrix cores
  // run while the exponentials do.  Loads go two tiles ahead for V, three for K.
  //
  // Tiles lo .. hi - 1 are seen whole by all of the wave's rows, none of tile `stop` and
  // later.
  int lo = i0, hi = blocks.first + (wmin + 1) / TK - blocks.second;
  if (c.window > 0) lo = max(blocks.first, blocks.first + (max(0, wmax - c.window + 1) + TK - 1) / TK - blocks.second);
  const int stop = wmax < 0 ? 0 : min(i1, blocks.first + wmax / TK + 1 - blocks.second);
  f32x16 st;           // a turn's first scores,
  float top = kNegInf;  // their maximum before masks,
  u32x4 kf[steps];      // and the next keys
  if (i0 < i1) {
    fill_list(i0);
    missing = *lds_at<int>(flags);
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      if (x < 2 && i0 + x < i1) load_v(x, x);
      if (i0 + x < i1) load_k(x, x);
    }
    arrived(i0, false);
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0;
#pragma unroll
    for (int n = 0; n < steps; ++n) st = Half<T>::mma32(read_k(0, 0, n), q[n], st);
#pragma unroll
    for (int n = 0; n < steps; ++n) kf[n] = read_k(TK == 64 ? 0 : 1, TK == 64 ? 1 : 0, n);
    top = top_of(st);
  }
  const auto turn = [&](int i, auto slot_constant) {
    constexpr int slot = decltype(slot_constant)::value;  // of tile i
    const int at = i - i0;
    const auto more_v = [&] {
      if (i + 2 < i1) load_v(at + 2, (slot + 2) % kRing);
    };
    const auto more_k = [&] {
      if (i + AHEAD < i1) load_k(at + AHEAD, (slot + AHEAD) % kRing);
    };
    if (i + AHEAD < i1 && (at + AHEAD) * GROUPS % (kGroups / 2) == 0) {
      fill_list(i + AHEAD);  // over groups that are long done
      missing = *lds_at<int>(flags);
    }
    if (i < stop) {
      const bool whole = i >= lo && i < hi && !missing;
#pragma unroll
      for (int t = 0; t < TK / 32; ++t) {
        if (!whole) {
          const int kb = blocks.at(i) * TK + 32 * t;
          const uint32_t held = groups_of(at) >> 2 * t;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 8 * (r >> 2) + 4 * half + (r & 3), j = kb + key;
            const bool sees = (j <= place) & ((j > from) | (j < c.sinks)) & bool(held >> (key >> 4) & 1);
            st[r] = sees ? st[r] : kNegInf;
          }
          top = top_of(st);
        }
        raise<T, blocks32>(top, o, m, l, c.scale, a.lower);
        // What follows runs as it stands, each product with what fills its time: the next
        // scores' with exponentials of these, reads of V and the loads; O's with the next
        // scores' maximum and reads of the keys after them.  (The last turn's next keys are
        // what LDS holds, and their scores unused.)
        f32x16 after;
        u32x4 p[2], vf[2][blocks32];
        const float base = -origin(m) * c.scale;
#pragma unroll
        for (int r = 0; r < 16; ++r) after[r] = 0;
        // The wave goes first while it has exponentials to fill, the SIMD's other one then has
        // its O's products beside them (8192 tokens of 16 heads of 128: 272 us, without 281;
        // first in O's products, or in both: no faster).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int n = 0; n < steps; ++n) {
          after = Half<T>::mma32(kf[n], q[n], after);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x2 x = read_v(slot, t, n / blocks32, n % blocks32, e);
            vf[n / blocks32][n % blocks32][2 * e] = x[0];
            vf[n / blocks32][n % blocks32][2 * e + 1] = x[1];
          }
#pragma unroll
          for (int r = 16 * n / steps & ~1; r + 1 < 16 * (n + 1) / steps; r += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(st[r], c.scale, base)), p1 = __builtin_amdgcn_exp2f(fmaf(st[r + 1], c.scale, base));
            l += p0 + p1;
            p[r >> 3][(r & 7) >> 1] = pack2<T>(p0, p1);
          }
          if (t == 0 && n == 0) more_v();
          if (t == 0 && n == steps / 2) more_k();
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        top = kNegInf;
#pragma unroll
        for (int n = 0; n < 2 * blocks32; ++n) {
          o[n % blocks32] = Half<T>::mma32(vf[n / blocks32][n % blocks32], p[n / blocks32], o[n % blocks32]);
          __builtin_amdgcn_sched_barrier(0);
          if (TK == 64)
            kf[n] = t == 0 ? read_k((slot + 1) % kRing, 0, n) : read_k((slot + 1) % kRing, 1, n);
          else
            kf[n] = read_k((slot + 2) % kRing, 0, n);
#pragma unroll
          for (int r = 8 * n / blocks32; r < 8 * (n + 1) / blocks32; ++r) top = __builtin_elementwise_maximum(top, after[r]);
          __builtin_amdgcn_sched_barrier(0);
        }
        st = after;
      }
    } else {
      more_v();
      more_k();
    }
    if (i + 1 < i1) arrived(i + 1, i + AHEAD < i1);
  };
  for (int i = i0; i < i1; i += kRing) {
    turn(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) turn(i + 1, std::integral_constant<int, 1>{});
    if (i + 2 < i1) turn(i + 2, std::integral_constant<int, 2>{});
    if (i + 3 < i1) turn(i + 3, std::integral_constant<int, 3>{});
  }
  // The arguments once more: held across the loop they cost registers that it lacks, and a
  // kernel with anything in scratch memory starts later.
  typedef const __attribute__((address_space(4))) PromptArgs* Again;
  Again again = (Again)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(again));
  // V may hold values that are not finite, and of keys that only some rows of a tile see the
  // others' P of 0 makes NaN.  Where O is not finite it is formed again from the cache, with
  // the maximum known: 32 keys at a time, those with such values one by one, each added where
  // the row sees it.  (8192 tokens that see an infinity take 2 ms.  In the loop above the same
  // test took 3% of every long prompt's time.)
  bool finite = true;
#pragma unroll
  for (int b = 0; b < blocks32; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) finite &= __builtin_fabsf(o[b][r]) < __builtin_inff();
  if (__any(!finite)) {
#pragma unroll
    for (int b = 0; b < blocks32; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] = 0;
    const float base = -origin(m) * c.scale;
#pragma unroll 1
    for (int x = i0 * (TK / 32); x < i1 * (TK / 32); ++x) {
      const int kb = blocks.at(x / (TK / 32)) * TK + 32 * (x % (TK / 32));
      const T *kp[2], *vp[2];  // of either 16 keys
      uint32_t held = 0;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int key = kb + 16 * n, entry = key >> again->c.page_shift;
        const int page = entry < width ? again->c.tables[s * again->c.table_stride + entry] : -1;
        const bool none = page < 0 || page >= again->c.pages;
        const uint64_t at = none ? 0 : page, in = key & ((1 << again->c.page_shift) - 1);
        held |= uint32_t(!none) << n;
        kp[n] = static_cast<const T*>(again->c.k) + uint64_t(kvh) * again->c.k_head + at * again->c.k_page + in * again->c.k_token;
        vp[n] = static_cast<const T*>(again->c.v) + uint64_t(kvh) * again->c.v_head + at * again->c.v_page + in * again->c.v_token;
      }
      const auto seen = [&](int key) {
        const int j = kb + key;
        return bool((j <= place) & ((j > from) | (j < again->c.sinks)) & bool(held >> (key >> 4) & 1));
      };
      f32x16 score;
#pragma unroll
      for (int r = 0; r < 16; ++r) score[r] = 0;
#pragma unroll
      for (int n = 0; n < steps; ++n) {
        u32x4 k = {0, 0, 0, 0};
        const int d = 16 * n + 8 * half;
        if (EXACT || d < again->c.dim) k = *reinterpret_cast<const u32x4*>((col < 16 ? kp[0] : kp[1]) + uint64_t(col & 15) * again->c.k_token + d);
        score = Half<T>::mma32(k, q[n], score);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool sees = seen(8 * (r >> 2) + 4 * half + (r & 3));
        score[r] = sees ? __builtin_amdgcn_exp2f(fmaf(score[r], c.scale, base)) : 0.f;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        u32x4 p;
#pragma unroll
        for (int w = 0; w < 4; ++w) p[w] = pack2<T>(score[8 * n + 2 * w], score[8 * n + 2 * w + 1]);
#pragma unroll
        for (int b = 0; b < blocks32; ++b) {
          const int d = 32 * b + col;
          u32x4 v = {0, 0, 0, 0};
          bool apart = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = 8 * (e >> 2) + 4 * half + (e & 3);
            uint32_t bits = 0;
            if ((EXACT || d < again->c.dim) && (held >> n & 1) && kb + 16 * n + key < len)
              bits = *reinterpret_cast<const uint16_t*>(vp[n] + uint64_t(key) * again->c.v_token + d);
            constexpr uint32_t exponent = std::is_same<T, __bf16>::value ? 0x7f80 : 0x7c00;
            apart |= (bits & exponent) == exponent;
            v[e >> 1] |= bits << 16 * (e & 1);
          }
          if (!__any(apart)) {
            o[b] = Half<T>::mma32(v, p, o[b]);
            continue;
          }
#pragma unroll 1
          for (int y = 0; y < 16; ++y) {  // key y is slot 4 (y / 8) + y % 4 of half y / 4 % 2
            const int e = (y >> 3) * 4 + (y & 3);
            const bool sees = seen(16 * n + y);
            u32x4 pick;
#pragma unroll
            for (int w = 0; w < 4; ++w) pick[w] = ((half == (y >> 2 & 1)) & (w == e >> 1)) ? 0xffffu << 16 * (e & 1) : 0;
            f32x16 add;
#pragma unroll
            for (int r = 0; r < 16; ++r) add[r] = 0;
            add = Half<T>::mma32(v & pick, p & pick, add);
#pragma unroll
            for (int r = 0; r < 16; ++r) o[b][r] += sees ? add[r] : 0.f;
          }
        }
      }
    }
  }
  l = sum32(l);
  m *= c.scale;

  int place_in = lane;  // (the row's place in the output is found again, too)
  asm volatile("" : "+v"(place_in));
  const int64_t out_row = row0 + wave * 32 + (place_in & 31);
  if (out_row >= nrow) return;
  if (again->splits == 1) {
    const int out_token = int(out_row / again->c.group), out_head = kvh * again->c.group + int(out_row - int64_t(out_token) * again->c.group);
    const float r = l > 0 || l != l ? 1.f / l : 0.f;
    T* out = static_cast<T*>(again->out) + (begin + out_token) * again->out_token + out_head * again->out_head;
#pragma unroll
    for (int b = 0; b < blocks32; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * b + 8 * e + 4 * half;
        if (EXACT || d < again->c.dim)
          *reinterpret_cast<u32x2*>(out + d) = u32x2{pack2<T>(o[b][4 * e] * r, o[b][4 * e + 1] * r), pack2<T>(o[b][4 * e + 2] * r, o[b][4 * e + 3] * r)};
      }
    if (again->lse && half == 0)
      again->lse[int64_t(begin + out_token) * again->c.kv_heads * again->c.group + out_head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
  } else {
    float* to = again->work + (((int64_t(s) * ntile + tile) * again->c.kv_heads + kvh) * again->splits + split) * ROWS * (D + 2);
    const int r = wave * 32 + col;
    // o passes the caches by, which the kernel's end would wait to clean (1024 rows of 32 heads
    // of 64: 24.4 us against 27.2; the few of 16 rows after 30000 keys 38 against 36)
#pragma unroll
    for (int b = 0; b < blocks32; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        __builtin_nontemporal_store(f32x4{o[b][4 * e], o[b][4 * e + 1], o[b][4 * e + 2], o[b][4 * e + 3]},
                                    reinterpret_cast<f32x4*>(to + ((8 * b + 2 * e + half) * ROWS + r) * 4));
    if (half == 0) {
      to[ROWS * D + r] = m;
      to[ROWS * D + ROWS + r] = l;
    }
  }
}

// The splits' m, l and o in order, four values of a row a thread: with the next splits'
// loads under way, and rows side by side as the workspace has them.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptArgs a, int ntile) {
  constexpr int WG = 1024 / D;  // rows of a workgroup
  const CacheArgs& c = a.c;
  int64_t index = int64_t(blockIdx.x) * WG;
  const int chunk = threadIdx.x / WG, r = int(index % ROWS) + threadIdx.x % WG;
  index /= ROWS;
  const size_t piece = size_t(ROWS) * (D + 2);
  const float* const from = a.work + index * a.splits * piece;
  const int kvh = int(index % c.kv_heads);
  index /= c.kv_heads;
  const int tile = int(index % ntile), s = int(index / ntile);
  const int begin = min(max(a.starts[s], 0), a.total), count = min(max(a.starts[s + 1], begin), a.total) - begin;
  const int64_t row = int64_t(tile) * ROWS + r;
  if (row >= int64_t(count) * c.group) return;
  const int token = int(row / c.group), head = kvh * c.group + int(row - int64_t(token) * c.group);
  float m = kNegInf, l = 0;
  f32x4 o = {0, 0, 0, 0};
  constexpr int AT_ONCE = 4;
  for (int i = 0; i < a.splits; i += AT_ONCE) {
    f32x4 po[AT_ONCE];
    float pm[AT_ONCE], pl[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {  // (of the last split again where there are no more, as nothing)
      const float* const p = from + size_t(min(i + j, a.splits - 1)) * piece;
      po[j] = *reinterpret_cast<const f32x4*>(p + (size_t(chunk) * ROWS + r) * 4);
      pm[j] = i + j < a.splits ? p[ROWS * D + r] : kNegInf;
      pl[j] = p[ROWS * D + ROWS + r];
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (i + j >= a.splits) break;
      const float top = fmaxf(m, pm[j]);
      const float f = __builtin_amdgcn_exp2f(m - origin(top)), pf = __builtin_amdgcn_exp2f(pm[j] - origin(top));
      o = o * f + po[j] * pf;
      l = l * f + pl[j] * pf;
      m = top;
    }
  }
  const float inv = l > 0 || l != l ? 1.f / l : 0.f;
  T* const out = static_cast<T*>(a.out) + (begin + token) * a.out_token + head * a.out_head;
  if (4 * chunk < c.dim) *reinterpret_cast<u32x2*>(out + 4 * chunk) = u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  if (a.lse && chunk == 0) a.lse[int64_t(begin + token) * c.kv_heads * c.group + head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
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
  const size_t lds = size_t(2) * kRing * tile_keys<D>() * D * sizeof(T) + 16 * kGroups + kFlags;
  const auto kernel = a.c.dim == D ? paged_prompt_kernel<T, D, NW, true> : paged_prompt_kernel<T, D, NW, false>;
  const unsigned groups = unsigned(ntile) * a.c.seqs * a.c.kv_heads;
  hipLaunchKernelGGL(kernel, dim3(groups * a.splits), dim3(NW * 64), lds, s, a, ntile);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL((prompt_join_kernel<T, D, 32 * NW>), dim3(groups * (32 * NW * D / 1024)), dim3(256), 0, s, a, ntile);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_dim(PromptArgs a, hipStream_t s) {
  a.lower = kLift<T> / a.c.scale;
  return a.c.dim <= 64 ? launch<T, 64, 8>(a, s) : a.c.dim <= 128 ? launch<T, 128, 8>(a, s) : launch<T, 256, 4>(a, s);
}

}  // namespace

int prompt_splits(size_t seqs, size_t kv_heads, size_t group, size_t dim, size_t max_rows, size_t keys) {
  const size_t tiles = size_t(tiles_of(max_rows, group, dim)) * seqs * kv_heads;
  // One tile alone has a CU; more than one of them there gained nothing (16 query heads of
  // 128 over 8, 512 rows after 4000 keys: 37 us, with twice the splits 14 more, with none 130).
  // Shorter stretches than 256 keys cost the join more than they save (16 rows after 300:
  // 13.4, of 128 keys 14.7), in rows of 256 values, whose tiles take longer, than 128 (64
  // rows after 1000: 25.1, of 256 keys 30.4).
  if (!tiles || tiles > 128) return 1;
  return int(std::max<size_t>(1, std::min<size_t>(256 / tiles, keys / (dim > 128 ? 128 : 256))));
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
