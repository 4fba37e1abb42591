// Attention of one new token per sequence where groups of sequences share a prefix: the
// keys and values of the prefix are read once for the group, what follows for each
// sequence.
//   o = sum_j 2^(s_j - m) v_j / l over the prefix's keys and the sequence's own, as in
//   attention_decode.hip, with the two parts' m, l and o joined at the end.
//
// 4 dim bytes of K and V a key and key/value head against 4 dim operations a query: reading
// them bounds it up to some hundred queries, and what decides is again that every CU has loads
// under way.  A workgroup a CU works on one kind of keys, the prefixes' or the sequences' own,
// as many on each as its share of the work, of which each takes an equal stretch, counted in
// blocks of 32 keys that a wave takes (and some for the start of another head's keys):
// * own keys by single waves, as in attention_decode.hip, but with no LDS: pieces of a head
//   that several waves have part of go to the workspace;
// * a prefix's keys by whole workgroups.  All its sequences' heads of one key/value head are
//   columns, spread over 1, 2, 4 or 8 waves of 32 columns each (16 in rows of more than 128 values),
//   which read the same keys one soon after the other (a cache answers); the others take every 8th, 4th or 2nd block, and
//   waves that have the same columns add up through LDS.  A workgroup has at most two pieces
//   of heads that it shares with others.
// The products are attention_decode.hip's, with up to two tiles of 16 columns for one load of K and
// V and one transposition of V.  The join kernel adds the pieces in order, so results do not
// depend on timing.
//
// Measured, with the join (7 and 6 us of it): 64 sequences over one prefix of 8,192 keys and up
// to 512 of their own, 16 heads of 128 over 8, 37 us for 103 MB, where attention_decode.hip takes
// 310; five groups of 1 to 12 over prefixes of up to 30,000, 32 heads of 64 over 4, 35 us for
// 114 MB (85).  The prefix of the first is 128 columns, four waves that each read the same keys:
// its loads from the caches, and its products beside them, are what is left.
// Columns of 64 a wave halve those loads, but leave registers for one wave a SIMD (62 us for 42),
// and keys staged in LDS are read as often from there (no gain).
#include "attention.hpp"
#include "shared_rule.hpp"

namespace praghip {
namespace {

template <int D>
struct SharedShape {
  static constexpr int waves = D > 128 ? 4 : 8;  // (rows of 256 values take more than 256 registers)
  // Tiles of 16 columns that a wave has.  Two of them in rows of 256 values take more registers
  // than there are, so that some are kept in accumulator registers: where the compiler copies one
  // there while only some lanes are active, the others' value is lost (tests/test_asm_spills.py).  One
  // is faster too: 8 sequences over 4,000 keys, 8 heads of 256 over 2, 22.7 us for 27.6, 32 31 for 37.
  static constexpr int tiles = D > 128 ? 1 : 2, columns = 16 * tiles;
  static constexpr int steps = D / 32;           // of the first product
  static constexpr int per = D / 16;             // values of a key's row that a lane holds
  static constexpr int words = per / 2;
  static constexpr int row = D + 4;              // a row of o, then m and l
};

// units of a head's keys before its first block (its start takes about as long), and the
// shortest stretch
constexpr int kPrefixStart = 8, kOwnStart = 2, kPrefixLeast = 8, kOwnLeast = 3;

// Keys lo .. hi - 1 of the pages of sequence `first`, for the heads of the sequences from
// it on: `columns` columns of a key/value head.
struct Entry {
  int first, columns, lo, hi;
  __device__ __forceinline__ int begin() const { return lo >> 5; }
  __device__ __forceinline__ int blocks() const { return hi > lo ? ((hi + 31) >> 5) - (lo >> 5) : 0; }
};

// The prefix of a group: as long as its first sequence, whose pages it is read from, at most;
// a group of one has none.
__device__ __forceinline__ Entry prefix_of(const SharedArgs& a, int g) {
  const int first = min(max(a.groups[g], 0), a.c.seqs), end = min(max(a.groups[g + 1], first), a.c.seqs);
  Entry e{first, (end - first) * a.c.group, 0, 0};
  if (end - first > 1) e.hi = min(max(a.shared[g], 0), length_of(a.c, first));
  return e;
}
// What sequence s has of its own, and its group (-1: it takes part in none: a sequence that
// is shorter than the prefix reads all its keys itself).
__device__ __forceinline__ Entry own_of(const SharedArgs& a, int s, int& group) {
  Entry e{s, a.c.group, 0, length_of(a.c, s)};
  group = -1;
  int lo = 0, hi = a.count - 1;  // the last group that starts at or before s
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.groups[mid] <= s)
      lo = mid;
    else
      hi = mid - 1;
  }
  if (a.count > 0 && a.groups[lo] <= s && s < a.groups[lo + 1]) {
    const int prefix = prefix_of(a, lo).hi;
    if (prefix > 0 && e.hi >= prefix) {
      e.lo = prefix;
      group = lo;
    }
  }
  return e;
}

// How many parts a head's columns are cut into, waves (a power of two) that have the columns
// of one part at the same time, units of one part of one head.
template <typename S>
struct Parts {
  int parts, shift;
  uint32_t units;
  __device__ __forceinline__ Parts(bool prefix, int columns, int blocks) {
    shift = prefix ? (columns > S::columns) + (columns > 2 * S::columns) + (columns > 4 * S::columns && S::waves == 8) : 0;
    parts = prefix ? (columns + S::columns * S::waves - 1) / (S::columns * S::waves) : (columns + 15) >> 4;
    units = blocks ? (uint32_t(blocks) << shift) + (prefix ? kPrefixStart : kOwnStart) : 0;
  }
  __device__ __forceinline__ uint32_t all(int kv_heads) const { return units * parts * kv_heads; }
};

// the sum of the lanes up to each, by moves within rows of 16 lanes and from their last ones
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CONTROL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  return v + moved<0x143, 0xc>(v);
}

// Units over workgroups, or waves: each of the first `extra` has one more than the others.
struct Stretches {
  uint32_t count, each, extra;
  __device__ __forceinline__ Stretches(uint32_t units, uint32_t most, uint32_t least) {
    count = max(1u, min(most, units / least));
    each = units / count;
    extra = units - each * count;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return each * w + min(w, extra); }
  // the stretch that holds unit u
  __device__ __forceinline__ uint32_t of(uint32_t u) const {
    const uint32_t longer = extra * (each + 1);
    return u < longer ? u / (each + 1) : extra + (u - longer) / each;
  }
};
// blocks of a head (one of whose blocks is 2^shift units, after its start) before unit u
__device__ __forceinline__ int blocks_before(uint32_t u, uint32_t first, int shift) {
  return u > first ? int((u - first + (1u << shift) - 1) >> shift) : 0;
}
// A column's sequence, from the entry's first, and head of the key/value head (by a product
// where that is exact).
struct Column {
  int member, head;
  __device__ __forceinline__ Column(const SharedArgs& a, int i) {
    member = a.inverse ? int(__umulhi(uint32_t(i), a.inverse)) : i / a.c.group;
    head = i - member * a.c.group;
  }
};

// The workgroups for the prefixes, as their share of the work is: a unit of theirs takes about a
// quarter longer, most of them with two tiles of columns (groups of 5, 1, 9 and 2 over 8,192 keys,
// 512 of their own: 29 us for 33 at the same weight; 64 over 8,192 41.6 for 42.9; 8 over 2,048,
// one tile, and 2,048 of their own 18.9 for 18.2; at half as much again 64 over 32,768 98 for 88).
__device__ __forceinline__ uint32_t prefix_groups(uint32_t prefix, uint32_t own, uint32_t groups) {
  if (!prefix || !own || groups < 2) return prefix ? groups : 0;
  const int less = max(0, 9 - int(__clz(prefix | own)));  // (below 2^23 each, whose products with groups 32 bits hold)
  prefix >>= less, own >>= less;
  prefix += prefix >> 2;
  const uint32_t all = prefix + own, n = (groups * prefix + all / 2) / max(all, 1u);
  return min(max(n, 1u), groups - 1);
}

// The keys of one key/value head h in an entry's blocks first, first + step .. below last,
// for 16 TILES columns from column0 on: o, m and l as of keys in powers of two.
template <typename T, int D, bool EXACT, int TILES>
__device__ __forceinline__ void take_blocks(const SharedArgs& a, const Entry& x, int h, int column0, int first, int last, int step,
                                            f32x4 (&o)[SharedShape<D>::tiles][D / 16], float (&m)[SharedShape<D>::tiles],
                                            float (&l)[SharedShape<D>::tiles]) {
  using S = SharedShape<D>;
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  u32x4 q[TILES][S::steps];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int column = column0 + 16 * t + col;
    const Column of(a, column);
    const int seq = x.first + of.member, head = h * c.group + of.head;
#pragma unroll
    for (int i = 0; i < S::steps; ++i) {
      q[t][i] = u32x4{0, 0, 0, 0};
      const int d = 32 * i + 8 * quad;
      if (column < x.columns && (EXACT || d < c.dim))
        q[t][i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + seq * a.q_seq + head * a.q_head + d);
      q[t][i] ^= c.flip;
    }
  }
  const int32_t* named = c.tables + x.first * c.table_stride;
  const int most = int(c.capacity >> c.page_shift) - 1;
  const auto page_at = [&](int block, int half) { return named[entry_at(x.begin() + block, half, c.page_shift, most)]; };
  int next[2] = {page_at(first, 0), page_at(first, 1)};
  for (int i = first; i < last; i += step) {
    const int kb = (x.begin() + i) << 5;
    u32x4 kf[2][S::steps];
    uint32_t vr[8][S::words];
    bool page_ok[2];
    int pages[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      page_ok[t] = (next[t] >= 0) & (next[t] < c.pages) & ((kb + 16 * t) >> c.page_shift <= most);
      pages[t] = page_ok[t] ? next[t] : 0;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = (kb + 16 * t) & ((1 << c.page_shift) - 1);
      const T* kp = static_cast<const T*>(c.k) + uint64_t(pages[t]) * c.k_page + uint64_t(h) * c.k_head + uint64_t(row + col) * c.k_token + 8 * quad;
#pragma unroll
      for (int n = 0; n < S::steps; ++n) {
        kf[t][n] = u32x4{0, 0, 0, 0};
        if (EXACT || 32 * n + 8 * quad < c.dim) kf[t][n] = *reinterpret_cast<const u32x4*>(kp + 32 * n);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = (kb + 16 * t) & ((1 << c.page_shift) - 1);
      const T* vp = static_cast<const T*>(c.v) + uint64_t(pages[t]) * c.v_page + uint64_t(h) * c.v_head + uint64_t(row + 4 * quad) * c.v_token + S::per * col;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int w = 0; w < S::words; ++w) vr[4 * t + r][w] = 0;
        if (EXACT || S::per * col < c.dim) {
          if constexpr (S::words == 2) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(vp + uint64_t(r) * c.v_token);
            vr[4 * t + r][0] = v[0];
            vr[4 * t + r][1] = v[1];
          } else {
#pragma unroll
            for (int w = 0; w < S::words; w += 4) {
              if (!EXACT && S::per * col + 2 * w >= c.dim) continue;
              const u32x4 v = *reinterpret_cast<const u32x4*>(vp + uint64_t(r) * c.v_token + 2 * w);
#pragma unroll
              for (int b = 0; b < 4; ++b) vr[4 * t + r][w + b] = v[b];
            }
          }
        }
      }
    }
    // (the next block's entries, beside these loads; past the last they are the table's last)
#pragma unroll
    for (int t = 0; t < 2; ++t) next[t] = page_at(i + step, t);
    const bool whole = page_ok[0] && page_ok[1] && kb >= x.lo && kb + 32 <= x.hi;
    u32x4 ph[TILES], pl[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      f32x4 st[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (int n = 0; n < S::steps; ++n) {
        st[0] = Half<T>::mma16(kf[0][n], q[t][n], st[0]);
        st[1] = Half<T>::mma16(kf[1][n], q[t][n], st[1]);
      }
      float s[8];  // before the scale, which is above 0
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = st[r >> 2][r & 3];
      if (!whole) {  // keys that are not the entry's count as nothing, whatever their page holds
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int at = kb + 16 * (r >> 2) + 4 * quad + (r & 3);
          const bool sees = bool(page_ok[r >> 2]) & (at >= x.lo) & (at < x.hi);
          s[r] = sees ? s[r] : kNegInf;
#pragma unroll
          for (int w = 0; w < S::words; ++w) vr[r][w] = sees ? vr[r][w] : 0;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      const float peak = max32(max16(top));
      float by = c.scale;
      top = peak * c.scale - Half<T>::most;
      if (__any(__builtin_fabsf(top) >= kLarge)) {  // scores and their maximum, rounded alike
        by = 1, top = peak * c.scale;
        top -= below_most<T>(top);
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] *= c.scale;
      }
      top = fmaxf(m[t], top);
      if (__any(top > m[t])) {
        const float f = __builtin_amdgcn_exp2f(m[t] - origin(top));
        l[t] *= f;
#pragma unroll
        for (int j = 0; j < S::per; ++j) o[t][j] *= f;
        m[t] = top;
      }
      uint32_t hi[4], rest[4];
      const float from = -origin(m[t]);
#pragma unroll
      for (int r = 0; r < 8; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], by, from)), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], by, from));
        l[t] += p0 + p1;
        hi[r / 2] = pack2<T>(p0, p1);
        rest[r / 2] = pack2<T>(p0 - low<T>(hi[r / 2]), p1 - high<T>(hi[r / 2]));
      }
      ph[t] = u32x4{hi[0], hi[1], hi[2], hi[3]}, pl[t] = u32x4{rest[0], rest[1], rest[2], rest[3]};
    }
#pragma unroll
    for (int j = 0; j < S::per; ++j) {
      u32x4 vt;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        vt[p] = __builtin_amdgcn_perm(vr[2 * p + 1][j / 2], vr[2 * p][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t][j] = Half<T>::mma16(vt, ph[t], o[t][j]);
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t][j] = Half<T>::mma16(vt, pl[t], o[t][j]);
    }
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) l[t] = sum32(sum16(l[t]));
}

// A lane's rows of o, and m and l, at `to` (for the columns of a wave).
template <int D>
__device__ __forceinline__ void store_columns(float* to, int columns, const f32x4 (&o)[SharedShape<D>::tiles][D / 16],
                                              const float (&m)[SharedShape<D>::tiles], const float (&l)[SharedShape<D>::tiles]) {
  using S = SharedShape<D>;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
#pragma unroll
  for (int t = 0; t < S::tiles; ++t) {
    if (16 * t + col >= columns) continue;
    float* p = to + (16 * t + col) * S::row;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < S::per; j += 4)
        *reinterpret_cast<f32x4*>(p + (4 * quad + r) * S::per + j) = f32x4{o[t][j][r], o[t][j + 1][r], o[t][j + 2][r], o[t][j + 3][r]};
    if (quad == 0) {
      p[D] = m[t];
      p[D + 1] = l[t];
    }
  }
}

template <typename T, int D, bool EXACT>
__global__ void __launch_bounds__(SharedShape<D>::waves * 64) paged_shared_kernel(SharedArgs a) {
  using S = SharedShape<D>;
  constexpr int W = S::waves;
  extern __shared__ __attribute__((aligned(16))) float lds[];  // [W][columns] rows
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = c.kv_heads * c.group;

  // units before each stretch of groups, and of sequences, one stretch per lane; every wave
  // counts for itself
  const int per_group = (a.count + 63) >> 6, per_seq = (c.seqs + 63) >> 6;
  uint32_t mine_p = 0, mine_o = 0;
  Entry last_p{0, 0, 0, 0}, last_o{0, 0, 0, 0};  // a lane's one entry, where it has one
  int group = -1;
  const bool few = per_group <= 1 && per_seq == 1;
  if (few) {  // all loads at once; what they depend on is in the lanes
    const bool has = lane < a.count;
    int begin = 0, stop = 0, shared = 0;
    if (a.count > 0) {  // (all lanes load, as others read them)
      begin = a.groups[min(lane, a.count)], stop = a.groups[min(lane + 1, a.count)], shared = a.shared[min(lane, a.count - 1)];
    }
    const int length = length_of(c, min(lane, c.seqs - 1));
    const int first = min(max(begin, 0), c.seqs), end = min(max(stop, first), c.seqs);
    const int longest = __shfl(length, min(first, 63), 64);
    last_p = {first, (end - first) * c.group, 0, end - first > 1 ? min(max(shared, 0), longest) : 0};
    last_o = {lane, c.group, 0, length};
    for (int g = 0; g < a.count; ++g) {
      const int prefix = __builtin_amdgcn_readlane(last_p.hi, g);
      if (lane >= __builtin_amdgcn_readlane(begin, g) && lane < __builtin_amdgcn_readlane(stop, g)) {
        const bool part = prefix > 0 && length >= prefix;
        last_o.lo = part ? prefix : 0;
        group = part ? g : -1;
      }
    }
    if (has) mine_p = Parts<S>(true, last_p.columns, last_p.blocks()).all(c.kv_heads);
    if (lane < c.seqs) mine_o = Parts<S>(false, last_o.columns, last_o.blocks()).all(c.kv_heads);
  } else {
    for (int i = 0; i < per_group; ++i)
      if (lane * per_group + i < a.count) {
        const Entry x = prefix_of(a, lane * per_group + i);
        mine_p += Parts<S>(true, x.columns, x.blocks()).all(c.kv_heads);
      }
    for (int i = 0; i < per_seq; ++i)
      if (lane * per_seq + i < c.seqs) {
        const Entry x = own_of(a, lane * per_seq + i, group);
        mine_o += Parts<S>(false, x.columns, x.blocks()).all(c.kv_heads);
      }
  }
  const uint32_t sum_p = wave_scan(mine_p), sum_o = wave_scan(mine_o);  // inclusive
  const uint32_t total_p = uint32_t(__builtin_amdgcn_readlane(int(sum_p), 63)), total_o = uint32_t(__builtin_amdgcn_readlane(int(sum_o), 63));
  if (blockIdx.x == 0 && wave == 0) {  // for the join
    if (lane == 0) a.entries[a.count + c.seqs] = uint4{total_p, total_o, 0, 0};
    uint32_t at_p = sum_p - mine_p, at_o = sum_o - mine_o;
    if (few) {
      if (lane < a.count) a.entries[lane] = uint4{at_p, uint32_t(last_p.blocks()), uint32_t(last_p.first), uint32_t(last_p.columns)};
      if (lane < c.seqs) a.entries[a.count + lane] = uint4{at_o, uint32_t(last_o.blocks()), uint32_t(group), uint32_t(last_o.columns)};
    } else {
      for (int e = lane * per_group; e < min((lane + 1) * per_group, a.count); ++e) {
        const Entry x = prefix_of(a, e);
        a.entries[e] = uint4{at_p, uint32_t(x.blocks()), uint32_t(x.first), uint32_t(x.columns)};
        at_p += Parts<S>(true, x.columns, x.blocks()).all(c.kv_heads);
      }
      for (int e = lane * per_seq; e < min((lane + 1) * per_seq, c.seqs); ++e) {
        const Entry x = own_of(a, e, group);
        a.entries[a.count + e] = uint4{at_o, uint32_t(x.blocks()), uint32_t(group), uint32_t(x.columns)};
        at_o += Parts<S>(false, x.columns, x.blocks()).all(c.kv_heads);
      }
    }
  }
  const uint32_t prefixes = prefix_groups(total_p, total_o, gridDim.x);
  const bool kind = blockIdx.x >= prefixes;  // own keys
  const uint32_t total = kind ? total_o : total_p;
  const Stretches stretches(total, kind ? (gridDim.x - prefixes) * W : prefixes, kind ? kOwnLeast : kPrefixLeast);
  // (stretch i of the own keys: waves of different workgroups first)
  const uint32_t mine_at = kind ? (blockIdx.x - prefixes) + wave * (gridDim.x - prefixes) : blockIdx.x;
  if (mine_at >= stretches.count || !total) return;
  const uint32_t u_begin = stretches.begin(mine_at), u_end = stretches.begin(mine_at + 1);
  uint32_t u = u_begin;
  const uint32_t to_lane = kind ? sum_o : sum_p;
  const Entry last{kind ? last_o.first : last_p.first, kind ? last_o.columns : last_p.columns, kind ? last_o.lo : last_p.lo, kind ? last_o.hi : last_p.hi};
  const int from_lane = __popcll(__ballot(to_lane <= u)), each = kind ? per_seq : per_group, entries = kind ? c.seqs : a.count;
  int e = from_lane * each;
  uint32_t base = uint32_t(__builtin_amdgcn_readlane(int(to_lane - (kind ? mine_o : mine_p)), from_lane));

  for (; u < u_end && e < entries; ++e) {
    Entry x;
    if (few) {  // the lanes have them
      x = {__builtin_amdgcn_readlane(last.first, e), __builtin_amdgcn_readlane(last.columns, e), __builtin_amdgcn_readlane(last.lo, e),
           __builtin_amdgcn_readlane(last.hi, e)};
    } else {
      int none;
      x = kind ? own_of(a, e, none) : prefix_of(a, e);
      x = {__builtin_amdgcn_readfirstlane(x.first), __builtin_amdgcn_readfirstlane(x.columns), __builtin_amdgcn_readfirstlane(x.lo),
           __builtin_amdgcn_readfirstlane(x.hi)};
    }
    const int nb = x.blocks();
    const Parts<S> parts(!kind, x.columns, nb);
    const uint32_t all = parts.all(c.kv_heads);
    while (u < min(u_end, base + all)) {
      const int index = int((u - base) / parts.units), h = parts.parts == 1 ? index : index / parts.parts, column0 = (index - h * parts.parts) * (kind ? 16 : S::columns * W);
      const uint32_t start = base + index * parts.units + (kind ? kOwnStart : kPrefixStart), stop = min(u_end, base + (index + 1) * parts.units);
      const int first = blocks_before(u, start, parts.shift), end = blocks_before(stop, start, parts.shift);
      u = stop;
      if (first >= end) continue;
      f32x4 o[S::tiles][S::per];
      float m[S::tiles], l[S::tiles];
#pragma unroll
      for (int t = 0; t < S::tiles; ++t) {
        m[t] = kNegInf, l[t] = 0;
#pragma unroll
        for (int j = 0; j < S::per; ++j) o[t][j] = f32x4{0, 0, 0, 0};
      }
      const bool complete = first == 0 && end == nb;
      const int cw = 1 << parts.shift, kw = kind ? 1 : W >> parts.shift, part = kind ? 0 : wave >> parts.shift;
      const int mine0 = kind ? column0 : column0 + (wave & (cw - 1)) * S::columns;
      if (mine0 < x.columns && first + part < end) {
        if (S::tiles == 1 || kind || x.columns <= 16)
          take_blocks<T, D, EXACT, 1>(a, x, h, mine0, first + part, end, kw, o, m, l);
        else if constexpr (S::tiles > 1)
          take_blocks<T, D, EXACT, S::tiles>(a, x, h, mine0, first + part, end, kw, o, m, l);
      }
      if (kind) {
        float* to = complete ? a.rows + ((int64_t(c.seqs) + x.first) * heads + h * c.group + column0) * S::row
                             : a.own_pieces + (int64_t(mine_at) * 2 + (start >= u_begin)) * a.own_columns * S::row;
        store_columns<D>(to, min(x.columns - column0, 16), o, m, l);
        continue;
      }
      // the sums of waves that have the same columns
      __syncthreads();  // the rows of the head before have been read
      store_columns<D>(lds + wave * S::columns * S::row, x.columns - mine0, o, m, l);
      __syncthreads();
      const int have = min(x.columns - column0, S::columns * cw), waves = min(kw, end - first);
      float* const to = complete ? a.rows : a.pieces + (int64_t(mine_at) * 2 + (start >= u_begin)) * a.columns * S::row;
#pragma unroll 2
      for (int i = threadIdx.x; i < have * (D / 4); i += W * 64) {
        const int column = i / (D / 4), d = i % (D / 4) * 4;
        const float* from = lds + column * S::row;  // (one wave's columns after the other's)
        float top = from[D], ls = from[D + 1];
        f32x4 sums = *reinterpret_cast<const f32x4*>(from + d);
        for (int n = 1; n < waves; ++n) {
          const float* p = from + n * cw * S::columns * S::row;
          const float m = p[D], l = p[D + 1], most = fmaxf(top, m);
          const f32x4 o = *reinterpret_cast<const f32x4*>(p + d);
          const float f0 = __builtin_amdgcn_exp2f(top - origin(most)), f1 = __builtin_amdgcn_exp2f(m - origin(most));
          sums = sums * f0 + o * f1;
          ls = ls * f0 + l * f1;
          top = most;
        }
        int64_t row = column;
        if (complete) {
          const Column of(a, column0 + column);
          row = int64_t(x.first + of.member) * heads + h * c.group + of.head;
        }
        // (past the caches: a kernel's end waits for the lines that they hold)
        __builtin_nontemporal_store(sums, reinterpret_cast<f32x4*>(to + row * S::row + d));
        if (d == 0) __builtin_nontemporal_store(f32x4{top, ls, 0, 0}, reinterpret_cast<f32x4*>(to + row * S::row + D));
      }
    }
    base += all;
  }
}

// One workgroup per sequence and head: the pieces of its prefix and of its own keys, in
// order.  Each D / 4 threads take every (1024 / D)-th piece.
template <typename T, int D>
__global__ void __launch_bounds__(256) shared_join_kernel(SharedArgs a, unsigned workgroups) {
  using S = SharedShape<D>;
  constexpr int per = D / 4, sets = 256 / per, W = S::waves;
  __shared__ __attribute__((aligned(16))) float part[sets][D];
  __shared__ float tops[sets], sums[sets];
  const CacheArgs& c = a.c;
  const int all = c.kv_heads * c.group, s = blockIdx.x / all, head = blockIdx.x - s * all, kvh = head / c.group;
  const int set = threadIdx.x / per, d = threadIdx.x % per * 4;
  const uint4 totals = a.entries[a.count + c.seqs], own = a.entries[a.count + s];
  const uint32_t prefixes = prefix_groups(totals.x, totals.y, workgroups);
  float m = kNegInf, l = 0;
  f32x4 o = {0, 0, 0, 0};
  int turn = 0;  // pieces before this kind's
  for (int kind = 0; kind < 2; ++kind) {
    if (kind == 0 && int(own.z) < 0) continue;
    const uint4 x = kind ? own : a.entries[own.z];
    const int nb = int(x.y), columns = int(x.w), cut = kind ? 16 : S::columns * W;
    if (!nb) continue;
    const Parts<S> parts(!kind, columns, nb);
    const Stretches stretches = kind ? Stretches(totals.y, (workgroups - prefixes) * W, kOwnLeast) : Stretches(totals.x, prefixes, kPrefixLeast);
    const int column = (kind ? 0 : (s - int(x.z)) * c.group) + head - kvh * c.group;
    const uint32_t start = x.x + (uint32_t(kvh) * parts.parts + column / cut) * parts.units + (kind ? kOwnStart : kPrefixStart);
    const uint32_t stop = start + (uint32_t(nb) << parts.shift);
    const uint32_t w0 = stretches.of(start), w1 = stretches.of(stop - 1);
    const bool complete = blocks_before(min(stop, stretches.begin(w0 + 1)), start, parts.shift) == nb;
    const uint32_t count = complete ? 1 : w1 - w0 + 1;
    for (uint32_t i = (set + sets - turn % sets) % sets; i < count; i += sets) {
      const uint32_t w = w0 + i, from = stretches.begin(w);
      if (blocks_before(from, start, parts.shift) >= blocks_before(min(stop, stretches.begin(w + 1)), start, parts.shift)) continue;  // no block of it
      const int64_t piece = int64_t(w) * 2 + (start >= from);
      const float* p = complete ? a.rows + ((int64_t(kind) * c.seqs + s) * all + head) * S::row
                       : kind   ? a.own_pieces + (piece * a.own_columns + column % cut) * S::row
                                : a.pieces + (piece * a.columns + column % cut) * S::row;
      const f32x4 po = *reinterpret_cast<const f32x4*>(p + d);
      const float pm = p[D], pl = p[D + 1], top = fmaxf(m, pm);
      const float f = __builtin_amdgcn_exp2f(m - origin(top)), pf = __builtin_amdgcn_exp2f(pm - origin(top));
      o = o * f + po * pf;
      l = l * f + pl * pf;
      m = top;
    }
    turn += int(count);
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
  if (int(threadIdx.x) < c.dim) static_cast<T*>(a.out)[s * a.out_seq + head * a.out_head + threadIdx.x] = T(sum * inv);
  if (a.lse && threadIdx.x == 0) a.lse[int64_t(s) * all + head] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int D>
hipError_t launch(const SharedArgs& a, unsigned workgroups, hipStream_t s) {
  using S = SharedShape<D>;
  constexpr size_t lds = size_t(S::waves) * S::columns * S::row * sizeof(float);
  const auto kernel = a.c.dim == D ? paged_shared_kernel<T, D, true> : paged_shared_kernel<T, D, false>;
  hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(S::waves * 64), lds, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3(unsigned(a.c.seqs) * a.c.kv_heads * a.c.group), dim3(256), 0, s, a, workgroups);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_dim(const SharedArgs& a, unsigned workgroups, hipStream_t s) {
  return a.c.dim <= 64 ? launch<T, 64>(a, workgroups, s) : a.c.dim <= 128 ? launch<T, 128>(a, workgroups, s) : launch<T, 256>(a, workgroups, s);
}

int width_of(size_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

}  // namespace

// One workgroup a CU, and no more than there is work for.
unsigned shared_workgroups(size_t entries, size_t kv_heads, size_t group, size_t keys) {
  const size_t units = entries * kv_heads * ((group + 15) / 16) * ((keys + 31) / 32 + kPrefixStart);
  return unsigned(std::max<size_t>(2, std::min<size_t>(units / kPrefixLeast, 256)));
}
size_t shared_own_columns(size_t group) { return std::min<size_t>(group, 16); }
size_t shared_waves(size_t dim) { return dim > 128 ? SharedShape<256>::waves : SharedShape<128>::waves; }
size_t shared_columns(size_t seqs, size_t group, size_t dim) {
  using Wide = SharedShape<256>;
  using Narrow = SharedShape<128>;
  return std::min<size_t>((seqs * group + 31) / 32 * 32, dim > 128 ? Wide::waves * Wide::columns : Narrow::waves * Narrow::columns);
}
// an exact i / group of i below seqs * group as a product's upper half, or 0
uint32_t shared_inverse(size_t seqs, size_t group) {
  return group > 1 && seqs * group * group < (uint64_t(1) << 32) ? uint32_t(((uint64_t(1) << 32) + group - 1) / group) : 0;
}
size_t shared_row_floats(size_t dim) { return width_of(dim) + 4; }

hipError_t launch_paged_shared(const SharedArgs& a, int type, unsigned workgroups, hipStream_t s) {
  return type == PRAGHIP_F16 ? launch_dim<_Float16>(a, workgroups, s) : launch_dim<__bf16>(a, workgroups, s);
}

}  // namespace praghip
