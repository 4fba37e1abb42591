// Pages of a key/value cache: writing new tokens, reserving, forking, freeing,
// trimming, compacting and copying.
//
// Who holds what is on the device too (tables, lengths, reference counts), so that a
// call needs no answer from the GPU and can stand in a captured graph.  One
// workgroup decides (checks the lists, finds free pages by counting over the
// reference counts, lowest index first), and a grid moves the bytes; a call that has
// only tables to change is one launch.  What is refused changes nothing and leaves
// its code in `status`.
//
// Moving pages is bound by memory: 2 bytes of traffic a byte, 16-byte accesses, four
// loads of a thread under way.  Their stores pass the caches by: a kernel's end waits for
// the dirty lines of all L2s (a fork's 29 MB of copies: 8.1 us, through the caches 21).  A
// fork takes 5 us of plan before its copies, a compaction's 92 us and 5 of plan.  New tokens
// go through the caches, where the attention finds them: 34 MB in 12.4 us (5.4 TB/s with
// their reads), one token of 64 sequences in 4.1 of the host's 10.
#include "pages.hpp"

#include <algorithm>

#include "page_rule.hpp"
#include "praghip.h"

namespace praghip {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ void refuse(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// Whether the ids of a list are rows of the tables, each once.  All threads of the
// workgroup call it; `seen` is a bit per row.
__device__ __forceinline__ bool distinct(const int32_t* list, int n, int seqs, uint32_t* seen, int* bad) {
  if (threadIdx.x == 0) *bad = 0;
  for (int i = threadIdx.x; i < (seqs + 31) / 32; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = list[i];
    if (s < 0 || s >= seqs || (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1)) *bad = 1;
  }
  __syncthreads();
  const bool fine = *bad == 0;
  __syncthreads();  // the caller may use the flag again
  return fine;
}

// Sum over the workgroup of a wave's value (the same in its lanes), and the sum of
// the waves before; all threads call it.
template <typename T>
__device__ __forceinline__ T waves_before(T value, T* lds, T& total) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave] = value;
  __syncthreads();
  T before = 0;
  total = 0;
  for (int w = 0; w < kWaves; ++w) {
    const T x = lds[w];
    total += x;
    if (w < wave) before += x;
  }
  return before;
}

// A wave's stretch of the pages, in turns of 256: calls f(first page of 64, ballot
// of lanes whose page is held).
template <typename F>
__device__ __forceinline__ void over_pages(const int32_t* refs, int pages, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (pages + kWaves * 64 - 1) / (kWaves * 64) * 64, lo = wave * per, hi = min(pages, lo + per);
  for (int p = lo; p < hi; p += 256) {
    int32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = p + 64 * i + lane < hi ? refs[p + 64 * i + lane] : 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + 64 * i < hi) f(p + 64 * i, min(64, hi - p - 64 * i), __ballot(r[i] > 0));
  }
}

__device__ __forceinline__ uint64_t lanes(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ int below(uint64_t mask) { return __popcll(mask & ((1ull << (threadIdx.x & 63)) - 1)); }

// The free pages of index 0 .. need - 1 by rising page number, given to
// f(index, page); false, and nothing given, where there are fewer.
template <typename F>
__device__ __forceinline__ bool give_free(const int32_t* refs, int pages, int need, int* lds, F f) {
  int mine = 0, total;
  over_pages(refs, pages, [&](int, int n, uint64_t held) { mine += __popcll(~held & lanes(n)); });
  int at = waves_before(mine, lds, total);
  if (total < need) return false;
  over_pages(refs, pages, [&](int p, int n, uint64_t held) {
    const uint64_t free = ~held & lanes(n);
    const int index = at + below(free);
    if ((free >> (threadIdx.x & 63) & 1) && index < need) f(index, p + int(threadIdx.x & 63));
    at += __popcll(free);
  });
  return true;
}

// ----------------------------------------------------------------- free, trim
// Every workgroup checks the whole list and takes its share of the entries.
__global__ void __launch_bounds__(256) page_free_kernel(TableArgs t, const int32_t* list, int n, int window, int sinks,
                                                        bool all) {
  __shared__ uint32_t seen[kMaxSequences / 32];
  __shared__ int bad;
  if (!distinct(list, n, t.seqs, seen, &bad)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) refuse(t.status, PRAGHIP_PAGES_SEQUENCE);
    return;
  }
  const int64_t items = int64_t(n) * t.width, step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += step) {
    const int s = list[i / t.width], at = int(i % t.width);
    if (!all) {  // what the next token, at position length, or a later one sees stays
      const int64_t first = int64_t(at) << t.page_shift, end = first + (1 << t.page_shift);
      if (first < sinks || end - 1 > int64_t(t.lengths[s]) - window) continue;
    }
    int32_t* entry = t.tables + s * t.stride + at;
    const int page = *entry;
    if (page >= 0) {
      if (page < t.pages) atomicSub(t.refs + page, 1);
      *entry = -1;
    }
    if (all && at == 0) t.lengths[s] = 0;
  }
}

// -------------------------------------------------------------------- reserve
__global__ void __launch_bounds__(kThreads) page_reserve_kernel(TableArgs t, const int32_t* list, const int32_t* counts,
                                                                int n) {
  __shared__ uint32_t seen[kMaxSequences / 32];
  __shared__ int start[kMaxList + 1];  // new pages before each sequence's
  __shared__ int64_t sums[kWaves];
  __shared__ int bad, part[kWaves];
  if (!distinct(list, n, t.seqs, seen, &bad)) {
    if (threadIdx.x == 0) refuse(t.status, PRAGHIP_PAGES_SEQUENCE);
    return;
  }
  const int per = (n + kThreads - 1) / kThreads;
  int64_t mine = 0;
  for (int i = threadIdx.x * per; i < min(n, int(threadIdx.x + 1) * per); ++i) {
    const int64_t pages = new_pages(t.lengths[list[i]], counts[i], t.width, t.page_shift);
    if (pages < 0)
      bad = 1;
    else
      mine += pages;
  }
  int64_t sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(sum, d, 64);
    if (int(threadIdx.x & 63) >= d) sum += up;
  }
  int64_t all;
  const int64_t first = waves_before(__shfl(sum, 63, 64), sums, all) + sum - mine;
  if (bad) {
    if (threadIdx.x == 0) refuse(t.status, PRAGHIP_PAGES_CAPACITY);
    return;
  }
  if (all > t.pages) {  // (below that 32 bits hold it)
    if (threadIdx.x == 0) refuse(t.status, PRAGHIP_PAGES_EXHAUSTED);
    return;
  }
  const int need = int(all);
  int before = int(first);
  for (int i = threadIdx.x * per; i < min(n, int(threadIdx.x + 1) * per); ++i) {
    start[i] = before;
    before += int(new_pages(t.lengths[list[i]], counts[i], t.width, t.page_shift));
  }
  if (threadIdx.x == 0) start[n] = need;
  __syncthreads();
  // a stretch's own references are written while others still count: a page that is
  // given has been counted by its own wave, the only one that looks at it again
  const bool done = give_free(t.refs, t.pages, need, part, [&](int index, int page) {
    int lo = 0, hi = n - 1;  // the last sequence with start <= index
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= index)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int s = list[lo];
    t.tables[s * t.stride + pages_for(t.lengths[s], t.page_shift) + index - start[lo]] = page;
    t.refs[page] = 1;
  });
  if (!done) {
    if (threadIdx.x == 0) refuse(t.status, PRAGHIP_PAGES_EXHAUSTED);
    return;
  }
  __syncthreads();  // the old lengths have been read
  for (int i = threadIdx.x; i < n; i += kThreads) t.lengths[list[i]] += counts[i];
}

// i / by and i % by of an i below `most`, in 32 bits where that holds all (a division in 64
// takes some hundred instructions).
struct Parts {
  int64_t whole, rest;
};
__device__ __forceinline__ Parts parts(int64_t i, int64_t by, int64_t most) {
  if (most >> 32 == 0) {
    const uint32_t q = uint32_t(i) / uint32_t(by);
    return {q, uint32_t(i) - q * uint32_t(by)};
  }
  return {i / by, i % by};
}

// ----------------------------------------------------------------------- copy
// moves[i] of all planes, 16 KiB a turn of a workgroup
__device__ __forceinline__ void copy_pages(const PoolArgs& p, const int32_t* from, const int32_t* to, int moves, unsigned block,
                                           unsigned blocks) {
  constexpr int kTurn = 256 * 64;
  const int64_t turns = (p.page_bytes + kTurn - 1) / kTurn, items = turns * p.planes * moves;
  for (int64_t i = block; i < items; i += blocks) {
    const Parts x0 = parts(i, turns, items), x1 = parts(x0.whole, moves, items);
    const int64_t turn = x0.rest;
    const int move = int(x1.rest), plane = int(x1.whole), src = from[move], dst = to[move];
    if (src < 0 || src >= p.pages || dst < 0 || dst >= p.pages || src == dst) continue;
    const char* a = p.base + plane * p.plane_bytes + src * p.page_bytes;
    char* b = p.base + plane * p.plane_bytes + dst * p.page_bytes;
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (no load behind a condition: the compiler would keep x in LDS)
      x[j] = *reinterpret_cast<const u32x4*>(a + min(turn * kTurn + (j * 256 + int64_t(threadIdx.x)) * 16, p.page_bytes - 16));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = turn * kTurn + (j * 256 + threadIdx.x) * 16;
      if (at < p.page_bytes) __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4*>(b + at));
    }
  }
}

__global__ void __launch_bounds__(256) page_copy_kernel(PoolArgs p, const int32_t* from, const int32_t* to, int n) {
  copy_pages(p, from, to, n, blockIdx.x, gridDim.x);
}

// ----------------------------------------------------------------------- fork
// work: kPlanHead words, then n pages to copy from and n to copy to (-1: none)
__global__ void __launch_bounds__(kThreads) fork_plan_kernel(TableArgs t, const int32_t* parents, const int32_t* children,
                                                             int n, int32_t* work) {
  __shared__ uint32_t seen[kMaxSequences / 32];
  __shared__ int bad, part[kWaves];
  int32_t *from = work + kPlanHead, *to = from + n;
  bool fine = distinct(children, n, t.seqs, seen, &bad);
  if (fine) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int s = parents[i];
      if (s < 0 || s >= t.seqs || (seen[s >> 5] >> (s & 31) & 1) || t.lengths[children[i]] != 0 || t.lengths[s] < 0 ||
          t.lengths[s] > int64_t(t.width) << t.page_shift)
        bad = 1;
    }
    __syncthreads();
    fine = bad == 0;
  }
  if (!fine) {
    if (threadIdx.x == 0) {
      work[kPlanAllowed] = 0;
      refuse(t.status, PRAGHIP_PAGES_SEQUENCE);
    }
    return;
  }
  // children whose last page is not full, in order: a wave's stretch of the list each
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (n + kWaves * 64 - 1) / (kWaves * 64) * 64;
  int mine = 0, need;
  for (int i = wave * per + lane; i < (wave + 1) * per; i += 64) {
    int page = -1;
    if (i < n) {
      const int len = t.lengths[parents[i]];
      if (len & ((1 << t.page_shift) - 1)) page = t.tables[parents[i] * t.stride + (len >> t.page_shift)];
      if (page >= t.pages) page = -1;
      from[i] = page;
      to[i] = -1;
    }
    mine += __popcll(__ballot(page >= 0));
  }
  int at = waves_before(mine, part, need);
  // which child takes the k-th free page: kept in `to` until the page is known
  __shared__ int taker[kMaxList];
  for (int i = wave * per + lane; i < (wave + 1) * per; i += 64) {
    const bool takes = i < n && from[i] >= 0;
    const uint64_t mask = __ballot(takes);
    if (takes) taker[at + below(mask)] = i;
    at += __popcll(mask);
  }
  __syncthreads();
  const bool done = give_free(t.refs, t.pages, need, part, [&](int index, int page) {
    to[taker[index]] = page;
    t.refs[page] = 1;
  });
  if (threadIdx.x == 0) {
    work[kPlanAllowed] = done;
    if (!done) refuse(t.status, PRAGHIP_PAGES_EXHAUSTED);
  }
}

__global__ void __launch_bounds__(256) fork_apply_kernel(TableArgs t, PoolArgs p, const int32_t* parents,
                                                         const int32_t* children, int n, const int32_t* work, unsigned table_blocks) {
  if (!work[kPlanAllowed]) return;
  const int32_t *from = work + kPlanHead, *to = from + n;
  const int64_t items = int64_t(n) * t.width;
  if (blockIdx.x >= table_blocks) return copy_pages(p, from, to, n, blockIdx.x - table_blocks, gridDim.x - table_blocks);
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += int64_t(table_blocks) * blockDim.x) {
    const Parts x = parts(i, t.width, items);
    const int child = int(x.whole), at = int(x.rest), s = parents[child], len = t.lengths[s];
    const int count = pages_for(len, t.page_shift);
    int page = at < count ? t.tables[s * t.stride + at] : -1;
    if (at == count - 1 && to[child] >= 0)
      page = to[child];
    else if (page >= 0 && page < t.pages)
      atomicAdd(t.refs + page, 1);
    t.tables[children[child] * t.stride + at] = page;
    if (at == 0) t.lengths[children[child]] = len;
  }
}

// -------------------------------------------------------------------- compact
// work: kPlanHead words, pages / 2 + 1 sources and as many targets, then the new
// index of every page from the count of held pages on
__global__ void __launch_bounds__(kThreads) compact_plan_kernel(int32_t* refs, int pages, int32_t* work) {
  __shared__ int part[kWaves];
  const int most = pages / 2 + 1;
  int32_t *from = work + kPlanHead, *to = from + most, *place = to + most;
  int mine = 0, live, holes = 0, moved = 0, moves, unused;
  over_pages(refs, pages, [&](int, int n, uint64_t held) { mine += __popcll(held & lanes(n)); });
  waves_before(mine, part, live);
  // held pages at `live` or above move into holes below it, both in rising order
  const auto lower = [&](int p, int n) { return lanes(max(0, min(n, live - p))); };
  over_pages(refs, pages, [&](int p, int n, uint64_t held) {
    holes += __popcll(~held & lower(p, n));
    moved += __popcll(held & lanes(n) & ~lower(p, n));
  });
  int hole = waves_before(holes, part, unused), move = waves_before(moved, part, moves);
  over_pages(refs, pages, [&](int p, int n, uint64_t held) {
    const uint64_t empty = ~held & lower(p, n), up = held & lanes(n) & ~lower(p, n), bit = 1ull << (threadIdx.x & 63);
    const int page = p + int(threadIdx.x & 63);
    if (empty & bit) to[hole + below(empty)] = page;
    if (up & bit) from[move + below(up)] = page;
    if (page < p + n && page >= live) place[page] = -1;
    hole += __popcll(empty);
    move += __popcll(up);
  });
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kThreads) {
    place[from[i]] = to[i];
    refs[to[i]] = refs[from[i]];
    refs[from[i]] = 0;
  }
  if (threadIdx.x == 0) {
    work[kPlanMoves] = moves;
    work[kPlanLive] = live;
  }
}

__global__ void __launch_bounds__(256) compact_apply_kernel(TableArgs t, PoolArgs p, const int32_t* work) {
  const int most = t.pages / 2 + 1, moves = work[kPlanMoves], live = work[kPlanLive];
  if (!moves) return;
  const int32_t *from = work + kPlanHead, *to = from + most, *place = to + most;
  const int64_t items = int64_t(t.seqs) * t.width, step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += step) {
    const Parts x = parts(i, t.width, items);
    int32_t* entry = t.tables + x.whole * t.stride + x.rest;
    const int page = *entry;
    if (page >= live && page < t.pages) *entry = place[page];
  }
  copy_pages(p, from, to, moves, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------- write
// One thread per 16 bytes of K and the same of V.
__global__ void __launch_bounds__(256) page_write_kernel(WriteArgs a) {
  const int chunks = a.row_bytes / 16;
  const int64_t items = int64_t(a.tokens) * a.kv_heads * chunks, step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += step) {
    const Parts x0 = parts(i, chunks, items), x1 = parts(x0.whole, a.kv_heads, items);
    const int x = int(x0.rest), h = int(x1.rest), token = int(x1.whole);
    int lo = 0, hi = a.seqs - 1;  // the last sequence that starts at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.starts[mid] <= token)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int begin = a.starts[lo], end = a.starts[lo + 1];
    const int64_t at = int64_t(a.lengths[lo]) - end + token;
    if (token < begin || token >= end || at < 0 || at >> a.page_shift >= a.width) continue;
    const int page = a.tables[lo * a.table_stride + (at >> a.page_shift)];
    if (page < 0 || page >= a.pages) continue;
    const int64_t in = at & ((1 << a.page_shift) - 1);
    *reinterpret_cast<uint4*>(a.k_pages + page * a.kp_page + h * a.kp_head + in * a.kp_token + 16 * x) =
        *reinterpret_cast<const uint4*>(a.k + token * a.k_token + h * a.k_head + 16 * x);
    *reinterpret_cast<uint4*>(a.v_pages + page * a.vp_page + h * a.vp_head + in * a.vp_token + 16 * x) =
        *reinterpret_cast<const uint4*>(a.v + token * a.v_token + h * a.v_head + 16 * x);
  }
}

unsigned grid_of(int64_t items, int64_t per) { return unsigned(std::min<int64_t>(std::max<int64_t>(1, (items + per - 1) / per), 2048)); }
int64_t copy_items(const PoolArgs& p, int64_t moves) { return (p.page_bytes + 256 * 64 - 1) / (256 * 64) * p.planes * moves; }

}  // namespace

hipError_t launch_page_write(const WriteArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(page_write_kernel, dim3(grid_of(int64_t(a.tokens) * a.kv_heads * (a.row_bytes / 16), 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}
hipError_t launch_page_free(const TableArgs& t, const int32_t* list, int n, int window, int sinks, bool all, hipStream_t s) {
  hipLaunchKernelGGL(page_free_kernel, dim3(grid_of(int64_t(n) * t.width, 256)), dim3(256), 0, s, t, list, n, window, sinks, all);
  return hipGetLastError();
}
hipError_t launch_page_reserve(const TableArgs& t, const int32_t* list, const int32_t* counts, int n, hipStream_t s) {
  hipLaunchKernelGGL(page_reserve_kernel, dim3(1), dim3(kThreads), 0, s, t, list, counts, n);
  return hipGetLastError();
}
hipError_t launch_page_fork(const TableArgs& t, const PoolArgs& p, const int32_t* parents, const int32_t* children, int n,
                            int32_t* work, hipStream_t s) {
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kThreads), 0, s, t, parents, children, n, work);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // the tables by workgroups of their own, whose chain of reads is as long as a copy's
  const unsigned tables = std::min(grid_of(int64_t(n) * t.width, 256), 256u);
  hipLaunchKernelGGL(fork_apply_kernel, dim3(tables + grid_of(copy_items(p, n), 1)), dim3(256), 0, s, t, p, parents, children, n, work, tables);
  return hipGetLastError();
}
hipError_t launch_page_compact(const TableArgs& t, const PoolArgs& p, int32_t* work, hipStream_t s) {
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kThreads), 0, s, t.refs, t.pages, work);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_apply_kernel, dim3(2048), dim3(256), 0, s, t, p, work);
  return hipGetLastError();
}
hipError_t launch_page_copy(const PoolArgs& p, const int32_t* from, const int32_t* to, int n, hipStream_t s) {
  hipLaunchKernelGGL(page_copy_kernel, dim3(grid_of(copy_items(p, n), 1)), dim3(256), 0, s, p, from, to, n);
  return hipGetLastError();
}

}  // namespace praghip
