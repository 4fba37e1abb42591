// The cache's pages: their copies, and the tables, lengths and reference counts that
// say who holds them (pages.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace praghip {

constexpr int kMaxList = 8192;        // sequences of one call
constexpr int kMaxSequences = 131072;  // rows of the tables
// first words of the workspace of a fork or a compaction
enum { kPlanMoves, kPlanAllowed, kPlanLive, kPlanHead = 4 };

struct TableArgs {
  int32_t* tables;   // [seqs][width], -1: no page
  int64_t stride;
  int width, seqs;
  int32_t* lengths;  // [seqs]
  int32_t* refs;     // [pages]: table entries that name the page
  int pages, page_shift;
  int32_t* status;   // or null: the first refusal's code stays
};
struct PoolArgs {
  char* base;  // [planes][pages] pages of page_bytes, a multiple of 16
  int64_t plane_bytes, page_bytes;
  int planes, pages;
};
struct WriteArgs {
  const char *k, *v;  // [tokens][kv_heads][dim]
  int64_t k_token, k_head, v_token, v_head;  // all strides in bytes
  char *k_pages, *v_pages;
  int64_t kp_page, kp_head, kp_token, vp_page, vp_head, vp_token;
  const int32_t *tables, *lengths, *starts;
  int64_t table_stride;
  int width, seqs, pages, page_shift, kv_heads, row_bytes, tokens;
};

hipError_t launch_page_write(const WriteArgs& a, hipStream_t s);
hipError_t launch_page_free(const TableArgs& t, const int32_t* list, int n, int window, int sinks, bool all, hipStream_t s);
hipError_t launch_page_reserve(const TableArgs& t, const int32_t* list, const int32_t* counts, int n, hipStream_t s);
hipError_t launch_page_fork(const TableArgs& t, const PoolArgs& p, const int32_t* parents, const int32_t* children, int n,
                            int32_t* work, hipStream_t s);
hipError_t launch_page_compact(const TableArgs& t, const PoolArgs& p, int32_t* work, hipStream_t s);
hipError_t launch_page_copy(const PoolArgs& p, const int32_t* from, const int32_t* to, int n, hipStream_t s);

}  // namespace praghip
