// C ABI of the serving operators (include/praghip.h): checks of arguments, and the
// launches of attention_decode.hip, attention_prompt.hip, pages.hip and matvec.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "praghip.h"
#include "attention.hpp"
#include "host.hpp"
#include "matvec.hpp"
#include "pages.hpp"

using namespace praghip;
using namespace praghip::host;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
bool power_of_two(size_t n) { return n && !(n & (n - 1)); }
bool eights(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8) return false;
  return true;
}
// strides that the kernels hold in 32 bits: 16 tokens' bytes in one number
bool words(const int64_t* s) {
  return s[0] >= 0 && s[0] <= INT_MAX && s[1] >= 0 && s[1] <= INT_MAX && s[2] >= 0 && s[2] < (1 << 26);
}
int log2_of(size_t n) { return 63 - __builtin_clzll(n); }

// positions that a row of the tables holds, as the kernels count them (32 bits, and
// room for one block of keys beyond)
int64_t capacity_of(size_t width, size_t page_size) {
  return int64_t(std::min<size_t>(width, (INT_MAX - 64) / page_size) * page_size);
}

int check_cache(const praghip_cache* c) {
  if (!c || !c->k || !c->v || !c->tables || !c->lengths) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (c->type != PRAGHIP_BF16 && c->type != PRAGHIP_F16) return fail(PRAGHIP_E_ARGUMENT, "E_ATTENTION_TYPE");
  if (!power_of_two(c->page_size) || c->page_size < 16 || c->page_size > 32768 || !c->head_dim || c->head_dim % 8 ||
      c->head_dim > 256 || !c->pages || c->pages > INT_MAX || !c->kv_heads || c->kv_heads > 65536 || c->seqs > (1u << 20) ||
      !c->table_width || c->table_width > INT_MAX || !words(c->k_strides) || !words(c->v_strides))
    return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_SHAPE");
  if (!aligned16(c->k) || !aligned16(c->v) || !eights(c->k_strides, 3) || !eights(c->v_strides, 3) || !aligned4(c->tables) ||
      !aligned4(c->lengths))
    return fail(PRAGHIP_E_ARGUMENT, "E_ATTENTION_ALIGNMENT");
  return PRAGHIP_OK;
}

CacheArgs cache_args(const praghip_cache& c, size_t heads, float scale, size_t window, size_t sinks) {
  CacheArgs a{};
  a.k = c.k;
  a.v = c.v;
  a.k_page = uint32_t(c.k_strides[0]), a.k_head = uint32_t(c.k_strides[1]), a.k_token = uint32_t(c.k_strides[2]);
  a.v_page = uint32_t(c.v_strides[0]), a.v_head = uint32_t(c.v_strides[1]), a.v_token = uint32_t(c.v_strides[2]);
  a.tables = c.tables;
  a.table_stride = c.table_stride;
  a.lengths = c.lengths;
  a.pages = int(c.pages), a.page_shift = log2_of(c.page_size), a.seqs = int(c.seqs), a.kv_heads = int(c.kv_heads);
  a.group = int(heads / c.kv_heads), a.dim = int(c.head_dim);
  a.capacity = capacity_of(c.table_width, c.page_size);
  // a window that every position fits in is none
  a.window = window >= size_t(a.capacity) ? 0 : int(window);
  a.sinks = int(std::min(sinks, size_t(a.capacity)));
  // a scale of 0 as one that leaves no score above rounding: -inf times it stays -inf
  a.scale = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);
  a.flip = scale < 0 ? 0x80008000u : 0;
  return a;
}

// (a launch's threads are counted in 32 bits: 256 for a sequence's head, 512 for a
// prompt's tile)
bool heads_fit(const praghip_cache& c, size_t heads) {
  return heads && heads % c.kv_heads == 0 && heads <= 65536 && c.seqs * heads < (size_t(1) << 24);
}
bool tiles_fit(const praghip_cache& c, size_t heads, size_t max_rows) {
  const size_t group = heads / c.kv_heads;
  return max_rows <= INT_MAX && max_rows * group / 128 + 1 <= ((size_t(1) << 23) - 1) / std::max<size_t>(1, c.seqs * c.kv_heads);
}
size_t bound_of(const praghip_cache& c, size_t max_length) {
  const size_t most = size_t(capacity_of(c.table_width, c.page_size));
  return max_length ? std::min(max_length, most) : most;
}
// the decode counts blocks of 32 keys over all sequences and heads in 32 bits
bool blocks_fit(const praghip_cache& c, size_t heads) {
  const size_t blocks = size_t(capacity_of(c.table_width, c.page_size)) / 32 + 1;
  return c.seqs * c.kv_heads * ((heads / c.kv_heads + 15) / 16) <= (size_t(1) << 31) / blocks;
}
// keys that a query, or the queries of `rows` neighbours, can see at most
size_t keys_of(size_t bound, size_t rows, size_t window, size_t sinks) {
  return window && window < bound ? std::min(bound, window + std::min(sinks, bound) + rows) : bound;
}

// Workgroups that share a tile's keys, by the arguments that both the call and its workspace
// function have: with the call's smaller max_rows (no longer than its tokens) fewer tiles would
// take more splits than the workspace has room for.
int splits_of(const praghip_cache& c, size_t heads, size_t max_rows, size_t window, size_t sinks, size_t max_length) {
  if (!tiles_fit(c, heads, max_rows)) return 1;
  return prompt_splits(c.seqs, c.kv_heads, heads / c.kv_heads, c.head_dim, max_rows,
                       keys_of(bound_of(c, max_length), max_rows, window, sinks));
}

struct DecodePlan {
  unsigned workgroups;
  size_t base_bytes, bytes;
};
// the same whatever window a call has, so that one workspace serves all of a model's layers
DecodePlan decode_plan(const praghip_cache& c, size_t heads, size_t max_length) {
  DecodePlan p;
  const size_t group = heads / c.kv_heads;
  p.workgroups = decode_workgroups(c.seqs, c.kv_heads, group, bound_of(c, max_length));
  p.base_bytes = ((c.seqs + 1) * sizeof(uint32_t) + 15) / 16 * 16;
  p.bytes = p.base_bytes + decode_work_floats(p.workgroups, group, c.head_dim) * sizeof(float);
  return p;
}

int hip_result(const char* what, hipError_t e) { return e == hipSuccess ? PRAGHIP_OK : hip_fail(what, e); }

int check_table(const praghip_page_table* t, const void* a, const void* b, size_t n) {
  if (!t || !t->tables || !t->lengths || !t->refs || !a || !b) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (!power_of_two(t->page_size) || t->page_size > 32768 || !t->width || t->width > INT_MAX || !t->pages ||
      t->pages > (1u << 28) || t->seqs > size_t(kMaxSequences) || n > size_t(kMaxList))
    return fail(PRAGHIP_E_SHAPE, "E_PAGES_SHAPE");
  if (!aligned4(t->tables) || !aligned4(t->lengths) || !aligned4(t->refs) || !aligned4(t->status) || !aligned4(a) || !aligned4(b))
    return fail(PRAGHIP_E_ARGUMENT, "E_PAGES_ALIGNMENT");
  return PRAGHIP_OK;
}
TableArgs table_args(const praghip_page_table& t) {
  return {t.tables, t.stride, int(t.width), int(t.seqs), t.lengths, t.refs, int(t.pages), log2_of(t.page_size), t.status};
}
int check_pool(const praghip_page_pool* p) {
  if (!p || !p->base) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (!p->page_bytes || p->page_bytes % 16 || p->page_bytes > (1u << 30) || !p->planes || p->planes > INT_MAX || !p->pages ||
      p->pages > (1u << 28))
    return fail(PRAGHIP_E_SHAPE, "E_PAGES_SHAPE");
  if (!aligned16(p->base) || p->plane_bytes % 16) return fail(PRAGHIP_E_ARGUMENT, "E_PAGES_ALIGNMENT");
  return PRAGHIP_OK;
}
PoolArgs pool_args(const praghip_page_pool& p) {
  return {static_cast<char*>(p.base), p.plane_bytes, int64_t(p.page_bytes), int(p.planes), int(p.pages)};
}

}  // namespace

extern "C" {

size_t praghip_paged_decode_workspace(const praghip_cache* c, size_t heads, size_t max_length) {
  if (!c || check_cache(c) || !heads_fit(*c, heads)) return 0;
  return decode_plan(*c, heads, max_length).bytes;
}

int praghip_paged_decode(int device, const praghip_cache* c, const void* q, const int64_t* q_strides, size_t heads, void* out,
                         const int64_t* out_strides, float* lse, float scale, size_t window, size_t sinks, size_t max_length,
                         void* work, size_t work_bytes, void* stream) {
  if (c && c->seqs == 0) return PRAGHIP_OK;
  if (const int rc = check_cache(c)) return rc;
  if (!q || !q_strides || !out || !out_strides || !work) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (!heads_fit(*c, heads) || !blocks_fit(*c, heads) || !std::isfinite(scale)) return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_SHAPE");
  if (!aligned16(q) || !aligned16(out) || !aligned16(work) || !aligned4(lse) || !eights(q_strides, 2) || !eights(out_strides, 2))
    return fail(PRAGHIP_E_ARGUMENT, "E_ATTENTION_ALIGNMENT");
  const DecodePlan p = decode_plan(*c, heads, max_length);
  if (work_bytes < p.bytes) return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_WORKSPACE");
  DecodeArgs a{};
  a.c = cache_args(*c, heads, scale, window, sinks);
  a.q = q, a.q_seq = q_strides[0], a.q_head = q_strides[1];
  a.out = out, a.out_seq = out_strides[0], a.out_head = out_strides[1];
  a.lse = lse;
  a.base = static_cast<uint32_t*>(work);
  a.work = reinterpret_cast<float*>(static_cast<char*>(work) + p.base_bytes);
  // A layer's keys and values that no cache holds until the next token are read past all of
  // them (627 MB: 119 us against 131; 134 MB: 35.5 against 37; 8 MB, which the next call finds
  // there: 15.0 against 13.8).  The host knows a bound of the lengths and not which pages the
  // sequences share: where the bound is far off, or answers share their prompt, the call takes
  // the form that finds less in the caches.
  const double keys = double(keys_of(bound_of(*c, max_length), 1, window, sinks));
  a.past = keys * double(c->seqs * c->kv_heads * c->head_dim) * 4 > double(64 << 20);
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_paged_decode(a, c->type, p.workgroups, pick(stream));
  return hip_result("E_ATTENTION_HIP: ", e);
}

size_t praghip_paged_prompt_workspace(const praghip_cache* c, size_t heads, size_t max_rows, size_t window, size_t sinks,
                                      size_t max_length) {
  if (!c || check_cache(c) || !heads_fit(*c, heads) || !tiles_fit(*c, heads, max_rows)) return 0;
  const int splits = splits_of(*c, heads, max_rows, window, sinks, max_length);
  return prompt_work_floats(splits, c->seqs, c->kv_heads, heads / c->kv_heads, c->head_dim, max_rows) * sizeof(float);
}

int praghip_paged_prompt(int device, const praghip_cache* c, const void* q, const int64_t* q_strides, size_t heads,
                         const int32_t* starts, size_t tokens, size_t max_rows, void* out, const int64_t* out_strides, float* lse,
                         float scale, size_t window, size_t sinks, size_t max_length, void* work, size_t work_bytes,
                         void* stream) {
  if (tokens == 0 || max_rows == 0 || (c && c->seqs == 0)) return PRAGHIP_OK;
  if (const int rc = check_cache(c)) return rc;
  if (!q || !q_strides || !starts || !out || !out_strides) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  const size_t given = max_rows;
  max_rows = std::min(max_rows, tokens);
  if (!heads_fit(*c, heads) || !tiles_fit(*c, heads, max_rows) || !std::isfinite(scale) || tokens > INT_MAX)
    return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_SHAPE");
  if (!aligned16(q) || !aligned16(out) || !aligned16(work) || !aligned4(lse) || !aligned4(starts) || !eights(q_strides, 2) ||
      !eights(out_strides, 2))
    return fail(PRAGHIP_E_ARGUMENT, "E_ATTENTION_ALIGNMENT");
  PromptArgs a{};
  a.splits = splits_of(*c, heads, given, window, sinks, max_length);
  const size_t need =
      prompt_work_floats(a.splits, c->seqs, c->kv_heads, heads / c->kv_heads, c->head_dim, max_rows) * sizeof(float);
  if (need && (!work || work_bytes < need)) return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_WORKSPACE");
  a.c = cache_args(*c, heads, scale, window, sinks);
  a.q = q, a.q_token = q_strides[0], a.q_head = q_strides[1];
  a.out = out, a.out_token = out_strides[0], a.out_head = out_strides[1];
  a.lse = lse;
  a.starts = starts;
  a.total = int(tokens), a.max_rows = int(max_rows);
  a.work = static_cast<float*>(work);
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_paged_prompt(a, c->type, pick(stream));
  return hip_result("E_ATTENTION_HIP: ", e);
}

int praghip_page_reserve(int device, const praghip_page_table* t, const int32_t* list, const int32_t* counts, size_t n,
                         void* stream) {
  if (n == 0) return PRAGHIP_OK;
  if (const int rc = check_table(t, list, counts, n)) return rc;
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_page_reserve(table_args(*t), list, counts, int(n), pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

int praghip_page_free(int device, const praghip_page_table* t, const int32_t* list, size_t n, void* stream) {
  if (n == 0) return PRAGHIP_OK;
  if (const int rc = check_table(t, list, list, n)) return rc;
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_page_free(table_args(*t), list, int(n), 0, 0, true, pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

int praghip_page_trim(int device, const praghip_page_table* t, const int32_t* list, size_t n, size_t window, size_t sinks,
                      void* stream) {
  if (n == 0) return PRAGHIP_OK;
  if (const int rc = check_table(t, list, list, n)) return rc;
  if (!window) return fail(PRAGHIP_E_ARGUMENT, "E_PAGES_WINDOW");
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess)
    e = launch_page_free(table_args(*t), list, int(n), int(std::min<size_t>(window, INT_MAX)), int(std::min<size_t>(sinks, INT_MAX)),
                         false, pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

size_t praghip_page_fork_workspace(size_t n) { return (kPlanHead + 2 * n) * sizeof(int32_t); }

int praghip_page_fork(int device, const praghip_page_table* t, const praghip_page_pool* pool, const int32_t* parents,
                      const int32_t* children, size_t n, void* work, size_t work_bytes, void* stream) {
  if (n == 0) return PRAGHIP_OK;
  if (const int rc = check_table(t, parents, children, n)) return rc;
  if (const int rc = check_pool(pool)) return rc;
  if (!work) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (pool->pages != t->pages) return fail(PRAGHIP_E_SHAPE, "E_PAGES_SHAPE");
  if (!aligned4(work)) return fail(PRAGHIP_E_ARGUMENT, "E_PAGES_ALIGNMENT");
  if (work_bytes < praghip_page_fork_workspace(n)) return fail(PRAGHIP_E_SHAPE, "E_PAGES_WORKSPACE");
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess)
    e = launch_page_fork(table_args(*t), pool_args(*pool), parents, children, int(n), static_cast<int32_t*>(work), pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

size_t praghip_page_compact_workspace(size_t pages) { return (kPlanHead + 2 * (pages / 2 + 1) + pages) * sizeof(int32_t); }

int praghip_page_compact(int device, const praghip_page_table* t, const praghip_page_pool* pool, void* work, size_t work_bytes,
                         void* stream) {
  if (const int rc = check_table(t, work, work, 0)) return rc;
  if (const int rc = check_pool(pool)) return rc;
  if (pool->pages != t->pages) return fail(PRAGHIP_E_SHAPE, "E_PAGES_SHAPE");
  if (work_bytes < praghip_page_compact_workspace(t->pages)) return fail(PRAGHIP_E_SHAPE, "E_PAGES_WORKSPACE");
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_page_compact(table_args(*t), pool_args(*pool), static_cast<int32_t*>(work), pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

int praghip_page_copy(int device, const praghip_page_pool* pool, const int32_t* from, const int32_t* to, size_t n, void* stream) {
  if (n == 0) return PRAGHIP_OK;
  if (const int rc = check_pool(pool)) return rc;
  if (!from || !to) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (n > (1u << 28)) return fail(PRAGHIP_E_SHAPE, "E_PAGES_SHAPE");
  if (!aligned4(from) || !aligned4(to)) return fail(PRAGHIP_E_ARGUMENT, "E_PAGES_ALIGNMENT");
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_page_copy(pool_args(*pool), from, to, int(n), pick(stream));
  return hip_result("E_PAGES_HIP: ", e);
}

int praghip_page_write(int device, const praghip_cache* c, const void* k, const int64_t* k_strides, const void* v,
                       const int64_t* v_strides, const int32_t* starts, size_t tokens, void* stream) {
  if (tokens == 0 || (c && c->seqs == 0)) return PRAGHIP_OK;
  if (const int rc = check_cache(c)) return rc;
  if (!k || !v || !k_strides || !v_strides || !starts) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (tokens > INT_MAX) return fail(PRAGHIP_E_SHAPE, "E_ATTENTION_SHAPE");
  if (!aligned16(k) || !aligned16(v) || !aligned4(starts) || !eights(k_strides, 2) || !eights(v_strides, 2))
    return fail(PRAGHIP_E_ARGUMENT, "E_ATTENTION_ALIGNMENT");
  WriteArgs a{};
  a.k = static_cast<const char*>(k), a.v = static_cast<const char*>(v);
  a.k_token = 2 * k_strides[0], a.k_head = 2 * k_strides[1], a.v_token = 2 * v_strides[0], a.v_head = 2 * v_strides[1];
  a.k_pages = static_cast<char*>(c->k), a.v_pages = static_cast<char*>(c->v);
  a.kp_page = 2 * c->k_strides[0], a.kp_head = 2 * c->k_strides[1], a.kp_token = 2 * c->k_strides[2];
  a.vp_page = 2 * c->v_strides[0], a.vp_head = 2 * c->v_strides[1], a.vp_token = 2 * c->v_strides[2];
  a.tables = c->tables, a.lengths = c->lengths, a.starts = starts, a.table_stride = c->table_stride;
  a.width = int(c->table_width), a.seqs = int(c->seqs), a.pages = int(c->pages), a.page_shift = log2_of(c->page_size);
  a.kv_heads = int(c->kv_heads), a.row_bytes = int(2 * c->head_dim), a.tokens = int(tokens);
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_page_write(a, pick(stream));
  return hip_result("E_ATTENTION_HIP: ", e);
}

int praghip_matvec_w4(int device, const praghip_w4* w, const void* x, int64_t x_stride, size_t m, void* y, int64_t y_stride,
                      void* stream) {
  if (m == 0 || (w && w->n == 0)) return PRAGHIP_OK;
  if (!w || !y || (w->k && (!w->w || !w->scales || !x))) return fail(PRAGHIP_E_ARGUMENT, "E_NULL");
  if (w->type != PRAGHIP_BF16 && w->type != PRAGHIP_F16) return fail(PRAGHIP_E_ARGUMENT, "E_W4_TYPE");
  if (!w->group || w->group % 32 || w->group > (1u << 30) || w->k > (1u << 30) || w->n > (1u << 27) || m > (1u << 20) ||
      w->width > (1u << 30) || w->width < (w->k + 1) / 2)
    return fail(PRAGHIP_E_SHAPE, "E_W4_SHAPE");
  const auto odd = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 1; };
  if (odd(x) || odd(y) || odd(w->scales)) return fail(PRAGHIP_E_ARGUMENT, "E_W4_ALIGNMENT");
  MatvecArgs a{};
  a.x = x, a.x_stride = x_stride;
  a.w = w->w, a.w_stride = w->w_stride;
  a.scales = w->scales, a.scale_stride = w->scale_stride;
  a.zeros = w->zeros, a.zero_stride = w->zero_stride;
  a.y = y, a.y_stride = y_stride;
  a.m = int(m), a.k = int(w->k), a.n = int(w->n), a.group = int(w->group), a.width = int(w->width);
  a.aligned = aligned16(x) && x_stride % 8 == 0 && aligned16(w->w) && w->w_stride % 16 == 0 && w->width % 16 == 0;
  a.vector_scales = aligned16(w->scales) && w->scale_stride % 8 == 0 &&
                    (!w->zeros || ((reinterpret_cast<uintptr_t>(w->zeros) & 7) == 0 && w->zero_stride % 8 == 0));
  DeviceScope scope(device);
  hipError_t e = scope.status();
  if (e == hipSuccess) e = launch_matvec_w4(a, w->type, pick(stream));
  return hip_result("E_W4_HIP: ", e);
}

}  // extern "C"
