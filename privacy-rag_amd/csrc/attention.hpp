// What the attention kernels (attention_decode.hip, attention_shared.hip, attention_prompt.hip) share:
// the cache as a kernel sees it, which keys a query sees, 16-bit vectors of both
// types with their matrix instructions, and reductions across a wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#include "praghip.h"

namespace praghip {

// Keys and values of one layer in pages: token p of sequence s is row p mod
// page_size of page tables[s][p / page_size], by strides in elements.
struct CacheArgs {
  const void* k;
  const void* v;
  uint32_t k_page, k_head, k_token, v_page, v_head, v_token;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  int pages, page_shift, seqs, kv_heads, group, dim;
  int64_t capacity;  // positions that a row of the table has room for
  int window, sinks;
  float scale;       // of q.k, times log2 e (the kernels work in powers of two), positive:
  uint32_t flip;     // its sign is in the bits that q's values are flipped by
};

struct DecodeArgs {
  CacheArgs c;
  const void* q;
  int64_t q_seq, q_head;
  void* out;
  int64_t out_seq, out_head;
  float* lse;  // [seqs][heads] or null
  float* work;
  uint32_t* base;  // [seqs + 1] key blocks before each sequence
  bool past;       // whether keys and values are read past the caches
};

struct SharedArgs {
  CacheArgs c;
  const void* q;
  int64_t q_seq, q_head;
  void* out;
  int64_t out_seq, out_head;
  float* lse;             // [seqs][heads] or null
  const int32_t* groups;  // [count + 1] first sequences
  const int32_t* shared;  // [count] positions that a group's sequences have in common
  int count;
  // the workspace, in rows of o, m and l
  uint4* entries;                          // [count + seqs + 1]
  float* rows;                             // heads of one piece: [2][seqs][heads]
  float *pieces, *own_pieces;              // in several: [workgroups][2][columns], [waves][2][own_columns]
  int columns, own_columns;
  uint32_t inverse;  // of the heads of a key/value head, or 0
};

struct PromptArgs {
  CacheArgs c;
  const void* q;
  int64_t q_token, q_head;
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens][heads] or null
  const int32_t* starts;
  int total, max_rows, splits;
  float* work;
  float lower;  // how far a score's origin is kept below the maximum, before the scale
};

hipError_t launch_paged_decode(const DecodeArgs& a, int type, unsigned workgroups, hipStream_t s);
hipError_t launch_paged_shared(const SharedArgs& a, int type, unsigned workgroups, hipStream_t s);
hipError_t launch_paged_prompt(const PromptArgs& a, int type, hipStream_t s);
unsigned decode_workgroups(size_t seqs, size_t kv_heads, size_t group, size_t keys);
size_t decode_work_floats(unsigned workgroups, size_t group, size_t dim);
unsigned shared_workgroups(size_t entries, size_t kv_heads, size_t group, size_t keys);
size_t shared_columns(size_t seqs, size_t group, size_t dim);  // of a piece, at most
size_t shared_own_columns(size_t group);
uint32_t shared_inverse(size_t seqs, size_t group);
size_t shared_waves(size_t dim);  // of a workgroup
size_t shared_row_floats(size_t dim);
int prompt_splits(size_t seqs, size_t kv_heads, size_t group, size_t dim, size_t max_rows, size_t keys);
size_t prompt_work_floats(int splits, size_t seqs, size_t kv_heads, size_t group, size_t dim, size_t max_rows);

// ------------------------------------------------------------ 16-bit vectors
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Vectors and matrix instructions of one 16-bit type, and the power of two that P may
// reach in it.
//
// P = 2^(x - m) of a score x in powers of two goes into a product in the type.  bfloat16 has
// as many powers below 1 as 32 bits have, so m is the maximum.  float16 ends at 2^-24: keys 18
// below the strongest in the natural exponent (2^-26) would vanish from O while l counts them,
// 10^5 of them 2e-3 of the output, and all of it where the strongest key's value is 0.  So m
// is kept below the maximum there and P goes up to 2^15; l, O and lse hold the same m.
template <typename T>
struct Half;
template <>
struct Half<__bf16> {
  static constexpr float most = 0;
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Half<_Float16> {
  static constexpr float most = 15;
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// two floats rounded to nearest even and packed
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename Half<T>::v2));
}
template <typename T>
__device__ __forceinline__ float low(uint32_t v) {
  return float(__builtin_bit_cast(typename Half<T>::v2, v)[0]);
}
template <typename T>
__device__ __forceinline__ float high(uint32_t v) {
  return float(__builtin_bit_cast(typename Half<T>::v2, v)[1]);
}

// A value and its partner's, of lanes l and l ^ 32 (l ^ 16).  (The results go through
// variables: a bit cast of a vector's element takes element 0 whatever its index.)
struct Two {
  float a, b;
};
__device__ __forceinline__ Two swap32(float x) {
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t a = r[0], b = r[1];
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Two swap16(float x) {
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  const uint32_t a = r[0], b = r[1];
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float max32(float x) {
  const Two t = swap32(x);
  return fmaxf(t.a, t.b);
}
__device__ __forceinline__ float sum32(float x) {
  const Two t = swap32(x);
  return t.a + t.b;
}
__device__ __forceinline__ float max16(float x) {
  const Two t = swap16(x);
  return fmaxf(t.a, t.b);
}
__device__ __forceinline__ float sum16(float x) {
  const Two t = swap16(x);
  return t.a + t.b;
}

// Scores in powers of two of which 32 bits hold no fraction below 2^-3.  The exponent of one is the
// difference of two numbers that are rounded alike (half a step of 2^24 is twice a probability,
// half a step of 2^31 2^128 times it), and its origin the maximum itself: in float16 what it lies
// below that could be some steps.
constexpr float kLarge = 1 << 20;
template <typename T>
__device__ __forceinline__ float below_most(float top) {  // how far an origin is kept below a maximum
  return Half<T>::most > 0 && __builtin_fabsf(top) < kLarge ? Half<T>::most : 0.f;
}

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_inff();

// A maximum as the exponent's origin: rows that have seen nothing take 0, so that
// their terms are exp2(-inf) = 0 and not exp2(-inf + inf).
__device__ __forceinline__ float origin(float m) { return m == kNegInf ? 0.f : m; }

// Length of a sequence as the kernels use it: inside 0 .. capacity whatever the
// tensor holds.
__device__ __forceinline__ int length_of(const CacheArgs& c, int s) {
  const int64_t n = c.lengths[s];
  return int(n < 0 ? 0 : n > c.capacity ? c.capacity : n);
}

// The key blocks of size 2^shift that queries at positions lo .. hi may see: 0 ..
// first - 1 (the sinks) and second .. end - 1 (the window); first <= second.
struct Blocks {
  int first, second, end;
  __device__ __forceinline__ int count() const { return first + end - second; }
  __device__ __forceinline__ int at(int i) const { return i < first ? i : i - first + second; }
};
__device__ __forceinline__ Blocks visible_blocks(const CacheArgs& c, int lo, int hi, int shift) {
  Blocks b{0, 0, 0};
  if (hi < 0) return b;
  const int size = 1 << shift;
  b.end = (hi >> shift) + 1;
  if (c.window > 0) {
    const int from = max(0, lo - c.window + 1);
    b.first = min((min(c.sinks, from) + size - 1) >> shift, b.end);
    b.second = max(b.first, min(from >> shift, b.end));
  }
  return b;
}

}  // namespace praghip
