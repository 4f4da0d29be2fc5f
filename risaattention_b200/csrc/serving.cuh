// What the serving kernels share: the view of a step (sequences, their new tokens, their pages), the
// contract checks of the C-ABI's descriptions, and the word in which kernels report a bad page.
#pragma once
#include "../../include/risa_b200_cache.h"
#include "common.cuh"

namespace risa_b200 {
namespace serving {

constexpr int kInt8 = 4;  // dtype code of a cache of codes

// Address on the current device of the word that records a page outside the pool (sequence + 1 of the
// first one seen); nullptr with the error set where it cannot be had.  Defined in cache_ops.cu.
unsigned int* status_word();

inline int check_cache(const risa_b200_cache* c, const char* what) {
  RISA_REQUIRE(c != nullptr && c->keys != nullptr && c->values != nullptr, "%s: null cache", what);
  RISA_REQUIRE(c->pages > 0 && c->kv_heads > 0, "%s: the cache needs pages and heads", what);
  RISA_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
               "%s: page_size must be 16, 32, 64 or 128", what);
  RISA_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256,
               "%s: head_dim must be 64, 128 or 256", what);
  RISA_REQUIRE(c->dtype_code == 1 || c->dtype_code == 2 || c->dtype_code == kInt8,
               "%s: the cache holds float16, bfloat16 or int8", what);
  RISA_REQUIRE(c->dtype_code != kInt8 || (c->key_scales != nullptr && c->value_scales != nullptr),
               "%s: an int8 cache needs scales", what);
  RISA_REQUIRE((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) % 16 == 0,
               "%s: pages must be 16-byte aligned", what);
  return RISA_B200_OK;
}

inline int check_step(const risa_b200_step* s, const risa_b200_cache* c, const char* what) {
  RISA_REQUIRE(s != nullptr && s->page_table != nullptr && s->lengths != nullptr, "%s: null step", what);
  RISA_REQUIRE(s->batch > 0 && s->batch <= 65535 && s->table_width > 0,
               "%s: batch must be in 1..65535 and the page table must have columns", what);
  RISA_REQUIRE(int64_t(s->table_width) * c->page_size < RISA_B200_CACHE_MOST_SLOTS,
               "%s: a sequence may hold fewer than 2^31 - 8192 keys", what);
  RISA_REQUIRE(s->query_offsets != nullptr || s->tokens == s->batch,
               "%s: without query_offsets every sequence has one token", what);
  RISA_REQUIRE(s->tokens > 0, "%s: no tokens", what);
  return RISA_B200_OK;
}

#ifdef __CUDACC__

// A launch that failed ends its call: what comes behind it reads what it would have written, or relies on its wait.
inline int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return RISA_B200_OK;
  cudaGetLastError();
  return fail(RISA_B200_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// A divisor known to the host: numbers below 2^31 are divided by a multiplication.
struct Divisor {
  int value;
  uint32_t mul, shift;
  __host__ __device__ Divisor() : value(1), mul(0), shift(0) {}
  explicit Divisor(int d) : value(d) {
    uint32_t l = 0;
    while ((int64_t(1) << l) < d) ++l;
    mul = uint32_t((uint64_t(1) << (31 + l)) / uint32_t(d) + 1);
    shift = 31 + l;
  }
  __host__ __device__ __forceinline__ operator int() const { return value; }
};
__device__ __forceinline__ int operator/(int n, const Divisor& d) { return int((uint64_t(uint32_t(n)) * d.mul) >> d.shift); }
__device__ __forceinline__ int operator%(int n, const Divisor& d) { return n - (n / d) * d.value; }

// ---- a step as the kernels see it -----------------------------------------------------------------
struct StepView {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* offsets;
  int batch, width, tokens, page_shift;
};

inline StepView view_of(const risa_b200_step& s, int page_size) {
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  return {s.page_table, s.lengths, s.query_offsets, s.batch, s.table_width, s.tokens, shift};
}

// New tokens of sequence s and its cached length, clamped to what the tensors hold.
struct Sequence {
  int first, count, length;
};
__device__ __forceinline__ Sequence sequence_of(const StepView& v, int s) {
  Sequence q;
  if (v.offsets == nullptr) {
    q.first = s;
    q.count = 1;
  } else {
    q.first = min(max(__ldg(v.offsets + s), 0), v.tokens);
    q.count = max(min(__ldg(v.offsets + s + 1), v.tokens) - q.first, 0);
  }
  q.length = min(max(__ldg(v.lengths + s), 0), v.width << v.page_shift);
  return q;
}

// Keys [lo, hi) that the query at place `place` (may be negative: such a token sees nothing) of a
// sequence of `length` keys sees.
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange visible(int place, int length, bool causal, int window) {
  if (!causal) return {0, length};
  const int hi = min(place + 1, length);
  const int lo = window > 0 ? max(hi - window, 0) : 0;
  return {min(lo, max(hi, 0)), max(hi, 0)};
}

// ---- 16-bit types ------------------------------------------------------------------------------------
template <typename T> struct Half2;
template <> struct Half2<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};
template <> struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};

// D (fp32, 16 x 8) += A (16 x 16) * B (16 x 8).
template <typename T>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, const uint32_t* b);
template <>
__device__ __forceinline__ void mma16816<__half>(float* d, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

#endif  // __CUDACC__
}  // namespace serving
}  // namespace risa_b200
