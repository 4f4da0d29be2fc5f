// The cache in 4 bits, as its writers and readers share it.
//
// A value is code * group scale * token scale.  Codes are whole numbers -7..7, 8 of them in a 32-bit word as u = code + 8:
// channel 8 w + 2 i + j in bits 16 j + 4 i of word w, so that a mask leaves neighbouring channels in the halves of a register.
// A group is 16 channels; its scale is an e4m3 number in 0..448.  A token's scale (of one head) is a power of two, held as the
// exponent field of a 32-bit float: 0 for a scale of zero, 255 (infinity) for a row that is not finite.  Code times group scale
// has seven significant bits at most and so is exact in both 16-bit types; the power of two multiplies scores and
// probabilities in 32 bits.  The scales of a page and head lie together: page_size bytes of exponents, then
// page_size * head_dim / 16 bytes of e4m3.
#pragma once
#include "serving.cuh"

namespace risa_b200 {
namespace serving {

// Group scales are read as 16-bit numbers by their bits alone, which makes them 2^-8 of what they are.
constexpr float kGroupUnit = 256.0f;

template <int D>
__host__ __device__ constexpr int token_scale_bytes() { return 1 + D / 16; }

// Where the scales of page `id` and head `head` begin, and those of a slot's groups.
template <int D>
__device__ __forceinline__ const uint8_t* scales4(const void* pool, int64_t id, int kv_heads, int head, int page_shift) {
  return static_cast<const uint8_t*>(pool) + (((id * kv_heads + head) * token_scale_bytes<D>()) << page_shift);
}
template <int D>
__device__ __forceinline__ const uint8_t* groups4(const uint8_t* scales, int page_shift, int slot) {
  return scales + (1 << page_shift) + slot * (D / 16);
}
__device__ __forceinline__ float power_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }
// Its logarithm in units of group scales as they are read, for the running maximum of probabilities times scales.  A scale of zero
// must not let its key's own probability overflow, nor may the largest ones (up to 2^125) leave denominators no room above
// 2^-126: probabilities times scales then grow to 2^15, which fp16 holds.  (Rows that see one that is not finite become NaN.  Where all
// scales that a row sees are below 2^-108 its largest product is below 1, and fp16's smallest numbers leave errors of 2^-133 of a
// probability times scale, 2^-121 of a value, for each key.)
__device__ __forceinline__ float lift_of(uint32_t exponent) {
  return fminf(fmaxf(__uint_as_float(0x4b000000u | exponent) - (8388608.0f + 119.0f), -100.f), 110.f);
}

// Group scales as a pair of 16-bit numbers, and what multiplies the bias of codes + 8 + 2^n.
template <typename M> struct GroupScale;
template <> struct GroupScale<__half> {
  __half2 s, c0, c1;
  // pair: two e4m3 numbers in the low bytes of the halves, zeros above
  __device__ __forceinline__ explicit GroupScale(uint32_t pair) {
    const uint32_t bits = pair << 7;
    s = *reinterpret_cast<const __half2*>(&bits);
    c0 = __hmul2(s, __float2half2_rn(-1032.f));  // exact: 129 times four bits
    c1 = __hmul2(s, __float2half2_rn(-72.f));
  }
};
template <> struct GroupScale<__nv_bfloat16> {
  __nv_bfloat162 s, c0;
  // times 2^(exponent - 127) beside that 2^-8: the token's scale, for whom that range of exponents is no matter
  __device__ __forceinline__ GroupScale(uint32_t pair, float power) {
    const uint32_t bits = pair << 4;  // 2^-120 of the scale
    s = __hmul2(__hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), __float2bfloat162_rn(0x1p112f)), __float2bfloat162_rn(power));
    c0 = __hmul2(s, __float2bfloat162_rn(-136.f));  // exact: 17 times four bits
  }
  __device__ __forceinline__ explicit GroupScale(uint32_t pair) : GroupScale(pair, 1.0f) {}
};
__device__ __forceinline__ uint32_t twice(uint32_t byte) { return byte * 0x00010001u; }

// (a & mask) | bits: one instruction (left to itself the compiler takes two).
__device__ __forceinline__ uint32_t masked(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
// Codes times scales: element i of the result holds field i of both halves of the word.  fp16: 0x6400 + u is 1024 + u, and
// 0x5400 + 16 u is 64 + u; one fused multiply-add removes the bias and scales, exactly.
__device__ __forceinline__ void scaled_codes(uint32_t word, const GroupScale<__half>& g, uint32_t (&x)[4]) {
  const uint32_t above = word >> 8;
  const uint32_t b[4] = {masked(word, 0x000f000fu, 0x64006400u), masked(word, 0x00f000f0u, 0x54005400u), masked(above, 0x000f000fu, 0x64006400u),
                         masked(above, 0x00f000f0u, 0x54005400u)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&b[i]), g.s, i & 1 ? g.c1 : g.c0);
    x[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
// bf16: 0x4300 + u is 128 + u.
__device__ __forceinline__ void scaled_codes(uint32_t word, const GroupScale<__nv_bfloat16>& g, uint32_t (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = masked(word >> (4 * i), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&b), g.s, g.c0);
    x[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

}  // namespace serving
}  // namespace risa_b200
