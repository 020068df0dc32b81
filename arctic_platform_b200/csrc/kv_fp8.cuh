// The 8-bit key/value cache: layout and conversions that its kernels share.
//
// A block holds the 16 tokens of one (page, key head): 16 rows of D key codes (e4m3), 16 rows of value codes, 32 bytes of exponents.
// A row stands for code * 2^(byte - 127).  Its exponent is a power of two of its own: codes are floating-point numbers, so a finer
// scale would gain nothing but the last half step below 448, while every value of the cache is exactly a bf16 number this way, and
// scaling by it rounds nothing.  One exponent per token, not per page: a page fills one token at a time, and a larger token must
// not touch the codes of the smaller ones before it.  The bytes of tokens t and t + 8 lie side by side, keys then values, as the
// lanes of an MMA tile want them: one 32-bit word per t.
#pragma once
#include "common.cuh"

namespace apb {

constexpr int kKv8Page = 16;
constexpr int kKv8Least = -100, kKv8Most = 119;      // exponents: 2^-100 times the least code and 448 times 2^119 are bf16 numbers

template <int D>
struct Kv8 {
  static constexpr int kHalf = kKv8Page * D;         // key codes of a block
  static constexpr int kBlock = 2 * kHalf + 2 * kKv8Page;
};
__device__ __forceinline__ int kv8_exponent_at(int token, int value) { return 4 * (token & 7) + 2 * value + (token >> 3); }

// The least exponent with which `most` is no more than 448 = 1.75 * 2^8 (infinities take the largest).
__device__ __forceinline__ int kv8_exponent(float most) {
  const int e = static_cast<int>((__float_as_uint(most) + 0x1FFFFFu) >> 23) - (127 + 8);
  return min(max(e, kKv8Least), kKv8Most);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126 to 127

// Two numbers to codes, the nearest ones, ties to even; what is larger than 448 becomes 448, what is no number stays none.
__device__ __forceinline__ uint16_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes to fp16, exact.
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Four codes to two pairs of fp16.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t"
      ".reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ int lds8(uint32_t a) {
  int v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

}  // namespace apb
