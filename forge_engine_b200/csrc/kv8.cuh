// The 8-bit cache: what its writers, its readers and its attention kernels agree on.
//
// One layer's keys are k_codes[num_pages][num_kv_heads][page_size][head_dim], e4m3 numbers (4 significant
// bits, largest 448, steps of 2^-9 below 2^-6), with k_scales[num_pages][num_kv_heads][page_size] beside
// them, e8m0 numbers (a byte b stands for 2^(b - 127)); values likewise.  A cached number is code * scale.
//
// The scale of a vector x is 2^e with the least e for which max |x| <= 448 * 2^e, so the largest element
// lands in (224, 448].  A power of two costs an e4m3 number nothing but range: every code keeps its 4
// significant bits, scaling is exact in both directions, and code * scale is an exact bfloat16.  One scale
// per token, head and matrix: a token is written once and never read again to be scaled anew, and a scale
// is one factor of a column of scores (keys) or of weights (values).  e is held to [-64, 64]: elements below
// 2^-74 become zero and what is beyond 448 * 2^64 that value.
// A vector that holds an infinity or a NaN gets scale byte 255 (the e8m0 NaN) and codes of zero: it reads
// back as NaN, a query that sees it gets NaN, and a query that does not see it is not reached, because
// masked scores are replaced and a zero weight times a zero code is zero.
#pragma once
#include <cuda_fp16.h>

#include "attention_common.cuh"

constexpr int KV8_LEAST = -64, KV8_MOST = 64;     // bounds of e
constexpr int KV8_BIAS = 127;
constexpr int KV8_NAN = 255;

// 2^(b - 127); the NaN byte gives a NaN
__device__ __forceinline__ float kv8_scale(int b) {
  return b == KV8_NAN ? __int_as_float(0x7fffffff) : __int_as_float(b << 23);
}

// e of a vector whose largest magnitude has these (finite) bits: 448 = 1.75 * 2^8
__device__ __forceinline__ int kv8_exponent(unsigned bits) {
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, KV8_LEAST), KV8_MOST);
}
// The same for a row that is not stored: every size a 32-bit number has, as far as 2^e and 2^-e are ones (rows below
// 448 * 2^-120 lose bits).
__device__ __forceinline__ int kv8_row_exponent(unsigned bits) {
  return max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -120);
}

// two codes of two 32-bit numbers, rounded to nearest even, `lo` in the low byte
__device__ __forceinline__ unsigned short kv8_codes(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// the same of two half-precision numbers
__device__ __forceinline__ unsigned kv8_codes_of_half2(__half2 v) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const unsigned*>(&v)));
  return r;
}

// two codes as two half-precision numbers (exact)
__device__ __forceinline__ unsigned kv8_half2(unsigned short codes) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}

// four codes as two pairs of half-precision numbers
__device__ __forceinline__ void kv8_halves(unsigned codes, unsigned& lo, unsigned& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
