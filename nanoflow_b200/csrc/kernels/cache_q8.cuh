// The 8-bit cache's numbers: conversions between them and the types that the kernels compute with.
//
// A cached vector is head_dim numbers of 8 bits (e4m3 or whole numbers) and one fp32 scale; value = number * scale. Both kinds
// are exact in f16 (e4m3 has four significant bits and exponents from -9 to 8, whole numbers go to 127), so the tensor cores take
// them as they are and the scales join in fp32.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace nf {

// What the largest entry of a vector becomes.
template <int KIND>
__device__ __forceinline__ constexpr float q8_largest() { return KIND == NFK_Q8_E4M3 ? 448.f : 127.f; }

// Vectors whose largest entry is below this are stored as zeros: 1 / scale and products of scales stay finite.
constexpr float kQ8Smallest = 8.271806e-25f;   // 2^-80

// Four numbers of a word as two f16 pairs: (bytes 0, 1) and (bytes 2, 3).
template <int KIND>
__device__ __forceinline__ void q8_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (KIND == NFK_Q8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // 0x6400 + u is 1024 + u in f16 for u < 1024: with u = b + 128, take off 1152
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Four values, already divided by their scale, as four numbers; round to nearest, ties to even, and nothing beyond the largest.
template <int KIND>
__device__ __forceinline__ uint32_t q8_from_f32(float a, float b, float c, float d) {
  if (KIND == NFK_Q8_E4M3) {
    uint32_t w;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
  }
  // 1.5 * 2^23 + x has round(x) in its low bits
  const float k = 12582912.f;
  const auto n = [&](float x) { return __float_as_uint(fminf(fmaxf(x, -127.f), 127.f) + k); };
  return __byte_perm(__byte_perm(n(a), n(b), 0x0040), __byte_perm(n(c), n(d), 0x0040), 0x5410);
}

// Two fp32 operations by one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(f32x2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest magnitude; NaN where there is one.
__device__ __forceinline__ float max3_magnitude(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

// Power of two of a row's largest magnitude `most`, for queries as f16: row * q_down lies within (-2, 2), and q_up takes that
// back. Rows of zeros, infinities or NaN keep a finite factor.
__device__ __forceinline__ void q_powers(float most, float& q_down, float& q_up) {
  const uint32_t e = min(max(__float_as_uint(most) >> 23 & 255u, 1u), 253u);
  q_down = __uint_as_float((254u - e) << 23);
  q_up = __uint_as_float(e << 23);
}

}  // namespace nf
