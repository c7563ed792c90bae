// Device functions of the 4-bit format (its definition and the reasons for it stand
// in fp4.cu): rounding of a block of 16, and the values of codes and scales.
#pragma once

#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace fp4 {

// x / s rounded to nearest even, r = 1/s rounded to nearest (quant.cu's div_rn_by).
__device__ __forceinline__ float div_by(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-s, q, x), r, q);
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, float2 (&v)[8], bool vec) {
  constexpr int NV = 16 * sizeof(T) / 16;
  T e[16];
  if (vec) {
    uint4 u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    memcpy(e, u, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = make_float2(to_float(e[2 * i]), to_float(e[2 * i + 1]));
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Largest magnitude as the integer of its bits: an infinity or NaN orders above
// every finite value, so none is lost.
__device__ __forceinline__ uint32_t absmax16(const float2 (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu));
  return m;
}

__device__ __forceinline__ uint32_t e2m1x8(const float* q) {
  uint32_t d;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(d)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return d;
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)byte));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

// Exponent of the row scale from the bits of a finite absmax.
__device__ __forceinline__ int row_exponent(uint32_t bits) {
  if (bits < 0x00800000u) return -100;  // 0 or subnormal: below 2^-126
  const int e = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7fffffu) > 0x280000u ? 1 : 0);  // 0.3125 * 2^23
  return max(e, -100);
}


__device__ __forceinline__ long long block_offset(long long row, int b, int nk64) {
  return ((row >> 7) * nk64 + (b >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (b & 3);
}

// One block: its scale byte and 16 codes, from its absmax and the row's exponent.
// The quotients x / (block scale) are x r + x r', r + r' the reciprocal to 2^-45, in
// packed pairs: off by 2^-44 before their rounding, and x / s (24 bits by at most four) is
// at least 2^-29 from the middle of two floats, so they are the correctly rounded ones.
// (x r alone misses the borders of two codes at s = 15 / 8; three operations with the
// remainder took 227 us where these two take 209.)  r and r' carry the row's power of two; rows so large that r'
// would be subnormal are brought down first (exactly: what underflows is far below a code).
__device__ __forceinline__ uint32_t round_block(float2 (&x)[8], uint32_t top, int e, uint2& code) {
  // e4m3 of absmax / (6 scale): the division by 6 is the only rounding before it
  const float raw = div_by(__uint_as_float(top) * pow2f(-e), 6.0f, 1.0f / 6.0f);
  const uint32_t s8 = cvt_e4m3x2_f32(0.0f, raw) & 0xffu;
  if (s8 != 0) {
    if (e > 60) {  // of 117 at most
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmul2(x[i], both(pow2f(-64)));
      e -= 64;
    }
    const float s = e4m3_value(s8), r = rcp_approx(s);
    const float2 r2 = both(r * pow2f(-e)), t2 = both(fmaf(-s, r, 1.0f) * r * pow2f(-e));
    float q[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 c = ffma2(x[i], r2, fmul2(x[i], t2));
      q[2 * i] = c.x;
      q[2 * i + 1] = c.y;
    }
    code = make_uint2(e2m1x8(q), e2m1x8(q + 8));
  }
  return s8;
}

// A block as loaded, in pairs.
template <typename T>
__device__ __forceinline__ void pairs16(const uint4 (&u)[sizeof(T)], float2 (&v)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (std::is_same<T, __half>::value) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
}

// absmax16 of a block as loaded: 16-bit types compare two magnitudes at a time as
// integers, and only the larger one is widened.
template <typename T>
__device__ __forceinline__ uint32_t absmax_raw(const uint4 (&u)[sizeof(T)]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    uint32_t m = __vimax3_u16x2(w[0] & kAbs, w[1] & kAbs, w[2] & kAbs);
    m = __vimax3_u16x2(m, w[3] & kAbs, w[4] & kAbs);
    m = __vimax3_u16x2(m, w[5] & kAbs, w[6] & kAbs);
    m = __vimax3_u16x2(m, w[7] & kAbs, 0u);
    m = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<T, __half>::value)
      return m >= 0x7c00u ? 0x7f800000u | m : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    return m << 16;
  }
}

// Two e2m1 codes of a byte as two f16 (exact).
__device__ __forceinline__ void e2m1x8_halves(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

}  // namespace fp4
}  // namespace mh3
