// Head vectors to codes and scales (quantized.hip says which), from the elements that a lane holds:
// shared by the kernels that write quantised rows.
#pragma once

#include "codes.h"

namespace hs {

constexpr int QZ_E = 8;  // elements of a head vector per lane

// Adding it rounds a small float to a whole number (ties to even) and leaves that in the low bits.
constexpr float WHOLE = 12582912.f;  // 1.5 * 2^23

// Four floats of the code's range as codes, rounded to nearest; int8's come with WHOLE added.
template <int CODE>
__device__ __forceinline__ uint32_t codes4(const float (&q)[4]) {
  if constexpr (CODE == HS_DTYPE_I8) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(q[1]), __float_as_uint(q[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(q[3]), __float_as_uint(q[2]), 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  } else {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], p, true));
  }
}

// largest / top, correctly rounded: one Newton step on the product with the reciprocal (with the
// remainder exact; checked for every significand), or the division where it would underflow.
template <int CODE>
__device__ __forceinline__ float scale_of(float largest) {
  constexpr float TOP = code_top<CODE>(), RECIPROCAL = 1.f / TOP;
  if (largest < 0x1p-90f) return largest / TOP;
  const float q = largest * RECIPROCAL;
  return fmaf(fmaf(-TOP, q, largest), RECIPROCAL, q);
}

// A quotient next to a border between two codes, settled: the border t is exact in fp32, the sign
// of x - t * scale is that of one rounded multiply-add, and the result is t, or a value past
// it on x's side, which rounds as the exact quotient does.  (64-bit divisions here, in the one
// wave in 30 that comes by, took 8 of 19 us of a 16k-token prompt.)
template <int CODE>
__device__ __forceinline__ float settle(float q, float x, float scale) {
  if constexpr (CODE == HS_DTYPE_I8) {
    const float t = floorf(q) + 0.5f;
    if (!(fabsf(q - t) < 0x1p-15f)) return q;
    const float r = fmaf(-t, scale, x);
    return r > 0.f ? t + 0.25f : (r < 0.f ? t - 0.25f : t);
  } else {
    // five significand bits hold codes and borders; below 2^-6 the grid keeps the spacing of
    // [2^-6, 2^-5), to which the value is moved and moved back
    const float a = fabsf(q), up = a < 0x1p-6f ? 0x1p-6f : 0.f;
    const uint32_t b = __float_as_uint(a + up);
    if (((b + 0x80004u) & 0xfffffu) > 8u) return q;
    const float t = __uint_as_float((b + 0x40000u) & 0xfff80000u) - up;
    const float r = fmaf(-t, scale, fabsf(x));
    const float v = __uint_as_float(__float_as_uint(t) + (r > 0.f ? 1u : 0u) - (r < 0.f ? 1u : 0u));
    return copysignf(v, x);
  }
}

// A quotient in 64 bits, for scales whose inverse overflows: two 24-bit values' quotient that
// is no border of the grid is at least 2^-34 of itself away from one.  It is rounded on to
// fp32 towards zero, with the last bit set where that lost something: no border has that bit.
template <int CODE>
__device__ __forceinline__ float quotient64(float x, float scale) {
  constexpr double TOP = static_cast<double>(code_top<CODE>());
  const double q = fmin(fmax(static_cast<double>(x) / static_cast<double>(scale), -TOP), TOP);
  const float f = static_cast<float>(q);
  const double f64 = static_cast<double>(f);
  if (f64 == q) return f;
  return __uint_as_float((__float_as_uint(f) - (fabs(f64) > fabs(q) ? 1u : 0u)) | 1u);
}

// The codes of a lane's elements.  x * (1 / scale) in 32 bits (the reciprocal to one step) is within
// 1.5 * 2^-23 of the quotient, so the code it rounds to is the right one unless it lies that close
// to a border between two codes (one wave in 30 of int8's, in 200 of e4m3's, for normal values).
template <int CODE, typename X>
__device__ __forceinline__ u32x2 encode8(const X& x, float scale) {
  constexpr float ADD = CODE == HS_DTYPE_I8 ? WHOLE : 0.f;
  float q[2][4];
  if (scale >= 0x1p-100f) {
    const float inverse = __builtin_amdgcn_rcpf(scale);
    bool near;
    if constexpr (CODE == HS_DTYPE_I8) {
      float off = 0.f;
#pragma unroll
      for (int e = 0; e < QZ_E; ++e) {
        const float v = x.get(e), t = fmaf(v, inverse, WHOLE);
        q[e >> 2][e & 3] = t;
        off = fmaxf(off, fabsf(fmaf(v, inverse, WHOLE - t)));  // |quotient - code|
      }
      near = off > 0.5f - 0x1p-15f;
    } else {
      uint32_t off = 0xffffffffu;
#pragma unroll
      for (int e = 0; e < QZ_E; ++e) {
        const float v = x.get(e) * inverse, a = fabsf(v), b = a < 0x1p-6f ? a + 0x1p-6f : a;
        q[e >> 2][e & 3] = v;
        const uint32_t d = (__float_as_uint(b) + 0x80004u) & 0xfffffu;  // 4 at a border
        off = d < off ? d : off;
      }
      near = off <= 8u;
    }
    if (near) {
#pragma unroll
      for (int e = 0; e < QZ_E; ++e) q[e >> 2][e & 3] = settle<CODE>(x.get(e) * inverse, x.get(e), scale) + ADD;
    }
  } else {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) q[e >> 2][e & 3] = quotient64<CODE>(x.get(e), scale) + ADD;
  }
  return u32x2{codes4<CODE>(q[0]), codes4<CODE>(q[1])};
}

// Where a head vector of K lies in the pool (vectors; V's is P * Hkv further): 32-bit division
// unless the pool has more rows than that.
__device__ __forceinline__ int64_t vector_at(int64_t row, int64_t head, int64_t pool_rows, int64_t P, int64_t Hkv) {
  if (pool_rows <= 0xffffffffll) {
    const uint32_t r = static_cast<uint32_t>(row), p = static_cast<uint32_t>(P), block = r / p;
    return (static_cast<int64_t>(block) * 2 * P + (r - block * p)) * Hkv + head;
  }
  const int64_t block = row / P;
  return (block * 2 * P + (row - block * P)) * Hkv + head;
}

// The scale byte of 32 neighbours of largest magnitude `top` (float bits): the smallest power of two,
// from 2^-126 on, of at least a seventh of it (7 = 1.75 * 2^2; what lies between 6 and 7 rounds to 6,
// no further off than 5 is), or NaN's.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int byte = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return byte < 1 ? 1u : static_cast<uint32_t>(byte);
}

// The word of eight elements' 4-bit codes.  The quotient by a power of two is exact, and the
// instruction rounds it to nearest, ties to even, at most 6 (checked on both sides of every border,
// for subnormal elements too).
template <typename X>
__device__ __forceinline__ uint32_t encode_fp4(const X& x, uint32_t byte) {
  if (byte == 255u) return 0u;
  const float scale = __uint_as_float(byte << 23);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x.get(0), x.get(1), scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.get(2), x.get(3), scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.get(4), x.get(5), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.get(6), x.get(7), scale, 3);
}

}  // namespace hs
