// Codes of quantised caches and weights, shared by the kernels that write and read them: 8-bit ones,
// int8 and e4m3 (four significand bits, largest 448), and 4-bit ones, e2m1 (0, 0.5, 1, 1.5, 2, 3,
// 4, 6 and a sign) with a power of two for every 32 neighbours, held as a byte e for 2^(e - 127)
// (255: NaN).  gfx950 widens two e2m1 codes with their power of two in one instruction, which takes
// the power from the exponent of a float and reads no other bit of it.
#pragma once

#include "hs_common.h"

namespace hs {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int FP4_GROUP = 32;

inline bool valid_code(int code) { return code == HS_DTYPE_I8 || code == HS_DTYPE_E4M3; }

// The largest code: a head vector's scale is its largest magnitude over this.
template <int CODE>
constexpr __device__ __forceinline__ float code_top() {
  return CODE == HS_DTYPE_I8 ? 127.f : 448.f;
}

// The four codes of a word as floats (exact).
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, float (&v)[4]) {
  if constexpr (CODE == HS_DTYPE_I8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int32_t>(w << (24 - 8 * i)) >> 24);
  } else {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    v[0] = lo[0];
    v[1] = lo[1];
    v[2] = hi[0];
    v[3] = hi[1];
  }
}

template <int CODE>
__device__ __forceinline__ float decode1(unsigned char c) {
  if constexpr (CODE == HS_DTYPE_I8) return static_cast<float>(static_cast<signed char>(c));
  else return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c), false)[0];
}

// A scale byte as a float.
__device__ __forceinline__ float fp4_scale(uint32_t e) {
  return __uint_as_float(e == 0 ? 0x00400000u : (e == 255 ? 0x7fc00000u : e << 23));
}

// The two codes of the low byte, and of byte `byte` (a constant) as a bf16 pair, times the power of
// two in `scale`'s exponent (as byte << 23 gives it, 0 and 255 too).  Exact.
__device__ __forceinline__ f32x2 widen_fp4(uint32_t w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
}
__device__ __forceinline__ uint32_t widen_fp4_bf16(uint32_t w, float scale, int byte) {
  switch (byte) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  }
}
// The eight codes of a word as bf16 pairs.
__device__ __forceinline__ void widen_fp4_bf16x8(uint32_t w, float scale, u32x4& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = widen_fp4_bf16(w, scale, i);
}

}  // namespace hs
