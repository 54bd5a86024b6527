// 8-bit cache codes: int8 and e4m3 (four significand bits, largest 448), shared by the
// quantised cache's kernels (quantized.hip) and the attention over page tables (pages.hip).
#pragma once

#include "hs_common.h"

namespace hs {

typedef float f32x2 __attribute__((ext_vector_type(2)));

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

}  // namespace hs
