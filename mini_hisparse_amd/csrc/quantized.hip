// 8-bit K/V rows of a paged pool: quantised as they are written, widened as they are read.
//
// A quantised pool is two tensors, codes [blocks, 2, P, Hkv, D] (int8 or e4m3) and scales
// [blocks, 2, P, Hkv] float32: the layout of a plain pool with one scale per (row, plane,
// head).  For a head vector x of largest magnitude a,
//
//   scale = f32(a / top),  top = 127 (int8) or 448 (e4m3),
//   code  = the code nearest to the exact quotient x / scale, ties to even,
//
// and it reads back as code * scale.  A vector of zeros has scale 0 and codes 0; one with
// a NaN or an infinity has scale NaN and codes 0, so it reads back as NaN throughout.
// The scale is held in 32 bits, so a vector costs D + 4 bytes (132 for 256 of a 16-bit
// vector at D = 128).
//
// Both kernels move bytes and are bound by them.  A head vector is held by the smallest
// power of two of lanes that covers it at 8 elements a lane (16 at D = 128), so that a
// 16-bit row is one 16-byte load and one 8-byte store a lane, and the largest magnitude
// is a butterfly within those lanes.
#include <math.h>

#include "codes.h"

namespace hs {

constexpr int QZ_T = 256;
constexpr int QZ_E = 8;  // elements of a head vector per lane

struct QuantArgs {
  const void *k, *v;  // [tokens, Hkv, D], element strides per token and head
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t* rows;  // [tokens] physical rows
  unsigned char* codes;
  float* scales;
  int64_t tokens, pool_rows, P, Hkv;
  int D, lanes_log2;  // lanes per head vector: 1 << lanes_log2
};

struct ReadArgs {
  const unsigned char* codes;
  const float* scales;
  const int64_t* rows;  // [n]
  void *k, *v;          // [n, Hkv, D] contiguous
  int64_t n, pool_rows, P, Hkv;
  int D, lanes_log2;
};

// Element index of the lane's e-th element: VEC, the lane's 8 neighbours; else strided.
template <bool VEC>
__device__ __forceinline__ int elem_index(int lane, int lanes, int e) {
  return VEC ? lane * QZ_E + e : lane + lanes * e;
}

template <int DT, bool VEC>
__device__ __forceinline__ void load_vector(const void* base, int64_t at, int lane, int lanes, int D,
                                            float (&x)[QZ_E]) {
  if constexpr (VEC) {
    const bool in = lane * QZ_E < D;
    const int64_t i = at + (in ? lane * QZ_E : 0);
    if constexpr (DT == HS_DTYPE_F32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i);
      const f32x4 b = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = in ? a[e] : 0.f;
        x[4 + e] = in ? b[e] : 0.f;
      }
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const unsigned short*>(base) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t p = in ? w[e] : 0u;
        const unsigned short lo = static_cast<unsigned short>(p), hi = static_cast<unsigned short>(p >> 16);
        x[2 * e] = DT == HS_DTYPE_BF16 ? bf16_bits_to_f32(lo) : f16_bits_to_f32(lo);
        x[2 * e + 1] = DT == HS_DTYPE_BF16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) {
      const int d = lane + lanes * e;
      x[e] = d < D ? load_elem<DT>(base, at + d) : 0.f;
    }
  }
}

// Magnitude of the e4m3 code nearest to a (0 <= a <= 448), ties to even, as a float.
__device__ __forceinline__ float e4m3_nearest(double a) {
  const int ex = a > 0.0 ? __builtin_amdgcn_frexp_exp(a) : -99;  // a = m 2^ex, m in [0.5, 1)
  const int step = (ex - 1 < -6 ? -6 : ex - 1) - 3;              // log2 of the grid's spacing at a
  return static_cast<float>(ldexp(rint(ldexp(a, -step)), step));
}

// Code of one element by the exact quotient (64 bits hold it well enough: a quotient of
// two 24-bit values that is no border of the grid is at least 2^-34 of itself away from one).
template <int CODE>
__device__ __forceinline__ float code_exact(float x, float scale) {
  double q = static_cast<double>(x) / static_cast<double>(scale);
  q = fmin(fmax(q, -static_cast<double>(code_top<CODE>())), static_cast<double>(code_top<CODE>()));
  if constexpr (CODE == HS_DTYPE_I8) return static_cast<float>(rint(q));
  else return copysignf(e4m3_nearest(fabs(q)), x);
}

// The quotient x * (1 / scale) in 32 bits is within 2^-22 of itself; the code it rounds to
// is the right one unless it lies that close to a border between two codes.
template <int CODE>
__device__ __forceinline__ bool near_border(float q) {
  if constexpr (CODE == HS_DTYPE_I8) {
    return fabsf(fabsf(q - rintf(q)) - 0.5f) < 0x1p-14f;  // |q| <= 127: off by at most 2^-15
  } else {
    const uint32_t below = __float_as_uint(q) & 0xfffffu;  // significand bits under e4m3's
    const float t = fabsf(q) * 512.f;                      // multiples of 2^-9 below 2^-6
    const bool normal = below - 0x7fff0u <= 0x20u;
    return t >= 8.f ? normal : fabsf(t - floorf(t) - 0.5f) < 0x1p-16f;
  }
}

template <int CODE>
__device__ __forceinline__ u32x2 encode8(const float (&x)[QZ_E], float scale) {
  float c[QZ_E];
  const float inverse = 1.f / scale;
  // a scale so small that its inverse overflows takes the exact way throughout
  bool exact = !(scale >= 0x1p-100f);
#pragma unroll
  for (int e = 0; e < QZ_E; ++e) {
    const float q = x[e] * inverse;
    exact = exact || near_border<CODE>(q);
    c[e] = CODE == HS_DTYPE_I8 ? rintf(q) : q;
  }
  if (exact) {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) c[e] = code_exact<CODE>(x[e], scale);
  }
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (CODE == HS_DTYPE_I8) {
      w[h] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[h] |= (static_cast<uint32_t>(static_cast<int32_t>(c[4 * h + e])) & 0xffu) << (8 * e);
    } else {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h], c[4 * h + 1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h + 2], c[4 * h + 3], p, true);
      w[h] = static_cast<uint32_t>(p);
    }
  }
  return w;
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

template <bool VEC>
__device__ __forceinline__ void store_codes(unsigned char* codes, int64_t at, int lane, int lanes, int D, u32x2 w) {
  if constexpr (VEC) {
    if (lane * QZ_E < D) *reinterpret_cast<u32x2*>(codes + at * D + lane * QZ_E) = w;
  } else {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) {
      const int d = lane + lanes * e;
      if (d < D) codes[at * D + d] = static_cast<unsigned char>(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// The K and the V vector of one (token, head) per group of 1 << lanes_log2 lanes: they share
// the row and the index arithmetic, and their loads go out with the row's, together.
template <int DT, int CODE, bool VEC>
__global__ __launch_bounds__(QZ_T) void append_quantized_kernel(QuantArgs a) {
  const int lanes = 1 << a.lanes_log2;
  const uint32_t vec = (blockIdx.x * static_cast<uint32_t>(QZ_T) + threadIdx.x) >> a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t Hkv = static_cast<uint32_t>(a.Hkv), token = vec / Hkv, head = vec - token * Hkv;
  if (token >= a.tokens) return;  // whole groups leave: the butterfly stays within a group
  const int64_t row = a.rows[token];
  float x[2][QZ_E];
  load_vector<DT, VEC>(a.k, token * a.k_st + head * a.k_sh, lane, lanes, a.D, x[0]);
  load_vector<DT, VEC>(a.v, token * a.v_st + head * a.v_sh, lane, lanes, a.D, x[1]);
  // the largest magnitude as bits: NaN > infinity > every finite value
  uint32_t top[2] = {0u, 0u};
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) {
      const uint32_t bits = __float_as_uint(x[p][e]) & 0x7fffffffu;
      top[p] = bits > top[p] ? bits : top[p];
    }
  }
  for (int off = lanes >> 1; off > 0; off >>= 1) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint32_t other = __shfl_xor(top[p], off, 64);
      top[p] = other > top[p] ? other : top[p];
    }
  }
  if (row < 0 || row >= a.pool_rows) return;
  const int64_t at = vector_at(row, head, a.pool_rows, a.P, a.Hkv);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const bool finite = top[p] < 0x7f800000u;
    const float scale = finite ? __uint_as_float(top[p]) / code_top<CODE>() : __uint_as_float(0x7fc00000u);
    u32x2 w = {0u, 0u};
    if (finite && scale > 0.f) w = encode8<CODE>(x[p], scale);
    const int64_t to = at + (p ? a.P * a.Hkv : 0);
    if (lane == 0) a.scales[to] = scale;
    store_codes<VEC>(a.codes, to, lane, lanes, a.D, w);
  }
}

template <int DT, int CODE, bool VEC>
__device__ __forceinline__ void widen_vector(void* dst, int64_t to, u32x2 w, float scale, int lane, int lanes, int D) {
  float x[2][4];
  decode4<CODE>(w[0], x[0]);
  decode4<CODE>(w[1], x[1]);
  if constexpr (!VEC) {
#pragma unroll
    for (int e = 0; e < QZ_E; ++e) {
      const int d = lane + lanes * e;
      if (d < D) store_elem<DT>(dst, to + d, mul_rn(x[e >> 2][e & 3], scale));
    }
  } else if constexpr (DT == HS_DTYPE_F32) {
    float* p = static_cast<float*>(dst) + to + lane * QZ_E;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<f32x4*>(p + 4 * h) = f32x4{x[h][0] * scale, x[h][1] * scale, x[h][2] * scale, x[h][3] * scale};
  } else {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = pack16<DT == HS_DTYPE_F16>(mul_rn(x[e >> 1][2 * (e & 1)], scale), mul_rn(x[e >> 1][2 * (e & 1) + 1], scale));
    *reinterpret_cast<u32x4*>(static_cast<unsigned short*>(dst) + to + lane * QZ_E) = o;
  }
}

template <int DT, int CODE, bool VEC>
__global__ __launch_bounds__(QZ_T) void read_quantized_kernel(ReadArgs a) {
  const int lanes = 1 << a.lanes_log2;
  const uint32_t vec = (blockIdx.x * static_cast<uint32_t>(QZ_T) + threadIdx.x) >> a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t Hkv = static_cast<uint32_t>(a.Hkv), i = vec / Hkv, head = vec - i * Hkv;
  if (i >= a.n || (VEC && lane * QZ_E >= a.D)) return;
  const int64_t row = a.rows[i];
  const bool there = row >= 0 && row < a.pool_rows;  // else the row reads as zeros
  const int64_t at = there ? vector_at(row, head, a.pool_rows, a.P, a.Hkv) : 0;
  const int64_t to = (static_cast<int64_t>(i) * a.Hkv + head) * a.D;
  u32x2 w[2];
  float scale[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t from = at + (p ? a.P * a.Hkv : 0);
    scale[p] = a.scales[from];
    if constexpr (VEC) {
      w[p] = *reinterpret_cast<const u32x2*>(a.codes + from * a.D + lane * QZ_E);
    } else {
      w[p] = u32x2{0u, 0u};
#pragma unroll
      for (int e = 0; e < QZ_E; ++e) {
        const int d = lane + lanes * e;
        if (d < a.D) w[p][e >> 2] |= static_cast<uint32_t>(a.codes[from * a.D + d]) << (8 * (e & 3));
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
    widen_vector<DT, CODE, VEC>(p ? a.v : a.k, to, there ? w[p] : u32x2{0u, 0u}, there ? scale[p] : 0.f, lane, lanes,
                                a.D);
}

// log2 of the lanes of a head vector: 8 elements a lane, or a whole wave when strided.
static int vector_lanes_log2(bool vec, int64_t D) {
  if (!vec) return 6;
  int l = 0;
  while ((int64_t{QZ_E} << l) < D) ++l;
  return l;
}

static int check_quantized(int64_t rows_n, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t pool_rows,
                           int32_t dtype, int32_t code, const void* codes, const void* scales) {
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(valid_code(code), "invalid cache code %d", code);
  HS_CHECK_ARG(rows_n >= 0 && kv_heads >= 1 && head_dim >= 1 && head_dim <= 512 && page_size >= 1 && pool_rows >= 1,
               "quantised rows need positive sizes and a head_dim of at most 512");
  // head vectors, at up to 64 lanes each, are counted in 32 bits
  HS_CHECK_ARG(kv_heads <= (int64_t{1} << 20) && rows_n <= (int64_t{1} << 25) / kv_heads,
               "too many quantised head vectors in one call");
  HS_CHECK_ARG(codes && scales, "null quantised pool pointer");
  HS_CHECK_ARG((reinterpret_cast<uintptr_t>(scales) & 3) == 0, "scales must be 4-byte aligned");
  return HS_OK;
}

static bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace hs

using namespace hs;

#define HS_QUANT_LAUNCH(kernel, DT, CODE, vec, grid, stream, args)                                              \
  do {                                                                                                          \
    if (vec) hipLaunchKernelGGL((kernel<DT, CODE, true>), grid, dim3(QZ_T), 0, stream, args);                   \
    else hipLaunchKernelGGL((kernel<DT, CODE, false>), grid, dim3(QZ_T), 0, stream, args);                      \
  } while (0)
#define HS_QUANT_CODE(kernel, DT, code, vec, grid, stream, args)                                                \
  do {                                                                                                          \
    if ((code) == HS_DTYPE_I8) HS_QUANT_LAUNCH(kernel, DT, HS_DTYPE_I8, vec, grid, stream, args);               \
    else HS_QUANT_LAUNCH(kernel, DT, HS_DTYPE_E4M3, vec, grid, stream, args);                                   \
  } while (0)
#define HS_QUANT_DISPATCH(kernel, dtype, code, vec, grid, stream, args)                                         \
  do {                                                                                                          \
    if ((dtype) == HS_DTYPE_BF16) HS_QUANT_CODE(kernel, HS_DTYPE_BF16, code, vec, grid, stream, args);          \
    else if ((dtype) == HS_DTYPE_F16) HS_QUANT_CODE(kernel, HS_DTYPE_F16, code, vec, grid, stream, args);       \
    else HS_QUANT_CODE(kernel, HS_DTYPE_F32, code, vec, grid, stream, args);                                    \
  } while (0)

extern "C" int hs_append_quantized(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v,
                                   int64_t v_stride_t, int64_t v_stride_h, int32_t dtype, const int64_t* rows,
                                   int64_t tokens, void* codes, float* scales, int32_t code, int64_t pool_rows,
                                   int64_t page_size, int64_t kv_heads, int64_t head_dim, hipStream_t stream) {
  const int rc = check_quantized(tokens, kv_heads, head_dim, page_size, pool_rows, dtype, code, codes, scales);
  if (rc) return rc;
  if (tokens == 0) return HS_OK;
  HS_CHECK_ARG(k && v && rows, "null K/V or row pointer");
  HS_CHECK_ARG(k_stride_t >= 0 && k_stride_h >= 0 && v_stride_t >= 0 && v_stride_h >= 0, "negative K/V stride");
  const int64_t unit = 16 / elem_bytes(dtype);  // a vector load: 16 bytes
  const bool vec = head_dim % QZ_E == 0 && aligned(k, 16) && aligned(v, 16) && aligned(codes, QZ_E) &&
                   k_stride_t % unit == 0 && k_stride_h % unit == 0 && v_stride_t % unit == 0 &&
                   v_stride_h % unit == 0;
  QuantArgs a{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, rows, static_cast<unsigned char*>(codes), scales,
              tokens, pool_rows, page_size, kv_heads, static_cast<int>(head_dim), vector_lanes_log2(vec, head_dim)};
  const int64_t per = QZ_T >> a.lanes_log2;
  const int64_t blocks = (tokens * kv_heads + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(blocks));
  HS_QUANT_DISPATCH(append_quantized_kernel, dtype, code, vec, grid, stream, a);
  HS_CHECK_LAUNCH("append_quantized");
  return HS_OK;
}

extern "C" int hs_read_quantized(const void* codes, const float* scales, int32_t code, int64_t pool_rows,
                                 int64_t page_size, int64_t kv_heads, int64_t head_dim, const int64_t* rows, int64_t n,
                                 void* k, void* v, int32_t dtype, hipStream_t stream) {
  const int rc = check_quantized(n, kv_heads, head_dim, page_size, pool_rows, dtype, code, codes, scales);
  if (rc) return rc;
  if (n == 0) return HS_OK;
  HS_CHECK_ARG(k && v && rows, "null K/V or row pointer");
  const bool vec = head_dim % QZ_E == 0 && aligned(k, 16) && aligned(v, 16) && aligned(codes, QZ_E);
  ReadArgs a{static_cast<const unsigned char*>(codes), scales, rows, k, v, n, pool_rows, page_size, kv_heads,
             static_cast<int>(head_dim), vector_lanes_log2(vec, head_dim)};
  const int64_t per = QZ_T >> a.lanes_log2;
  const int64_t blocks = (n * kv_heads + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(blocks));
  HS_QUANT_DISPATCH(read_quantized_kernel, dtype, code, vec, grid, stream, a);
  HS_CHECK_LAUNCH("read_quantized");
  return HS_OK;
}
