// 8- and 4-bit K/V rows of a paged pool: quantised as they are written, widened as they are read.
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
// Both kernels move bytes and are bound by them: 16384 rows of 4 heads of 128 (bfloat16, int8;
// 51 MB) are written in 12 us, 4.2 TB/s, and read in 10, 5.0; 33768 of 8 heads (e4m3 to float16,
// 210 MB) are read in 31, 6.7 TB/s (a copy of 64 MiB that the last-level cache holds runs at 6.9, of
// 256 MiB at 5.35); one row is written in 2.4 us and read in 1.5.  A head vector is held by the smallest
// power of two of lanes that covers it at 8 elements a lane (16 at D = 128), so that a
// 16-bit row is one 16-byte load and one 8-byte store a lane, and the largest magnitude
// is a butterfly within those lanes.
//
// A 4-bit pool holds codes [blocks, 2, P, Hkv, D / 2], two to a byte, and scale bytes
// [blocks, 2, P, Hkv, D / 32]: a power of two for every 32 neighbours, so that a quotient is exact, a
// code is one conversion instruction's half and a value is widened with its scale by another's.  A
// vector of 128 costs 68 bytes.  Lanes hold eight neighbours as above, four lanes a scale.  16384 rows
// of 4 heads of 128 (bfloat16, 43 MB) are written in 9.6 us, 4.4 TB/s, and read in 9.4; one row is
// written in 1.8 us and read in 1.6.
#include <math.h>

#include "quantize.h"

namespace hs {

constexpr int QZ_T = 256;

struct QuantArgs {
  const void *k, *v;  // [tokens, Hkv, D], element strides per token and head
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t* rows;  // [tokens] physical rows
  unsigned char* codes;
  void* scales;
  int64_t tokens, pool_rows, P, Hkv;
  int D, lanes_log2;  // lanes per head vector: 1 << lanes_log2
};

struct ReadArgs {
  const unsigned char* codes;
  const void* scales;
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

// A lane's elements of a head vector, and the largest magnitude of them as float bits (their
// order is that of the magnitudes: NaN > infinity > every finite value).  16-bit elements are
// compared as they are, two at a time.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {  // of two pairs, or of two float32
  if constexpr (DT == HS_DTYPE_F32) return a > b ? a : b;
  else
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

template <int DT, bool VEC>
struct Elements {
  static constexpr int WORDS = VEC && DT != HS_DTYPE_F32 ? QZ_E / 2 : QZ_E;
  uint32_t w[WORDS];  // as stored (VEC), else floats

  __device__ __forceinline__ void load(const void* base, int64_t at, int lane, int lanes, int D) {
    if constexpr (VEC) {
      const bool in = lane * QZ_E < D;
      const char* p = static_cast<const char*>(base) + (at + (in ? lane * QZ_E : 0)) * (DT == HS_DTYPE_F32 ? 4 : 2);
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i + e] = in ? v[e] : 0u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < QZ_E; ++e) {
        const int d = lane + lanes * e;
        w[e] = __float_as_uint(d < D ? load_elem<DT>(base, at + d) : 0.f);
      }
    }
  }
  __device__ __forceinline__ uint32_t largest(int lanes) const {  // over the head vector's lanes
    constexpr int T = WORDS == QZ_E ? HS_DTYPE_F32 : DT;
    constexpr uint32_t MAGNITUDE = T == HS_DTYPE_F32 ? 0x7fffffffu : 0x7fff7fffu;
    uint32_t top = w[0] & MAGNITUDE;
#pragma unroll
    for (int i = 1; i < WORDS; ++i) top = larger<T>(top, w[i] & MAGNITUDE);
    top = group_reduce(top, lanes, [](uint32_t a, uint32_t b) { return larger<T>(a, b); });
    if constexpr (T == HS_DTYPE_F32) return top;
    const uint32_t lo = top & 0xffffu, hi = top >> 16, one = lo > hi ? lo : hi;
    return T == HS_DTYPE_BF16 ? one << 16 : __float_as_uint(f16_bits_to_f32(static_cast<unsigned short>(one)));
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (WORDS == QZ_E) return __uint_as_float(w[e]);
    else if constexpr (DT == HS_DTYPE_BF16) return e & 1 ? __uint_as_float(w[e >> 1] & 0xffff0000u) : __uint_as_float(w[e >> 1] << 16);
    else return f16_bits_to_f32(static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1))));
  }
};

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
// the row and the index arithmetic, and their loads go out with the row's, together.  (A grid
// of the workgroups that run at once, striding with the next pair's loads in flight, took
// 16.8 us for a 16k-token prompt at the 7B shape, this 14.0.)
template <int DT, int CODE, bool VEC>
__global__ __launch_bounds__(QZ_T) void append_quantized_kernel(QuantArgs a) {
  const int lanes = 1 << a.lanes_log2;
  const uint32_t vec = (blockIdx.x * static_cast<uint32_t>(QZ_T) + threadIdx.x) >> a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t Hkv = static_cast<uint32_t>(a.Hkv), token = vec / Hkv, head = vec - token * Hkv;
  if (token >= a.tokens) return;  // whole groups leave: the butterfly stays within a group
  const int64_t row = a.rows[token];
  Elements<DT, VEC> x[2];
  x[0].load(a.k, token * a.k_st + head * a.k_sh, lane, lanes, a.D);
  x[1].load(a.v, token * a.v_st + head * a.v_sh, lane, lanes, a.D);
  const uint32_t top[2] = {x[0].largest(lanes), x[1].largest(lanes)};
  if (row < 0 || row >= a.pool_rows) return;
  const int64_t at = vector_at(row, head, a.pool_rows, a.P, a.Hkv);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const bool finite = top[p] < 0x7f800000u;
    const float scale = finite ? scale_of<CODE>(__uint_as_float(top[p])) : __uint_as_float(0x7fc00000u);
    u32x2 w = {0u, 0u};
    if (finite && scale > 0.f) w = encode8<CODE>(x[p], scale);
    const int64_t to = at + (p ? a.P * a.Hkv : 0);
    if (lane == 0) static_cast<float*>(a.scales)[to] = scale;
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
    scale[p] = static_cast<const float*>(a.scales)[from];
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

// The 4-bit forms.  VEC: 16-byte loads and stores of K and V and 4-byte ones of codes, else single
// elements and bytes; either way a lane holds eight neighbours.
template <int DT, bool VEC>
__global__ __launch_bounds__(QZ_T) void append_fp4_kernel(QuantArgs a) {
  const int lanes = 1 << a.lanes_log2;
  const uint32_t vec = (blockIdx.x * static_cast<uint32_t>(QZ_T) + threadIdx.x) >> a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t Hkv = static_cast<uint32_t>(a.Hkv), token = vec / Hkv, head = vec - token * Hkv;
  if (token >= a.tokens || lane * QZ_E >= a.D) return;  // whole groups of four lanes leave
  const int64_t row = a.rows[token];
  Elements<DT, VEC> x[2];
  const int64_t from[2] = {token * a.k_st + head * a.k_sh, token * a.v_st + head * a.v_sh};
  if constexpr (VEC) {
    x[0].load(a.k, from[0], lane, lanes, a.D);
    x[1].load(a.v, from[1], lane, lanes, a.D);
  } else {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < QZ_E; ++e)
        x[p].w[e] = __float_as_uint(load_elem<DT>(p ? a.v : a.k, from[p] + lane * QZ_E + e));
  }
  const uint32_t top[2] = {x[0].largest(4), x[1].largest(4)};
  if (row < 0 || row >= a.pool_rows) return;
  const int64_t at = vector_at(row, head, a.pool_rows, a.P, a.Hkv);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint32_t byte = fp4_scale_byte(top[p]), w = encode_fp4(x[p], byte);
    const int64_t to = at + (p ? a.P * a.Hkv : 0);
    if ((lane & 3) == 0) static_cast<unsigned char*>(a.scales)[to * (a.D / FP4_GROUP) + (lane >> 2)] = static_cast<unsigned char>(byte);
    unsigned char* codes = a.codes + to * (a.D / 2) + lane * (QZ_E / 2);
    if constexpr (VEC) {
      *reinterpret_cast<uint32_t*>(codes) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) codes[e] = static_cast<unsigned char>(w >> (8 * e));
    }
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(QZ_T) void read_fp4_kernel(ReadArgs a) {
  const int lanes = 1 << a.lanes_log2;
  const uint32_t vec = (blockIdx.x * static_cast<uint32_t>(QZ_T) + threadIdx.x) >> a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t Hkv = static_cast<uint32_t>(a.Hkv), i = vec / Hkv, head = vec - i * Hkv;
  if (i >= a.n || lane * QZ_E >= a.D) return;
  const int64_t row = a.rows[i];
  const bool there = row >= 0 && row < a.pool_rows;  // else the row reads as zeros
  const int64_t at = there ? vector_at(row, head, a.pool_rows, a.P, a.Hkv) : 0;
  const int64_t to = (static_cast<int64_t>(i) * a.Hkv + head) * a.D + lane * QZ_E;
  uint32_t w[2], byte[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t from = at + (p ? a.P * a.Hkv : 0);
    byte[p] = static_cast<const unsigned char*>(a.scales)[from * (a.D / FP4_GROUP) + (lane >> 2)];
    const unsigned char* codes = a.codes + from * (a.D / 2) + lane * (QZ_E / 2);
    if constexpr (VEC) {
      w[p] = *reinterpret_cast<const uint32_t*>(codes);
    } else {
      w[p] = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[p] |= static_cast<uint32_t>(codes[e]) << (8 * e);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    void* dst = p ? a.v : a.k;
    const uint32_t codes = there ? w[p] : 0u;
    const float scale = __uint_as_float(there ? byte[p] << 23 : 0u);
    if constexpr (VEC && DT == HS_DTYPE_BF16) {
      u32x4 o;
      widen_fp4_bf16x8(codes, scale, o);
      *reinterpret_cast<u32x4*>(static_cast<unsigned short*>(dst) + to) = o;
    } else {
      float v[QZ_E];
#pragma unroll
      for (int e = 0; e < QZ_E; e += 2) {
        const f32x2 pair = widen_fp4(codes >> (4 * e), scale);
        v[e] = pair[0];
        v[e + 1] = pair[1];
      }
      if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < QZ_E; ++e) store_elem<DT>(dst, to + e, v[e]);
      } else if constexpr (DT == HS_DTYPE_F32) {
        float* out = static_cast<float*>(dst) + to;
        *reinterpret_cast<f32x4*>(out) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(out + 4) = f32x4{v[4], v[5], v[6], v[7]};
      } else {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack16<true>(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<u32x4*>(static_cast<unsigned short*>(dst) + to) = o;
      }
    }
  }
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
  HS_CHECK_ARG(valid_code(code) || code == HS_DTYPE_E2M1, "invalid cache code %d", code);
  HS_CHECK_ARG(code != HS_DTYPE_E2M1 || head_dim % FP4_GROUP == 0, "4-bit rows need a head_dim of a multiple of 32");
  HS_CHECK_ARG(rows_n >= 0 && kv_heads >= 1 && head_dim >= 1 && head_dim <= 512 && page_size >= 1 && pool_rows >= 1,
               "quantised rows need positive sizes and a head_dim of at most 512");
  // a page's V rows lie past its K rows, and the kernels divide rows by a page size of at most the rows
  HS_CHECK_ARG(pool_rows % page_size == 0, "pool_rows must be those of whole pages");
  // head vectors, at up to 64 lanes each, are counted in 32 bits
  HS_CHECK_ARG(kv_heads <= (int64_t{1} << 20) && rows_n <= (int64_t{1} << 25) / kv_heads,
               "too many quantised head vectors in one call");
  HS_CHECK_ARG(codes && scales, "null quantised pool pointer");
  HS_CHECK_ARG(code == HS_DTYPE_E2M1 || (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "scales must be 4-byte aligned");
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

#define HS_FP4_LAUNCH(kernel, DT, vec, grid, stream, args)                                                      \
  do {                                                                                                          \
    if (vec) hipLaunchKernelGGL((kernel<DT, true>), grid, dim3(QZ_T), 0, stream, args);                         \
    else hipLaunchKernelGGL((kernel<DT, false>), grid, dim3(QZ_T), 0, stream, args);                            \
  } while (0)
#define HS_FP4_DISPATCH(kernel, dtype, vec, grid, stream, args)                                                 \
  do {                                                                                                          \
    if ((dtype) == HS_DTYPE_BF16) HS_FP4_LAUNCH(kernel, HS_DTYPE_BF16, vec, grid, stream, args);                \
    else if ((dtype) == HS_DTYPE_F16) HS_FP4_LAUNCH(kernel, HS_DTYPE_F16, vec, grid, stream, args);             \
    else HS_FP4_LAUNCH(kernel, HS_DTYPE_F32, vec, grid, stream, args);                                          \
  } while (0)

extern "C" int hs_append_quantized(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v,
                                   int64_t v_stride_t, int64_t v_stride_h, int32_t dtype, const int64_t* rows,
                                   int64_t tokens, void* codes, void* scales, int32_t code, int64_t pool_rows,
                                   int64_t page_size, int64_t kv_heads, int64_t head_dim, hipStream_t stream) {
  const int rc = check_quantized(tokens, kv_heads, head_dim, page_size, pool_rows, dtype, code, codes, scales);
  if (rc) return rc;
  if (tokens == 0) return HS_OK;
  HS_CHECK_ARG(k && v && rows, "null K/V or row pointer");
  HS_CHECK_ARG(k_stride_t >= 0 && k_stride_h >= 0 && v_stride_t >= 0 && v_stride_h >= 0, "negative K/V stride");
  const int64_t unit = 16 / elem_bytes(dtype);  // a vector load: 16 bytes
  const bool fp4 = code == HS_DTYPE_E2M1;
  const bool vec = head_dim % QZ_E == 0 && aligned(k, 16) && aligned(v, 16) && aligned(codes, fp4 ? QZ_E / 2 : QZ_E) &&
                   k_stride_t % unit == 0 && k_stride_h % unit == 0 && v_stride_t % unit == 0 &&
                   v_stride_h % unit == 0;
  QuantArgs a{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, rows, static_cast<unsigned char*>(codes), scales,
              tokens, pool_rows, page_size, kv_heads, static_cast<int>(head_dim), vector_lanes_log2(vec || fp4, head_dim)};
  const int64_t per = QZ_T >> a.lanes_log2;
  const int64_t blocks = (tokens * kv_heads + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (fp4) HS_FP4_DISPATCH(append_fp4_kernel, dtype, vec, grid, stream, a);
  else HS_QUANT_DISPATCH(append_quantized_kernel, dtype, code, vec, grid, stream, a);
  HS_CHECK_LAUNCH("append_quantized");
  return HS_OK;
}

extern "C" int hs_read_quantized(const void* codes, const void* scales, int32_t code, int64_t pool_rows,
                                 int64_t page_size, int64_t kv_heads, int64_t head_dim, const int64_t* rows, int64_t n,
                                 void* k, void* v, int32_t dtype, hipStream_t stream) {
  const int rc = check_quantized(n, kv_heads, head_dim, page_size, pool_rows, dtype, code, codes, scales);
  if (rc) return rc;
  if (n == 0) return HS_OK;
  HS_CHECK_ARG(k && v && rows, "null K/V or row pointer");
  const bool fp4 = code == HS_DTYPE_E2M1;
  const bool vec = head_dim % QZ_E == 0 && aligned(k, 16) && aligned(v, 16) && aligned(codes, fp4 ? QZ_E / 2 : QZ_E);
  ReadArgs a{static_cast<const unsigned char*>(codes), scales, rows, k, v, n, pool_rows, page_size, kv_heads,
             static_cast<int>(head_dim), vector_lanes_log2(vec || fp4, head_dim)};
  const int64_t per = QZ_T >> a.lanes_log2;
  const int64_t blocks = (n * kv_heads + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (fp4) HS_FP4_DISPATCH(read_fp4_kernel, dtype, vec, grid, stream, a);
  else HS_QUANT_DISPATCH(read_quantized_kernel, dtype, code, vec, grid, stream, a);
  HS_CHECK_LAUNCH("read_quantized");
  return HS_OK;
}
