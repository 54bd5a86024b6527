// Dense-layer helpers of the layer-major decode engine for gfx950.
//
// A decode step of B tokens runs, per layer, RMSNorm -> q/k/v projections ->
// rotary embedding -> sparse attention -> o_proj -> residual -> RMSNorm ->
// SiLU MLP -> residual (the reference's MiniModel.decode, model.py:183-226,
// with its Qwen2 layer math).  With B rows of a few thousand elements every
// elementwise PyTorch op is one launch of negligible work, and a layer issues
// ~30 of them.  These kernels fuse them around the projections (which stay
// PyTorch-ROCm GEMMs, with q/k/v and gate/up packed into one weight each):
//
//   add_rms_norm   x <- x + delta (in the model dtype), y = RMSNorm(x)
//   rotary_split   fused q|k|v projection output -> rotated q, rotated k, v
//   silu_mul       fused gate|up projection output -> silu(gate) * up
//   norm_rotary_split  rotary_split with a per-head RMSNorm of q and k before the rotation
//
// Rounding follows the PyTorch ops they replace: the residual add rounds to
// the model dtype; RMSNorm squares and averages in fp32, rounds x * rsqrt to
// the model dtype and multiplies by the weight in that dtype; rotary rounds
// cos/sin, each product and the sum to the model dtype; SiLU rounds its fp32
// result before the product with `up`; norm_rotary_split has no chain of ops to follow
// and rounds its fp32 result once.  Only the fp32 sum order of the norm
// and the device's transcendental functions differ from PyTorch's.
#include <math.h>

#include "hs_common.h"

namespace hs {

constexpr int DN_T = 256;

// One workgroup per row.  `delta` may be null (no residual add); `x_out` may
// alias `x`.  A row of at most NR_REG * DN_T elements is held in registers: every
// load of x, delta and the weight is issued before the first is used, so the row
// costs one memory round trip (a store to x_out may alias the next load of x, so a
// loop that stores as it goes would wait out a round trip per element).  Longer
// rows go in rounds of NR_CH elements per thread, loads of a round issued together.
constexpr int NR_REG = 24;
constexpr int NR_CH = 8;

__device__ __forceinline__ float block_sum_dn(float v, float* partial) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < DN_T / 64; ++w) total += partial[w];
  return total;
}

template <int DT>
__global__ __launch_bounds__(DN_T) void add_rms_norm_kernel(const void* x, const void* delta, void* x_out, void* y,
                                                            const void* weight, int64_t width, int64_t x_stride,
                                                            int64_t y_stride, float eps) {
  __shared__ float partial[DN_T / 64];
  const int64_t row = blockIdx.x;
  const int64_t xo = row * x_stride, yo = row * y_stride;
  const bool add = delta != nullptr;
  const void* dsrc = add ? delta : x;  // always a valid row: no load sits under a branch
  if (width <= static_cast<int64_t>(NR_REG) * DN_T) {
    float v[NR_REG], dl[NR_REG], wv[NR_REG];
#pragma unroll
    for (int k = 0; k < NR_REG; ++k) {
      // unconditional loads of in-bounds elements (a load under a branch would be
      // waited for before the next), masked afterwards
      const int64_t i = threadIdx.x + static_cast<int64_t>(k) * DN_T;
      const bool in = i < width;
      const int64_t ic = in ? i : 0;
      const float xv = load_elem<DT>(x, xo + ic), wvv = load_elem<DT>(weight, ic);
      const float dv = load_elem<DT>(dsrc, xo + ic);
      v[k] = in ? xv : 0.f;
      dl[k] = in ? dv : 0.f;
      wv[k] = in ? wvv : 0.f;
    }
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < NR_REG; ++k) {
      const int64_t i = threadIdx.x + static_cast<int64_t>(k) * DN_T;
      if (i >= width) break;
      if (add) {
        v[k] = round_to<DT>(v[k] + dl[k]);
        store_elem<DT>(x_out, xo + i, v[k]);
      }
      sq += v[k] * v[k];
    }
    const float r = rsqrtf(block_sum_dn(sq, partial) / static_cast<float>(width) + eps);
#pragma unroll
    for (int k = 0; k < NR_REG; ++k) {
      const int64_t i = threadIdx.x + static_cast<int64_t>(k) * DN_T;
      if (i >= width) break;
      store_elem<DT>(y, yo + i, round_to<DT>(mul_rn(v[k], r)) * wv[k]);
    }
    return;
  }
  float sq = 0.f;
  for (int64_t base = threadIdx.x; base < width; base += static_cast<int64_t>(DN_T) * NR_CH) {
    float a[NR_CH], b[NR_CH];
#pragma unroll
    for (int k = 0; k < NR_CH; ++k) {
      const int64_t i = base + static_cast<int64_t>(k) * DN_T;
      const int64_t ic = i < width ? i : 0;
      const float xv = load_elem<DT>(x, xo + ic);
      const float dv = load_elem<DT>(dsrc, xo + ic);
      a[k] = i < width ? xv : 0.f;
      b[k] = i < width ? dv : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NR_CH; ++k) {
      const int64_t i = base + static_cast<int64_t>(k) * DN_T;
      if (i >= width) break;
      float s = a[k];
      if (add) {
        s = round_to<DT>(s + b[k]);
        store_elem<DT>(x_out, xo + i, s);
      }
      sq += s * s;
    }
  }
  const float r = rsqrtf(block_sum_dn(sq, partial) / static_cast<float>(width) + eps);
  const void* src = add ? x_out : x;
  for (int64_t base = threadIdx.x; base < width; base += static_cast<int64_t>(DN_T) * NR_CH) {
    float a[NR_CH], b[NR_CH];
#pragma unroll
    for (int k = 0; k < NR_CH; ++k) {
      const int64_t i = base + static_cast<int64_t>(k) * DN_T;
      const int64_t ic = i < width ? i : 0;
      const float sv = load_elem<DT>(src, xo + ic), wvv = load_elem<DT>(weight, ic);
      a[k] = i < width ? sv : 0.f;
      b[k] = i < width ? wvv : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NR_CH; ++k) {
      const int64_t i = base + static_cast<int64_t>(k) * DN_T;
      if (i >= width) break;
      store_elem<DT>(y, yo + i, round_to<DT>(mul_rn(a[k], r)) * b[k]);
    }
  }
}

// Grid (heads + 2 * kv_heads, rows); one thread per rotation pair (d, d + D/2).
// Heads [0, heads) are q, [heads, heads + kv_heads) k (both rotated at the
// row's position), the rest v (copied).
template <int DT>
__global__ __launch_bounds__(DN_T) void rotary_split_kernel(const void* qkv, int64_t qkv_stride, void* q, void* k,
                                                            void* v, const int64_t* positions, int64_t heads,
                                                            int64_t kv_heads, int64_t D, float theta) {
  const int64_t h = blockIdx.x, row = blockIdx.y;
  const int64_t half = D / 2;
  const int64_t src = row * qkv_stride + h * D;
  void* dst;
  int64_t doff;
  if (h < heads) {
    dst = q;
    doff = (row * heads + h) * D;
  } else if (h < heads + kv_heads) {
    dst = k;
    doff = (row * kv_heads + (h - heads)) * D;
  } else {
    dst = v;
    doff = (row * kv_heads + (h - heads - kv_heads)) * D;
  }
  if (h >= heads + kv_heads) {
    for (int64_t d = threadIdx.x; d < D; d += blockDim.x) store_elem<DT>(dst, doff + d, load_elem<DT>(qkv, src + d));
    return;
  }
  const float pos = static_cast<float>(positions[row]);
  for (int64_t i = threadIdx.x; i < half; i += blockDim.x) {
    float lo, hi;
    rotary_pair<DT>(load_elem<DT>(qkv, src + i), load_elem<DT>(qkv, src + i + half), pos, i, D, theta, lo, hi);
    store_elem<DT>(dst, doff + i, lo);
    store_elem<DT>(dst, doff + i + half, hi);
  }
}

// Per-head RMS norm of q and k, then the rotary embedding, with the split of a packed
// q|k|v row: for a q or k head vector x with norm weight w,
//
//   n_d = x_d rsqrt(mean(x^2) + eps) w_d,
//   (y_i, y_{i+D/2}) = (n_i cos a - n_{i+D/2} sin a, n_{i+D/2} cos a + n_i sin a),
//   a = position * theta^(-2i/D),
//
// in fp32, rounded once.  The angle is reduced to a part of one turn in 64 bits: at
// position 10^5 an fp32 angle is off by up to 4e-3, more than a bf16 step of the result.
// A head vector is held by `lanes` lanes of NE pairs each, so both halves of a pair meet in
// one lane and the norm's sum is a butterfly within the lanes.  A workgroup takes `brows` rows:
// its threads first fill the rows' cos/sin table in LDS (one 64-bit reduction per row and pair,
// shared by all heads), then walk the rows' heads, the next head's loads in flight.
// Bound by its bytes: 16384 rows of 28 query and 2 x 4 KV heads of 128 in bf16 move 302 MB in
// 58 us, 5.2 TB/s, where a copy of 256 MiB runs at 5.35.  A decode batch is bound by its chain of
// loads, table and stores: 16 rows of these heads take 3.9 us, one row of 14 and 2 x 2 heads of
// 64 takes 2.8.
constexpr int NH_TAB = 512;  // cos/sin pairs of a workgroup's table

struct NormRotaryArgs {
  const void *qkv, *wq, *wk;
  void *q, *k, *v;
  const int64_t* positions;
  int64_t qkv_stride, rows, heads, kv_heads;
  double log2_theta;
  float eps;
  int D, lanes_log2, brows;
};

// Elements of half a head vector that a lane holds, as loaded: NE neighbours (VEC), or one of
// every `lanes` (then as floats).
template <int DT, int NE, bool VEC>
struct HalfVector {
  static constexpr int WORDS = VEC && DT != HS_DTYPE_F32 ? NE / 2 : NE;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const void* base, int64_t at, int lane, int lanes, int half) {
    if constexpr (VEC) {
      const char* p = static_cast<const char*>(base) + (at + (lane * NE < half ? lane * NE : 0)) * (DT == HS_DTYPE_F32 ? 4 : 2);
      if constexpr (WORDS == 4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v[i];
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(p);
        w[0] = v[0];
        w[1] = v[1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = lane + lanes * e;
        w[e] = __float_as_uint(i < half ? load_elem<DT>(base, at + i) : 0.f);
      }
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t at, int lane, int lanes, int half) const {
    if constexpr (VEC) {
      if (lane * NE >= half) return;
      char* p = static_cast<char*>(base) + (at + lane * NE) * (DT == HS_DTYPE_F32 ? 4 : 2);
      if constexpr (WORDS == 4) *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
      else *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = lane + lanes * e;
        if (i < half) store_elem<DT>(base, at + i, __uint_as_float(w[e]));
      }
    }
  }
  __device__ __forceinline__ void floats(float (&x)[NE], bool in) const {  // zeros past the vector's end
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      if constexpr (WORDS == NE) {
        x[e] = __uint_as_float(w[e]);
      } else {
        const unsigned short b = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
        x[e] = DT == HS_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
      }
      if constexpr (VEC) x[e] = in ? x[e] : 0.f;
    }
  }
  __device__ __forceinline__ void round_from(const float (&x)[NE]) {
#pragma unroll
    for (int e = 0; e < WORDS; ++e) {
      if constexpr (WORDS == NE) w[e] = __float_as_uint(x[e]);
      else w[e] = pack16<DT == HS_DTYPE_F16>(x[2 * e], x[2 * e + 1]);
    }
  }
};

template <int DT, int NE, bool VEC>
__global__ __launch_bounds__(DN_T) void norm_rotary_split_kernel(NormRotaryArgs a) {
  using Half = HalfVector<DT, NE, VEC>;
  __shared__ __attribute__((aligned(16))) float s_cos[NH_TAB], s_sin[NH_TAB];
  const int half = a.D / 2, lanes = 1 << a.lanes_log2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.brows;
  const int nrows = static_cast<int>(a.rows - row0 < a.brows ? a.rows - row0 : a.brows);
  const int H = static_cast<int>(a.heads), K = static_cast<int>(a.kv_heads), total = H + 2 * K;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> a.lanes_log2, groups = DN_T >> a.lanes_log2;
  const bool in = !VEC || lane * NE < half;
  // this group's heads: h = first, first + step, ... of every row in turn; the next head's loads
  // go out before the current one is worked on
  const int step = static_cast<int>(gridDim.y) * groups;
  int r = 0, h = static_cast<int>(blockIdx.y) * groups + group;
  auto settle = [&]() {
    while (h >= total && r < nrows) {
      h -= total;
      ++r;
    }
  };
  Half lo, hi, wq[2], wk[2];
  auto fetch = [&](Half& x, Half& y) {
    const int64_t src = (row0 + r) * a.qkv_stride + static_cast<int64_t>(h) * a.D;
    x.load(a.qkv, src, lane, lanes, half);
    y.load(a.qkv, src + half, lane, lanes, half);
  };
  settle();
  if (r < nrows) fetch(lo, hi);
  for (int i = 0; i < 2; ++i) {
    wq[i].load(a.wq, i * half, lane, lanes, half);
    wk[i].load(a.wk, i * half, lane, lanes, half);
  }
  for (int t = threadIdx.x; t < nrows * half; t += DN_T) {
    const int tr = t / half, i = t - tr * half;
    // turns = position * theta^(-2i/D) / 2 pi
    const double turns = static_cast<double>(a.positions[row0 + tr]) *
                         (exp2(-(2.0 * i / a.D) * a.log2_theta) * 0.15915494309189535);
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    s_cos[t] = c;
    s_sin[t] = s;
  }
  __syncthreads();
  while (r < nrows) {
    const int cr = r, ch = h;
    Half cur[2] = {lo, hi};
    h += step;
    settle();
    if (r < nrows) fetch(lo, hi);
    const int64_t row = row0 + cr;
    void* dst = ch < H ? a.q : (ch < H + K ? a.k : a.v);
    const int64_t to = (ch < H ? row * H + ch : (ch < H + K ? row * K + ch - H : row * K + ch - H - K)) * a.D;
    if (ch < H + K) {  // one condition for all lanes of the head
      float x[NE], y[NE], u[NE], v[NE], sq = 0.f;
      cur[0].floats(x, in);
      cur[1].floats(y, in);
#pragma unroll
      for (int e = 0; e < NE; ++e) sq += x[e] * x[e] + y[e] * y[e];
      sq = group_reduce(sq, lanes, [](float p, float q) { return p + q; });
      const float norm = rsqrtf(sq / static_cast<float>(a.D) + a.eps);
      (ch < H ? wq[0] : wk[0]).floats(u, in);
      (ch < H ? wq[1] : wk[1]).floats(v, in);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = VEC ? lane * NE + e : lane + lanes * e;
        const int at = i < half ? cr * half + i : 0;
        const float p = x[e] * norm * u[e], q = y[e] * norm * v[e], c = s_cos[at], s = s_sin[at];
        x[e] = p * c - q * s;
        y[e] = q * c + p * s;
      }
      cur[0].round_from(x);
      cur[1].round_from(y);
    }
    cur[0].store(dst, to, lane, lanes, half);
    cur[1].store(dst, to + half, lane, lanes, half);
  }
}

// out[row, j] = silu(gate[row, j]) * up[row, j] with gate = gate_up[row, :width],
// up = gate_up[row, width:].
template <int DT>
__global__ __launch_bounds__(DN_T) void silu_mul_kernel(const void* gate_up, int64_t gu_stride, void* out,
                                                        int64_t out_stride, int64_t width) {
  const int64_t row = blockIdx.y;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * DN_T + threadIdx.x;
  if (j >= width) return;
  const float g = load_elem<DT>(gate_up, row * gu_stride + j);
  const float u = load_elem<DT>(gate_up, row * gu_stride + width + j);
  const float act = round_to<DT>(g / (1.f + expf(-g)));
  store_elem<DT>(out, row * out_stride + j, act * u);
}

}  // namespace hs

using namespace hs;

#define HS_DENSE_DISPATCH(dtype, kernel, grid, block, stream, ...)                                              \
  do {                                                                                                          \
    if ((dtype) == HS_DTYPE_BF16) hipLaunchKernelGGL((kernel<HS_DTYPE_BF16>), grid, block, 0, stream, __VA_ARGS__); \
    else if ((dtype) == HS_DTYPE_F16) hipLaunchKernelGGL((kernel<HS_DTYPE_F16>), grid, block, 0, stream, __VA_ARGS__); \
    else hipLaunchKernelGGL((kernel<HS_DTYPE_F32>), grid, block, 0, stream, __VA_ARGS__);                     \
  } while (0)

extern "C" int hs_add_rms_norm(const void* x, const void* delta, void* x_out, void* y, const void* weight,
                               int64_t rows, int64_t width, int64_t x_stride, int64_t y_stride, float eps,
                               int32_t dtype, hipStream_t stream) {
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(rows >= 1 && rows <= 65535 && width >= 1, "invalid norm shape");
  HS_CHECK_ARG(x_stride >= width && y_stride >= width, "row strides below the width");
  HS_CHECK_ARG(x && y && weight && (delta == nullptr || x_out != nullptr), "null norm pointer");
  HS_DENSE_DISPATCH(dtype, add_rms_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(DN_T), stream, x, delta,
                    x_out, y, weight, width, x_stride, y_stride, eps);
  HS_CHECK_LAUNCH("add_rms_norm");
  return HS_OK;
}

extern "C" int hs_rotary_split(const void* qkv, int64_t qkv_stride, void* q, void* k, void* v,
                               const int64_t* positions, int64_t rows, int64_t heads, int64_t kv_heads,
                               int64_t head_dim, float theta, int32_t dtype, hipStream_t stream) {
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(rows >= 1 && rows <= 65535 && heads >= 1 && kv_heads >= 1 && head_dim >= 2 && head_dim % 2 == 0,
               "invalid rotary shape");
  HS_CHECK_ARG(qkv_stride >= (heads + 2 * kv_heads) * head_dim, "q|k|v row stride below its width");
  HS_CHECK_ARG(qkv && q && k && v && positions, "null rotary pointer");
  const unsigned threads = head_dim / 2 >= DN_T ? DN_T : static_cast<unsigned>(((head_dim / 2 + 63) / 64) * 64);
  HS_DENSE_DISPATCH(dtype, rotary_split_kernel, dim3(static_cast<unsigned>(heads + 2 * kv_heads), static_cast<unsigned>(rows)),
                    dim3(threads), stream, qkv, qkv_stride, q, k, v, positions, heads, kv_heads, head_dim, theta);
  HS_CHECK_LAUNCH("rotary_split");
  return HS_OK;
}

extern "C" int hs_norm_rotary_split(const void* qkv, int64_t qkv_stride, const void* q_weight, const void* k_weight,
                                    float eps, void* q, void* k, void* v, const int64_t* positions, int64_t rows,
                                    int64_t heads, int64_t kv_heads, int64_t head_dim, double theta, int32_t dtype,
                                    hipStream_t stream) {
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(rows >= 1 && heads >= 1 && kv_heads >= 1 && head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 512,
               "invalid normed rotary shape");
  HS_CHECK_ARG(rows <= 0x7fffffff && heads <= 0xffff && kv_heads <= 0xffff, "too many rows or heads in one call");
  HS_CHECK_ARG(qkv_stride >= (heads + 2 * kv_heads) * head_dim, "q|k|v row stride below its width");
  HS_CHECK_ARG(qkv && q_weight && k_weight && q && k && v && positions, "null normed rotary pointer");
  HS_CHECK_ARG(theta > 0.0 && isfinite(theta) && eps >= 0.f, "theta must be positive and eps not negative");
  const int half = static_cast<int>(head_dim / 2);
  const uintptr_t all = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_weight) |
                        reinterpret_cast<uintptr_t>(k_weight) | reinterpret_cast<uintptr_t>(q) |
                        reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  // pairs of a lane: a load of 16 bytes where the head dim and the addresses allow it, else of 8
  // (16-bit types), else element by element over a whole wave
  int ne = 0;
  for (const int n : {16 / elem_bytes(dtype), 4})
    if (ne == 0 && half % n == 0 && qkv_stride % n == 0 && all % (n * elem_bytes(dtype)) == 0) ne = n;
  NormRotaryArgs a{qkv, q_weight, k_weight, q, k, v, positions, qkv_stride, rows, heads, kv_heads, log2(theta), eps,
                   static_cast<int>(head_dim), 6, 1};
  if (ne) {
    a.lanes_log2 = 0;
    while ((ne << a.lanes_log2) < half) ++a.lanes_log2;
  }
  const int64_t groups = DN_T >> a.lanes_log2, total = heads + 2 * kv_heads;
  // Rows per workgroup: as many as give every thread one cos/sin pair, once that still
  // leaves two workgroups per CU; fewer rows go one to a workgroup, their heads spread.
  const int64_t fill = DN_T / half > 1 ? DN_T / half : 1;
  a.brows = rows >= 512 * fill ? static_cast<int>(fill) : 1;
  int64_t spread = 1;
  if (rows < 512) {
    spread = (total + groups - 1) / groups;
    const int64_t most = (512 + rows - 1) / rows;
    if (spread > most) spread = most;
  }
  HS_CHECK_ARG((rows + a.brows - 1) / a.brows < (int64_t{1} << 32) / DN_T, "too many rows in one call");
  const dim3 grid(static_cast<unsigned>((rows + a.brows - 1) / a.brows), static_cast<unsigned>(spread));
#define HS_NORM_ROTARY(DT, NE, VEC) \
  hipLaunchKernelGGL((norm_rotary_split_kernel<DT, NE, VEC>), grid, dim3(DN_T), 0, stream, a)
  if (dtype == HS_DTYPE_F32) {
    if (ne) HS_NORM_ROTARY(HS_DTYPE_F32, 4, true);
    else HS_NORM_ROTARY(HS_DTYPE_F32, 4, false);
  } else if (dtype == HS_DTYPE_BF16) {
    if (ne == 8) HS_NORM_ROTARY(HS_DTYPE_BF16, 8, true);
    else if (ne) HS_NORM_ROTARY(HS_DTYPE_BF16, 4, true);
    else HS_NORM_ROTARY(HS_DTYPE_BF16, 4, false);
  } else {
    if (ne == 8) HS_NORM_ROTARY(HS_DTYPE_F16, 8, true);
    else if (ne) HS_NORM_ROTARY(HS_DTYPE_F16, 4, true);
    else HS_NORM_ROTARY(HS_DTYPE_F16, 4, false);
  }
#undef HS_NORM_ROTARY
  HS_CHECK_LAUNCH("norm_rotary_split");
  return HS_OK;
}

extern "C" int hs_silu_mul(const void* gate_up, int64_t gu_stride, void* out, int64_t out_stride, int64_t rows,
                           int64_t width, int32_t dtype, hipStream_t stream) {
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(rows >= 1 && rows <= 65535 && width >= 1, "invalid silu_mul shape");
  HS_CHECK_ARG(gu_stride >= 2 * width && out_stride >= width, "row strides below the width");
  HS_CHECK_ARG(gate_up && out, "null silu_mul pointer");
  const int64_t blocks = (width + DN_T - 1) / DN_T;
  HS_CHECK_ARG(blocks <= 0x7fffffff, "silu_mul width too large");
  HS_DENSE_DISPATCH(dtype, silu_mul_kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(rows)),
                    dim3(DN_T), stream, gate_up, gu_stride, out, out_stride, width);
  HS_CHECK_LAUNCH("silu_mul");
  return HS_OK;
}
