// Per-head RMS norm and rotary embedding of a packed q|k|v projection, with its split
// (norm_rotary_split) or with K and V written to a paged pool on the way (norm_rotary_append):
// the kernel and its launch shape.
#pragma once

#include <math.h>

#include "quantize.h"

namespace hs {

constexpr int DN_T = 256;

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
  const void *qkv, *wq, *wk;  // into a pool: no weights, no norm
  void *q, *k, *v;
  const int64_t* positions;
  int64_t qkv_stride, rows, heads, kv_heads;
  double log2_theta;
  float eps;
  int D, lanes_log2, brows;
  // into a pool: K and V of a row go to physical row to_rows[row]
  const int64_t* to_rows;
  void *pool, *scales;
  int64_t pool_rows, P;
};

constexpr int NO_POOL = -1;  // K and V to k and v; else the pool's element code

// Elements of half a head vector that a lane holds: NE neighbours as loaded (VEC), or as floats
// loaded one by one, neighbours too (NEAR) or one of every `lanes`.
template <int DT, int NE, bool VEC, bool NEAR = VEC>
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
        const int i = NEAR ? lane * NE + e : lane + lanes * e;
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
        const int i = NEAR ? lane * NE + e : lane + lanes * e;
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
      if constexpr (NEAR) x[e] = in ? x[e] : 0.f;
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

// A lane's elements of the two halves as one run of eight, or of one half as eight.
template <int NE>
struct Run {
  const float *x, *y;
  __device__ __forceinline__ float get(int e) const { return e < NE ? x[e] : y[e - NE]; }
};

// Largest magnitudes (float bits) of the 32 neighbours that this lane's elements x of the first half and
// y of the second belong to, in a head vector of a multiple of 32.  Where the halves are whole
// groups of 32, a group is 32 / NE lanes of one half.  Else both halves are an odd number h of runs
// of 16, and the pair of run w (of the whole vector) is w ^ 1: the first half's last run pairs with
// the second half's first.
template <int NE>
__device__ __forceinline__ void group_tops(const float (&x)[NE], const float (&y)[NE], int lane, int lanes, int half,
                                           uint32_t& tx, uint32_t& ty) {
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  tx = ty = 0u;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    tx = larger(tx, __float_as_uint(x[e]) & 0x7fffffffu);
    ty = larger(ty, __float_as_uint(y[e]) & 0x7fffffffu);
  }
  if (half % FP4_GROUP == 0) {
    tx = group_reduce(tx, FP4_GROUP / NE, larger);
    ty = group_reduce(ty, FP4_GROUP / NE, larger);
    return;
  }
  constexpr int RUN = 16 / NE;  // lanes
  tx = group_reduce(tx, RUN, larger);
  ty = group_reduce(ty, RUN, larger);
  const int h = half / 16, u = lane / RUN, first = static_cast<int>(threadIdx.x & 63) - lane;
  auto run_of = [&](uint32_t t, int run) {  // (a run past the vector: any lane of this one, unused)
    return static_cast<uint32_t>(__shfl(static_cast<int>(t), first + ((run * RUN) & (lanes - 1)), 64));
  };
  const uint32_t x_pair = run_of(tx, u ^ 1), y_first = run_of(ty, 0), x_last = run_of(tx, h - 1);
  const uint32_t y_pair = run_of(ty, ((h + u) ^ 1) - h);
  tx = larger(tx, u == h - 1 ? y_first : x_pair);
  ty = larger(ty, u == 0 ? x_last : y_pair);
}

template <int BYTES>
__device__ __forceinline__ void store_code_bytes(unsigned char* p, uint32_t lo, uint32_t hi, bool wide) {
  if (!wide) {
#pragma unroll
    for (int e = 0; e < BYTES; ++e) p[e] = static_cast<unsigned char>((e < 4 ? lo : hi) >> (8 * (e & 3)));
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<u32x2*>(p) = u32x2{lo, hi};
  } else if constexpr (BYTES == 4) {
    *reinterpret_cast<uint32_t*>(p) = lo;
  } else {
    *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(lo);
  }
}

// One head vector (halves x and y, zeros past its end) into a quantised pool, as vector `to` of it.
// `wide`: the codes' address allows one store a run of NE (NEAR).
template <int POOL, int NE, bool NEAR>
__device__ __forceinline__ void store_quantised(const NormRotaryArgs& a, int64_t to, const float (&x)[NE], const float (&y)[NE],
                                                int lane, int lanes, int half, bool wide) {
  unsigned char* codes = static_cast<unsigned char*>(a.pool);
  if constexpr (POOL == HS_DTYPE_E2M1) {
    uint32_t top[2];
    group_tops<NE>(x, y, lane, lanes, half, top[0], top[1]);
    if (lane * NE >= half) return;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int d = (p ? half : 0) + lane * NE;
      const float* v = p ? y : x;
      const uint32_t byte = fp4_scale_byte(top[p]);
      if (d % FP4_GROUP == 0)
        static_cast<unsigned char*>(a.scales)[to * (a.D / FP4_GROUP) + d / FP4_GROUP] = static_cast<unsigned char>(byte);
      uint32_t w = 0u;
      if (byte != 255u) {
        const float scale = __uint_as_float(byte << 23);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        if constexpr (NE == 8) {
          w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
          w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        }
      }
      store_code_bytes<NE / 2>(codes + to * (a.D / 2) + d / 2, w, 0u, wide);
    }
  } else {
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const uint32_t mx = __float_as_uint(x[e]) & 0x7fffffffu, my = __float_as_uint(y[e]) & 0x7fffffffu;
      top = top > mx ? top : mx;
      top = top > my ? top : my;
    }
    top = group_reduce(top, lanes, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
    const bool finite = top < 0x7f800000u;
    const float scale = finite ? scale_of<POOL>(__uint_as_float(top)) : __uint_as_float(0x7fc00000u);
    const bool some = finite && scale > 0.f;
    if (lane == 0) static_cast<float*>(a.scales)[to] = scale;
    unsigned char* at = codes + to * a.D;
    if constexpr (NE == 8) {
      u32x2 lo = {0u, 0u}, hi = {0u, 0u};
      if (some) {
        lo = encode8<POOL>(Run<8>{x, x}, scale);
        hi = encode8<POOL>(Run<8>{y, y}, scale);
      }
      if (lane * NE >= half) return;
      store_code_bytes<8>(at + lane * NE, lo[0], lo[1], wide);
      store_code_bytes<8>(at + half + lane * NE, hi[0], hi[1], wide);
    } else {
      u32x2 w = {0u, 0u};
      if (some) w = encode8<POOL>(Run<NE>{x, y}, scale);
      if constexpr (NEAR) {
        if (lane * NE >= half) return;
        store_code_bytes<4>(at + lane * NE, w[0], 0u, wide);
        store_code_bytes<4>(at + half + lane * NE, w[1], 0u, wide);
      } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int i = lane + lanes * e;
          if (i >= half) continue;
          at[i] = static_cast<unsigned char>(w[0] >> (8 * e));
          at[half + i] = static_cast<unsigned char>(w[1] >> (8 * e));
        }
      }
    }
  }
}

// POOL: where K and V go (NO_POOL, or the element code of the pool that they are written to, as
// quantized.hip's append writes them, from the fp32 values).
template <int DT, int NE, bool VEC, int POOL = NO_POOL>
__global__ __launch_bounds__(DN_T) void norm_rotary_split_kernel(NormRotaryArgs a) {
  constexpr bool NEAR = VEC || POOL == HS_DTYPE_E2M1;  // two codes share a byte
  using Half = HalfVector<DT, NE, VEC, NEAR>;
  __shared__ __attribute__((aligned(16))) float s_cos[NH_TAB], s_sin[NH_TAB];
  __shared__ int64_t s_row[POOL == NO_POOL ? 1 : DN_T];
  const int half = a.D / 2, lanes = 1 << a.lanes_log2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.brows;
  const int nrows = static_cast<int>(a.rows - row0 < a.brows ? a.rows - row0 : a.brows);
  const int H = static_cast<int>(a.heads), K = static_cast<int>(a.kv_heads), total = H + 2 * K;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> a.lanes_log2, groups = DN_T >> a.lanes_log2;
  const bool in = !NEAR || lane * NE < half;
  const bool normed = POOL == NO_POOL || a.wq != nullptr;
  // this group's heads: h = first, first + step, ... of every row in turn; the next head's loads
  // go out before the current one is worked on
  // (into a pool: all rows' query heads, then their K and their V, so that a wave seldom holds vectors of
  // two kinds, whose work differs: 16383 rows of 28 and 4 heads of 128 into int8, and read back, 71.1 us
  // head after head, 69.0 so.  `past` heads come before this kind's, of `kind` a row.)
  const int step = static_cast<int>(gridDim.y) * groups;
  int r = 0, h = static_cast<int>(blockIdx.y) * groups + group;
  int past = 0, kind = POOL == NO_POOL ? total : H;
  auto settle = [&]() {
    if constexpr (POOL == NO_POOL) {
      while (h >= total && r < nrows) {
        h -= total;
        ++r;
      }
    } else {
      while (h >= kind && r < nrows) {
        h -= kind;
        if (++r == nrows && past < H + K) {
          r = 0;
          past += kind;
          kind = K;
        }
      }
    }
  };
  Half lo, hi, wq[2], wk[2];
  auto fetch = [&](Half& x, Half& y) {
    const int64_t src = (row0 + r) * a.qkv_stride + static_cast<int64_t>(past + h) * a.D;
    x.load(a.qkv, src, lane, lanes, half);
    y.load(a.qkv, src + half, lane, lanes, half);
  };
  settle();
  if (r < nrows) fetch(lo, hi);
  for (int i = 0; i < 2 && normed; ++i) {
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
  if constexpr (POOL != NO_POOL) {
    if (static_cast<int>(threadIdx.x) < nrows) s_row[threadIdx.x] = a.to_rows[row0 + threadIdx.x];
  }
  __syncthreads();
  // the normed (or not) and rotated halves of a q or k head vector (norm_rotary_split states the same
  // below: the compiler fuses other multiply-adds there, and its bits are to stay)
  auto turn = [&](const Half (&cur)[2], int cr, bool query, float (&x)[NE], float (&y)[NE]) {
    float u[NE], v[NE], sq = 0.f;
    cur[0].floats(x, in);
    cur[1].floats(y, in);
    if (normed) {
#pragma unroll
      for (int e = 0; e < NE; ++e) sq += x[e] * x[e] + y[e] * y[e];
      sq = group_reduce(sq, lanes, [](float p, float q) { return p + q; });
      const float norm = rsqrtf(sq / static_cast<float>(a.D) + a.eps);
      (query ? wq[0] : wk[0]).floats(u, in);
      (query ? wq[1] : wk[1]).floats(v, in);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        x[e] = x[e] * norm * u[e];
        y[e] = y[e] * norm * v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int i = NEAR ? lane * NE + e : lane + lanes * e;
      const int at = i < half ? cr * half + i : 0;
      const float p = x[e], q = y[e], c = s_cos[at], s = s_sin[at];
      x[e] = p * c - q * s;
      y[e] = q * c + p * s;
    }
  };
  while (r < nrows) {
    const int cr = r, ch = past + h;
    Half cur[2] = {lo, hi};
    h += step;
    settle();
    if (r < nrows) fetch(lo, hi);
    const int64_t row = row0 + cr;
    if constexpr (POOL == NO_POOL) {
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
    } else if (ch < H) {
      const int64_t to = (row * H + ch) * a.D;
      float x[NE], y[NE];
      turn(cur, cr, true, x, y);
      cur[0].round_from(x);
      cur[1].round_from(y);
      cur[0].store(a.q, to, lane, lanes, half);
      cur[1].store(a.q, to + half, lane, lanes, half);
    } else {
      const int64_t pool_row = s_row[cr];
      if (pool_row < 0 || pool_row >= a.pool_rows) continue;
      const bool key = ch < H + K;
      const int64_t to = vector_at(pool_row, key ? ch - H : ch - H - K, a.pool_rows, a.P, K) + (key ? 0 : a.P * K);
      if (POOL == DT && !key) {
        cur[0].store(a.pool, to * a.D, lane, lanes, half);
        cur[1].store(a.pool, to * a.D + half, lane, lanes, half);
        continue;
      }
      float x[NE], y[NE];
      if (key) {
        turn(cur, cr, false, x, y);
      } else {
        cur[0].floats(x, in);
        cur[1].floats(y, in);
      }
      if constexpr (POOL == DT) {
        cur[0].round_from(x);
        cur[1].round_from(y);
        cur[0].store(a.pool, to * a.D, lane, lanes, half);
        cur[1].store(a.pool, to * a.D + half, lane, lanes, half);
      } else {
        store_quantised<POOL, NE, NEAR>(a, to, x, y, lane, lanes, half, VEC);
      }
    }
  }
}

// Pairs of a lane: a load of 16 bytes where the head dim and the addresses allow it, else of 8 (16-bit
// types); 0: element by element.  `half_bytes`: half bytes of a quantised pool's element (0: no such
// pool), `codes` the address of its codes.
inline int norm_rotary_pairs(int dtype, int64_t half, int64_t stride, uintptr_t all, int half_bytes, uintptr_t codes) {
  for (const int n : {16 / elem_bytes(dtype), 4})
    if (half % n == 0 && stride % n == 0 && all % (n * elem_bytes(dtype)) == 0 &&
        (half_bytes == 0 || codes * 2 % (n * half_bytes) == 0))
      return n;
  return 0;
}

// Lanes of a head vector (for `ne` neighbours a lane, or a whole wave), rows of a workgroup and the
// grid.  Rows per workgroup: as many as give every thread one cos/sin pair, once that still leaves
// two workgroups per CU; fewer rows go one to a workgroup, their heads spread.
inline dim3 norm_rotary_grid(NormRotaryArgs& a, int ne) {
  const int half = a.D / 2;
  a.lanes_log2 = 6;
  if (ne) {
    a.lanes_log2 = 0;
    while ((ne << a.lanes_log2) < half) ++a.lanes_log2;
  }
  const int64_t groups = DN_T >> a.lanes_log2, total = a.heads + 2 * a.kv_heads;
  const int64_t fill = DN_T / half > 1 ? DN_T / half : 1;
  a.brows = a.rows >= 512 * fill ? static_cast<int>(fill) : 1;
  int64_t spread = 1;
  if (a.rows < 512) {
    spread = (total + groups - 1) / groups;
    const int64_t most = (512 + a.rows - 1) / a.rows;
    if (spread > most) spread = most;
  }
  return dim3(static_cast<unsigned>((a.rows + a.brows - 1) / a.brows), static_cast<unsigned>(spread));
}

}  // namespace hs
