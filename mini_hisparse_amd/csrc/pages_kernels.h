// The kernels of the attention over page tables, for every kind of pool: the vector-unit kernel,
// the matrix-core kernel, and their launches.  pages.hip holds the schedule of large batches, the
// join of the parts, the plans and the entry points, and describes the operator.
#pragma once

#include <math.h>

#include <type_traits>

#include "arrive.h"
#include "codes.h"
#include "page_parts.h"

namespace hs {

// Slots of a request's partials: [first, first + count).
struct SlotRange {
  int32_t first, count;
};
// A workgroup's share: part `part` of the `parts` of request b, which has n tokens.
struct alignas(16) Slot {
  int32_t b, part, parts, n;
};

struct PagesArgs {
  const void* q;
  int64_t q_sb, q_sh;
  int q_dtype;
  const void* pool;
  const float* scales;               // 8-bit pools only
  const unsigned char* scale_bytes;  // 4-bit pools only
  int64_t P, Hkv, D, blocks;
  const int32_t* tables;
  int64_t t_sb, t_sk, pages;
  const int32_t* lengths;
  int32_t window, sinks;  // the newest and the first tokens that count (page_parts.h); NO_WINDOW: all
  int64_t B, Hq, g;
  int head_chunks;
  int64_t splits, chunk;
  float scale;
  float *part_m, *part_l, *part_o;  // [slots, Hq], [slots, Hq], [slots, Hq, D]
  SlotRange* ranges;                // [B] written by the MFMA kernel; null: `splits` slots a request
  Slot* shares;                     // long, above PM_LANES requests: the schedule written out
  int units, waves_units, subs;     // MFMA kernel: (KV head, 16 heads) units; a workgroup's; waves of one
  int64_t target, min_tiles;        // long: workgroups aimed at; both: the fewest tiles of a part
  int q_vec, o_vec;  // query and output rows aligned for vector loads and stores
  // short: tagged partial words [B, max_parts, Hq] m and l, [B, max_parts, Hq, D] o, and the
  // arrival counters [B, units] (arrive.h)
  unsigned long long *word_m, *word_l, *word_o, *arrivals;
  unsigned long long epoch;
  int max_parts;
  void* out;
  int64_t o_sb, o_sh;
};

// Tokens of request b that the tables can name.
__device__ __forceinline__ int64_t request_length(const PagesArgs& a, int64_t b) {
  const int64_t n = a.lengths[b], most = a.pages * a.P;
  return n < 0 ? 0 : (n > most ? most : n);
}

__device__ __forceinline__ float load_any(const void* base, int64_t i, int dtype) {
  if (dtype == HS_DTYPE_F32) return load_elem<HS_DTYPE_F32>(base, i);
  if (dtype == HS_DTYPE_BF16) return load_elem<HS_DTYPE_BF16>(base, i);
  return load_elem<HS_DTYPE_F16>(base, i);
}
__device__ __forceinline__ void store_any(void* base, int64_t i, float v, int dtype) {
  if (dtype == HS_DTYPE_F32) store_elem<HS_DTYPE_F32>(base, i, v);
  else if (dtype == HS_DTYPE_BF16) store_elem<HS_DTYPE_BF16>(base, i, v);
  else store_elem<HS_DTYPE_F16>(base, i, v);
}

// 2^x on the transcendental unit; scores and maxima are held in powers of two.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Four neighbouring elements, rounded; `vec` when the address allows one store.
template <int DT>
__device__ __forceinline__ void store_quad(void* base, int64_t i, f32x4 v, bool vec) {
  if constexpr (DT == HS_DTYPE_F32) {
    float* p = static_cast<float*>(base) + i;
    if (vec) *reinterpret_cast<f32x4*>(p) = v;
    else
      for (int e = 0; e < 4; ++e) p[e] = v[e];
  } else {
    unsigned short* p = static_cast<unsigned short*>(base) + i;
    const u32x2 w = {pack16<DT == HS_DTYPE_F16>(v[0], v[1]), pack16<DT == HS_DTYPE_F16>(v[2], v[3])};
    if (vec) {
      *reinterpret_cast<u32x2*>(p) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

constexpr bool quantised(int S) { return S == HS_DTYPE_I8 || S == HS_DTYPE_E4M3; }  // with a float32 scale for a head vector
constexpr bool fp4(int S) { return S == HS_DTYPE_E2M1; }  // with a scale byte for every 32 of the head dim

constexpr int elem_bits(int S) { return S == HS_DTYPE_F32 ? 32 : (quantised(S) ? 8 : (fp4(S) ? 4 : 16)); }

// C neighbouring pool elements as floats.
template <int S, int C>
__device__ __forceinline__ void load_pool(const void* pool, int64_t i, float (&x)[C]) {
  if constexpr (C == 1) {
    if constexpr (quantised(S)) {
      x[0] = decode1<S>(static_cast<const unsigned char*>(pool)[i]);
    } else if constexpr (fp4(S)) {
      x[0] = widen_fp4(static_cast<uint32_t>(static_cast<const unsigned char*>(pool)[i >> 1]) >> (4 * (i & 1)), 1.f)[0];
    } else {
      x[0] = load_elem<S>(pool, i);
    }
  } else {
    static_assert(C == 4, "one or four elements");
    if constexpr (quantised(S)) {
      decode4<S>(*reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(pool) + i), x);
    } else if constexpr (fp4(S)) {
      const uint32_t w = *reinterpret_cast<const unsigned short*>(static_cast<const unsigned char*>(pool) + (i >> 1));
      const f32x2 lo = widen_fp4(w, 1.f), hi = widen_fp4(w >> 8, 1.f);
      x[0] = lo[0];
      x[1] = lo[1];
      x[2] = hi[0];
      x[3] = hi[1];
    } else if constexpr (S == HS_DTYPE_F32) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(pool) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = w[e];
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const unsigned short*>(pool) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned short h = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
        x[e] = S == HS_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
      }
    }
  }
}

// The general kernel: any head dim up to 512, page size, pool and query type; one
// workgroup of four waves per (split, KV head and G of its query heads, request).  A wave
// takes tiles of 64 tokens: a lane scores one token for the G heads (its K row against the
// queries in LDS, read as broadcasts), then the lanes turn to the head dim and add the
// tile's V rows, C elements a lane and 64 / (D / C) rows at once, weighted by the heads'
// probabilities from LDS.  Both products run on the vector unit in fp32 throughout,
// and bound the kernel: 16 requests of 4096 tokens, 32 query and 8 KV heads of 80 in int8, 88 MB,
// take 51.5 us, 1.7 TB/s; of 512 in bf16, 1.07 GB, 354, 3.0.  Odd head dims load single elements
// (81: 141 us).
constexpr int PG_W = 4;
constexpr int PG_T = 64 * PG_W;

static int64_t general_smem(int64_t G, int64_t D) {  // floats: queries, probabilities, offsets; or the waves' sums
  const int64_t tile = G * D + PG_W * G * 64 + PG_W * 64 * 2, sums = PG_W * G * D;
  return 4 * (tile > sums ? tile : sums);
}

template <int S, int C, int NC, int G>
__global__ __launch_bounds__(PG_T) void pages_general_kernel(PagesArgs a) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ float s_m[PG_W][G], s_l[PG_W][G];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int D = static_cast<int>(a.D);
  const int64_t split = blockIdx.x, b = blockIdx.z;
  const int64_t kv = blockIdx.y / a.head_chunks, h0 = static_cast<int64_t>(blockIdx.y % a.head_chunks) * G;
  const int heads = static_cast<int>(a.g - h0 < G ? a.g - h0 : G);
  const int32_t length = static_cast<int32_t>(request_length(a, b));
  const int32_t lo = seen_of(length, a.window, a.sinks).lo, skip = lo > a.sinks ? lo - a.sinks : 0;
  const int64_t n = length - skip, t0 = split * a.chunk;  // the tokens that count, one after another
  const int64_t t1 = n < t0 + a.chunk ? n : t0 + a.chunk;
  const int32_t* table = a.tables + b * a.t_sb + kv * a.t_sk;
  float* s_q = smem;                                       // [G][D]
  float* s_p = smem + G * D + wave * G * 64;               // [G][64] of this wave
  int32_t* s_at = reinterpret_cast<int32_t*>(smem + G * D + PG_W * G * 64) + wave * 128;  // [64] block, [64] row within
  for (int i = threadIdx.x; i < G * D; i += PG_T) {
    const int h = i / D;
    s_q[i] = h < heads ? load_any(a.q, b * a.q_sb + (kv * a.g + h0 + h) * a.q_sh + (i - h * D), a.q_dtype) : 0.f;
  }
  __syncthreads();

  const int lpr = (D + C - 1) / C < 64 ? (D + C - 1) / C : 64;  // lanes of a V row
  const int abreast = 64 / lpr;                                  // V rows at once
  const int sub = lane / lpr, first = lane - sub * lpr;          // this lane's row and first chunk of it
  float acc[G][NC * C];
#pragma unroll
  for (int h = 0; h < G; ++h)
#pragma unroll
    for (int e = 0; e < NC * C; ++e) acc[h][e] = 0.f;
  float m[G], l[G];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
  }

  for (int64_t base = t0 + wave * 64; base < t1; base += PG_T) {
    int64_t t = base + lane;
    int64_t block = -1, within = 0;
    if (t < t1) {
      if (t >= a.sinks) t += skip;
      const int64_t page = t / a.P;
      within = t - page * a.P;
      block = table[page];
    }
    const bool ok = block >= 0 && block < a.blocks;
    const int64_t row = ok ? (block * 2 * a.P + within) * a.Hkv + kv : 0;  // head vector of K; V: + P * Hkv
    float dot[G];
#pragma unroll
    for (int h = 0; h < G; ++h) dot[h] = 0.f;
    if (ok) {
      if constexpr (fp4(S)) {
        for (int g = 0; g < D / FP4_GROUP; ++g) {
          float part[G] = {};
#pragma unroll 4
          for (int d = g * FP4_GROUP; d < (g + 1) * FP4_GROUP; d += C) {
            float x[C];
            load_pool<S, C>(a.pool, row * D + d, x);
#pragma unroll
            for (int h = 0; h < G; ++h)
#pragma unroll
              for (int e = 0; e < C; ++e) part[h] += x[e] * s_q[h * D + d + e];
          }
          const float scale = fp4_scale(a.scale_bytes[row * (D / FP4_GROUP) + g]);
#pragma unroll
          for (int h = 0; h < G; ++h) dot[h] += part[h] * scale;
        }
      } else {
#pragma unroll 4
        for (int d = 0; d < D; d += C) {
          float x[C];
          load_pool<S, C>(a.pool, row * D + d, x);
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int e = 0; e < C; ++e) dot[h] += x[e] * s_q[h * D + d + e];
        }
      }
    }
    float k_scale = a.scale, v_scale = 1.f;
    if constexpr (quantised(S)) {
      k_scale = ok ? a.scales[row] * a.scale : 0.f;
      v_scale = ok ? a.scales[row + a.P * a.Hkv] : 0.f;
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const float s = ok ? dot[h] * k_scale : -INFINITY;
      float top = s;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
      const float m_new = fmaxf(m[h], top);
      const float alpha = m_new == -INFINITY ? 1.f : exp2_(m[h] - m_new);
      const float p = s == -INFINITY ? 0.f : exp2_(s - m_new);  // a NaN score stays NaN
      l[h] = l[h] * alpha + p;
      m[h] = m_new;
      s_p[h * 64 + lane] = ok ? p * v_scale : 0.f;
#pragma unroll
      for (int e = 0; e < NC * C; ++e) acc[h][e] *= alpha;
    }
    s_at[lane] = ok ? static_cast<int32_t>(block) : -1;
    s_at[64 + lane] = static_cast<int32_t>(within);
    wave_lds_sync();
    const int64_t left = t1 - base;
    const int rows = left < 64 ? static_cast<int>(left) : 64;
    if (sub < abreast) {
#pragma unroll 4
      for (int r = sub; r < rows; r += abreast) {
        const int64_t vb = s_at[r];
        if (vb < 0) continue;
        const int64_t at = ((vb * 2 + 1) * a.P + s_at[64 + r]) * a.Hkv + kv;
        float p[G];
#pragma unroll
        for (int h = 0; h < G; ++h) p[h] = s_p[h * 64 + r];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int d = (first + lpr * i) * C;
          if (d >= D) continue;
          float x[C];
          load_pool<S, C>(a.pool, at * D + d, x);
          if constexpr (fp4(S)) {
            const float scale = fp4_scale(a.scale_bytes[at * (D / FP4_GROUP) + d / FP4_GROUP]);
#pragma unroll
            for (int e = 0; e < C; ++e) x[e] *= scale;
          }
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int e = 0; e < C; ++e) acc[h][i * C + e] += p[h] * x[e];
        }
      }
    }
    wave_lds_sync();  // the tile's reads done before the next tile's writes
  }

  // the waves' sums, then this split's partial
#pragma unroll
  for (int h = 0; h < G; ++h) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) l[h] += __shfl_xor(l[h], off, 64);
    if (l[h] != l[h]) m[h] = 0.f;  // only NaN scores leave no maximum: keep the partial in the merge
    if (lane == 0) {
      s_m[wave][h] = m[h];
      s_l[wave][h] = l[h];
    }
  }
  __syncthreads();  // queries and probabilities are no longer read
  float* sum = smem + wave * G * D;
  for (int u = 0; u < abreast; ++u) {  // the rows read abreast add up in turn: a fixed order
    if (sub == u) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int d = (first + lpr * i) * C + e;
          if (d >= D) continue;
#pragma unroll
          for (int h = 0; h < G; ++h) sum[h * D + d] = (u == 0 ? 0.f : sum[h * D + d]) + acc[h][i * C + e];
        }
      }
    }
    wave_lds_sync();
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += PG_T) {
    const int h = i / D, d = i - h * D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < PG_W; ++w) M = fmaxf(M, s_m[w][h]);
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < PG_W; ++w) {
        const float f = s_m[w][h] == -INFINITY ? 0.f : exp2_(s_m[w][h] - M);
        L += f * s_l[w][h];
        O += f * smem[(w * G + h) * D + d];
      }
    }
    const int64_t head = kv * a.g + h0 + h;
    if (a.splits == 1) {
      store_any(a.out, b * a.o_sb + head * a.o_sh + d, L != 0.f ? O / L : 0.f, a.q_dtype);
      continue;
    }
    const int64_t at = (b * a.splits + split) * a.Hq + head;
    if (d == 0) {
      a.part_m[at] = M;
      a.part_l[at] = L;
    }
    a.part_o[at * D + d] = O;
  }
}

// ---- the matrix-core kernel ---------------------------------------------------------------
// Head dims of 32, 64, 96, 128 and 256.  A wave owns one unit (a KV head and up to 16 of its query
// heads) and walks tiles of 32 tokens, with no shared memory:
//
//   S^T = K Q^T   A: K rows (lane (j, c): row c, 8 of the head dim), B: the heads' queries;
//                 lane (j, c) receives head c's scores of tokens 4j .. 4j+3 and 16 + those
//   O^T += V^T P  B: those eight scores' weights, held already where the product wants them;
//                 A: lane (j, c) the same eight tokens' V at dims (D/16) c .., so that a V row
//                 is one contiguous load of the 16 lanes of a group (of 96 dims two: 4c .. and
//                 64 + 2c ..) and the transpose is the pairing of two tokens in a register
//
// with (j, c) = (lane / 16, lane % 16).  Codes widen to bf16 in registers (exact); queries and
// weights go in as sums of bf16 parts: as many of the query as its type has significand (1
// for bf16, 2 for float16, 3 for float32) and of the weights two (which hold a weight to 2^-16 of
// itself, a 256th of a bf16 output's half step and a 32nd of a float16's; three for float32
// queries).  float16 pools use float16 products, float32 pools float32 ones (four
// of the head dim, or four tokens, at a time; the same lanes hold the same values).  float16's
// range is short for weights, so they are held at 2^LIFT times their size, what the first part
// leaves at 2^LOW times that, and the products of the two are added in fp32: at most 2^-22 of a
// weight and 2^-(25 + LIFT + LOW) = 2^-45 of the largest one are lost.  (Two parts at one scale
// lose any weight below 2^-25 of the largest, which a long history behind one leading key adds
// up.  16 requests of 4096 tokens, 32 query and 8 KV heads, us at head dim 64, 128 and 256: 31.5
// 48.1 98 with these scales, as without.)  A tile's
// scales are one dword a lane, spread over the group by the broadcast of the multiply itself.
// The running maximum moves only when a score passes it by more than SLACK (the sums then
// hold weights up to 2^SLACK, no less precise): no cross-lane step in most tiles.

// Waves of a workgroup: half as many for 256 of the head dim, with twice the registers each.
constexpr int mfma_waves(int64_t D) { return D > 128 ? 4 : 8; }
// Waves a SIMD that the register allocator is held to (1: it decides).  float16 queries of 64 of the head
// dim in the short launch stand at the border between one workgroup a CU and two (126 to 130 registers)
// and fit below it without a spill (us with it and without, 14 and 2 heads on e4m3, 256 requests of
// 1024 tokens 22.9 and 24.3, 1024 of 256 26.4 and 32.5); a pair's 157 do not.
constexpr int mfma_least(int QD, int64_t D, bool SHORT, bool PAIR) {
  return QD == HS_DTYPE_F16 && D == 64 && SHORT && !PAIR ? 4 : 1;
}
constexpr int PM_PARTS = 8;  // parts of a short request
constexpr int PM_LANES = 64;  // requests whose schedule a wave derives by itself
constexpr float PM_SLACK = 6.f;
constexpr float PM_LIFT = 9.f;  // weights reach 2^(SLACK + LIFT) = 2^15, float16 65504
constexpr int PM_LOW = 11;      // what a float16 leaves of 2^15 is at most 2^4

// The power of two by which weights are held above the running maximum m's scale.  From 2^20 on
// float32 holds scores to 2^-3 at best and their distance to m - LIFT no longer exactly: none then.
template <bool F16>
__device__ __forceinline__ float lift_at(float m) { return F16 && fabsf(m) < 0x1p20f ? PM_LIFT : 0.f; }

// Parts of a query, and of a weight.  Two parts of a weight lose at most 2^-16 of it, and the output's
// own rounding is off by up to 2^-8 (bf16) or 2^-11 (float16) of it: 0.2% of bf16 outputs and 1.4% of
// float16's (8-bit pools) are another neighbour than the 64-bit result rounded, with a third part
// 0.03% and 0.12%, where the mean distance to it is the rounding's in all of them.  The third part
// took 16 requests of 4096 tokens, 8 KV heads of 64 in int8, from 22.0 to 23.0 us, 8 of 131072 with
// 4 of 128 from 195.0 to 195.6, and nothing at 256; float32 outputs need it.
template <int S, int QD>
constexpr int query_parts() { return !quantised(S) && !fp4(S) ? 1 : (QD == HS_DTYPE_BF16 ? 1 : (QD == HS_DTYPE_F16 ? 2 : 3)); }
template <int S, int QD>
constexpr int weight_parts() { return (quantised(S) || fp4(S)) && QD == HS_DTYPE_F32 ? 3 : 2; }

template <bool F16>
__device__ __forceinline__ float low16(uint32_t w) {
  return F16 ? f16_bits_to_f32(static_cast<unsigned short>(w)) : __uint_as_float(w << 16);
}
template <bool F16>
__device__ __forceinline__ float high16(uint32_t w) {
  return F16 ? f16_bits_to_f32(static_cast<unsigned short>(w >> 16)) : __uint_as_float(w & 0xffff0000u);
}

// Two pairs' low halves, or high halves, as one pair.
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Two small floats as a bf16 pair, exactly (codes have at most 8 significand bits).
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
  return high_halves(__float_as_uint(lo), __float_as_uint(hi));
}

template <bool F16>
__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The value of lane n of each group of 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t group_word(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x150 + N, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ float group_lane(float v) { return __uint_as_float(group_word<N>(__float_as_uint(v))); }

// BYTES bytes (1, 2, 4, 8 or 16 a load) as words.
template <int BYTES>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (BYTES == 1) {
    w[0] = *reinterpret_cast<const unsigned char*>(p);
  } else if constexpr (BYTES == 2) {
    w[0] = *reinterpret_cast<const unsigned short*>(p);
  } else if constexpr (BYTES == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0];
    w[1] = v[1];
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
  }
}

// The scale bytes of one head vector, in order.
template <int GS>
__device__ __forceinline__ void load_scales(const unsigned char* p, uint32_t* w) {
  if constexpr (GS == 3) w[0] = p[0] | static_cast<uint32_t>(p[1]) << 8 | static_cast<uint32_t>(p[2]) << 16;
  else load_words<GS>(reinterpret_cast<const char*>(p), w);
}

struct Share {
  int64_t b;
  int32_t slot, part, parts;  // this workgroup's slot; its part of the request's
  int32_t n;                  // the request's tokens
};

// Inclusive sum over the wave's lanes on the vector unit (no LDS permutes: this runs before
// the first load of a workgroup).
template <typename T>
__device__ __forceinline__ T scan_lanes(T v) {
  auto step = [&](auto ctrl, auto rows) {
    const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value,
                                              0xf, true);
    v += __builtin_bit_cast(T, o);
  };
  step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from 1, 2, 4, 8 lanes below
  step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // a row's last lane to the next row
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // lane 31 to the upper half
  return v;
}

// The request and part of workgroup w, of up to PM_LANES requests: every wave derives the same
// schedule from the lengths, one request a lane.
template <bool WINDOW>
__device__ __forceinline__ bool share_of(const PagesArgs& a, int32_t w, Share& out) {
  const int lane = threadIdx.x & 63;
  const int32_t n = lane < a.B ? clamp_length(a.lengths[lane], a.pages * a.P) : 0;
  const int32_t tiles = WINDOW ? seen_tiles(n, a.window, a.sinks) : tiles_of(n);
  const float total =
      __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scan_lanes(static_cast<float>(tiles))), 63));
  const uint32_t target = static_cast<uint32_t>(a.target), min_tiles = static_cast<uint32_t>(a.min_tiles);
  const uint32_t sure = sure_size(total, sure_room(a.target, a.B));
  uint32_t per = tried_size(sure, sure, 0, min_tiles);
  if (total < 0x1p24f && a.B * 4 > a.target) {
    const uint32_t least = (static_cast<uint32_t>(total) + target - 1) / target;
    uint32_t count[PM_TRIES / 2];  // two sizes' parts in 16 bits each: at most target + B
#pragma unroll
    for (int k = 0; k < PM_TRIES; k += 2) {
      const int32_t lo = parts_of(tiles, tried_size(least, sure, k, min_tiles));
      const int32_t hi = parts_of(tiles, tried_size(least, sure, k + 1, min_tiles));
      count[k / 2] = __builtin_amdgcn_readlane(scan_lanes(lane < a.B ? lo | hi << 16 : 0), 63);
    }
#pragma unroll
    for (int k = PM_TRIES - 1; k >= 0; --k)
      if ((count[k / 2] >> (16 * (k & 1)) & 0xffffu) <= target) per = tried_size(least, sure, k, min_tiles);
  }
  const int32_t parts = lane < a.B ? parts_of(tiles, per) : 0, through = scan_lanes(parts);
  const uint64_t owners = __ballot(through > w);
  if (!owners) return false;
  const int src = __ffsll(static_cast<unsigned long long>(owners)) - 1;
  out.b = src;
  out.n = __builtin_amdgcn_readlane(n, src);
  out.parts = __builtin_amdgcn_readlane(parts, src);
  out.part = w - (__builtin_amdgcn_readlane(through, src) - out.parts);
  out.slot = w;
  return true;
}

// SHORT: few tokens in all.  Every unit has workgroups of its own (all waves on its tiles), a
// request `max_parts` at most, in a fixed grid, so that the table, the length and the query
// load together; a part alone writes the output, several are joined by the last to arrive.
// Else the schedule of share_of over workgroups of up to four units (a page's rows are
// contiguous over the KV heads), joined by pages_merge_kernel.
// PAIR (4-bit pools, one table for all KV heads, at most 8 query heads a KV head): a unit is two
// neighbouring KV heads, whose vectors are one of 2D, with the first one's query heads in columns 0 ..
// 7 of the products and the second one's in 8 .. 15.  Scores are taken from either's product; of V's
// the quarter in which rows and columns are of one head counts, half of the lanes' sums.  So a wave
// reads whole lines of the cache (a head's row is 64 bytes at D = 128: two waves that each read one
// half of a line take it from memory twice where they drift apart), and one exponential a lane
// serves two heads.  us with one head a unit and with two: 8 requests of 131072 tokens, 28 and 4
// heads of 128, 112 (the loads alone 111) and 106; 16 of 65536 .. 20521, 40 and 8 heads, float16
// queries, 166 and 137.  (Small calls go one by one: pages.hip, one_by_one.)
// WINDOW: whole histories have kernels without its arithmetic, which takes up to ten registers and
// with them one of two workgroups a CU where a kernel stands at the border.  us with it and without,
// 14 query and 2 KV heads of 64, whole histories: float16, 512 requests of 1024 tokens 47.3 and 42.8,
// 1024 of 256 37.5 and 30.2; float16 queries on e4m3, 256 of 1 .. 4096 41.4 and 40.4 (but 96 of 4096
// each, 40 and 8 heads, 112 with one workgroup a CU and 121 with two).
template <int S, int QD, int D, bool UNIFORM, bool SHORT, bool WINDOW, bool PAIR = false>
__global__ __launch_bounds__(64 * mfma_waves(D), mfma_least(QD, D, SHORT, PAIR)) void pages_mfma_kernel(PagesArgs a) {
  static_assert(!PAIR || (fp4(S) && D <= 128 && D != 96), "pairs of 4-bit head vectors of 32, 64 or 128");
  constexpr int KVS = PAIR ? 2 : 1, DD = KVS * D;  // KV heads of a unit; their vectors' elements
  constexpr int W = mfma_waves(D), T = 64 * W;
  constexpr bool F16 = S == HS_DTYPE_F16, F32 = S == HS_DTYPE_F32;
  constexpr int BITS = elem_bits(S), VECTOR = D * BITS / 8;  // of an element; bytes of a head vector
  constexpr int KK = F32 ? D / 4 : D / 32;   // products over the head dim
  constexpr int E = DD / 16;                 // V elements of a lane and token
  constexpr int NQ = query_parts<S, QD>(), NP = weight_parts<S, QD>();
  constexpr int KROW = VECTOR / 4;           // K bytes of a lane and row
  constexpr int KL = KROW < 16 ? KROW & -KROW : (KROW % 16 ? 8 : 16);  // a K load
  constexpr int KN = KROW / KL;
  constexpr int E0 = D == 96 ? 4 : E;        // V elements of a lane and token in its first load(s)
  constexpr int VB = E0 * BITS / 8;          // their bytes
  constexpr int VL = VB < 16 ? VB : 16;      // a V load
  constexpr int VB1 = (E - E0) * BITS / 8;   // bytes of the second part, from dim 16 E0
  constexpr int VW0 = VB < 4 ? 1 : VB / 4, VW = VW0 + (VB1 + 3) / 4;
  constexpr int GS1 = D / FP4_GROUP, GS = KVS * GS1;  // 4-bit pools: scales of a head vector, and of a unit's
  constexpr int SD = D + 4;                  // row stride of the waves' sums in LDS: no bank conflicts
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ float s_m[W][16], s_l[W][16];
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  Share sh;
  if constexpr (SHORT) {
    sh.b = blockIdx.z;
    sh.part = static_cast<int32_t>(blockIdx.x);
  } else {
    if (a.shares) {
      const Slot t = a.shares[blockIdx.x];
      if (t.b < 0) return;
      sh = Share{t.b, static_cast<int32_t>(blockIdx.x), t.part, t.parts, t.n};
    } else {
      if (!share_of<WINDOW>(a, static_cast<int32_t>(blockIdx.x), sh)) return;  // the same for every wave
      if (sh.part == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.ranges[sh.b] = SlotRange{sh.slot, sh.parts};
    }
  }
  const int64_t b = sh.b;
  const int unit = SHORT ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.y) * a.waves_units + wave % a.waves_units;
  const int sub = SHORT ? wave : wave / a.waves_units;
  const int subs = SHORT ? W : a.subs;
  const int kv = PAIR ? 2 * unit : unit / a.head_chunks, h0 = PAIR ? 0 : unit % a.head_chunks * 16;
  const int heads = PAIR ? static_cast<int>(2 * a.g) : static_cast<int>(a.g - h0 < 16 ? a.g - h0 : 16);
  const int32_t* table = a.tables + b * a.t_sb + kv * a.t_sk;
  const uint32_t P = static_cast<uint32_t>(a.P), pages = static_cast<uint32_t>(a.pages);
  const char* pool = static_cast<const char*>(a.pool);
  const uint32_t row_bytes = static_cast<uint32_t>(a.Hkv) * VECTOR;  // the host keeps 16 of them in 31 bits
  const int64_t v_plane = a.P * static_cast<int64_t>(row_bytes);

  // Everything that needs no other load goes out first: the length, the first table entries
  // (whatever the length: an index past the table reads its first entry, unused) and the query.
  const int64_t limit = a.pages * a.P;
  const int32_t length = SHORT ? a.lengths[b] : sh.n;
  unsigned long long* counter = nullptr;
  unsigned long long seen = 0;
  int32_t share, tile0;
  if constexpr (SHORT) {
    if (a.max_parts > 1) {  // else there is no workspace
      counter = a.arrivals + b * a.units + unit;
      seen = __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    share = static_cast<int32_t>(a.min_tiles);
    tile0 = sh.part * share;
  }
  // Tiles are counted over those that the window shows; `tile_at` says which of the request's one is.
  int32_t n = 0, tiles = 0;
  Seen view{0, 0, 0};
  auto measure = [&]() {  // waits for the length
    n = __builtin_amdgcn_readfirstlane(length < 0 ? 0 : (length > limit ? static_cast<int32_t>(limit) : length));
    if constexpr (WINDOW) view = seen_of(n, a.window, a.sinks);
    tiles = tiles_of(n) - view.gap;
    if constexpr (SHORT) sh.parts = tiles > share ? (tiles + share - 1) / share : 1;
  };
  if constexpr (!SHORT) {
    measure();
    share = (tiles + sh.parts - 1) / sh.parts;
    tile0 = sh.part * share;
  } else if constexpr (WINDOW) {
    measure();  // which table entries come first depends on the length then
  }
  auto tile_at = [&](int32_t tile) { return WINDOW && tile >= view.front ? tile + view.gap : tile; };

  // UNIFORM: pages of a multiple of 16 rows, so a tile's two halves lie in one page each.  A wave
  // reads the table for 32 of its tiles at once (lane l: half l), keeps the halves' first rows
  // in a register and takes each tile's from there; tiles without a page are passed over.
  // Else lanes 0-31 find their token's row, one tile ahead, and the others take it from them.
  // Table entry, and row within its page, of this lane's half (UNIFORM: in the next batch) or
  // token (in the next tile).
  int32_t entry = 0;
  uint32_t within = 0;
  auto half_token = [&](int32_t batch) {  // first token of this lane's half in the batch
    return static_cast<uint32_t>(tile_at(tile0 + sub + (batch + (lane >> 1)) * subs)) * 32u + 16u * (lane & 1);
  };
  auto token_of = [&](int32_t tile) { return static_cast<uint32_t>(tile_at(tile)) * 32u + (lane & 31); };
  auto fetch = [&](uint32_t token) {
    const uint32_t page = token / P;
    within = token - page * P;
    entry = table[page < pages ? page : 0u];
  };
  int32_t at_tile = tile0 + sub;  // !UNIFORM: the tile `entry` belongs to
  if constexpr (UNIFORM) fetch(half_token(0));
  else fetch(token_of(at_tile));

  // Q of head c, 8 of the head dim from d0(kk) for each product kk; or float32's one, at the dim
  // of the lane's kk-th K word
  auto d0_of = [&](int kk) {
    if constexpr (fp4(S)) return 2 * KL * (4 * (kk / (KL / 4)) + j) + 8 * (kk % (KL / 4));
    return F32 ? 16 * (kk >> 2) + 4 * j + (kk & 3)
               : (BITS == 8 && KL == 16 ? 64 * (kk >> 1) + 16 * j + 8 * (kk & 1) : 32 * kk + 8 * j);
  };
  const bool live = PAIR ? (c & 7) < a.g : c < heads;
  // (this column's query head past the unit's first; not held through the loop: two registers)
  auto column = [&](int v) { return PAIR ? (v >> 3) * a.g + (v & 7) : v; };
  const int64_t q_at = b * a.q_sb + (kv * a.g + h0 + column(live ? c : 0)) * a.q_sh;
  constexpr int QE = F32 ? 1 : 8;
  constexpr int QW = QD == HS_DTYPE_F32 ? QE : 4;  // words of a product's elements
  uint32_t qw[KK][QW];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if constexpr (QD == HS_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < QE; ++i)
        qw[kk][i] = __float_as_uint(static_cast<const float*>(a.q)[q_at + d0_of(kk) + i]);
    } else {
      const unsigned short* q = static_cast<const unsigned short*>(a.q) + q_at + d0_of(kk);
      if (a.q_vec) {
        load_words<16>(reinterpret_cast<const char*>(q), qw[kk]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) qw[kk][i] = q[2 * i] | static_cast<uint32_t>(q[2 * i + 1]) << 16;
      }
    }
  }
  if constexpr (SHORT && !WINDOW) measure();
  const int32_t tile1 = tile0 + share < tiles ? tile0 + share : tiles;
  if (SHORT && sh.part > 0 && tile0 >= tiles) return;  // past the request's tiles: the whole workgroup

  f32x4 acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  // A tile's registers: scales, K and V.  Loads of the next tile go out as soon as the registers
  // of this one are consumed.
  uint32_t kw[2][KVS * KN * KL / 4], vw[8][VW];
  float sc = 0.f;
  // 4-bit pools: the scale bytes of a lane's K loads, and all those of one token's V
  uint32_t kb[2][fp4(S) ? KVS * KN : 1], vb[fp4(S) && GS > 4 ? 2 : 1];
  // token of the scale this lane holds (lanes 0-7 of a group: keys, 8-15: values)
  const int s_token = 4 * j + (c & 3), s_half = (c >> 2) & 1;
  float qs[F32 ? KK : 1];
  u32x4 qf[F32 ? 1 : NQ][F32 ? 1 : KK];
  auto split_query = [&]() {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (F32) {
        qs[kk] = live ? __uint_as_float(qw[kk][0]) : 0.f;
      } else if constexpr (NQ == 1) {  // a 16-bit query goes in as it is
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[0][kk][i] = live ? qw[kk][i] : 0u;
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (QD == HS_DTYPE_F32) x[i] = __uint_as_float(qw[kk][i]);
          else x[i] = i & 1 ? high16<true>(qw[kk][i >> 1]) : low16<true>(qw[kk][i >> 1]);
          x[i] = live ? x[i] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qf[q][kk][i] = pack16<F16>(x[2 * i], x[2 * i + 1]);
            x[2 * i] -= low16<F16>(qf[q][kk][i]);
            x[2 * i + 1] -= high16<F16>(qf[q][kk][i]);
          }
        }
      }
    }
  };

  // One tile; bit t of `valid`: its token t counts.
  auto use_tile = [&](uint32_t valid, auto next_k, auto next_v) {
    // this tile's scales leave the register that the next tile's load writes (a copy made at
    // the end of the tile instead would wait for that load there)
    float sct = 0.f;
    if constexpr (quantised(S)) asm volatile("v_mov_b32 %0, %1" : "=v"(sct) : "v"(sc));
    float s[8];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
      if constexpr (PAIR) {
        f32x4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          u32x4 kf, kg;
          widen_fp4_bf16x8(kw[rt][kk], __uint_as_float(kb[rt][0] << 23), kf);
          widen_fp4_bf16x8(kw[rt][KK + kk], __uint_as_float(kb[rt][1] << 23), kg);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            t = mfma_16x16x32<false>(kf, qf[q][kk], t);
            u = mfma_16x16x32<false>(kg, qf[q][kk], u);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = c < 8 ? t[i] : u[i];
      } else {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if constexpr (F32) {
            t = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[rt][kk]), qs[kk], t, 0, 0, 0);
          } else {
            u32x4 kf;
            if constexpr (fp4(S)) {
              widen_fp4_bf16x8(kw[rt][kk], __uint_as_float(kb[rt][kk / (KL / 4)] << 23), kf);
            } else if constexpr (quantised(S)) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float x[4];
                decode4<S>(kw[rt][2 * kk + h], x);
                kf[2 * h] = pair_bf16(x[0], x[1]);
                kf[2 * h + 1] = pair_bf16(x[2], x[3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) kf[i] = kw[rt][4 * kk + i];
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q) t = mfma_16x16x32<F16>(kf, qf[q][kk], t);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * rt + i] = t[i];
    }
    next_k();
    const bool whole = valid == 0xffffffffu;
    if (!whole) {  // a row past the end may hold anything
      if constexpr (quantised(S)) sct = valid >> (16 * s_half + s_token) & 1 ? sct : 0.f;
      if constexpr (fp4(S)) {
        const bool in = valid >> (16 * s_half + s_token) & 1;
        vb[0] = in ? vb[0] : 0u;
        if constexpr (GS > 4) vb[1] = in ? vb[1] : 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = valid >> (16 * (e >> 2) + 4 * j + (e & 3)) & 1;
#pragma unroll
        for (int w = 0; w < VW; ++w) vw[e][w] = in ? vw[e][w] : 0u;  // its weight is 0, but 0 * NaN is not
      }
    }
    if constexpr (quantised(S)) {
      const float ks = sct * a.scale;
      s[0] *= group_lane<0>(ks);
      s[1] *= group_lane<1>(ks);
      s[2] *= group_lane<2>(ks);
      s[3] *= group_lane<3>(ks);
      s[4] *= group_lane<4>(ks);
      s[5] *= group_lane<5>(ks);
      s[6] *= group_lane<6>(ks);
      s[7] *= group_lane<7>(ks);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] *= a.scale;
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = valid >> (16 * (e >> 2) + 4 * j + (e & 3)) & 1 ? s[e] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e]);
    if (__any(top > m_run + PM_SLACK)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m_new = fmaxf(m_run, top);
      const float alpha =
          m_new == -INFINITY ? 1.f : exp2_((m_run - lift_at<F16>(m_run)) - (m_new - lift_at<F16>(m_new)));
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run - lift_at<F16>(m_run);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = exp2_(s[e] - m_use);
    l_run += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    if constexpr (quantised(S)) {
      s[0] *= group_lane<8>(sct);
      s[1] *= group_lane<9>(sct);
      s[2] *= group_lane<10>(sct);
      s[3] *= group_lane<11>(sct);
      s[4] *= group_lane<12>(sct);
      s[5] *= group_lane<13>(sct);
      s[6] *= group_lane<14>(sct);
      s[7] *= group_lane<15>(sct);
    }
    if constexpr (F32) {  // four tokens a product: token slot t of the four groups
#pragma unroll
      for (int t = 0; t < 8; ++t) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vw[t][e]), s[t], acc[e], 0, 0, 0);
      }
    } else {
      u32x4 pf[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pf[q][i] = pack16<F16>(s[2 * i], s[2 * i + 1]);
          if (q + 1 < NP) {
            constexpr float UP = F16 ? 1 << PM_LOW : 1;
            s[2 * i] = (s[2 * i] - low16<F16>(pf[q][i])) * UP;
            s[2 * i + 1] = (s[2 * i + 1] - high16<F16>(pf[q][i])) * UP;
          }
        }
      }
      // 4-bit V: the scales of the eight tokens at this lane's dims (of 96 dims two parts), in the
      // exponent's place; the instruction that widens reads no other bit of them
      float vs[8][VB1 > 0 ? 2 : 1];
      if constexpr (fp4(S)) {
        const uint32_t group = static_cast<uint32_t>(c * E0) / FP4_GROUP;
        auto spread = [&](auto token) {
          constexpr int T = decltype(token)::value;
          uint32_t w = group_word<T>(vb[0]);
          if constexpr (GS > 4) {
            const uint32_t high = group_word<T>(vb[1]);  // taken by every lane: its source lanes must be on
            w = c >= 8 ? high : w;
          }
          vs[T][0] = __uint_as_float(GS == 1 ? w << 23 : __builtin_amdgcn_alignbit(w, w, 8 * (group & 3) + 9));
          if constexpr (VB1 > 0) vs[T][1] = __uint_as_float(w << 7);
        };
        spread(std::integral_constant<int, 0>{});
        spread(std::integral_constant<int, 1>{});
        spread(std::integral_constant<int, 2>{});
        spread(std::integral_constant<int, 3>{});
        spread(std::integral_constant<int, 4>{});
        spread(std::integral_constant<int, 5>{});
        spread(std::integral_constant<int, 6>{});
        spread(std::integral_constant<int, 7>{});
      }
      // V^T fragments: pairs of tokens (2i, 2i + 1) at one dim
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        u32x4 even, odd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (fp4(S)) {
            const int part = e < E0 ? 0 : 1, word = e < E0 ? e >> 3 : VW0, byte = e < E0 ? (e >> 1) & 3 : (e - E0) >> 1;
            const uint32_t x = widen_fp4_bf16(vw[2 * i][word], vs[2 * i][part], byte);
            const uint32_t y = widen_fp4_bf16(vw[2 * i + 1][word], vs[2 * i + 1][part], byte);
            even[i] = low_halves(x, y);
            odd[i] = high_halves(x, y);
          } else if constexpr (quantised(S)) {
            float x[4], y[4];
            decode4<S>(vw[2 * i][e >> 2], x);
            decode4<S>(vw[2 * i + 1][e >> 2], y);
            even[i] = pair_bf16(x[e & 3], y[e & 3]);
            odd[i] = pair_bf16(x[(e & 3) + 1], y[(e & 3) + 1]);
          } else {
            even[i] = low_halves(vw[2 * i][e >> 1], vw[2 * i + 1][e >> 1]);
            odd[i] = high_halves(vw[2 * i][e >> 1], vw[2 * i + 1][e >> 1]);
          }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          if (F16 && q) {
            constexpr float DOWN = 1.f / (1 << PM_LOW);
            const f32x4 none = {0.f, 0.f, 0.f, 0.f};
            acc[e] += mfma_16x16x32<F16>(even, pf[q], none) * DOWN;
            acc[e + 1] += mfma_16x16x32<F16>(odd, pf[q], none) * DOWN;
          } else {
            acc[e] = mfma_16x16x32<F16>(even, pf[q], acc[e]);
            acc[e + 1] = mfma_16x16x32<F16>(odd, pf[q], acc[e + 1]);
          }
        }
      }
    }
    next_v();
  };

  if constexpr (UNIFORM) {
    const int32_t mine = tile1 - tile0 > sub ? (tile1 - tile0 - sub + subs - 1) / subs : 0;  // tiles of this wave
    int32_t batch = -32;  // none yet
    uint64_t present = 0;
    int64_t offset = 0;  // the half's first K row of this KV head, in head vectors
    auto open = [&]() {  // the batch of `entry` becomes current, and the next one's table loads start
      const uint32_t t = half_token(batch);
      const bool ok = batch + (lane >> 1) < mine && t < static_cast<uint32_t>(n) && entry >= 0 && entry < a.blocks;
      offset = ok ? (static_cast<int64_t>(entry) * 2 * P + within) * a.Hkv + kv : 0;
      present = __ballot(ok);
      if (batch + 32 < mine) fetch(half_token(batch + 32));
    };
    uint32_t valid = 0;
    uint64_t off0 = 0, off1 = 0;
    auto advance = [&]() {  // the next tile with a page; false at the end
      uint64_t some = (present | present >> 1) & 0x5555555555555555ull;
      while (some == 0) {
        batch += 32;
        if (batch >= mine) return false;
        open();
        some = (present | present >> 1) & 0x5555555555555555ull;
      }
      const int at = __ffsll(static_cast<unsigned long long>(some)) - 1;
      const int32_t base = 32 * tile_at(tile0 + sub + (batch + (at >> 1)) * subs), left = n - base;
      valid = left >= PM_TILE ? 0xffffffffu : (1u << left) - 1u;
      if (WINDOW && base < view.lo) valid &= seen_mask(base, view.lo, a.sinks);
      const uint32_t has = static_cast<uint32_t>(present >> at) & 3u;
      if (!(has & 1u)) valid &= 0xffff0000u;
      if (!(has & 2u)) valid &= 0x0000ffffu;
      const uint32_t lo = static_cast<uint32_t>(offset), hi = static_cast<uint32_t>(offset >> 32);
      auto from = [&](int l) {
        return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, l))) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, l));
      };
      off0 = from(at);
      off1 = from(at + 1);
      present &= ~(3ull << at);
      return true;
    };
    // A load is a base every lane shares and a 32-bit offset of the lane's own.
    const uint32_t k_lane = c * row_bytes + j * KL;
    const uint32_t s_lane = static_cast<uint32_t>(s_token) * static_cast<uint32_t>(a.Hkv);
    const uint32_t kb_lane = static_cast<uint32_t>(c) * static_cast<uint32_t>(a.Hkv) * GS1 + KL * j / 16;
    uint32_t v_lane[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v_lane[e] = (4 * j + e) * row_bytes;
    const uint32_t v_col = c * VB, v_col1 = 16 * VB + c * VB1;
    auto load_k = [&]() {
      if constexpr (quantised(S)) {
        const uint64_t row = (s_half ? off1 : off0) + (c >= 8 ? a.P * a.Hkv : 0);
        sc = a.scales[row + s_lane];
      }
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const char* p = pool + (rt ? off1 : off0) * VECTOR;
#pragma unroll
        for (int i = 0; i < KVS * KN; ++i) load_words<KL>(p + k_lane + 4 * KL * i, &kw[rt][i * (KL / 4)]);
        if constexpr (fp4(S)) {
          const unsigned char* b = a.scale_bytes + (rt ? off1 : off0) * GS1;
#pragma unroll
          for (int i = 0; i < KVS * KN; ++i) kb[rt][i] = b[kb_lane + (PAIR ? GS1 * i : KL * i / 4)];
        }
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const char* p = pool + v_plane + (e < 4 ? off0 : off1) * VECTOR;
#pragma unroll
        for (int i = 0; i < VB / VL; ++i) load_words<VL>(p + (v_lane[e & 3] + v_col) + VL * i, &vw[e][i * 4]);
        if constexpr (VB1 > 0) load_words<VB1>(p + (v_lane[e & 3] + v_col1), &vw[e][VW0]);
      }
      if constexpr (fp4(S))
        load_scales<GS>(a.scale_bytes + ((s_half ? off1 : off0) + a.P * a.Hkv + s_lane) * GS1, vb);
    };
    if (advance()) {
      load_k();
      load_v();
      split_query();
      bool more = true;
      while (more) {
        const uint32_t now = valid;
        more = advance();  // past the end the offsets stay: the last tile is read again, unused
        use_tile(now, load_k, load_v);
      }
    }
  } else {
    int64_t row = 0;  // head vector of K of this lane's token; a masked token reads row 0
    uint32_t valid = 0;
    auto advance = [&]() {
      const uint32_t t = token_of(at_tile);
      const bool ok = at_tile < tile1 && t < static_cast<uint32_t>(n) && entry >= 0 && entry < a.blocks &&
                      (!WINDOW || t >= static_cast<uint32_t>(view.lo) || t < static_cast<uint32_t>(a.sinks));
      row = ok ? (static_cast<int64_t>(entry) * 2 * P + within) * a.Hkv + kv : 0;
      valid = static_cast<uint32_t>(__ballot(ok));
      at_tile += subs;
      fetch(token_of(at_tile));
    };
    auto row_of = [&](int t) { return static_cast<int64_t>(__shfl(static_cast<long long>(row), t, 64)); };
    auto load_k = [&]() {
      if constexpr (quantised(S)) sc = a.scales[row_of(16 * s_half + s_token) + (c >= 8 ? a.P * a.Hkv : 0)];
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int64_t from = row_of(16 * rt + c);
        const char* p = pool + from * VECTOR + j * KL;
#pragma unroll
        for (int i = 0; i < KVS * KN; ++i) load_words<KL>(p + 4 * KL * i, &kw[rt][i * (KL / 4)]);
        if constexpr (fp4(S)) {
#pragma unroll
          for (int i = 0; i < KVS * KN; ++i) kb[rt][i] = a.scale_bytes[from * GS1 + KL * j / 16 + (PAIR ? GS1 * i : KL * i / 4)];
        }
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const char* p = pool + row_of(16 * (e >> 2) + 4 * j + (e & 3)) * VECTOR + v_plane;
#pragma unroll
        for (int i = 0; i < VB / VL; ++i) load_words<VL>(p + c * VB + VL * i, &vw[e][i * 4]);
        if constexpr (VB1 > 0) load_words<VB1>(p + 16 * VB + c * VB1, &vw[e][VW0]);
      }
      if constexpr (fp4(S)) load_scales<GS>(a.scale_bytes + (row_of(16 * s_half + s_token) + a.P * a.Hkv) * GS1, vb);
    };
    if (at_tile < tile1) {
      int32_t left = (tile1 - at_tile + subs - 1) / subs;
      advance();
      load_k();
      load_v();
      split_query();
      while (left > 0) {
        const uint32_t now = valid;
        advance();  // past the end every token is masked and reads row 0
        use_tile(now, load_k, load_v);
        --left;
      }
    }
  }

  // (of a pair, the lanes whose rows are of their column's head)
  const bool mine = live && (!PAIR || (j < 2) == (c < 8));
  auto dim_of = [](int v_lane, int e) {
    if constexpr (PAIR) return E * (v_lane & 7) + e;
    return e < E0 ? E0 * v_lane + e : 16 * E0 + (E - E0) * v_lane + e - E0;
  };
  m_run -= lift_at<F16>(m_run);  // the scale that the sums are at
  // the totals of a head over the four groups, then the waves of a unit, then the partial
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (l_run != l_run) m_run = 0.f;  // NaN scores set no maximum: keep the partial in the merge
  if (!SHORT && a.subs == 1) {
    if (mine) {
      const int64_t at = sh.slot * a.Hq + kv * a.g + h0 + column(c);
      if (j == 0 || (PAIR && j == 2)) {
        a.part_m[at] = m_run;
        a.part_l[at] = l_run;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) a.part_o[at * D + dim_of(4 * j + i, e)] = acc[e][i];
      }
    }
    return;
  }
  const int rows = PAIR ? 16 : static_cast<int>(a.g < 16 ? a.g : 16);
  if (mine) {
    if (j == 0 || (PAIR && j == 2)) {
      s_m[wave][c] = m_run;
      s_l[wave][c] = l_run;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) smem[(wave * rows + c) * SD + dim_of(4 * j + i, e)] = acc[e][i];
    }
  }
  __syncthreads();
  const int stride = SHORT ? 1 : a.waves_units, waves = SHORT ? W : a.waves_units * a.subs;
  const uint32_t tag = SHORT ? group_tag(a.epoch, counter_round(seen, a.epoch)) : 0u;
  constexpr int QUADS = D / 4;
  for (int i = threadIdx.x; i < stride * rows * QUADS; i += blockDim.x) {
    const int d = i % QUADS * 4, hu = i / QUADS;
    const int u = SHORT ? 0 : hu / rows, h = SHORT ? hu : hu % rows;
    const int un = SHORT ? unit : static_cast<int>(blockIdx.y) * a.waves_units + u;
    const int first = PAIR ? 0 : un % a.head_chunks * 16;
    if (PAIR ? (h & 7) >= a.g : first + h >= a.g) continue;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (u + w * stride < waves) M = fmaxf(M, s_m[u + w * stride][h]);
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int at = u + w * stride;
        if (at >= waves) continue;
        const float f = exp2_(s_m[at][h] - M);  // 0 where a wave had no token
        L += f * s_l[at][h];
        O += f * *reinterpret_cast<const f32x4*>(smem + (at * rows + h) * SD + d);
      }
    }
    const int64_t head = PAIR ? (2 * static_cast<int64_t>(un) + (h >> 3)) * a.g + (h & 7)
                              : static_cast<int64_t>(un / a.head_chunks) * a.g + first + h;
    if constexpr (SHORT) {
      if (sh.parts == 1) {
        store_quad<QD>(a.out, b * a.o_sb + head * a.o_sh + d, L != 0.f ? O * (1.f / L) : f32x4{0.f, 0.f, 0.f, 0.f}, a.o_vec);
      } else {
        const int64_t at = (b * a.max_parts + sh.part) * a.Hq + head;
        if (d == 0) {
          store_partial(a.word_m + at, M, tag);
          store_partial(a.word_l + at, L, tag);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) store_partial(a.word_o + at * D + d + e, O[e], tag);
      }
    } else {
      const int64_t at = sh.slot * a.Hq + head;
      if (d == 0) {
        a.part_m[at] = M;
        a.part_l[at] = L;
      }
      *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = O;
    }
  }
  if constexpr (SHORT) {
    if (sh.parts == 1) return;
    // The unit's last part joins all of them.  A slot is one (request, unit, part)'s at any
    // length, and its words are cleared as they are taken: a replay of the launch finds no
    // word of an earlier one, also where other work used the counters' memory in between.
    __shared__ int s_last;
    __shared__ float s_w[PM_PARTS][16], s_sum[16];
    __syncthreads();  // every wave's stores are out before the arrival
    if (threadIdx.x == 0) s_last = arrive_last(counter, seen, a.epoch, sh.parts) ? 1 : 0;
    __syncthreads();
    if (!s_last) return;
    const int64_t base = b * a.max_parts * a.Hq + kv * a.g + h0;  // word of head h, part p: base + p * Hq + h
    const int64_t next = a.Hq * D;                                // from a part's o word to the next part's
    // Every word goes out before any is used, with no branch between them (a part past the last
    // reads part 0's again): o words of the thread's (head, dim) pairs, then its m and its l.
    constexpr int PAIRS = (16 * D + T - 1) / T;
    unsigned long long w[PAIRS][PM_PARTS];
    auto pair_word = [&](int r) {
      const int i = threadIdx.x + T * r < heads * D ? threadIdx.x + T * r : 0;
      return a.word_o + (base + i / D) * D + i % D;
    };
#pragma unroll
    for (int r = 0; r < PAIRS; ++r) {
      if (T * r >= heads * D) continue;
#pragma unroll
      for (int u = 0; u < PM_PARTS; ++u)
        w[r][u] = __hip_atomic_load(pair_word(r) + (u < sh.parts ? u : 0) * next, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    auto taken = [&](unsigned long long* p, unsigned long long v) {  // a word's value, the word cleared
      if (static_cast<uint32_t>(v >> 32) != tag) v = partial_reread(p, tag);
      __hip_atomic_store(p, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return partial_value(v);
    };
    if (threadIdx.x < sh.parts * 16 && (threadIdx.x & 15) < heads) {
      const int i = threadIdx.x, p = i >> 4, h = i & 15;
      unsigned long long *pm = a.word_m + base + p * a.Hq + h, *pl = a.word_l + base + p * a.Hq + h;
      const unsigned long long vm = __hip_atomic_load(pm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const unsigned long long vl = __hip_atomic_load(pl, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_w[p][h] = taken(pm, vm);
      smem[i] = taken(pl, vl);
    }
    __syncthreads();
    if (threadIdx.x < heads) {
      const int h = threadIdx.x;
      float M = -INFINITY, L = 0.f;
      for (int p = 0; p < sh.parts; ++p) M = fmaxf(M, s_w[p][h]);
      for (int p = 0; p < sh.parts; ++p) {
        const float f = s_w[p][h] == -INFINITY ? 0.f : exp2_(s_w[p][h] - M);
        s_w[p][h] = f;
        L += f * smem[p * 16 + h];
      }
      s_sum[h] = L;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PAIRS; ++r) {
      const int i = threadIdx.x + T * r;
      if (i >= heads * D) continue;
      const int h = i / D, d = i % D;
      unsigned long long* const at = pair_word(r);
      float O = 0.f;
#pragma unroll
      for (int u = 0; u < PM_PARTS; ++u)
        if (u < sh.parts) O += s_w[u][h] * taken(at + u * next, w[r][u]);
      const float L = s_sum[h];
      store_elem<QD>(a.out, b * a.o_sb + (kv * a.g + h0 + h) * a.o_sh + d, L != 0.f ? O / L : 0.f);
    }
    if (threadIdx.x == 0)  // a replay of this launch counts from zero in the next round
      __hip_atomic_store(counter,
                         static_cast<unsigned long long>(counter_id(a.epoch)) << 32 |
                             static_cast<unsigned long long>((counter_round(seen, a.epoch) + 1) & 0xffffu) << 16,
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// ---- launches -------------------------------------------------------------------

struct PagesPlan {
  bool mfma, brief, pair;
  int G, head_chunks;
  int64_t splits, chunk;                 // general kernel
  int units, waves_units, subs;          // MFMA kernel
  int64_t target, min_tiles, slots;
};

template <int S, int QD, bool WINDOW>
static void launch_mfma_pages(const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  const int64_t waves = p.brief ? mfma_waves(a.D) : p.waves_units * p.subs, heads = p.pair || a.g > 16 ? 16 : a.g;
  const dim3 grid = p.brief ? dim3(static_cast<unsigned>(p.slots), static_cast<unsigned>(p.units), static_cast<unsigned>(a.B))
                            : dim3(static_cast<unsigned>(p.slots), static_cast<unsigned>(p.units / p.waves_units));
  const dim3 block(static_cast<unsigned>(64 * waves));
  // the waves' sums; a short request's joins need PM_PARTS x 16 floats of it
  int64_t bytes = !p.brief && p.subs == 1 ? 0 : waves * heads * (a.D + 4) * 4;
  if (p.brief && bytes < PM_PARTS * 16 * 4) bytes = PM_PARTS * 16 * 4;
  const unsigned smem = static_cast<unsigned>(bytes);
#define HS_PAGES_RUN(DIM, U, SHORT)                                                                   \
  do {                                                                                                \
    if constexpr (fp4(S) && DIM <= 128 && DIM != 96) {                                                \
      if (p.pair) hipLaunchKernelGGL((pages_mfma_kernel<S, QD, DIM, U, SHORT, WINDOW, true>), grid, block, smem, s, a); \
      else hipLaunchKernelGGL((pages_mfma_kernel<S, QD, DIM, U, SHORT, WINDOW>), grid, block, smem, s, a); \
    } else {                                                                                          \
      hipLaunchKernelGGL((pages_mfma_kernel<S, QD, DIM, U, SHORT, WINDOW>), grid, block, smem, s, a); \
    }                                                                                                 \
  } while (0)
#define HS_PAGES_D(DIM)                                         \
  do {                                                          \
    if (a.P % 16 == 0 && p.brief) HS_PAGES_RUN(DIM, true, true); \
    else if (a.P % 16 == 0) HS_PAGES_RUN(DIM, true, false);     \
    else if (p.brief) HS_PAGES_RUN(DIM, false, true);           \
    else HS_PAGES_RUN(DIM, false, false);                       \
  } while (0)
  if (a.D == 32) HS_PAGES_D(32);
  else if (a.D == 64) HS_PAGES_D(64);
  else if (a.D == 96) HS_PAGES_D(96);
  else if (S == HS_DTYPE_F32 || a.D == 128) HS_PAGES_D(128);
  else if constexpr (S != HS_DTYPE_F32) HS_PAGES_D(256);
#undef HS_PAGES_D
#undef HS_PAGES_RUN
}

// The matrix-core launch over a pool of element code S; WINDOW where a.window is one.
template <int S, bool WINDOW>
static void launch_mfma_pool(const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  if constexpr (quantised(S) || fp4(S)) {  // any query type
    if (a.q_dtype == HS_DTYPE_BF16) launch_mfma_pages<S, HS_DTYPE_BF16, WINDOW>(p, a, s);
    else if (a.q_dtype == HS_DTYPE_F16) launch_mfma_pages<S, HS_DTYPE_F16, WINDOW>(p, a, s);
    else launch_mfma_pages<S, HS_DTYPE_F32, WINDOW>(p, a, s);
  } else {
    launch_mfma_pages<S, S, WINDOW>(p, a, s);
  }
}

template <int S>
static void launch_general(const PagesPlan& p, const PagesArgs& a, bool vec, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.splits), static_cast<unsigned>(a.Hkv * p.head_chunks),
                  static_cast<unsigned>(a.B));
  const unsigned smem = static_cast<unsigned>(general_smem(p.G, a.D));
#define HS_PAGES_RUN(C, NC, G) \
  hipLaunchKernelGGL((pages_general_kernel<S, C, NC, G>), grid, dim3(PG_T), smem, s, a)
  if (p.G == 4) {
    if (vec && a.D <= 256) HS_PAGES_RUN(4, 1, 4);
    else if (vec) HS_PAGES_RUN(4, 2, 4);
    else HS_PAGES_RUN(1, 8, 4);
  } else {
    if (vec && a.D <= 256) HS_PAGES_RUN(4, 1, 2);
    else if (vec) HS_PAGES_RUN(4, 2, 2);
    else HS_PAGES_RUN(1, 8, 2);
  }
#undef HS_PAGES_RUN
}

// The launches of other files: whole histories in 4 bits (pages_fp4.hip; `vec`, for the vector-unit
// kernel), and windows, for which the vector-unit kernel has no forms of its own (pages_window.hip).
void launch_fp4_pages(const PagesPlan& p, const PagesArgs& a, bool vec, hipStream_t s);
void launch_window_pages(int pool_code, const PagesPlan& p, const PagesArgs& a, hipStream_t s);
void launch_fp4_window_pages(const PagesPlan& p, const PagesArgs& a, hipStream_t s);

}  // namespace hs
