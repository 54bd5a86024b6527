// Attention of one new token per request over a paged KV cache (page tables).
//
// Token t of request b sits in row t % P of block table[b][t / P] of a pool
// [blocks, 2, P, Hkv, D]; a table entry outside the pool (-1) is an absent page, whose
// tokens are masked.  The table may differ by KV head (each head's selected pages).  Per
// query head h with KV head h // g, over the request's first length[b] tokens:
//
//   out = sum_t e^(s_t - m) V_t / sum_t e^(s_t - m),  s_t = (K_t . q) D^-1/2,  m = max_t s_t,
//
// and 0 when no token is left.  The pool is plain (float32, float16, bfloat16) or
// quantised (codes with a float32 scale per row, plane and head): a K row's scale
// multiplies its score, a V row's its weight, so codes are never widened in memory.
//
// The cache is read once and everything else is small, so the kernels are bound by its
// bytes.  The token axis is split over workgroups; every split leaves its running
// (m, l, sum e^(s - m) V) in fp32 and `pages_merge_kernel` joins them.  Scores carry the
// factor log2(e), so every exponential is a power of two.
#include <math.h>

#include "codes.h"

namespace hs {

// Slots of a request's partials: [first, first + count).
struct SlotRange {
  int32_t first, count;
};

struct PagesArgs {
  const void* q;
  int64_t q_sb, q_sh;
  int q_dtype;
  const void* pool;
  const float* scales;  // quantised pools only
  int64_t P, Hkv, D, blocks;
  const int32_t* tables;
  int64_t t_sb, t_sk, pages;
  const int32_t* lengths;
  int64_t B, Hq, g;
  int head_chunks;
  int64_t splits, chunk;
  float scale;
  float *part_m, *part_l, *part_o;  // [slots, Hq], [slots, Hq], [slots, Hq, D]
  SlotRange* ranges;                // [B] written by the MFMA kernel; null: `splits` slots a request
  int units, waves_units, subs;     // MFMA kernel: (KV head, 16 heads) units, of a workgroup, waves of one
  int64_t target, min_tiles;
  int q_vec;
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

constexpr bool quantised(int S) { return S == HS_DTYPE_I8 || S == HS_DTYPE_E4M3; }

// C neighbouring pool elements as floats.
template <int S, int C>
__device__ __forceinline__ void load_pool(const void* pool, int64_t i, float (&x)[C]) {
  if constexpr (C == 1) {
    if constexpr (quantised(S)) x[0] = decode1<S>(static_cast<const unsigned char*>(pool)[i]);
    else x[0] = load_elem<S>(pool, i);
  } else {
    static_assert(C == 4, "one or four elements");
    if constexpr (quantised(S)) {
      decode4<S>(*reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(pool) + i), x);
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
// probabilities from LDS.  Both products run on the vector unit in fp32 throughout.
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
  const int64_t n = request_length(a, b), t0 = split * a.chunk;
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
    const int64_t t = base + lane;
    int64_t block = -1, within = 0;
    if (t < t1) {
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
    const int64_t at = (b * a.splits + split) * a.Hq + kv * a.g + h0 + h;
    if (d == 0) {
      a.part_m[at] = M;
      a.part_l[at] = L;
    }
    a.part_o[at * D + d] = O;
  }
}

// ---- the matrix-core kernel ---------------------------------------------------------------
// 8- and 16-bit pools with a head dim of 32, 64 or 128.  A wave owns one unit (a KV head and
// up to 16 of its query heads) and walks tiles of 32 tokens, with no shared memory:
//
//   S^T = K Q^T   A: K rows (lane (j, c): row c, 8 of the head dim), B: the heads' queries;
//                 lane (j, c) receives head c's scores of tokens 4j .. 4j+3 and 16 + those
//   O^T += V^T P  B: those eight scores' weights, held already where the product wants them;
//                 A: lane (j, c) the same eight tokens' V at dims (D/16) c .., so that a V row
//                 is one contiguous load of the 16 lanes of a group and the transpose is the
//                 pairing of two tokens in a register
//
// with (j, c) = (lane / 16, lane % 16).  Codes widen to bf16 in registers (exact); queries and
// weights go in as sums of bf16 parts: as many of the query as its type has significand (1
// for bf16, 2 for float16, 3 for float32) and of the weights two (2^-16 of a weight; three
// for float32 queries).  float16 pools use float16 products.  A tile's scales are one dword a
// lane, spread over the group by the broadcast of the multiply itself.
// The running maximum moves only when a score passes it by more than SLACK (the sums then
// hold weights up to 2^SLACK, no less precise): no cross-lane step in most tiles.

constexpr int PM_TILE = 32;
constexpr float PM_SLACK = 6.f;

template <int S>
constexpr int elem_size() { return S == HS_DTYPE_F32 ? 4 : (quantised(S) ? 1 : 2); }

// Parts of a query, and of a weight.
template <int S, int QD>
constexpr int query_parts() { return !quantised(S) ? 1 : (QD == HS_DTYPE_BF16 ? 1 : (QD == HS_DTYPE_F16 ? 2 : 3)); }
template <int S, int QD>
constexpr int weight_parts() { return quantised(S) && QD == HS_DTYPE_F32 ? 3 : 2; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two floats as a pair of 16-bit values, rounded to nearest.
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
  else return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}
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
__device__ __forceinline__ float group_lane(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x150 + N, 0xf, 0xf, true));
}

// BYTES bytes (2, 4, 8 or 16 a load) as words.
template <int BYTES>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (BYTES == 2) {
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

struct Share {
  int64_t b;
  int32_t slot, part, parts;  // this workgroup's slot; its part of the request's
};

// The request and part of workgroup w: every wave derives the same schedule from the lengths.
// Parts are of `per` tiles, the fewest for which all requests together need at most `target`
// workgroups (sum ceil(n_b / per) <= sum n_b / per + B); an empty request has one part.
__device__ __forceinline__ bool share_of(const PagesArgs& a, int32_t w, Share& out) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += 64)
    if (b0 + lane < a.B) total += (request_length(a, b0 + lane) + PM_TILE - 1) / PM_TILE;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(static_cast<long long>(total), off, 64);
  const int64_t room = a.target - (a.B < a.target / 2 ? a.B : a.target / 2);
  int64_t per = (total + room - 1) / room;
  if (per < a.min_tiles) per = a.min_tiles;
  int32_t before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += 64) {
    int32_t parts = 0;
    if (b0 + lane < a.B) {
      const int64_t tiles = (request_length(a, b0 + lane) + PM_TILE - 1) / PM_TILE;
      parts = tiles > per ? static_cast<int32_t>((tiles + per - 1) / per) : 1;
    }
    const int32_t through = before + wave_inclusive_sum(parts);
    const uint64_t owners = __ballot(through > w);
    if (owners) {
      const int src = __ffsll(static_cast<unsigned long long>(owners)) - 1;
      out.b = b0 + src;
      out.parts = __builtin_amdgcn_readlane(parts, src);
      out.part = w - (__builtin_amdgcn_readlane(through, src) - out.parts);
      out.slot = w;
      return true;
    }
    before = __builtin_amdgcn_readlane(through, 63);
  }
  return false;
}

template <int S, int QD, int D, bool UNIFORM>
__global__ __launch_bounds__(512) void pages_mfma_kernel(PagesArgs a) {
  constexpr bool F16 = S == HS_DTYPE_F16;
  constexpr int ES = elem_size<S>();
  constexpr int KK = D / 32;                 // products over the head dim
  constexpr int E = D / 16;                  // V elements of a lane and token
  constexpr int NQ = query_parts<S, QD>(), NP = weight_parts<S, QD>();
  constexpr int KROW = D / 4 * ES;           // K bytes of a lane and row
  constexpr int KL = KROW < 16 ? KROW : 16;  // a K load
  constexpr int KN = KROW / KL;
  constexpr int VB = E * ES;                 // V bytes of a lane and token: one load
  constexpr int VW = VB < 4 ? 1 : VB / 4;
  extern __shared__ __attribute__((aligned(16))) float smem[];
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  Share sh;
  if (!share_of(a, static_cast<int32_t>(blockIdx.x), sh)) return;  // the same for every wave
  const int64_t b = sh.b;
  if (sh.part == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.ranges[b] = SlotRange{sh.slot, sh.parts};
  const int unit = static_cast<int>(blockIdx.y) * a.waves_units + wave % a.waves_units;
  const int sub = wave / a.waves_units;
  const int64_t kv = unit / a.head_chunks;
  const int h0 = unit % a.head_chunks * 16;
  const int heads = static_cast<int>(a.g - h0 < 16 ? a.g - h0 : 16);
  const int32_t n = static_cast<int32_t>(request_length(a, b));
  const int32_t tiles = (n + PM_TILE - 1) / PM_TILE;
  const int32_t share = (tiles + sh.parts - 1) / sh.parts;
  const int32_t tile0 = sh.part * share;
  const int32_t tile1 = tile0 + share < tiles ? tile0 + share : tiles;
  const int32_t* table = a.tables + b * a.t_sb + kv * a.t_sk;
  const uint32_t P = static_cast<uint32_t>(a.P);
  const char* pool = static_cast<const char*>(a.pool);

  // Q fragments of head c: part, product kk, 8 of the head dim from d0(kk)
  auto d0_of = [&](int kk) { return ES == 1 && D >= 64 ? 64 * (kk >> 1) + 16 * j + 8 * (kk & 1) : 32 * kk + 8 * j; };
  u32x4 qf[NQ][KK];
  {
    const bool in = c < heads;
    const int64_t at = b * a.q_sb + (kv * a.g + h0 + (in ? c : 0)) * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      float x[8];
      if (QD != HS_DTYPE_F32 && a.q_vec) {
        uint32_t w[4];
        load_words<16>(static_cast<const char*>(a.q) + (at + d0_of(kk)) * 2, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = low16<QD == HS_DTYPE_F16>(w[i]);
          x[2 * i + 1] = high16<QD == HS_DTYPE_F16>(w[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_elem<QD>(a.q, at + d0_of(kk) + i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = in ? x[i] : 0.f;
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

  f32x4 acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  // A tile's registers: K, V and scales.  Loads of the next tile go out as soon as the
  // registers of this one are consumed.
  uint32_t kw[2][KN * KL / 4], vw[8][VW];
  float sc = 0.f;
  const int64_t row_bytes = a.Hkv * D * ES;
  const int64_t v_plane = static_cast<int64_t>(P) * row_bytes;
  // token of the scale this lane holds (lanes 0-7 of a group: keys, 8-15: values)
  const int s_token = 4 * j + (c & 3), s_half = (c >> 2) & 1;

  // One tile; bit t of `valid`: its token t counts.
  auto use_tile = [&](uint32_t valid, auto next_k, auto next_v) {
    float sct = sc;
    float s[8];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        u32x4 kf;
        if constexpr (quantised(S)) {
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
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * rt + i] = t[i];
    }
    next_k();
    const bool whole = valid == 0xffffffffu;
    if constexpr (quantised(S)) {
      if (!(valid >> (16 * s_half + s_token) & 1)) sct = 0.f;  // a row past the end may hold anything
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
      for (int e = 0; e < 8; ++e) {
        if (!(valid >> (16 * (e >> 2) + 4 * j + (e & 3)) & 1)) {
          s[e] = -INFINITY;
#pragma unroll
          for (int w = 0; w < VW; ++w) vw[e][w] = 0u;  // weight 0, but 0 * NaN is none
        }
      }
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e]);
    if (__any(top > m_run + PM_SLACK)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_new == -INFINITY ? 1.f : exp2_(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] = exp2_(s[e] - m_use);
      l_run += s[e];
    }
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
    u32x4 pf[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pf[q][i] = pack16<F16>(s[2 * i], s[2 * i + 1]);
        if (q + 1 < NP) {
          s[2 * i] -= low16<F16>(pf[q][i]);
          s[2 * i + 1] -= high16<F16>(pf[q][i]);
        }
      }
    }
    // V^T fragments: pairs of tokens (2i, 2i + 1) at one dim
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      u32x4 even, odd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (quantised(S)) {
          float x[4], y[4];
          const int shift = 8 * (e & 3);
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
        acc[e] = mfma_16x16x32<F16>(even, pf[q], acc[e]);
        acc[e + 1] = mfma_16x16x32<F16>(odd, pf[q], acc[e + 1]);
      }
    }
    next_v();
  };

  if constexpr (UNIFORM) {
    // Pages of a multiple of 16 rows: a tile's two halves lie in one page each.  The wave reads
    // the table for 32 of its tiles at once (lane l: half l), keeps the byte offsets in a
    // register and takes each tile's from there; tiles without a page are passed over.
    const int32_t mine = tile1 - tile0 > sub ? (tile1 - tile0 - sub + a.subs - 1) / a.subs : 0;  // tiles of this wave
    auto half_token = [&](int32_t batch) {  // first token of this lane's half in the batch
      return 32 * (tile0 + sub + (batch + (lane >> 1)) * a.subs) + 16 * (lane & 1);
    };
    auto fetch = [&](int32_t batch, int32_t& block) {
      const int32_t t = half_token(batch);
      const bool in = batch + (lane >> 1) < mine && t < n;
      block = table[in ? static_cast<uint32_t>(t) / P : 0u];
      if (!in) block = -1;
    };
    int32_t batch = 0, block, ahead;
    uint64_t present = 0;
    int64_t offset = 0;  // byte offset of the half's first K row of this KV head
    auto open = [&]() {  // the batch in `block` becomes current, the next one's table loads start
      const int32_t t = half_token(batch);
      const bool ok = block >= 0 && block < a.blocks;
      const uint32_t within = static_cast<uint32_t>(t) % P;
      offset = ok ? ((static_cast<int64_t>(block) * 2 * P + within) * a.Hkv + kv) * (D * ES) : 0;
      present = __ballot(ok);
      fetch(batch + 32, ahead);
    };
    uint32_t valid = 0;
    int64_t off0 = 0, off1 = 0;
    auto advance = [&]() {  // the next tile with a page; false at the end
      uint64_t tilebits = (present | present >> 1) & 0x5555555555555555ull;
      while (tilebits == 0) {
        batch += 32;
        if (batch >= mine) return false;
        block = ahead;
        open();
        tilebits = (present | present >> 1) & 0x5555555555555555ull;
      }
      const int at = __ffsll(static_cast<unsigned long long>(tilebits)) - 1;
      const int32_t t = 32 * (tile0 + sub + (batch + (at >> 1)) * a.subs);
      const int left = n - t;
      valid = left >= PM_TILE ? 0xffffffffu : (1u << left) - 1u;
      if (!(present >> at & 1)) valid &= 0xffff0000u;
      if (!(present >> at & 2)) valid &= 0x0000ffffu;
      const uint32_t lo = static_cast<uint32_t>(offset), hi = static_cast<uint32_t>(offset >> 32);
      off0 = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, at))) << 32 |
                                  static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, at)));
      off1 = static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, at + 1))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, at + 1)));
      present &= ~(3ull << at);
      return true;
    };
    const int64_t k_lane = c * row_bytes + j * KL, v_lane = v_plane + 4 * j * row_bytes + c * VB;
    auto load_k = [&]() {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
        for (int i = 0; i < KN; ++i) load_words<KL>(pool + (rt ? off1 : off0) + k_lane + 64 * i, &kw[rt][i * (KL / 4)]);
      }
      if constexpr (quantised(S)) {
        const int64_t row = (s_half ? off1 : off0) / D + (c >= 8 ? a.P * a.Hkv : 0);
        sc = a.scales[row + s_token * a.Hkv];
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) load_words<VB>(pool + (e < 4 ? off0 : off1) + v_lane + (e & 3) * row_bytes, vw[e]);
    };
    if (mine > 0) {
      fetch(0, block);
      open();
      if (advance()) {
        load_k();
        load_v();
        bool more = true;
        while (more) {
          const uint32_t now = valid;
          more = advance();  // past the end the offsets stay: the last tile is read again, unused
          use_tile(now, load_k, load_v);
        }
      }
    }
  } else {
    // Any page size: lanes 0-31 find their token's row (head vectors of K from the pool's
    // start), the others take it from them.  A masked token reads row 0.
    int32_t tile = tile0 + sub;
    int32_t ahead = 0;  // table entry of this lane's token, one tile ahead
    uint32_t within = 0;
    bool in = false;
    int64_t row = 0;
    uint32_t valid = 0;
    auto fetch = [&](int32_t i) {
      const int32_t t = PM_TILE * i + (lane & 31);
      in = i < tile1 && t < n;
      const uint32_t page = in ? static_cast<uint32_t>(t) / P : 0u;
      within = in ? static_cast<uint32_t>(t) - page * P : 0u;
      ahead = table[page];
    };
    auto advance = [&]() {
      const bool ok = in && ahead >= 0 && ahead < a.blocks;
      row = ok ? (static_cast<int64_t>(ahead) * 2 * P + within) * a.Hkv + kv : 0;
      valid = static_cast<uint32_t>(__ballot(ok));
      tile += a.subs;
      fetch(tile);
    };
    auto row_of = [&](int t) { return static_cast<int64_t>(__shfl(static_cast<long long>(row), t, 64)); };
    auto load_k = [&]() {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const char* p = pool + row_of(16 * rt + c) * (D * ES) + j * KL;
#pragma unroll
        for (int i = 0; i < KN; ++i) load_words<KL>(p + 64 * i, &kw[rt][i * (KL / 4)]);
      }
      if constexpr (quantised(S)) sc = a.scales[row_of(16 * s_half + s_token) + (c >= 8 ? a.P * a.Hkv : 0)];
    };
    auto load_v = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        load_words<VB>(pool + row_of(16 * (e >> 2) + 4 * j + (e & 3)) * (D * ES) + v_plane + c * VB, vw[e]);
    };
    if (tile < tile1) {
      fetch(tile);
      advance();
      load_k();
      load_v();
      int32_t left = (tile1 - tile0 - sub + a.subs - 1) / a.subs;
      while (left > 0) {
        const uint32_t now = valid;
        advance();  // past the end every token is masked and reads row 0
        use_tile(now, load_k, load_v);
        --left;
      }
    }
  }

  // the totals of a head over the four groups, then the waves of a unit, then the partial
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (l_run != l_run) m_run = 0.f;  // NaN scores set no maximum: keep the partial in the merge
  __shared__ float s_m[8][16], s_l[8][16];
  const int most = static_cast<int>(a.g < 16 ? a.g : 16);
  if (a.subs == 1) {
    if (c < heads) {
      const int64_t at = sh.slot * a.Hq + kv * a.g + h0 + c;
      if (j == 0) {
        a.part_m[at] = m_run;
        a.part_l[at] = l_run;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) a.part_o[at * D + E * (4 * j + i) + e] = acc[e][i];
      }
    }
    return;
  }
  if (c < heads) {
    if (j == 0) {
      s_m[wave][c] = m_run;
      s_l[wave][c] = l_run;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) smem[(wave * most + c) * D + E * (4 * j + i) + e] = acc[e][i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.waves_units * most * D; i += blockDim.x) {
    const int u = i / (most * D), h = i / D % most, d = i % D;
    const int un = static_cast<int>(blockIdx.y) * a.waves_units + u;
    const int first = un % a.head_chunks * 16;
    if (first + h >= a.g) continue;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = u; w < a.waves_units * a.subs; w += a.waves_units) M = fmaxf(M, s_m[w][h]);
    if (M != -INFINITY) {
      for (int w = u; w < a.waves_units * a.subs; w += a.waves_units) {
        const float f = s_m[w][h] == -INFINITY ? 0.f : exp2_(s_m[w][h] - M);
        L += f * s_l[w][h];
        O += f * smem[(w * most + h) * D + d];
      }
    }
    const int64_t at = sh.slot * a.Hq + un / a.head_chunks * a.g + first + h;
    if (d == 0) {
      a.part_m[at] = M;
      a.part_l[at] = L;
    }
    a.part_o[at * D + d] = O;
  }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a head's slots; 0 if all are empty.
__global__ __launch_bounds__(256) void pages_merge_kernel(PagesArgs a) {
  const int64_t h = blockIdx.x, b = blockIdx.y;
  SlotRange r{static_cast<int32_t>(b * a.splits), static_cast<int32_t>(a.splits)};
  if (a.ranges) r = a.ranges[b];
  const int64_t base = r.first * a.Hq + h;
  float M = -INFINITY;
  for (int s = 0; s < r.count; ++s) M = fmaxf(M, a.part_m[base + s * a.Hq]);
  for (int64_t d = threadIdx.x; d < a.D; d += blockDim.x) {
    float L = 0.f, O = 0.f;
    for (int s = 0; s < r.count; ++s) {
      const int64_t at = base + s * a.Hq;
      const float ms = a.part_m[at];
      if (ms == -INFINITY) continue;
      const float f = exp2_(ms - M);
      L += f * a.part_l[at];
      O += f * a.part_o[at * a.D + d];
    }
    store_any(a.out, b * a.o_sb + h * a.o_sh + d, L != 0.f ? O / L : 0.f, a.q_dtype);
  }
}

// ---- host side ----------------------------------------------------------------

struct PagesPlan {
  bool mfma;
  int G, head_chunks;
  int64_t splits, chunk;                 // general kernel
  int units, waves_units, subs;          // MFMA kernel
  int64_t target, min_tiles, slots;
};

static bool pages_mfma_shape(int code, int64_t D) { return code != HS_DTYPE_F32 && (D == 32 || D == 64 || D == 128); }

// Splits of the token axis: about 2048 workgroups, each with at least one tile per wave.
static PagesPlan plan_pages(bool mfma, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t tokens) {
  PagesPlan p{};
  const int64_t g = Hq / Hkv;
  p.mfma = mfma;
  if (mfma) {
    p.head_chunks = static_cast<int>((g + 15) / 16);
    p.units = static_cast<int>(Hkv * p.head_chunks);
    p.waves_units = 8;
    while (p.units % p.waves_units) --p.waves_units;
    p.subs = 8 / p.waves_units;
    const int64_t groups = p.units / p.waves_units;
    p.target = (512 + groups - 1) / groups;
    p.min_tiles = 2 * p.subs;
    const int64_t tiles = (tokens + PM_TILE - 1) / PM_TILE;
    const int64_t most = B * ((tiles + p.min_tiles - 1) / p.min_tiles);
    p.slots = most < p.target + B ? most : p.target + B;
    return p;
  }
  p.G = g <= 4 || D > 256 ? 4 : 8;
  p.head_chunks = static_cast<int>((g + p.G - 1) / p.G);
  const int64_t groups = B * Hkv * p.head_chunks;
  int64_t splits = (2048 + groups - 1) / groups;
  const int64_t cap = (tokens + PG_T - 1) / PG_T;
  if (splits > cap) splits = cap;
  if (splits < 1) splits = 1;
  p.chunk = ((tokens + splits - 1) / splits + PG_T - 1) / PG_T * PG_T;
  if (p.chunk < PG_T) p.chunk = PG_T;
  p.splits = (tokens + p.chunk - 1) / p.chunk;
  if (p.splits < 1) p.splits = 1;
  p.slots = B * p.splits;
  return p;
}

// Partials (m, l, o) of every slot and query head, and the requests' slot ranges.
static int64_t pages_workspace(const PagesPlan& p, int64_t B, int64_t Hq, int64_t D) {
  return p.slots * Hq * (D + 2) * 4 + B * static_cast<int64_t>(sizeof(SlotRange)) + 8;
}

template <int S, int QD>
static void launch_mfma_pages(const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.slots), static_cast<unsigned>(p.units / p.waves_units));
  const dim3 block(static_cast<unsigned>(64 * p.waves_units * p.subs));
  const int64_t heads = a.g < 16 ? a.g : 16;
  const unsigned smem = p.subs == 1 ? 0u : static_cast<unsigned>(p.waves_units * p.subs * heads * a.D * 4);
#define HS_PAGES_D(DIM)                                                                                       \
  do {                                                                                                        \
    if (a.P % 16 == 0) hipLaunchKernelGGL((pages_mfma_kernel<S, QD, DIM, true>), grid, block, smem, s, a);    \
    else hipLaunchKernelGGL((pages_mfma_kernel<S, QD, DIM, false>), grid, block, smem, s, a);                 \
  } while (0)
  if (a.D == 32) HS_PAGES_D(32);
  else if (a.D == 64) HS_PAGES_D(64);
  else HS_PAGES_D(128);
#undef HS_PAGES_D
}

template <int S>
static void launch_mfma_codes(const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  if (a.q_dtype == HS_DTYPE_BF16) launch_mfma_pages<S, HS_DTYPE_BF16>(p, a, s);
  else if (a.q_dtype == HS_DTYPE_F16) launch_mfma_pages<S, HS_DTYPE_F16>(p, a, s);
  else launch_mfma_pages<S, HS_DTYPE_F32>(p, a, s);
}

template <int S>
static void launch_general(const PagesPlan& p, const PagesArgs& a, bool vec, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.splits), static_cast<unsigned>(a.Hkv * p.head_chunks),
                  static_cast<unsigned>(a.B));
  const unsigned smem = static_cast<unsigned>(general_smem(p.G, a.D));
  if (p.G == 4) {
    if (vec && a.D <= 256) hipLaunchKernelGGL((pages_general_kernel<S, 4, 1, 4>), grid, dim3(PG_T), smem, s, a);
    else if (vec) hipLaunchKernelGGL((pages_general_kernel<S, 4, 2, 4>), grid, dim3(PG_T), smem, s, a);
    else hipLaunchKernelGGL((pages_general_kernel<S, 1, 8, 4>), grid, dim3(PG_T), smem, s, a);
  } else {
    if (vec) hipLaunchKernelGGL((pages_general_kernel<S, 4, 1, 8>), grid, dim3(PG_T), smem, s, a);
    else hipLaunchKernelGGL((pages_general_kernel<S, 1, 4, 8>), grid, dim3(PG_T), smem, s, a);
  }
}

static int64_t pool_elem_bytes(int code) { return code == HS_DTYPE_F32 ? 4 : (quantised(code) ? 1 : 2); }

static int check_pages(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                       int64_t pages) {
  HS_CHECK_ARG(batch >= 1 && heads >= 1 && kv_heads >= 1 && head_dim >= 1 && page_size >= 1 && pages >= 1,
               "page attention needs positive sizes");
  HS_CHECK_ARG(heads % kv_heads == 0, "query heads must be a multiple of KV heads");
  HS_CHECK_ARG(head_dim <= 512, "head_dim above 512 is not supported");
  HS_CHECK_ARG(batch <= 65535 && heads <= 65535, "at most 65535 requests and query heads per call");
  HS_CHECK_ARG(page_size <= 0x7fffffff && pages <= 0x7fffffff / page_size, "a table may name at most 2^31 - 1 tokens");
  return HS_OK;
}

}  // namespace hs

using namespace hs;

extern "C" int64_t hs_attend_pages_workspace_bytes(int32_t query_dtype, int32_t pool_code, int64_t batch,
                                                   int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                   int64_t page_size, int64_t pages) {
  if (check_pages(batch, heads, kv_heads, head_dim, page_size, pages)) return 256;
  // either kernel may run on it (a pool that is not 16-byte aligned goes to the general one)
  int64_t need = 0;
  for (const bool mfma : {false, true}) {
    if (mfma && !pages_mfma_shape(pool_code, head_dim)) continue;
    const int64_t bytes = pages_workspace(plan_pages(mfma, batch, heads, kv_heads, head_dim, pages * page_size), batch,
                                          heads, head_dim);
    need = bytes > need ? bytes : need;
  }
  return need;
}

extern "C" int hs_attend_pages(const void* query, int64_t q_stride_b, int64_t q_stride_h, int32_t query_dtype,
                               const void* pool, const float* scales, int32_t pool_code, int64_t blocks,
                               int64_t page_size, int64_t kv_heads, int64_t head_dim, const int32_t* tables,
                               int64_t t_stride_b, int64_t t_stride_k, int64_t pages, const int32_t* lengths,
                               int64_t batch, int64_t heads, void* out, int64_t o_stride_b, int64_t o_stride_h,
                               void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const int rc = check_pages(batch, heads, kv_heads, head_dim, page_size, pages);
  if (rc) return rc;
  HS_CHECK_ARG(valid_dtype(query_dtype), "invalid dtype code %d", query_dtype);
  HS_CHECK_ARG(valid_dtype(pool_code) || valid_code(pool_code), "invalid pool code %d", pool_code);
  HS_CHECK_ARG(valid_code(pool_code) || pool_code == query_dtype, "a plain pool needs a query of its own dtype");
  HS_CHECK_ARG(query && pool && tables && lengths && out, "null page attention pointer");
  HS_CHECK_ARG(valid_code(pool_code) == (scales != nullptr), "scales go with a quantised pool, and only with one");
  HS_CHECK_ARG(blocks >= 1 && blocks <= 0x7fffffff, "a pool has 1 to 2^31 - 1 blocks");
  const bool mfma = pages_mfma_shape(pool_code, head_dim) && reinterpret_cast<uintptr_t>(pool) % 16 == 0;
  const PagesPlan p = plan_pages(mfma, batch, heads, kv_heads, head_dim, pages * page_size);
  const int64_t need = pages_workspace(p, batch, heads, head_dim);
  HS_CHECK_ARG(workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0,
               "page attention workspace too small or unaligned: need %lld bytes", static_cast<long long>(need));
  PagesArgs a{};
  a.q = query;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_dtype = query_dtype;
  a.pool = pool;
  a.scales = scales;
  a.P = page_size;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.blocks = blocks;
  a.tables = tables;
  a.t_sb = t_stride_b;
  a.t_sk = t_stride_k;
  a.pages = pages;
  a.lengths = lengths;
  a.B = batch;
  a.Hq = heads;
  a.g = heads / kv_heads;
  a.head_chunks = p.head_chunks;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.scale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(head_dim)));
  a.part_m = static_cast<float*>(workspace);
  a.part_l = a.part_m + p.slots * heads;
  a.part_o = a.part_l + p.slots * heads;
  a.ranges = nullptr;
  a.out = out;
  a.o_sb = o_stride_b;
  a.o_sh = o_stride_h;
  if (p.mfma) {
    const uintptr_t end = reinterpret_cast<uintptr_t>(a.part_o + p.slots * heads * head_dim);
    a.ranges = reinterpret_cast<SlotRange*>((end + 7) / 8 * 8);
    a.units = p.units;
    a.waves_units = p.waves_units;
    a.subs = p.subs;
    a.target = p.target;
    a.min_tiles = p.min_tiles;
    a.q_vec = reinterpret_cast<uintptr_t>(query) % 16 == 0 && q_stride_b % 8 == 0 && q_stride_h % 8 == 0;
    switch (pool_code) {
      case HS_DTYPE_F16: launch_mfma_pages<HS_DTYPE_F16, HS_DTYPE_F16>(p, a, stream); break;
      case HS_DTYPE_BF16: launch_mfma_pages<HS_DTYPE_BF16, HS_DTYPE_BF16>(p, a, stream); break;
      case HS_DTYPE_I8: launch_mfma_codes<HS_DTYPE_I8>(p, a, stream); break;
      default: launch_mfma_codes<HS_DTYPE_E4M3>(p, a, stream); break;
    }
  } else {
    const bool vec = head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(pool) % (4 * pool_elem_bytes(pool_code)) == 0;
    switch (pool_code) {
      case HS_DTYPE_F32: launch_general<HS_DTYPE_F32>(p, a, vec, stream); break;
      case HS_DTYPE_F16: launch_general<HS_DTYPE_F16>(p, a, vec, stream); break;
      case HS_DTYPE_BF16: launch_general<HS_DTYPE_BF16>(p, a, vec, stream); break;
      case HS_DTYPE_I8: launch_general<HS_DTYPE_I8>(p, a, vec, stream); break;
      default: launch_general<HS_DTYPE_E4M3>(p, a, vec, stream); break;
    }
  }
  HS_CHECK_LAUNCH("page attention");
  const unsigned threads = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256);
  hipLaunchKernelGGL(pages_merge_kernel, dim3(static_cast<unsigned>(heads), static_cast<unsigned>(batch)),
                     dim3(threads), 0, stream, a);
  HS_CHECK_LAUNCH("page attention merge");
  return HS_OK;
}
