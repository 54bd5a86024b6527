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
// (m, l, sum e^(s - m) V) in fp32 and `pages_merge_kernel` joins them.
#include <math.h>

#include "codes.h"

namespace hs {

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
  float *part_m, *part_l, *part_o;  // [B, Hq, splits], [B, Hq, splits], [B, Hq, splits, D]
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
      const float alpha = m_new == -INFINITY ? 1.f : __expf(m[h] - m_new);
      const float p = s == -INFINITY ? 0.f : __expf(s - m_new);  // a NaN score stays NaN
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
        const float f = s_m[w][h] == -INFINITY ? 0.f : __expf(s_m[w][h] - M);
        L += f * s_l[w][h];
        O += f * smem[(w * G + h) * D + d];
      }
    }
    const int64_t at = (b * a.Hq + kv * a.g + h0 + h) * a.splits + split;
    if (d == 0) {
      a.part_m[at] = M;
      a.part_l[at] = L;
    }
    a.part_o[at * D + d] = O;
  }
}

// out = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s over a head's splits; 0 if all are empty.
__global__ __launch_bounds__(256) void pages_merge_kernel(PagesArgs a) {
  const int64_t h = blockIdx.x, b = blockIdx.y;
  const int64_t base = (b * a.Hq + h) * a.splits;
  float M = -INFINITY;
  for (int64_t s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_m[base + s]);
  for (int64_t d = threadIdx.x; d < a.D; d += blockDim.x) {
    float L = 0.f, O = 0.f;
    for (int64_t s = 0; s < a.splits; ++s) {
      const float ms = a.part_m[base + s];
      if (ms == -INFINITY) continue;
      const float f = __expf(ms - M);
      L += f * a.part_l[base + s];
      O += f * a.part_o[(base + s) * a.D + d];
    }
    store_any(a.out, b * a.o_sb + h * a.o_sh + d, L != 0.f ? O / L : 0.f, a.q_dtype);
  }
}

// ---- host side ----------------------------------------------------------------

struct PagesPlan {
  int G, head_chunks;
  int64_t splits, chunk;
};

// Splits of the token axis: about 2048 workgroups, each with at least one tile per wave.
static PagesPlan plan_pages(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t tokens) {
  PagesPlan p{};
  const int64_t g = Hq / Hkv;
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
  return p;
}

static int64_t pages_workspace(const PagesPlan& p, int64_t B, int64_t Hq, int64_t D) {
  return B * Hq * p.splits * (D + 2) * 4;
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
  return pages_workspace(plan_pages(batch, heads, kv_heads, head_dim, pages * page_size), batch, heads, head_dim);
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
  const PagesPlan p = plan_pages(batch, heads, kv_heads, head_dim, pages * page_size);
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
  a.scale = 1.0f / sqrtf(static_cast<float>(head_dim));
  a.part_m = static_cast<float*>(workspace);
  a.part_l = a.part_m + batch * heads * p.splits;
  a.part_o = a.part_l + batch * heads * p.splits;
  a.out = out;
  a.o_sb = o_stride_b;
  a.o_sh = o_stride_h;
  const bool vec = head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(pool) % (4 * pool_elem_bytes(pool_code)) == 0;
  switch (pool_code) {
    case HS_DTYPE_F32: launch_general<HS_DTYPE_F32>(p, a, vec, stream); break;
    case HS_DTYPE_F16: launch_general<HS_DTYPE_F16>(p, a, vec, stream); break;
    case HS_DTYPE_BF16: launch_general<HS_DTYPE_BF16>(p, a, vec, stream); break;
    case HS_DTYPE_I8: launch_general<HS_DTYPE_I8>(p, a, vec, stream); break;
    default: launch_general<HS_DTYPE_E4M3>(p, a, vec, stream); break;
  }
  HS_CHECK_LAUNCH("page attention");
  const unsigned threads = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256);
  hipLaunchKernelGGL(pages_merge_kernel, dim3(static_cast<unsigned>(heads), static_cast<unsigned>(batch)),
                     dim3(threads), 0, stream, a);
  HS_CHECK_LAUNCH("page attention merge");
  return HS_OK;
}
