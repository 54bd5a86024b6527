// Decode projections with 4-bit weights: y[M, N] = x[M, K] . W[N, K]^T (+ bias[N]) with M <= 16,
// W[n, k] = code[n, k] * 2^(e[n, k / 32] - 127) (e2m1 codes, a scale byte for every 32 of a row).
//
// The weight is read once and is nearly all of the bytes, a quarter of a 16-bit weight's, so the
// kernel is a stream of W through v_mfma_f32_16x16x32_bf16 with 16 weight rows as the MFMA's M
// dimension and the token rows (padded) as its N dimension, as in gemm.hip.  W is laid out once
// (dense.QuantizedWeight): blocks of 16 rows x 128 k, a lane's 16 bytes one after another, so that
// a wave's load of a block is 1 KB of consecutive bytes and gives it four products' operands: lane
// (j, c) holds 32 neighbours in k, from 32 j on, of row c, which share one scale.  (The sum over k
// takes any order, so product i takes 8 of them, and x at the same k.)  A lane's scales of four
// blocks are one dword.  Two codes and their scale widen to a bf16 pair in one instruction, exactly;
// a float16 x goes in as the sum of two bf16 parts, which hold it exactly too.  Sums are fp32.
#include "codes.h"

namespace hs {

constexpr int F4_STEP = 128;  // k of a block
constexpr int F4_UNROLL = 4;  // blocks of a round: a dword of scales

struct Fp4GemmArgs {
  const unsigned short* x;
  int64_t x_stride;
  const unsigned char* tiles;   // [T][steps][64][16]
  const uint32_t* scales;       // [T][groups][64]
  int64_t N, K, T;
  int M, steps, groups;
  const unsigned short* bias;  // nullable
  void* out;
  int64_t out_stride;
};

__device__ __forceinline__ f32x4 fp4_mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight float16 as the sum of two bf16 (8 and then at most 3 significand bits: exact; an infinity keeps
// a finite second part, which an infinity less itself would not be).
__device__ __forceinline__ void split_f16x8(u32x4 v, u32x4 (&part)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo = f16_bits_to_f32(static_cast<unsigned short>(v[i])), hi = f16_bits_to_f32(static_cast<unsigned short>(v[i] >> 16));
    part[0][i] = pack16<false>(lo, hi);
    lo = __builtin_amdgcn_fmed3f(lo - __uint_as_float(part[0][i] << 16), -65504.f, 65504.f);
    hi = __builtin_amdgcn_fmed3f(hi - __uint_as_float(part[0][i] & 0xffff0000u), -65504.f, 65504.f);
    part[1][i] = pack16<false>(lo, hi);
  }
}

// A workgroup owns GT row tiles of 16; its NW waves take rounds of four blocks of k in turn, with all
// loads of a round out before its first product, and their sums meet in LDS.
template <int DT, int GT, int NW, bool NT>
__global__ __launch_bounds__(64 * NW) void fp4_gemm_kernel(Fp4GemmArgs a) {
  constexpr int U = F4_UNROLL;
  __shared__ float red[NW][16 * GT][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, j = lane >> 4;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * GT;
  const unsigned char* w[GT];
  const uint32_t* s[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const int64_t tile = t0 + t < a.T ? t0 + t : a.T - 1;  // a tile past the last reads it again; its rows are dropped
    w[t] = a.tiles + tile * a.steps * 1024 + lane * 16;
    s[t] = a.scales + tile * a.groups * 64 + lane;
  }
  const unsigned short* x = a.x + (c < a.M ? c : a.M - 1) * a.x_stride;
  const int K = static_cast<int>(a.K);
  f32x4 acc[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int g = wave; g < a.groups; g += NW) {
    u32x4 wf[U][GT], xf[U][4];
    uint32_t sc[GT];
#pragma unroll
    for (int t = 0; t < GT; ++t) sc[t] = s[t][g * 64];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int step = g * U + u < a.steps ? g * U + u : a.steps - 1;  // past the last: read again, unused
#pragma unroll
      for (int t = 0; t < GT; ++t) {
        const u32x4* at = reinterpret_cast<const u32x4*>(w[t] + static_cast<int64_t>(step) * 1024);
        wf[u][t] = NT ? __builtin_nontemporal_load(at) : *at;
      }
      const int k = F4_STEP * step + 32 * j;
#pragma unroll
      for (int i = 0; i < 4; ++i) xf[u][i] = *reinterpret_cast<const u32x4*>(x + (k < K ? k : 0) + 8 * i);
      if (k >= K) {  // the last block ends inside: its codes are 0 there, and so is x
#pragma unroll
        for (int i = 0; i < 4; ++i) xf[u][i] = u32x4{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g * U + u >= a.steps) break;  // the same for the wave
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 part[2];
        if constexpr (DT == HS_DTYPE_F16) split_f16x8(xf[u][i], part);
        else part[0] = xf[u][i];
#pragma unroll
        for (int t = 0; t < GT; ++t) {
          u32x4 wide;
          widen_fp4_bf16x8(wf[u][t][i], __uint_as_float(__builtin_amdgcn_alignbit(sc[t], sc[t], (8 * u + 9) & 31)), wide);
          acc[t] = fp4_mfma(wide, part[0], acc[t]);
          if constexpr (DT == HS_DTYPE_F16) acc[t] = fp4_mfma(wide, part[1], acc[t]);
        }
      }
    }
  }
  // lane (j, c) holds rows 4j .. 4j + 3 of token c; the waves' sums in wave order
#pragma unroll
  for (int t = 0; t < GT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][16 * t + 4 * j + i][c] = acc[t][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * GT * 16; i += 64 * NW) {
    const int r = i % (16 * GT), m = i / (16 * GT);
    const int64_t n = t0 * 16 + r;
    if (m >= a.M || n >= a.N) continue;
    float v = red[0][r][m];
#pragma unroll
    for (int q = 1; q < NW; ++q) v += red[q][r][m];
    if (a.bias) v += load_elem<DT>(a.bias, n);
    store_elem<DT>(a.out, m * a.out_stride + n, v);
  }
}

// The form for many rows of a K that eight waves hold in one round each (K <= 4096): one workgroup a CU
// keeps its waves' parts of x in registers and walks its share of the row tiles two at a time, the
// next two's loads out before this two's products.  The waves' sums meet in one of two LDS
// buffers, so that one barrier a turn, which waits for no load, is enough.
constexpr int F4_WAVES = 8;

template <int DT>
__global__ __launch_bounds__(64 * F4_WAVES) void fp4_gemm_walk_kernel(Fp4GemmArgs a) {
  constexpr int U = F4_UNROLL, PARTS = DT == HS_DTYPE_F16 ? 2 : 1;
  __shared__ float red[2][F4_WAVES][32][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane & 15, j = lane >> 4;
  const int64_t lo = a.T * blockIdx.x / gridDim.x, hi = a.T * (blockIdx.x + 1) / gridDim.x;
  const int busy = a.groups < F4_WAVES ? a.groups : F4_WAVES;  // waves with a part of K
  const int K = static_cast<int>(a.K), first = wave * U;
  // one turn's end: the waves' sums are in LDS, and the next turns' loads stay in flight
  auto finish = [&](int buffer, int64_t t) {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int r = threadIdx.x & 31, m = threadIdx.x >> 5;
    const int64_t n = t * 16 + r;
    if (m < a.M && n < hi * 16 && n < a.N) {
      float v = red[buffer][0][r][m];
      for (int q = 1; q < busy; ++q) v += red[buffer][q][r][m];
      if (a.bias) v += load_elem<DT>(a.bias, n);
      store_elem<DT>(a.out, m * a.out_stride + n, v);
    }
  };
  if (wave >= busy) {
    for (int64_t t = lo, buffer = 0; t < hi; t += 2, buffer ^= 1) finish(static_cast<int>(buffer), t);
    return;
  }
  struct Pair {
    u32x4 w[2][U];
    uint32_t sc[2];
  };
  auto load = [&](Pair& p, int64_t t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t tile = t + i < hi ? t + i : hi - 1;  // past the share: read again, dropped
      p.sc[i] = a.scales[(tile * a.groups + wave) * 64 + lane];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // past the last block: read again, where x is 0
        const int step = first + u < a.steps ? first + u : a.steps - 1;
        const u32x4* at = reinterpret_cast<const u32x4*>(a.tiles + (tile * a.steps + step) * 1024 + lane * 16);
        p.w[i][u] = __builtin_nontemporal_load(at);
      }
    }
  };
  u32x4 x[PARTS][U][4], raw[U][4];
  const unsigned short* row = a.x + (c < a.M ? c : a.M - 1) * a.x_stride;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = F4_STEP * (first + u) + 32 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[u][i] = *reinterpret_cast<const u32x4*>(row + (k < K ? k : 0) + 8 * i);
  }
  Pair one, two, three;
  load(one, lo);
  load(two, lo + 2);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool in = F4_STEP * (first + u) + 32 * j < K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 v = in ? raw[u][i] : u32x4{0u, 0u, 0u, 0u};
      if constexpr (DT == HS_DTYPE_F16) {
        u32x4 part[2];
        split_f16x8(v, part);
        x[0][u][i] = part[0];
        x[1][u][i] = part[1];
      } else {
        x[0][u][i] = v;
        // x is waited for here: a wait inside the loop would be one for younger loads too
        asm volatile("" : "+v"(x[0][u][i]));
      }
    }
  }
  auto turn = [&](const Pair& p, int buffer, int64_t t) {
    f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float scale = __uint_as_float(__builtin_amdgcn_alignbit(p.sc[i], p.sc[i], (8 * u + 9) & 31));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          u32x4 wide;
          widen_fp4_bf16x8(p.w[i][u][q], scale, wide);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) acc[i] = fp4_mfma(wide, x[part][u][q], acc[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[buffer][wave][16 * i + 4 * j + e][c] = acc[i][e];
    finish(buffer, t);
  };
  if constexpr (DT == HS_DTYPE_F16) {  // x takes twice the registers
    for (int64_t t = lo; t < hi; t += 4) {
      turn(one, 0, t);
      load(one, t + 4);
      if (t + 2 >= hi) break;
      turn(two, 1, t + 2);
      load(two, t + 6);
    }
  } else {
    int buffer = 0;
    for (int64_t t = lo; t < hi; t += 6) {
      load(three, t + 4);
      turn(one, buffer, t);
      if (t + 2 >= hi) break;
      load(one, t + 6);
      turn(two, buffer ^ 1, t + 2);
      if (t + 4 >= hi) break;
      load(two, t + 8);
      turn(three, buffer, t + 4);
      buffer ^= 1;
    }
  }
}

struct Fp4GemmPlan {
  int tiles, waves;
  bool stream, walk;
};

// Row tiles and waves of a workgroup (not by the token rows, so that a row's sums are the same in every
// batch).  Tiles share the reads of x, which at 16 token rows are four times a tile's own bytes, but
// a CU should have a workgroup.  us for 1 and for 16 token rows, one, two and four tiles in 8 waves:
// 3584 x 3584 3.95 4.41 5.33 and 5.8 6.3 7.6; 4608 x 3584 5.2 4.5 5.4 and 9.0 6.4 7.7; 8192 x 2048
// 4.2 4.0 4.7 and 6.4 5.0 5.8; 12288 x 4096 8.1 8.6 7.5 and 14.1 12.9 9.8.  Where several workgroups
// run on a CU in any case, those of four waves: four tiles of 55296 x 5120 in 8 waves 30.1 and 40.5,
// in 4 26.3 and 35.9.  The walk: 37888 x 3584 15.8 and 17.9, four tiles in four waves 14.7 and 19.4;
// 152064 x 3584 with 4 rows in float16 49.9 and 57.2; but 12288 x 4096 9.7 and 11.7, and where only
// two of its waves have a part of K, 151936 x 896, 19.5 and 21.4 (17.7 and 23.1 in four tiles).
static Fp4GemmPlan plan_fp4_gemm(int64_t T, int64_t groups) {
  Fp4GemmPlan p{};
  p.tiles = T > 512 ? 4 : (T > 256 ? 2 : 1);
  p.waves = T > 1024 ? 4 : 8;
  p.walk = T > 1024 && groups >= 4 && groups <= F4_WAVES;
  // a weight is read once per step: above the 4 MB of an XCD's L2 nothing of it is left for the next
  // (more than 1024 row tiles are always above: the forms for them have no other loads)
  p.stream = T * groups * 4096 > (4 << 20);
  return p;
}

template <int DT, int GT, int NW>
static void launch_fp4_gemm(const Fp4GemmPlan& p, const Fp4GemmArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.T + GT - 1) / GT));
  if constexpr (NW == 8) {
    if (!p.stream) {
      hipLaunchKernelGGL((fp4_gemm_kernel<DT, GT, NW, false>), grid, dim3(64 * NW), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((fp4_gemm_kernel<DT, GT, NW, true>), grid, dim3(64 * NW), 0, s, a);
}

template <int DT>
static void launch_fp4_gemm(const Fp4GemmPlan& p, const Fp4GemmArgs& a, hipStream_t s) {
  if (p.walk) {
    // one workgroup a CU; the plan gives each several tiles
    hipLaunchKernelGGL((fp4_gemm_walk_kernel<DT>), dim3(256), dim3(64 * F4_WAVES), 0, s, a);
    return;
  }
  if (p.tiles == 4) p.waves == 8 ? launch_fp4_gemm<DT, 4, 8>(p, a, s) : launch_fp4_gemm<DT, 4, 4>(p, a, s);
  else if (p.tiles == 2) launch_fp4_gemm<DT, 2, 8>(p, a, s);
  else launch_fp4_gemm<DT, 1, 8>(p, a, s);
}

}  // namespace hs

using namespace hs;

extern "C" int hs_skinny_gemm_fp4(const void* x, int64_t x_stride, const void* tiles, const void* scales, int64_t n,
                                  int64_t k, const void* bias, void* out, int64_t out_stride, int64_t rows, int32_t dtype,
                                  hipStream_t stream) {
  HS_CHECK_ARG(dtype == HS_DTYPE_BF16 || dtype == HS_DTYPE_F16, "4-bit projections take bf16 or f16 rows: dtype code %d", dtype);
  HS_CHECK_ARG(rows >= 1 && rows <= 16, "4-bit projections take 1 to 16 rows");
  // (n: the grid's threads stay below 2^32)
  HS_CHECK_ARG(n >= 1 && n <= (int64_t{1} << 28) && k >= 32 && k % 32 == 0 && k < (int64_t{1} << 30),
               "4-bit projections need n of 1 to 2^28 and k a multiple of 32 below 2^30");
  HS_CHECK_ARG(x && tiles && scales && out, "null 4-bit projection pointer");
  HS_CHECK_ARG(x_stride % 8 == 0 && (rows == 1 || x_stride >= k) && out_stride >= (rows == 1 ? 0 : n),
               "row strides below the width, or x rows not 16-byte aligned");
  HS_CHECK_ARG(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(tiles) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(scales) % 4 == 0,
               "4-bit projection operands must be aligned: x and tiles to 16 bytes, scales to 4");
  Fp4GemmArgs a{};
  a.x = static_cast<const unsigned short*>(x);
  a.x_stride = x_stride;
  a.tiles = static_cast<const unsigned char*>(tiles);
  a.scales = static_cast<const uint32_t*>(scales);
  a.N = n;
  a.K = k;
  a.T = (n + 15) / 16;
  a.M = static_cast<int>(rows);
  a.steps = static_cast<int>((k + F4_STEP - 1) / F4_STEP);
  a.groups = (a.steps + F4_UNROLL - 1) / F4_UNROLL;
  a.bias = static_cast<const unsigned short*>(bias);
  a.out = out;
  a.out_stride = out_stride;
  const Fp4GemmPlan p = plan_fp4_gemm(a.T, a.groups);
  if (dtype == HS_DTYPE_BF16) launch_fp4_gemm<HS_DTYPE_BF16>(p, a, stream);
  else launch_fp4_gemm<HS_DTYPE_F16>(p, a, stream);
  HS_CHECK_LAUNCH("skinny_gemm_fp4");
  return HS_OK;
}
