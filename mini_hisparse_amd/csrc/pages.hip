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
// bytes: 8 requests of 131072 tokens, 28 query and 4 KV heads of 128 in int8, 1.08 GB, take
// 183 .. 193 us and the join 5, 5.6 .. 5.9 TB/s where a plain read of 1 GiB runs at 6.07.  Small
// calls are bound by a chain of loads (length and table, page, K, V) and joins: 8.6 us for one
// request of 2000 tokens with 14 and 2 heads of 64, 0.5 MB.  The token axis is split over
// workgroups; every split leaves its running (m, l, sum e^(s - m) V) in fp32 and
// `pages_merge_kernel` joins them.  Scores carry the factor log2(e), so every exponential is a
// power of two.
#include "pages_kernels.h"

namespace hs {

// The same schedule for more requests, written out once: a workgroup's share (request -1: none)
// and the requests' slots.  One workgroup; 1024 requests at a time.  (Walked by every wave, 64
// lengths a step, it cost 16384 requests of 1 .. 1280 tokens 3033 us; they take 460 with this.)
constexpr int PS_T = 1024;

__global__ __launch_bounds__(PS_T) void pages_schedule_kernel(PagesArgs a, int64_t slots) {
  __shared__ int64_t s_tiles[PS_T / 64];
  __shared__ int32_t s_parts[2][PS_T / 64], s_count[PM_TRIES][PS_T / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t limit = a.pages * a.P;
  int64_t total = 0;
  for (int64_t b = threadIdx.x; b < a.B; b += PS_T) total += seen_tiles(clamp_length(a.lengths[b], limit), a.window, a.sinks);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(static_cast<long long>(total), off, 64);
  if (lane == 0) s_tiles[wave] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < PS_T / 64; ++w) total += s_tiles[w];
  const uint32_t least = static_cast<uint32_t>((total + a.target - 1) / a.target);
  const uint32_t sure = sure_size(total, sure_room(a.target, a.B)), min_tiles = static_cast<uint32_t>(a.min_tiles);
  uint32_t per = tried_size(sure, sure, 0, min_tiles);
  if (a.B <= a.target) {  // else every size gives more parts
    int32_t count[PM_TRIES] = {};
    for (int64_t b = threadIdx.x; b < a.B; b += PS_T) {
      const int32_t tiles = seen_tiles(clamp_length(a.lengths[b], limit), a.window, a.sinks);
#pragma unroll
      for (int k = 0; k < PM_TRIES; ++k) count[k] += parts_of(tiles, tried_size(least, sure, k, min_tiles));
    }
#pragma unroll
    for (int k = 0; k < PM_TRIES; ++k) {
      const int32_t all = scan_lanes(count[k]);
      if (lane == 63) s_count[k][wave] = all;
    }
    __syncthreads();
#pragma unroll
    for (int k = PM_TRIES - 1; k >= 0; --k) {
      int32_t all = 0;
#pragma unroll
      for (int w = 0; w < PS_T / 64; ++w) all += s_count[k][w];
      if (all <= a.target) per = tried_size(least, sure, k, min_tiles);
    }
  }
  int32_t before = 0;
  for (int64_t b0 = 0, turn = 0; b0 < a.B; b0 += PS_T, turn ^= 1) {
    const int64_t b = b0 + threadIdx.x;
    const int32_t n = b < a.B ? clamp_length(a.lengths[b], limit) : 0;
    const int32_t parts = b < a.B ? parts_of(seen_tiles(n, a.window, a.sinks), per) : 0;
    int32_t through = scan_lanes(parts);
    if (lane == 63) s_parts[turn][wave] = through;
    __syncthreads();  // the next turn writes the other half
    int32_t all = 0;
#pragma unroll
    for (int w = 0; w < PS_T / 64; ++w) {
      if (w == wave) through += before + all;
      all += s_parts[turn][w];
    }
    before += all;
    const int32_t first = through - parts;
    if (b < a.B) a.ranges[b] = SlotRange{first, parts};
    for (int32_t p = 0; p < parts; ++p) a.shares[first + p] = Slot{static_cast<int32_t>(b), p, parts, n};
  }
  for (int64_t w = before + threadIdx.x; w < slots; w += PS_T) a.shares[w] = Slot{-1, 0, 0, 0};
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a head's slots; 0 if all are empty.
// One workgroup per (query head, request; and 256 C of the head dim).  The slots' weights go to
// LDS, one slot a thread; then the sums: C elements a lane, 256 / (D / C) slots abreast and PJ_U of each in flight, so
// that a long history's slots are a few rounds of loads (one slot after another took 66 of
// 87 us at 128 slots of D = 64), joined over LDS in a fixed order.  Bound by its launch and two
// rounds of loads: 3.9 us for 4 requests of 14 heads of 64 in 61 slots each, 5.6 for 8 of 28 heads
// of 128 in 31.
constexpr int PJ_T = 256;
constexpr int PJ_U = 4;
constexpr int PJ_SLOTS = 1024;  // of a request, at most (plan_pages: as many splits, or `target` parts)

template <int C>
__global__ __launch_bounds__(PJ_T) void pages_merge_kernel(PagesArgs a) {
  __shared__ float s_w[PJ_SLOTS];
  __shared__ float s_part[PJ_T * C];
  __shared__ float s_red[PJ_T / 64];
  const int64_t h = blockIdx.x, b = blockIdx.y;
  const int D = static_cast<int>(a.D);
  SlotRange r{static_cast<int32_t>(b * a.splits), static_cast<int32_t>(a.splits)};
  if (a.ranges) r = a.ranges[b];
  const int64_t base = r.first * a.Hq + h;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto total = [&](float v, bool largest) {  // over the workgroup, in a fixed order
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float o = __shfl_xor(v, off, 64);
      v = largest ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if (lane == 0) s_red[wave] = v;
    __syncthreads();
    v = s_red[0];
#pragma unroll
    for (int w = 1; w < PJ_T / 64; ++w) v = largest ? fmaxf(v, s_red[w]) : v + s_red[w];
    return v;
  };
  float M = -INFINITY;
  for (int s = threadIdx.x; s < r.count; s += PJ_T) M = fmaxf(M, a.part_m[base + s * a.Hq]);
  M = total(M, true);
  const int columns = (D + C - 1) / C < PJ_T ? (D + C - 1) / C : PJ_T;  // lanes of a slot
  const int abreast = PJ_T / columns;
  const int g = threadIdx.x / columns, d = blockIdx.z * PJ_T * C + (threadIdx.x - g * columns) * C;
  float L = 0.f, O[C] = {};
  for (int s = threadIdx.x; s < r.count; s += PJ_T) {
    const int64_t at = base + s * a.Hq;
    const float m = a.part_m[at], l = a.part_l[at];
    const float w = m == -INFINITY ? 0.f : exp2_(m - M);
    s_w[s] = w;
    L += w * l;
  }
  __syncthreads();
  if (g < abreast && d < D) {
    for (int s = g; s < r.count; s += abreast * PJ_U) {
      float x[PJ_U][C];
#pragma unroll
      for (int u = 0; u < PJ_U; ++u) {
        const int at = s + u * abreast < r.count ? s + u * abreast : s;
        const float* p = a.part_o + (base + at * a.Hq) * D + d;
        if constexpr (C == 4) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] = v[e];
        } else {
          x[u][0] = *p;
        }
      }
#pragma unroll
      for (int u = 0; u < PJ_U; ++u) {
        const float w = s + u * abreast < r.count ? s_w[s + u * abreast] : 0.f;
#pragma unroll
        for (int e = 0; e < C; ++e) O[e] += w * x[u][e];
      }
    }
  }
  L = total(L, false);
#pragma unroll
  for (int e = 0; e < C; ++e) s_part[threadIdx.x * C + e] = O[e];
  __syncthreads();
  const int first = blockIdx.z * PJ_T * C;
  for (int i = threadIdx.x; i < columns * C && first + i < D; i += PJ_T) {
    float sum = 0.f;
    for (int u = 0; u < abreast; ++u) sum += s_part[u * columns * C + i];
    store_any(a.out, b * a.o_sb + h * a.o_sh + first + i, L != 0.f ? sum / L : 0.f, a.q_dtype);
  }
}

// ---- host side ----------------------------------------------------------------

// The MFMA kernel's shapes: its lane offsets within 16 rows are 32-bit.  (16 requests of 4096
// tokens, 32 query and 8 KV heads: of 96 on the vector unit 64.8 us in int8 and 78.5 in bf16, here
// 30.6 and 38.7; of 256 162 and 197, here 49 and 99; of 80, which the vector unit keeps, 51.5 in
// int8.  float32 rows of 256 would spill registers.)
static bool pages_mfma_shape(int64_t bits, int64_t Hkv, int64_t D) {
  return (D == 32 || D == 64 || D == 96 || D == 128 || (D == 256 && bits < 32)) && Hkv * D * bits < (int64_t{1} << 30);
}

// 4-bit pools whose KV heads share their tables may go two KV heads a unit where the products' 16 columns
// hold both's query heads.
static bool pages_pair_shape(int pool_code, int64_t Hq, int64_t Hkv, int64_t D) {
  return pool_code == HS_DTYPE_E2M1 && (D == 32 || D == 64 || D == 128) && Hkv % 2 == 0 && Hq / Hkv <= 8;
}

// `whole`: the general kernel takes a request in one split (the workspace was sized for a kernel
// that needs none).  `most`: tokens that the tables can name.
static PagesPlan plan_pages(bool mfma, bool pair, bool whole, int64_t bits, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                            int64_t most, int32_t window, int32_t sinks) {
  PagesPlan p{};
  const int64_t g = Hq / Hkv;
  p.mfma = mfma;
  if (mfma) {
    p.pair = pair;
    p.head_chunks = static_cast<int>((g + 15) / 16);
    p.units = static_cast<int>(pair ? Hkv / 2 : Hkv * p.head_chunks);
    const int64_t tiles = most_seen_tiles(most, window, sinks);
    // Short: as many parts of a request as give every CU a workgroup, 8 at most, of a tile for each
    // of its waves at least.  Taken while a wave has four tiles at most: us by this launch and by
    // the long one, 28 query and 4 KV heads of 128 in int8, for 1 request of 256, 1024 and 4096
    // tokens 7.2 11.2 14.0 and 13.5 13.9 14.6, for 16 of 1024, 4096 and 16384 13.3 21.0 62.7 and
    // 16.7 23.5 61.3.  The parts' join is one workgroup's work and loses above 16 of their words a
    // thread (16 heads of 128, 1 request of 512, 1024 and 2048 tokens, 8, 16 and 32 words: 8.7 13.3
    // 14.7 here, 12.8 12.9 13.0 in the long one; 4 heads of 256, 4 requests of 512 and 1024 tokens,
    // 16 and 32 words: 12.9 16.2 and 12.6 12.6).
    // A unit of at most 128 KiB stays one part (14 query and 2 KV heads of 64 in int8, 64 requests
    // of 1024 tokens: 10.4 in one part, 12.7 in two).
    // For windows and 4-bit pools both limits are a little wider: two tiles more, as a window begins and
    // its first tokens end inside a tile (16 windows of 4096, 28 and 4 heads of 128 in int8, 20.2 here and
    // 22.4 long), and one part of up to 288 KiB of head dims up to 64 (one window of 1024, 14 and 2
    // heads of 64 in bf16, 9.6 in one and 11.1 in eight; but of 28 and 4 heads of 128 in int8 11.3 and
    // 11.0, 1060 tokens of 40 and 8 heads of 128 in 4 bits 15.5 and 13.4).  Whole 4-bit histories
    // with and without the two, 64 and 256 of 1056 tokens: 14 and 2 heads of 64 8.1 10.4 and 10.6 26.7,
    // 40 and 8 of 128 18.5 69.8 and 29.1 85.7, but 8 and 8 of 64 15.2 51.3 and 19.3 47.8.
    const bool wider = bits == 4 || most_seen(most, window, sinks) < most;
    const int64_t W = mfma_waves(D), slack = wider ? 2 : 0, kib = wider && D <= 64 && tiles <= 4 * W + slack ? 288 : 128;
    const int64_t rows = pair ? 2 * g : (g < 16 ? g : 16), held = pair ? 2 * D : D;
    int64_t parts = 256 / (B * p.units);
    parts = parts < 1 || tiles * 2 * PM_TILE * held * bits <= kib * 1024 * 8 ? 1 : (parts > PM_PARTS ? PM_PARTS : parts);
    p.min_tiles = (tiles + parts - 1) / parts;
    if (p.min_tiles < W) p.min_tiles = W;
    p.slots = (tiles + p.min_tiles - 1) / p.min_tiles;
    p.brief = p.min_tiles <= 4 * W + slack && p.units <= 65535 && (p.slots == 1 || p.slots * rows * D < 16 * 64 * W);
    if (p.brief) return p;
    // Long: one workgroup a CU, over up to four units.  us at 4 histories of 32768
    // tokens, 14 query and 2 KV heads of 64 in bf16, for 256, 512 and 768 workgroups 20.4 21.4
    // 24.2; 28 and 4 heads of 128 in int8 32.5 38.9 45.4; 16 of 16384, 40 and 8 heads of 128 in
    // e4m3, with four units a workgroup 109, with eight 110, with one 192.
    p.waves_units = 4;
    while (p.units % p.waves_units) --p.waves_units;
    p.subs = static_cast<int>(W) / p.waves_units;
    const int64_t groups = p.units / p.waves_units;
    // Two of them for batches above a wave's lanes, whose ragged lengths then balance (28 and 4 heads
    // of 128 in int8, 256 requests of 1 .. 4096 tokens 162 us with one a CU, 137 with two, 136 with
    // three; 96 with 40 and 8 heads 120, 98, 98; 96 full ones of 4096 with 28 and 4 heads 90, 95, 101).
    p.target = ((B > PM_LANES ? 512 : 256) + groups - 1) / groups;
    p.min_tiles = p.subs;
    const int64_t sure = B * ((tiles + p.min_tiles - 1) / p.min_tiles);
    p.slots = sure < p.target + B ? sure : p.target + B;
    return p;
  }
  // Query heads of a workgroup: two where there are no more, or where four would leave CUs idle.
  // us with four and two, head dim 80 in int8: 16 requests of 4096 tokens, 8 KV heads of one, two
  // and four query heads each 54 54 57 and 47 47 75; 1 of 1024, four each, 22 and 17; 4 of 4096, 16
  // and 2 heads of 112, 26 and 22.  (Eight took 64 for 16 of 4096, 32 and 4 heads, four 56.)
  const int64_t tokens = most_seen(most, window, sinks), cap = (tokens + PG_T - 1) / PG_T;
  p.G = g <= 2 || B * Hkv * ((g + 3) / 4) * cap <= 256 ? 2 : 4;
  p.head_chunks = static_cast<int>((g + p.G - 1) / p.G);
  // Splits: about 1024 workgroups (16 requests of 16384 tokens, 32 and 8 heads of 80: 246 us with 768,
  // 194 with 1024, 272 with 1536, 197 with 2048), a split no shorter than a tile a wave.
  const int64_t groups = B * Hkv * p.head_chunks;
  int64_t splits = (1024 + groups - 1) / groups;
  if (splits > cap) splits = cap;
  if (whole || splits < 1) splits = 1;
  p.chunk = ((tokens + splits - 1) / splits + PG_T - 1) / PG_T * PG_T;
  if (p.chunk < PG_T) p.chunk = PG_T;
  p.splits = (tokens + p.chunk - 1) / p.chunk;
  if (p.splits < 1) p.splits = 1;
  p.slots = B * p.splits;
  return p;
}

// Whether a call whose KV heads could go in pairs goes one head a unit, by the plan for that: where the
// short launch then has at most a workgroup for every CU, pairs only halve their number, and a wave has
// both heads' work one after the other.  us in pairs and one by one, bf16 queries: 14 and 2 heads of 64,
// 1 request of 1000 tokens 8.6 7.5, 16 of 1 .. 4000 11.7 10.4, 256 of 1 .. 1000 (512 workgroups)
// 9.3 11.9; 28 and 4 heads of 128, 16 of 1 .. 1000 13.8 8.7, 64 of 1 .. 1000 15.7 10.8, 256 of
// 1 .. 1000 26.4 31.0; 40 and 8 heads, 1 of 4000 15.5 13.0, 64 of 1 .. 1000 16.0 20.4.  Not where the parts
// of a request are above four tiles a wave: 16 windows of 4096, 28 and 4 heads of 128, 17.8 and 19.9.
// (The long launch goes in pairs; some single requests would be faster one by one: of 16000 tokens,
// 40 and 8 heads of 128, 20.4 14.8; 28 and 4 heads 15.3 16.0; 64 of 1 .. 16000 tokens 66 73.)
static bool one_by_one(const PagesPlan& p, int64_t B, int64_t D) {
  return p.brief && B * p.units * p.slots <= 256 && (p.slots == 1 || p.min_tiles <= 4 * mfma_waves(D));
}

// Partials (m, l, o) of every slot and query head, the requests' slot ranges and the schedule.
static int64_t pages_workspace(const PagesPlan& p, int64_t B, int64_t Hq, int64_t D) {
  if (!p.mfma && p.splits == 1) return 0;
  if (p.mfma && p.brief) return p.slots == 1 ? 0 : (B * p.slots * Hq * (D + 2) + B * p.units) * 8;
  return p.slots * Hq * (D + 2) * 4 + B * static_cast<int64_t>(sizeof(SlotRange)) + 8 +
         (p.mfma && B > PM_LANES ? p.slots * static_cast<int64_t>(sizeof(Slot)) + 16 : 0);
}

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

static int check_window(int64_t window, int64_t sinks) {
  HS_CHECK_ARG(window >= 0 && sinks >= 0, "a window and its first tokens are not negative");
  HS_CHECK_ARG(window > 0 || sinks == 0, "first tokens that stay go with a window");
  return HS_OK;
}
// (a window of every token that the tables can name is none)
static int32_t window_of(int64_t window, int64_t tokens) {
  return window == 0 || window >= tokens ? NO_WINDOW : static_cast<int32_t>(window);
}
static int32_t sinks_of(int64_t sinks) { return clamp_length(sinks, NO_WINDOW); }

}  // namespace hs

using namespace hs;

extern "C" int64_t hs_attend_pages_window_workspace_bytes(int32_t query_dtype, int32_t pool_code, int64_t batch,
                                                          int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                          int64_t page_size, int64_t pages, int64_t window,
                                                          int64_t sinks) {
  if (check_pages(batch, heads, kv_heads, head_dim, page_size, pages) || check_window(window, sinks)) return 256;
  const int64_t bits = elem_bits(pool_code), tokens = pages * page_size;
  const int32_t newest = window_of(window, tokens), first = sinks_of(sinks);
  const bool shape = pages_mfma_shape(bits, kv_heads, head_dim);
  auto need_of = [&](bool mfma, bool pair, bool whole) {
    return pages_workspace(plan_pages(mfma, pair, whole, bits, batch, heads, kv_heads, head_dim, tokens, newest, first),
                           batch, heads, head_dim);
  };
  int64_t need = need_of(shape, false, false);
  if (!shape) return need;
  // a pool that is not aligned goes to the general kernel, and only tables that KV heads share to pairs
  const int64_t other = need_of(false, false, need == 0);
  if (other > need) need = other;
  const int64_t paired = pages_pair_shape(pool_code, heads, kv_heads, head_dim) ? need_of(true, true, false) : 0;
  return paired > need ? paired : need;
}

extern "C" int64_t hs_attend_pages_workspace_bytes(int32_t query_dtype, int32_t pool_code, int64_t batch,
                                                   int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                   int64_t page_size, int64_t pages) {
  return hs_attend_pages_window_workspace_bytes(query_dtype, pool_code, batch, heads, kv_heads, head_dim, page_size,
                                                pages, 0, 0);
}

extern "C" int hs_attend_pages(const void* query, int64_t q_stride_b, int64_t q_stride_h, int32_t query_dtype,
                               const void* pool, const void* scales, int32_t pool_code, int64_t blocks,
                               int64_t page_size, int64_t kv_heads, int64_t head_dim, const int32_t* tables,
                               int64_t t_stride_b, int64_t t_stride_k, int64_t pages, const int32_t* lengths,
                               int64_t batch, int64_t heads, void* out, int64_t o_stride_b, int64_t o_stride_h,
                               void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return hs_attend_pages_window(query, q_stride_b, q_stride_h, query_dtype, pool, scales, pool_code, blocks, page_size,
                                kv_heads, head_dim, tables, t_stride_b, t_stride_k, pages, lengths, batch, heads, 0, 0,
                                out, o_stride_b, o_stride_h, workspace, workspace_bytes, stream);
}

extern "C" int hs_attend_pages_window(const void* query, int64_t q_stride_b, int64_t q_stride_h, int32_t query_dtype,
                                      const void* pool, const void* scales, int32_t pool_code, int64_t blocks,
                                      int64_t page_size, int64_t kv_heads, int64_t head_dim, const int32_t* tables,
                                      int64_t t_stride_b, int64_t t_stride_k, int64_t pages, const int32_t* lengths,
                                      int64_t batch, int64_t heads, int64_t window, int64_t sinks, void* out,
                                      int64_t o_stride_b, int64_t o_stride_h, void* workspace, int64_t workspace_bytes,
                                      hipStream_t stream) {
  int rc = check_pages(batch, heads, kv_heads, head_dim, page_size, pages);
  if (rc == HS_OK) rc = check_window(window, sinks);
  if (rc) return rc;
  const bool quantised_pool = valid_code(pool_code) || pool_code == HS_DTYPE_E2M1;
  HS_CHECK_ARG(valid_dtype(query_dtype), "invalid dtype code %d", query_dtype);
  HS_CHECK_ARG(valid_dtype(pool_code) || quantised_pool, "invalid pool code %d", pool_code);
  HS_CHECK_ARG(quantised_pool || pool_code == query_dtype, "a plain pool needs a query of its own dtype");
  HS_CHECK_ARG(pool_code != HS_DTYPE_E2M1 || head_dim % FP4_GROUP == 0, "4-bit pools need a head_dim of a multiple of 32");
  HS_CHECK_ARG(query && pool && tables && lengths && out, "null page attention pointer");
  HS_CHECK_ARG(quantised_pool == (scales != nullptr), "scales go with a quantised pool, and only with one");
  HS_CHECK_ARG(blocks >= 1 && blocks <= 0x7fffffff, "a pool has 1 to 2^31 - 1 blocks");
  const int64_t bits = elem_bits(pool_code), tokens = pages * page_size;
  const int32_t newest = window_of(window, tokens), first = sinks_of(sinks);
  const bool shape = pages_mfma_shape(bits, kv_heads, head_dim);
  // (4-bit scales of 256 of the head dim are loaded eight at a time)
  const bool mfma = shape && reinterpret_cast<uintptr_t>(pool) % 16 == 0 &&
                    (pool_code != HS_DTYPE_E2M1 || reinterpret_cast<uintptr_t>(scales) % 8 == 0);
  PagesPlan p = plan_pages(shape, false, false, bits, batch, heads, kv_heads, head_dim, tokens, newest, first);
  if (mfma && t_stride_k == 0 && pages_pair_shape(pool_code, heads, kv_heads, head_dim) && !one_by_one(p, batch, head_dim))
    p = plan_pages(true, true, false, bits, batch, heads, kv_heads, head_dim, tokens, newest, first);
  if (shape && !mfma)
    p = plan_pages(false, false, pages_workspace(p, batch, heads, head_dim) == 0, bits, batch, heads, kv_heads, head_dim,
                   tokens, newest, first);
  HS_CHECK_ARG((p.mfma ? p.target : p.splits) <= PJ_SLOTS, "page attention plan with too many parts of a request");
  const int64_t need = pages_workspace(p, batch, heads, head_dim);
  HS_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                             (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "page attention workspace too small or unaligned: need %lld bytes", static_cast<long long>(need));
  PagesArgs a{};
  a.q = query;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_dtype = query_dtype;
  a.pool = pool;
  a.scales = static_cast<const float*>(scales);
  a.scale_bytes = static_cast<const unsigned char*>(scales);
  a.P = page_size;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.blocks = blocks;
  a.tables = tables;
  a.t_sb = t_stride_b;
  a.t_sk = t_stride_k;
  a.pages = pages;
  a.lengths = lengths;
  a.window = newest;
  a.sinks = first;
  a.B = batch;
  a.Hq = heads;
  a.g = heads / kv_heads;
  a.head_chunks = p.head_chunks;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.scale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(head_dim)));
  a.part_o = static_cast<float*>(workspace);
  a.part_m = a.part_o + p.slots * heads * head_dim;
  a.part_l = a.part_m + p.slots * heads;
  a.ranges = nullptr;
  a.out = out;
  a.o_sb = o_stride_b;
  a.o_sh = o_stride_h;
  if (p.mfma) {
    a.units = p.units;
    a.min_tiles = p.min_tiles;
    if (p.brief) {
      a.max_parts = static_cast<int>(p.slots);
      a.word_o = static_cast<unsigned long long*>(workspace);
      a.word_m = a.word_o + batch * p.slots * heads * head_dim;
      a.word_l = a.word_m + batch * p.slots * heads;
      a.arrivals = a.word_l + batch * p.slots * heads;
      a.epoch = next_epoch();
    } else {
      const uintptr_t end = reinterpret_cast<uintptr_t>(a.part_l + p.slots * heads);
      a.ranges = reinterpret_cast<SlotRange*>((end + 7) / 8 * 8);
      if (batch > PM_LANES) a.shares = reinterpret_cast<Slot*>((reinterpret_cast<uintptr_t>(a.ranges + batch) + 15) / 16 * 16);
      a.waves_units = p.waves_units;
      a.subs = p.subs;
      a.target = p.target;
    }
    a.o_vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && o_stride_b % 4 == 0 && o_stride_h % 4 == 0;
    a.q_vec = reinterpret_cast<uintptr_t>(query) % 16 == 0 && q_stride_b % 8 == 0 && q_stride_h % 8 == 0;
    if (a.shares) {
      hipLaunchKernelGGL(pages_schedule_kernel, dim3(1), dim3(PS_T), 0, stream, a, p.slots);
      HS_CHECK_LAUNCH("page attention schedule");
    }
    if (newest != NO_WINDOW) {
      launch_window_pages(pool_code, p, a, stream);
    } else {
      switch (pool_code) {
        case HS_DTYPE_F32: launch_mfma_pool<HS_DTYPE_F32, false>(p, a, stream); break;
        case HS_DTYPE_F16: launch_mfma_pool<HS_DTYPE_F16, false>(p, a, stream); break;
        case HS_DTYPE_BF16: launch_mfma_pool<HS_DTYPE_BF16, false>(p, a, stream); break;
        case HS_DTYPE_I8: launch_mfma_pool<HS_DTYPE_I8, false>(p, a, stream); break;
        case HS_DTYPE_E2M1: launch_fp4_pages(p, a, true, stream); break;
        default: launch_mfma_pool<HS_DTYPE_E4M3, false>(p, a, stream); break;
      }
    }
  } else {
    const bool vec = head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(pool) % (bits / 2) == 0;
    switch (pool_code) {
      case HS_DTYPE_F32: launch_general<HS_DTYPE_F32>(p, a, vec, stream); break;
      case HS_DTYPE_F16: launch_general<HS_DTYPE_F16>(p, a, vec, stream); break;
      case HS_DTYPE_BF16: launch_general<HS_DTYPE_BF16>(p, a, vec, stream); break;
      case HS_DTYPE_I8: launch_general<HS_DTYPE_I8>(p, a, vec, stream); break;
      case HS_DTYPE_E2M1: launch_fp4_pages(p, a, vec, stream); break;
      default: launch_general<HS_DTYPE_E4M3>(p, a, vec, stream); break;
    }
  }
  HS_CHECK_LAUNCH("page attention");
  if (p.mfma ? p.brief : p.splits == 1) return HS_OK;
  const int64_t columns = PJ_T * (head_dim % 4 == 0 ? 4 : 1);
  const dim3 joins(static_cast<unsigned>(heads), static_cast<unsigned>(batch),
                   static_cast<unsigned>((head_dim + columns - 1) / columns));
  if (head_dim % 4 == 0) hipLaunchKernelGGL(pages_merge_kernel<4>, joins, dim3(PJ_T), 0, stream, a);
  else hipLaunchKernelGGL(pages_merge_kernel<1>, joins, dim3(PJ_T), 0, stream, a);
  HS_CHECK_LAUNCH("page attention merge");
  return HS_OK;
}
