// The normed (or plain) rotary split of norm_rotary.h with K and V written to a paged pool on the way:
// q comes out, and no K or V is stored in between.  The pool is plain, of qkv's type, or quantised
// (quantized.hip), and then its codes are those of the fp32 values, which are rounded once.
// Bound by its bytes, or a short call by its chain of loads, table and stores: 16383 rows of 28 query
// and 4 KV heads of 128 in bf16 into int8, 285 MB, take 59 us, 4.8 TB/s; 16 rows into bf16 4 us.
#include "norm_rotary.h"

namespace hs {

template <int DT, int NE, bool VEC>
static void launch_rotary_append(int pool_code, dim3 grid, const NormRotaryArgs& a, hipStream_t s) {
#define HS_ROTARY_APPEND(POOL) hipLaunchKernelGGL((norm_rotary_split_kernel<DT, NE, VEC, POOL>), grid, dim3(DN_T), 0, s, a)
  if (pool_code == HS_DTYPE_I8) HS_ROTARY_APPEND(HS_DTYPE_I8);
  else if (pool_code == HS_DTYPE_E4M3) HS_ROTARY_APPEND(HS_DTYPE_E4M3);
  else if (pool_code == HS_DTYPE_E2M1) HS_ROTARY_APPEND(HS_DTYPE_E2M1);
  else HS_ROTARY_APPEND(DT);
#undef HS_ROTARY_APPEND
}

}  // namespace hs

using namespace hs;

extern "C" int hs_norm_rotary_append(const void* qkv, int64_t qkv_stride, const void* q_weight, const void* k_weight,
                                     float eps, void* q, const int64_t* positions, const int64_t* to_rows, int64_t rows,
                                     int64_t heads, double theta, int32_t dtype, void* pool, void* scales,
                                     int32_t pool_code, int64_t pool_rows, int64_t page_size, int64_t kv_heads,
                                     int64_t head_dim, hipStream_t stream) {
  const bool quantised = valid_code(pool_code) || pool_code == HS_DTYPE_E2M1;
  HS_CHECK_ARG(valid_dtype(dtype), "invalid dtype code %d", dtype);
  HS_CHECK_ARG(quantised || pool_code == dtype, "a plain pool holds the projection's dtype: pool code %d", pool_code);
  HS_CHECK_ARG(rows >= 0 && heads >= 1 && kv_heads >= 1 && head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 512 &&
                   page_size >= 1 && pool_rows >= 1,
               "invalid normed rotary append shape");
  HS_CHECK_ARG(pool_code != HS_DTYPE_E2M1 || head_dim % FP4_GROUP == 0, "4-bit rows need a head_dim of a multiple of 32");
  HS_CHECK_ARG(rows <= 0x7fffffff && heads <= 0xffff && kv_heads <= 0xffff, "too many rows or heads in one call");
  // a page's V rows lie past its K rows, and the kernel divides rows by a page size of at most the rows
  HS_CHECK_ARG(pool_rows % page_size == 0, "pool_rows must be those of whole pages");
  HS_CHECK_ARG(qkv_stride >= (heads + 2 * kv_heads) * head_dim, "q|k|v row stride below its width");
  HS_CHECK_ARG(pool != nullptr && quantised == (scales != nullptr), "scales go with a quantised pool, and only with one");
  HS_CHECK_ARG(!valid_code(pool_code) || reinterpret_cast<uintptr_t>(scales) % 4 == 0, "scales must be 4-byte aligned");
  HS_CHECK_ARG((q_weight == nullptr) == (k_weight == nullptr), "both norm weights, or none");
  HS_CHECK_ARG(theta > 0.0 && isfinite(theta) && (eps >= 0.f || !q_weight), "theta must be positive and eps not negative");
  if (rows == 0) return HS_OK;
  HS_CHECK_ARG(qkv && q && positions && to_rows, "null normed rotary append pointer");
  uintptr_t all = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_weight) |
                  reinterpret_cast<uintptr_t>(k_weight) | reinterpret_cast<uintptr_t>(q);
  if (!quantised) all |= reinterpret_cast<uintptr_t>(pool);
  const int half_bytes = quantised ? (pool_code == HS_DTYPE_E2M1 ? 1 : 2) : 0;
  const int ne = norm_rotary_pairs(dtype, head_dim / 2, qkv_stride, all, half_bytes, half_bytes ? reinterpret_cast<uintptr_t>(pool) : 0);
  NormRotaryArgs a{qkv, q_weight, k_weight, q, nullptr, nullptr, positions, qkv_stride, rows, heads, kv_heads,
                   log2(theta), eps, static_cast<int>(head_dim), 6, 1, to_rows, pool, scales, pool_rows, page_size};
  // element by element, 4-bit codes still share bytes: four neighbours a lane
  const dim3 grid = norm_rotary_grid(a, ne == 0 && pool_code == HS_DTYPE_E2M1 ? 4 : ne);
  HS_CHECK_ARG(grid.x < (int64_t{1} << 32) / DN_T, "too many rows in one call");
  if (dtype == HS_DTYPE_F32) {
    if (ne) launch_rotary_append<HS_DTYPE_F32, 4, true>(pool_code, grid, a, stream);
    else launch_rotary_append<HS_DTYPE_F32, 4, false>(pool_code, grid, a, stream);
  } else if (dtype == HS_DTYPE_BF16) {
    if (ne == 8) launch_rotary_append<HS_DTYPE_BF16, 8, true>(pool_code, grid, a, stream);
    else if (ne) launch_rotary_append<HS_DTYPE_BF16, 4, true>(pool_code, grid, a, stream);
    else launch_rotary_append<HS_DTYPE_BF16, 4, false>(pool_code, grid, a, stream);
  } else {
    if (ne == 8) launch_rotary_append<HS_DTYPE_F16, 8, true>(pool_code, grid, a, stream);
    else if (ne) launch_rotary_append<HS_DTYPE_F16, 4, true>(pool_code, grid, a, stream);
    else launch_rotary_append<HS_DTYPE_F16, 4, false>(pool_code, grid, a, stream);
  }
  HS_CHECK_LAUNCH("norm_rotary_append");
  return HS_OK;
}
