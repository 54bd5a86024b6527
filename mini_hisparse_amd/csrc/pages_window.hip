// The attention over page tables (pages.hip) through a window: the matrix-core kernels of
// pages_kernels.h that pass over the tiles between a request's first tokens and its newest.
#include "pages_kernels.h"

namespace hs {

void launch_window_pages(int pool_code, const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  switch (pool_code) {
    case HS_DTYPE_F32: launch_mfma_pool<HS_DTYPE_F32, true>(p, a, s); break;
    case HS_DTYPE_F16: launch_mfma_pool<HS_DTYPE_F16, true>(p, a, s); break;
    case HS_DTYPE_BF16: launch_mfma_pool<HS_DTYPE_BF16, true>(p, a, s); break;
    case HS_DTYPE_I8: launch_mfma_pool<HS_DTYPE_I8, true>(p, a, s); break;
    case HS_DTYPE_E2M1: launch_fp4_window_pages(p, a, s); break;
    default: launch_mfma_pool<HS_DTYPE_E4M3, true>(p, a, s); break;
  }
}

}  // namespace hs
