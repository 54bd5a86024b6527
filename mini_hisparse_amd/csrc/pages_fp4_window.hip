// pages_window.hip for 4-bit pools.
#include "pages_kernels.h"

namespace hs {

void launch_fp4_window_pages(const PagesPlan& p, const PagesArgs& a, hipStream_t s) {
  launch_mfma_pool<HS_DTYPE_E2M1, true>(p, a, s);
}

}  // namespace hs
