// The attention over page tables (pages.hip) for 4-bit pools: the kernels of pages_kernels.h over e2m1
// codes with a scale byte for every 32 of the head dim.
#include "pages_kernels.h"

namespace hs {

void launch_fp4_pages(const PagesPlan& p, const PagesArgs& a, bool vec, hipStream_t s) {
  if (p.mfma) launch_mfma_pool<HS_DTYPE_E2M1, false>(p, a, s);
  else launch_general<HS_DTYPE_E2M1>(p, a, vec, s);
}

}  // namespace hs
