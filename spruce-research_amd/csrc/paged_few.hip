// Attention over a paged K/V cache: few rows a sequence.
#include "paged_impl.h"

namespace spruce {

int launch_paged_few(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st) {
  if (D == 128)
    return f16 ? launch_paged<FewBody<128, true>, 128, true>(p, n, st)
               : launch_paged<FewBody<128, false>, 128, false>(p, n, st);
  return f16 ? launch_paged<FewBody<64, true>, 64, true>(p, n, st)
             : launch_paged<FewBody<64, false>, 64, false>(p, n, st);
}

}  // namespace spruce
