// Attention over a paged K/V cache: many rows, other pages.
#include "paged_impl.h"

namespace spruce {

int launch_paged_scattered(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st) {
  if (D == 128)
    return f16 ? launch_paged<ManyBody<128, true, false>, 128, true>(p, n, st)
               : launch_paged<ManyBody<128, false, false>, 128, false>(p, n, st);
  return f16 ? launch_paged<ManyBody<64, true, false>, 64, true>(p, n, st)
             : launch_paged<ManyBody<64, false, false>, 64, false>(p, n, st);
}

}  // namespace spruce
