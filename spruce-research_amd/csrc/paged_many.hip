// Attention over a paged K/V cache: many rows, pages of whole 64-key blocks.
#include "paged_impl.h"

namespace spruce {

int launch_paged_many(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st) {
  if (D == 128)
    return f16 ? launch_paged<ManyBody<128, true, true>, 128, true>(p, n, st)
               : launch_paged<ManyBody<128, false, true>, 128, false>(p, n, st);
  return f16 ? launch_paged<ManyBody<64, true, true>, 64, true>(p, n, st)
             : launch_paged<ManyBody<64, false, true>, 64, false>(p, n, st);
}

}  // namespace spruce
