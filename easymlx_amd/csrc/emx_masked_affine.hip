// Masked attention kernels over affine pages.
#include <hip/hip_runtime.h>

#include "masked_pick.hpp"

namespace emx {

// (64-wide heads have one group of 64)
template <int BITS>
static void pick(const MfmaCall& c, const MaskedArgs& a, const int cw, hipStream_t st) {
  if (c.gs == 64)
    launch_masked_kind<KvAffine<BITS, 64>>(a, c.D, cw, st);
  else if (c.D == 128)
    cw == 2 ? launch_masked_kernels<KvAffine<BITS, 128>, 128, 2, 2>(a, st)
            : launch_masked_kernels<KvAffine<BITS, 128>, 128, 2, 4>(a, st);
  else
    launch_masked_kernels<KvAffine<BITS, 128>, 256, 1, 4>(a, st);
}

void launch_masked_affine(const MfmaCall& c, const MaskedArgs& a, const int cw, hipStream_t st) {
  c.bits == 4 ? pick<4>(c, a, cw, st) : pick<8>(c, a, cw, st);
}

}  // namespace emx
