// Launches of masked_mfma and masked_merge for one cache kind.
#pragma once

#include "masked_mfma.hpp"

namespace emx {

template <class C, int D, int CT>
void launch_masked_kernels(const MaskedArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((masked_mfma<C, D, CT>), dim3((unsigned)(a.units * a.d.Hkv)), dim3(256), 0, st, a);
  if (a.share_of > 0)
    hipLaunchKernelGGL((masked_merge<C, D, CT>), dim3((unsigned)a.tiles, (unsigned)a.d.Hkv, CT), dim3(256), 0, st, a);
}

template <class C>
void launch_masked_kind(const MaskedArgs& a, const int D, const int ct, hipStream_t st) {
  if (D == 64)
    ct == 1 ? launch_masked_kernels<C, 64, 1>(a, st) : launch_masked_kernels<C, 64, 2>(a, st);
  else if (D == 128)
    ct == 1 ? launch_masked_kernels<C, 128, 1>(a, st) : launch_masked_kernels<C, 128, 2>(a, st);
  else
    launch_masked_kernels<C, 256, 1>(a, st);
}

}  // namespace emx
