// Launches of masked_wide and masked_merge for one cache kind.
#pragma once

#include "masked_wide.hpp"

namespace emx {

template <class C, int D, int KW>
void launch_masked_kernels(const MaskedArgs& a, hipStream_t st) {
  const int tiles = a.tiles * a.d.Hkv;
  hipLaunchKernelGGL((masked_wide<C, D, KW>), dim3((unsigned)(a.wgs > 0 ? a.wgs : tiles)), dim3(256), 0, st, a);
  if (a.wgs > 0)
    hipLaunchKernelGGL((masked_merge<C, D, KW>), dim3((unsigned)tiles, 4 / KW, D / 32), dim3(256), 0, st, a);
}

template <class C>
void launch_masked_kind(const MaskedArgs& a, const int D, const int kw, hipStream_t st) {
  if (D == 64)
    kw == 1 ? launch_masked_kernels<C, 64, 1>(a, st) : launch_masked_kernels<C, 64, 2>(a, st);
  else if (D == 128)
    kw == 1 ? launch_masked_kernels<C, 128, 1>(a, st) : launch_masked_kernels<C, 128, 2>(a, st);
  else
    launch_masked_kernels<C, 256, 1>(a, st);
}

}  // namespace emx
