// Launches of masked_wide and masked_merge for one cache kind.
#pragma once

#include "masked_wide.hpp"

namespace emx {

template <class C, int D, int KW, int CW>
void launch_masked_kernels(const MaskedArgs& a, hipStream_t st) {
  const int tiles = a.tiles * a.d.Hkv;
  hipLaunchKernelGGL((masked_wide<C, D, KW, CW>), dim3((unsigned)(a.wgs > 0 ? a.wgs : tiles)),
                     dim3((WideCfg<C, D, KW, CW>::TH)), 0, st, a);
  if (a.wgs > 0) {
    const unsigned n = tiles < a.wgs ? tiles : a.wgs;
    if (n * CW <= 128)
      hipLaunchKernelGGL((masked_merge<C, D, CW, 1>), dim3(n, CW, D / 32), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((masked_merge<C, D, CW, 4>), dim3(n, CW, D > 128 ? D / 128 : 1), dim3(D < 128 ? 2 * D : 256), 0,
                         st, a);
  }
}

// cw: waves side by side over the columns, as masked_shape has it
template <class C>
void launch_masked_kind(const MaskedArgs& a, const int D, const int cw, hipStream_t st) {
  if (D == 64) {
    cw == 2 ? launch_masked_kernels<C, 64, 2, 2>(a, st) : launch_masked_kernels<C, 64, 1, 4>(a, st);
  } else if (D == 256) {
    launch_masked_kernels<C, 256, 1, 4>(a, st);
  } else if (cw == 2) {
    launch_masked_kernels<C, 128, 2, 2>(a, st);
  } else if constexpr (C::kAffine) {
    launch_masked_kernels<C, 128, 2, 4>(a, st);
  } else if constexpr (C::kFp8) {
    launch_masked_kernels<C, 128, 1, 4>(a, st);
  } else {
    cw == 8 ? launch_masked_kernels<C, 128, 1, 8>(a, st) : launch_masked_kernels<C, 128, 1, 4>(a, st);
  }
}

}  // namespace emx
