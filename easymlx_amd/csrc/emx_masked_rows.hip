// Single-token rows with sinks: decode_mfma over every cache kind.
#include <hip/hip_runtime.h>

#include "decode_mfma.hpp"
#include "masked_launch.hpp"

namespace emx {
namespace {

typedef void (*RowsFn)(DecodeMfmaArgs);

template <class C>
RowsFn pick(int D) {
  return D == 64 ? decode_mfma<C, 64, true> : D == 128 ? decode_mfma<C, 128, true> : decode_mfma<C, 256, true>;
}
template <int BITS>
RowsFn pick_affine(int D, int gs) {
  if (gs == 64) return pick<KvAffine<BITS, 64>>(D);
  return D == 128 ? decode_mfma<KvAffine<BITS, 128>, 128, true> : decode_mfma<KvAffine<BITS, 128>, 256, true>;
}

}  // namespace

void launch_masked_rows(const MfmaCall& c, const int sinks, int* ws_cnt, float* partials, hipStream_t st) {
  RowsFn fn = nullptr;
  switch (c.kind) {
    case KvKind::f16: fn = pick<KvF16>(c.D); break;
    case KvKind::bf16: fn = pick<KvBF16>(c.D); break;
    case KvKind::fp8: fn = pick<KvFp8>(c.D); break;
    case KvKind::affine: fn = c.bits == 4 ? pick_affine<4>(c.D, c.gs) : pick_affine<8>(c.D, c.gs); break;
  }
  DecodeMfmaArgs a = decode_mfma_args(c, ws_cnt, partials);
  a.sinks = sinks;
  hipLaunchKernelGGL(fn, dim3((unsigned)decode_mfma_wgs(c.D)), dim3(256), 0, st, a);
}

}  // namespace emx
