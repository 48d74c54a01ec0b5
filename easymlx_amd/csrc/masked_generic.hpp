// Masked paged attention (masked_launch.hpp) for any head_dim <= 256, page size and cache type:
// the shapes outside masked_wide.hpp, fp32 among them.
//
// One wavefront per (token, kv_head, up to 16 query heads), keys 64 at a time: a key to a lane
// for the scores (with the lane's own walk up the tree where the block holds drafted nodes), then
// a dim to a lane for the values, the probabilities staged in LDS.  Keys that the row does not see
// are left out of both sums, so what they hold does not matter.  Blocks between the sinks and the
// window are skipped.  fp32 throughout; bound by the vector unit (one key element feeds at most
// 16 heads).
#pragma once

#include "common.hpp"
#include "masked_launch.hpp"
#include "paged_generic.hpp"

namespace emx {

template <typename QT, typename KV>
__global__ __launch_bounds__(64) void masked_generic(GenericArgs a, MaskRule mask, KV kv) {
  constexpr int MAXH = 16;
  constexpr int MAXD = 256;
  const int lane = threadIdx.x;
  const int token = blockIdx.x;
  const int kvh = blockIdx.y;
  const int HG = a.Hq / a.Hkv;
  const int h0 = blockIdx.z * MAXH;
  const int nh = min(MAXH, HG - h0);
  const int D = a.D;
  const QT* q = reinterpret_cast<const QT*>(a.q);
  QT* out = reinterpret_cast<QT*>(a.out) + ((size_t)token * a.Hq + (size_t)kvh * HG + h0) * D;

  __shared__ float qs[MAXH][MAXD];
  __shared__ float ps[MAXH][64];

  // ---- the row's sequence (the largest s with qsl[s] <= token)
  int s = -1, q0 = token, q_len = 1;
  if (a.decode) {
    s = token < a.S ? token : -1;
  } else if (a.S > 0 && a.qsl[0] <= token) {
    int lo = 0, hi = a.S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.qsl[mid] <= token) lo = mid; else hi = mid;
    }
    q0 = a.qsl[lo];
    q_len = a.qsl[lo + 1] - q0;
    if (q0 >= 0 && token < q0 + q_len) s = lo;
  }
  const int kv_len = s >= 0 ? min(max(a.kv_lens[s], 0), a.max_blocks * a.bs) : 0;
  const int past = kv_len - q_len, i = token - q0;
  const int max_k = past + i;
  if (s < 0 || max_k < 0) {
    for (int e = lane; e < nh * D; e += 64) from_f32(0.f, out + e);
    return;
  }
  const int32_t* par = mask.parents ? mask.parents + q0 : nullptr;
  const int depth = par && mask.window > 0 ? node_depth(par, i) : 0;
  const int start_k = mask.window > 0 ? max(0, past + (par ? depth : i) - mask.window + 1) : 0;

  for (int e = lane; e < nh * D; e += 64) {
    const int h = e / D, d = e % D;
    qs[h][d] = to_f32(q[((size_t)token * a.Hq + (size_t)kvh * HG + h0 + h) * D + d]);
  }
  __syncthreads();

  float m[MAXH], l[MAXH], acc[MAXH][MAXD / 64];
#pragma unroll
  for (int h = 0; h < MAXH; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < MAXD / 64; ++e) acc[h][e] = 0.f;
  }
  const int32_t* bt = a.block_tables + (size_t)s * a.max_blocks;

  for (int base = 0; base <= max_k; base += 64) {
    // (a window's first key lies in or past `past` only for nodes deeper than it is wide)
    if (base >= mask.sinks && base + 64 <= min(start_k, max(past, 0))) {
      base = min(start_k, max(past, 0)) / 64 * 64 - 64;
      continue;
    }
    const int pos = base + lane;
    const int blk = pos <= max_k ? bt[pos / a.bs] : -1;
    const bool ok = (unsigned)blk < (unsigned)a.nb && key_visible(mask, par, past, i, depth, pos);
    const uint64_t live = __ballot(ok);
    if (live == 0) continue;
    float sc[MAXH];
#pragma unroll
    for (int h = 0; h < MAXH; ++h) sc[h] = 0.f;
    if (ok) {
      const int off = pos % a.bs;
      for (int d = 0; d < D; ++d) {
        const float kd = kv.key(blk, off, kvh, d);
#pragma unroll
        for (int h = 0; h < MAXH; ++h)
          if (h < nh) sc[h] += qs[h][d] * kd;
      }
    }
#pragma unroll
    for (int h = 0; h < MAXH; ++h) {
      if (h < nh) {
        const float x = ok ? sc[h] * a.scale_log2 : -INFINITY;
        const float m_new = fmaxf(m[h], wave_max(x));
        float p = 0.f, alpha = 1.f;
        if (m_new != -INFINITY) {
          p = ok ? exp2f(x - m_new) : 0.f;
          alpha = exp2f(m[h] - m_new);
        } else if (x != x) {
          p = x;
        }
        l[h] = l[h] * alpha + wave_sum(p);
        m[h] = m_new;
        ps[h][lane] = p;
#pragma unroll
        for (int e = 0; e < MAXD / 64; ++e) acc[h][e] *= alpha;
      }
    }
    __syncthreads();
    for (uint64_t todo = live; todo; todo &= todo - 1) {
      const int t = __builtin_ctzll(todo);
      const int b = __builtin_amdgcn_readlane(blk, t);
      const int off = (base + t) % a.bs;
#pragma unroll
      for (int e = 0; e < MAXD / 64; ++e) {
        const int d = lane + 64 * e;
        if (d < D) {
          const float vd = kv.val(b, off, kvh, d);
#pragma unroll
          for (int h = 0; h < MAXH; ++h)
            if (h < nh) acc[h][e] += ps[h][t] * vd;
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int h = 0; h < MAXH; ++h) {
    if (h < nh) {
      const float inv = l[h] > 0.f || l[h] != l[h] ? 1.f / l[h] : 0.f;
#pragma unroll
      for (int e = 0; e < MAXD / 64; ++e) {
        const int d = lane + 64 * e;
        if (d < D) from_f32(acc[h][e] * inv, out + (size_t)h * D + d);
      }
    }
  }
}

}  // namespace emx
