// Masked paged attention (masked_launch.hpp) for any head_dim <= 256, page size and cache type:
// the shapes outside masked_wide.hpp, fp32 among them.
//
// A workgroup per (token, kv_head, up to 16 query heads), its eight waves take every eighth of the
// row's 64-key blocks (those between the sinks and the window are left out): a key to a lane for the
// scores (with the lane's own walk up the tree where the block holds drafted nodes), then a dim to a
// lane for the values, the probabilities staged in LDS; the waves' sums are joined in order.  Keys that
// the row does not see are left out of both sums, so what they hold does not matter.  fp32 throughout;
// bound by the latency of loads of one value a lane: a tree of 25 nodes over 1556 keys, 32 / 8 heads, D
// 128, fp32 404 us (2522 on one wave with one load in flight), bf16 on pages of 12 465 (2666).
#pragma once

#include "common.hpp"
#include "masked_launch.hpp"
#include "paged_generic.hpp"

namespace emx {

constexpr int kGenericWaves = 8;

template <typename QT, typename KV>
__global__ __launch_bounds__(64 * kGenericWaves) void masked_generic(GenericArgs a, MaskRule mask, KV kv) {
  constexpr int MAXH = 16;
  constexpr int MAXD = 256;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int token = blockIdx.x;
  const int kvh = blockIdx.y;
  const int HG = a.Hq / a.Hkv;
  const int h0 = blockIdx.z * MAXH;
  const int nh = min(MAXH, HG - h0);
  const int D = a.D;
  const QT* q = reinterpret_cast<const QT*>(a.q);
  QT* out = reinterpret_cast<QT*>(a.out) + ((size_t)token * a.Hq + (size_t)kvh * HG + h0) * D;

  __shared__ float qs[MAXH][MAXD];  // the queries, then a wave's sums on their way to the first wave
  __shared__ float pw[kGenericWaves][MAXH][64];
  __shared__ float mls[2][MAXH];
  float(*ps)[64] = pw[wv];

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
    for (int e = tid; e < nh * D; e += 64 * kGenericWaves) from_f32(0.f, out + e);
    return;
  }
  const int32_t* par = mask.parents ? mask.parents + q0 : nullptr;
  const int depth = par && mask.window > 0 ? node_depth(par, i) : 0;
  const int start_k = mask.window > 0 ? max(0, past + (par ? depth : i) - mask.window + 1) : 0;

  for (int e = tid; e < nh * D; e += 64 * kGenericWaves) {
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

  // (a window's first key lies in or past `past` only for nodes deeper than it is wide)
  const int lo = min(start_k, max(past, 0)) / 64, sinkb = min((mask.sinks + 63) / 64, lo), nb = max_k / 64 + 1 - lo + sinkb;
  for (int j = wv; j < nb; j += kGenericWaves) {
    const int base = 64 * (j < sinkb ? j : lo + j - sinkb);
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
#pragma unroll 8
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
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wave's LDS is its own, and served in order)
    __builtin_amdgcn_wave_barrier();
    for (int t0 = 0; t0 < 64; t0 += 4) {
      const uint32_t some = (uint32_t)(live >> t0) & 15u;
      if (!some) continue;
#pragma unroll
      for (int e = 0; e < MAXD / 64; ++e) {
        const int d = lane + 64 * e;
        if (d < D) {
          float vd[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            vd[t] = 0.f;
            if ((some >> t) & 1u)
              vd[t] = kv.val(__builtin_amdgcn_readlane(blk, t0 + t), (base + t0 + t) % a.bs, kvh, d);
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < MAXH; ++h)
              if (h < nh && ((some >> t) & 1u)) acc[h][e] += ps[h][t0 + t] * vd[t];
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // ---- the waves that had a block hand their sums to the first, in order
  const int waves = min(kGenericWaves, nb);
  for (int w = 1; w < waves; ++w) {
    __syncthreads();
    if (wv == w) {
#pragma unroll
      for (int h = 0; h < MAXH; ++h) {
        if (h < nh) {
#pragma unroll
          for (int e = 0; e < MAXD / 64; ++e) qs[h][lane + 64 * e] = acc[h][e];
          if (lane == 0) {
            mls[0][h] = m[h];
            mls[1][h] = l[h];
          }
        }
      }
    }
    __syncthreads();
    if (wv == 0) {
#pragma unroll
      for (int h = 0; h < MAXH; ++h) {
        if (h < nh) {
          const float m1 = mls[0][h], l1 = mls[1][h], top = fmaxf(m[h], m1);
          // (a wave without a live key has m = -inf and zeros, one of NaN scores only a sum that is NaN)
          const float f0 = m[h] == -INFINITY ? (l[h] == 0.f ? 0.f : l[h]) : exp2f(m[h] - top);
          const float f1 = m1 == -INFINITY ? (l1 == 0.f ? 0.f : l1) : exp2f(m1 - top);
          l[h] = l[h] * f0 + l1 * f1;
          m[h] = top;
#pragma unroll
          for (int e = 0; e < MAXD / 64; ++e) acc[h][e] = acc[h][e] * f0 + qs[h][lane + 64 * e] * f1;
        }
      }
    }
  }
  if (wv != 0) return;

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
