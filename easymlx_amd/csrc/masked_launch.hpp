// Paged attention whose rows see more, or less, than a causal run of keys: first tokens that
// stay visible beside a sliding window (sinks), trees of drafted tokens (emx_masked.hip, a
// translation unit of its own; called by its C entry points).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "mfma_launch.hpp"

namespace emx {

// What a row sees, beside the causal limit.  Query i of a sequence of kv_len keys and q query
// tokens stands at past + i, past = kv_len - q; a key stands at its position.  With `parents`
// the q tokens are a drafted tree: node i's place is past + depth(i), and of the keys from past
// on it sees its own and its ancestors'.  With a window, a key is seen when it stands less than
// `window` places before the query or below `sinks`.
struct MaskRule {
  const int32_t* parents;  // [T] node index within the row's own sequence, below the row's; else the row is a root
  int window;              // 0: none
  int sinks;               // tokens that stay visible (0 without a window)
};

// The parent of node i of the tree whose parents start at `par`; -1 for a root (an entry that is
// not the index of an earlier node).
__device__ __forceinline__ int parent_of(const int32_t* par, const int i) {
  const int p = par[i];
  return (unsigned)p < (unsigned)i ? p : -1;
}

// Whether key k is visible to query i (depth: of node i, used with a tree and a window).
__device__ __forceinline__ bool key_visible(const MaskRule& m, const int32_t* par, const int past, const int i,
                                            const int depth, const int k) {
  int place = k, at = past + i;
  if (par != nullptr) {
    at = past + depth;
    if (k >= past) {
      int cur = i, back = 0;
      while (cur > k - past) {
        cur = parent_of(par, cur);
        ++back;
      }
      if (cur != k - past) return false;
      place = at - back;
    }
  } else if (k > at) {
    return false;
  }
  return m.window <= 0 || place > at - m.window || place < m.sinks;
}

__device__ __forceinline__ int node_depth(const int32_t* par, int i) {
  int d = 0;
  while ((i = parent_of(par, i)) >= 0) ++d;
  return d;
}

struct MaskedArgs;  // masked_wide.hpp

// How a call is cut (sizes and types only).
struct MaskedShape {
  int cw, tokb;       // column waves of a workgroup (32 columns each), query tokens of a tile (0: not taken)
  long tiles;         // the most tiles per kv head
  int wgs;            // workgroups over which tiles are cut, 0: they are not
  size_t desc_bytes, part_bytes;
};
MaskedShape masked_shape(int T, int S, int Hq, int Hkv, int D, KvKind kind, bool cut);

// Single-token rows (c.qsl null) with a window and sinks > 0; buffers as launch_decode_mfma's (emx_masked_rows.hip).
void launch_masked_rows(const MfmaCall& c, int sinks, int* ws_cnt, float* partials, hipStream_t st);

void launch_masked_affine(const MfmaCall& c, const MaskedArgs& a, int cw, hipStream_t st);  // emx_masked_affine.hip

}  // namespace emx
