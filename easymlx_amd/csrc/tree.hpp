// Drafted trees beside the attention over them: the places of their nodes, the path that the
// target model agrees with, and the move of that path's rows to the front of the tree's place in
// the cache.
//
// A sequence's tree is the rows [query_start_loc[i], query_start_loc[i + 1]) of a call; parents[t] is
// the index, within its tree, of row t's parent: an earlier row, anything else makes a root.
#pragma once

#include "common.hpp"
#include "masked_launch.hpp"

namespace emx {

// The i in [0, n) with qsl[i] <= t < qsl[i + 1], -1 if none.
__device__ __forceinline__ int sequence_of(const int32_t* qsl, const int n, const int t) {
  if (n <= 0 || t < qsl[0] || t >= qsl[n]) return -1;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (qsl[mid] <= t) lo = mid;
    else hi = mid;
  }
  return t < qsl[lo + 1] ? lo : -1;
}

// positions[t], given as first + index (cache_slots), becomes first + depth: the position that node t has
// if its path is taken, by which it is rotated.  A thread to a node; bound by the latency of its walk.
__global__ __launch_bounds__(256) void tree_positions(const int32_t* parents, const int32_t* qsl, const int n,
                                                      const int T, int32_t* positions) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int s = sequence_of(qsl, n, t);
  if (s < 0) return;
  const int q0 = qsl[s];
  if (q0 < 0) return;
  positions[t] += node_depth(parents + q0, t - q0) - (t - q0);
}

// The accepted path of every tree: node 0 (the token that the model itself chose last), then of the last
// node's children the first whose token is the model's choice after that node, and so on.  path[q0 + k] is
// the k-th node (-1 past the path and in rows of no tree), accepted[s] their number, next[s] the model's
// choice after the last (-1 for an empty tree).
//
// One wave per tree, a node to a lane; every step is a comparison and a ballot over the nodes from the last
// one on, in registers for trees of up to 64 nodes.  Bound by its launch: 3 dependent loads, then some 20
// cycles per accepted node (one tree of 25: 1.5 us, 32 of up to 60: 3.6).
template <typename TT>
__global__ __launch_bounds__(64) void tree_accept(const TT* tokens, const TT* targets, const int32_t* parents,
                                                  const int32_t* qsl, const int n, const int T, int32_t* path,
                                                  int32_t* accepted, TT* next) {
  const int s = blockIdx.x, lane = threadIdx.x;
  if (s == n) {  // rows of no tree
    const int lo = n > 0 ? min(max(qsl[0], 0), T) : T, hi = n > 0 ? min(max(qsl[n], lo), T) : T;
    for (int t = lane; t < lo; t += 64) path[t] = -1;
    for (int t = hi + lane; t < T; t += 64) path[t] = -1;
    return;
  }
  const int q0 = qsl[s], q1 = min(qsl[s + 1], T), len = q0 < 0 ? 0 : q1 - q0;
  if (len <= 0) {
    if (lane == 0) {
      accepted[s] = 0;
      next[s] = (TT)-1;
    }
    return;
  }
  const int32_t* par = parents + q0;
  const TT *tok = tokens + q0, *tgt = targets + q0;
  // the first 64 nodes
  const int p0 = lane < len ? par[lane] : -1;
  const TT k0 = lane < len ? tok[lane] : 0;
  int count = 0, cur = 0;
  TT choice = tgt[0];
  int mine = -1;  // the path's node k at lane k % 64
  while (true) {
    if ((count & 63) == lane) mine = cur;
    ++count;
    if ((count & 63) == 0) path[q0 + count - 64 + lane] = mine;
    int found = -1;
    for (int base = (cur + 1) & ~63; base < len && found < 0; base += 64) {
      const int j = base + lane;
      const bool in = j > cur && j < len;
      const bool hit = base == 0 ? in && p0 == cur && k0 == choice : in && par[j] == cur && tok[j] == choice;
      const uint64_t b = __ballot(hit);
      if (b) found = base + __builtin_ctzll(b);
    }
    if (found < 0) break;
    cur = found;
    choice = tgt[cur];
  }
  for (int k = (count & ~63) + lane; k < len; k += 64) path[q0 + k] = k < count ? mine : -1;
  if (lane == 0) {
    accepted[s] = count;
    next[s] = choice;
  }
}

constexpr int kTreeLayers = 32;  // layers of one launch

// What the moves of all cache types have in common.
struct CommitArgs {
  const int32_t* slot_ids;  // [n] sequence of tree i; null: i
  const int32_t* path;      // [T]
  const int32_t* accepted;  // [n]
  const int32_t* qsl;       // [n + 1]
  int n, T, S, max_blocks, bs, nb;
  const int32_t* bt[kTreeLayers];
  int32_t* kv_lens[kTreeLayers];
};

// Tree i's place in layer l's cache.
struct TreePlace {
  const int32_t* bt;    // its sequence's row of the table
  const int32_t* path;  // its nodes
  int first, len, count;  // position of node 0, nodes, accepted nodes (0: nothing to move)
};

__device__ __forceinline__ TreePlace tree_place(const CommitArgs& a, const int i, const int l) {
  TreePlace p{};
  const int s = a.slot_ids ? a.slot_ids[i] : i;
  const int q0 = a.qsl[i], q1 = a.qsl[i + 1];
  if ((unsigned)s >= (unsigned)a.S || q0 < 0 || q1 > a.T || q1 <= q0) return p;
  p.bt = a.bt[l] + (size_t)s * a.max_blocks;
  p.path = a.path + q0;
  p.len = q1 - q0;
  p.first = a.kv_lens[l][s] - p.len;
  p.count = min(max(a.accepted[i], 0), p.len);
  return p;
}

// The rows of move k: page * bs + offset of its source and destination; false where nothing moves (the node is in
// its place, or a row lies outside the cache).
__device__ __forceinline__ bool tree_move(const CommitArgs& a, const TreePlace& p, const int k, int& src, int& dst) {
  const int node = p.path[k];
  if (node <= k || node >= p.len || p.first + k < 0) return false;
  const int ps = p.first + node, pd = p.first + k;
  const int cs = ps / a.bs, cd = pd / a.bs;
  if (cs >= a.max_blocks) return false;
  const int bs = p.bt[cs], bd = p.bt[cd];
  if ((unsigned)bs >= (unsigned)a.nb || (unsigned)bd >= (unsigned)a.nb) return false;
  src = bs * a.bs + ps % a.bs;
  dst = bd * a.bs + pd % a.bs;
  return true;
}

struct CommitRowArgs {
  CommitArgs c;
  char* cache[kTreeLayers][2];  // keys, values [nb, bs, row]
  int pieces;                   // of W per row
};

// Rows [Hkv, D] of a token-major cache.  Grid (chunks of a row, trees, 2 layers): a thread has one piece of the row
// and takes its moves in path order, eight loads ahead of their stores: a path ascends, so no store lands on the
// source of a later move, and no thread touches another's piece.  Bound by latency for one sequence (2 layers: 4.1 us), by
// the scattered rows' bandwidth for a batch (32 sequences, 32 layers, 61 MB read and written: 8 us, partly from cache).
template <typename W>
__global__ __launch_bounds__(128) void tree_commit_rows(CommitRowArgs a) {
  const int l = blockIdx.z >> 1;
  const TreePlace p = tree_place(a.c, blockIdx.y, l);
  const int e = blockIdx.x * 128 + threadIdx.x;
  if (e >= a.pieces) return;
  W* base = reinterpret_cast<W*>(a.cache[l][blockIdx.z & 1]) + e;
  for (int k0 = 0; k0 < p.count; k0 += 8) {
    W x[8];
    int dst[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int src = 0;
      dst[j] = -1;
      if (k0 + j < p.count && tree_move(a.c, p, k0 + j, src, dst[j])) x[j] = base[(size_t)src * a.pieces];
      else dst[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (dst[j] >= 0) base[(size_t)dst[j] * a.pieces] = x[j];
  }
}

struct CommitAffineArgs {
  CommitArgs c;
  void* arr[kTreeLayers][6];  // key codes, value codes, k_scales, k_biases, v_scales, v_biases
  int Hkv, D, G;
};

// One head's rows of affine pages.  Grid (Hkv, trees, layers).  A thread has one key word of the row, or one (array,
// group)'s scale or bias, or one dim of the values, whose codes sit in words that it shares with no other thread but
// with other tokens: the word that holds the destination is kept in a register over consecutive moves.
template <int BITS>
__global__ __launch_bounds__(256) void tree_commit_affine(CommitAffineArgs a) {
  constexpr int PW = 32 / BITS;
  constexpr uint32_t M = (1u << BITS) - 1u;
  const int h = blockIdx.x, l = blockIdx.z;
  const TreePlace p = tree_place(a.c, blockIdx.y, l);
  const int bs = a.c.bs, W = a.D / PW;
  for (int r = threadIdx.x; r < a.D + W + 4 * a.G; r += 256) {
    uint32_t* vc = static_cast<uint32_t*>(a.arr[l][1]);
    size_t held = ~(size_t)0;
    uint32_t word = 0;
    for (int k0 = 0; k0 < p.count; k0 += 8) {
      uint32_t x[8];
      int dst[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int src = 0;
        dst[j] = -1;
        if (k0 + j >= p.count || !tree_move(a.c, p, k0 + j, src, dst[j])) {
          dst[j] = -1;
          continue;
        }
        const size_t ph = (size_t)(src / bs) * a.Hkv + h;
        const int off = src % bs;
        if (r < a.D) {
          const size_t w = v_word_index<BITS>(ph, off, r, a.D, bs);
          // (a code of the word in the register is not in memory yet)
          x[j] = ((w == held ? word : vc[w]) >> v_shift<BITS>(off % PW)) & M;
        } else if (r < a.D + W) {
          x[j] = static_cast<const uint32_t*>(a.arr[l][0])[(ph * bs + off) * W + r - a.D];
        } else {
          const int q = r - a.D - W;
          x[j] = static_cast<const uint16_t*>(a.arr[l][2 + q / a.G])[(ph * a.G + q % a.G) * bs + off];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (dst[j] < 0) continue;
        const size_t ph = (size_t)(dst[j] / bs) * a.Hkv + h;
        const int off = dst[j] % bs;
        if (r < a.D) {
          const size_t w = v_word_index<BITS>(ph, off, r, a.D, bs);
          if (w != held) {
            if (held != ~(size_t)0) vc[held] = word;
            held = w;
            word = vc[w];
          }
          const int sh = v_shift<BITS>(off % PW);
          word = (word & ~(M << sh)) | (x[j] << sh);
        } else if (r < a.D + W) {
          static_cast<uint32_t*>(a.arr[l][0])[(ph * bs + off) * W + r - a.D] = x[j];
        } else {
          const int q = r - a.D - W;
          static_cast<uint16_t*>(a.arr[l][2 + q / a.G])[(ph * a.G + q % a.G) * bs + off] = (uint16_t)x[j];
        }
      }
    }
    if (held != ~(size_t)0) vc[held] = word;
  }
}

struct CommitLensArgs {
  const int32_t *slot_ids, *accepted, *qsl;
  int n, T, S, layers;
  int32_t* kv_lens[kTreeLayers];  // distinct
};

// kv_len - nodes + accepted, after the moves of every layer.
__global__ __launch_bounds__(256) void tree_commit_lens(CommitLensArgs a) {
  const int e = blockIdx.x * 256 + threadIdx.x, i = e / a.layers, l = e % a.layers;
  if (i >= a.n) return;
  const int s = a.slot_ids ? a.slot_ids[i] : i;
  const int q0 = a.qsl[i], q1 = a.qsl[i + 1];
  if ((unsigned)s >= (unsigned)a.S || q0 < 0 || q1 > a.T || q1 <= q0) return;
  a.kv_lens[l][s] += min(max(a.accepted[i], 0), q1 - q0) - (q1 - q0);
}

}  // namespace emx
