// Drafted trees: node positions, acceptance and the commit of accepted paths.  C entry points.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/emx_attn.h"
#include "entry.hpp"
#include "tree.hpp"

using namespace emx;

namespace {

// What the commits have in common, for layers [l0, l0 + layers).
int commit_args(int num_layers, const int32_t* const* block_tables, int32_t* const* kv_lens, int num_seqs,
                int max_blocks, int page_size, int num_blocks, const int32_t* slot_ids, int num_slots,
                const int32_t* path, const int32_t* accepted, const int32_t* qsl, int num_tokens, CommitArgs& a) {
  if (num_layers < 0 || num_slots < 0 || num_tokens < 0 || num_seqs < 0)
    return entry_fail(EMX_ERR_INVALID, "num_layers, num_slots, num_tokens and num_seqs must be >= 0");
  if (page_size <= 0 || num_blocks <= 0 || (max_blocks <= 0 && num_seqs > 0))
    return entry_fail(EMX_ERR_INVALID, "page_size, num_blocks and max_blocks_per_seq must be positive");
  if (!slot_ids && num_slots > num_seqs)
    return entry_fail(EMX_ERR_INVALID, "more trees than sequences");
  if ((long long)max_blocks * page_size >= (1LL << 31) || (long long)num_blocks * page_size >= (1LL << 31) ||
      num_slots > 65535)
    return entry_fail(EMX_ERR_UNSUPPORTED, "a table or pool of 2^31 tokens and more, or above 65535 trees");
  if (num_layers == 0 || num_slots == 0 || num_tokens == 0) return EMX_OK;
  if (!block_tables || !kv_lens || !path || !accepted || !qsl) return entry_fail(EMX_ERR_INVALID, "null pointer");
  for (int l = 0; l < num_layers; ++l)
    if (!block_tables[l] || !kv_lens[l]) return entry_fail(EMX_ERR_INVALID, "null pointer");
  a.slot_ids = slot_ids;
  a.path = path;
  a.accepted = accepted;
  a.qsl = qsl;
  a.n = num_slots;
  a.T = num_tokens;
  a.S = num_seqs;
  a.max_blocks = max_blocks;
  a.bs = page_size;
  a.nb = num_blocks;
  return EMX_OK;
}

// The lengths of every layer, each array once, after all moves.
int commit_lens(const CommitArgs& a, int num_layers, int32_t* const* kv_lens, hipStream_t st) {
  CommitLensArgs k{a.slot_ids, a.accepted, a.qsl, a.n, a.T, a.S, 0, {}};
  for (int l = 0; l < num_layers; ++l) {
    bool seen = false;
    for (int m = 0; m < l && !seen; ++m) seen = kv_lens[m] == kv_lens[l];
    if (!seen) k.kv_lens[k.layers++] = kv_lens[l];
    if (k.layers == kTreeLayers || (l + 1 == num_layers && k.layers > 0)) {
      hipLaunchKernelGGL(tree_commit_lens, dim3((unsigned)((a.n * k.layers + 255) / 256)), dim3(256), 0, st, k);
      if (int rc = entry_check_launch("tree_commit_lens")) return rc;
      k.layers = 0;
    }
  }
  return EMX_OK;
}

}  // namespace

extern "C" {

int emx_tree_positions(const int32_t* tree_parents, const int32_t* query_start_loc, int num_slots, int num_tokens,
                       int32_t* positions, void* stream) {
  if (num_slots < 0 || num_tokens < 0) return entry_fail(EMX_ERR_INVALID, "num_slots and num_tokens must be >= 0");
  if (num_slots == 0 || num_tokens == 0) return EMX_OK;
  if (!tree_parents || !query_start_loc || !positions) return entry_fail(EMX_ERR_INVALID, "null pointer");
  hipLaunchKernelGGL(tree_positions, dim3((unsigned)((num_tokens + 255) / 256)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), tree_parents, query_start_loc, num_slots, num_tokens,
                     positions);
  return entry_check_launch("tree_positions");
}

int emx_tree_accept(const void* tokens, const void* targets, int token_bytes, const int32_t* tree_parents,
                    const int32_t* query_start_loc, int num_slots, int num_tokens, int32_t* path, int32_t* accepted,
                    void* next_tokens, void* stream) {
  if (num_slots < 0 || num_tokens < 0) return entry_fail(EMX_ERR_INVALID, "num_slots and num_tokens must be >= 0");
  if (token_bytes != 4 && token_bytes != 8)
    return entry_fail(EMX_ERR_UNSUPPORTED, "tokens are 32-bit or 64-bit integers");
  if (num_slots == 0 && num_tokens == 0) return EMX_OK;
  if ((num_tokens > 0 && (!tokens || !targets || !tree_parents || !path)) ||
      (num_slots > 0 && (!query_start_loc || !accepted || !next_tokens)))
    return entry_fail(EMX_ERR_INVALID, "null pointer");
  const dim3 grid((unsigned)num_slots + 1);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (token_bytes == 4)
    hipLaunchKernelGGL(tree_accept<int32_t>, grid, dim3(64), 0, st, static_cast<const int32_t*>(tokens),
                       static_cast<const int32_t*>(targets), tree_parents, query_start_loc, num_slots, num_tokens,
                       path, accepted, static_cast<int32_t*>(next_tokens));
  else
    hipLaunchKernelGGL(tree_accept<int64_t>, grid, dim3(64), 0, st, static_cast<const int64_t*>(tokens),
                       static_cast<const int64_t*>(targets), tree_parents, query_start_loc, num_slots, num_tokens,
                       path, accepted, static_cast<int64_t*>(next_tokens));
  return entry_check_launch("tree_accept");
}

int emx_tree_commit_rows(int num_layers, void* const* key_caches, void* const* value_caches, int64_t row_bytes,
                         int page_size, int num_blocks, const int32_t* const* block_tables, int num_seqs,
                         int max_blocks_per_seq, int32_t* const* kv_lens, const int32_t* slot_ids, int num_slots,
                         const int32_t* path, const int32_t* accepted, const int32_t* query_start_loc, int num_tokens,
                         void* stream) {
  CommitRowArgs a{};
  if (int rc = commit_args(num_layers, block_tables, kv_lens, num_seqs, max_blocks_per_seq, page_size, num_blocks,
                           slot_ids, num_slots, path, accepted, query_start_loc, num_tokens, a.c))
    return rc;
  if (row_bytes <= 0 || row_bytes >= (1LL << 31)) return entry_fail(EMX_ERR_INVALID, "row_bytes must be positive");
  if (num_layers == 0 || num_slots == 0 || num_tokens == 0) return EMX_OK;
  if (!key_caches || !value_caches) return entry_fail(EMX_ERR_INVALID, "null cache pointer");
  uintptr_t bits = (uintptr_t)row_bytes;  // the piece that every row and cache is aligned to
  for (int l = 0; l < num_layers; ++l) {
    if (!key_caches[l] || !value_caches[l]) return entry_fail(EMX_ERR_INVALID, "null cache pointer");
    bits |= reinterpret_cast<uintptr_t>(key_caches[l]) | reinterpret_cast<uintptr_t>(value_caches[l]);
  }
  const int w = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  a.pieces = (int)(row_bytes / w);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int l0 = 0; l0 < num_layers; l0 += kTreeLayers) {
    const int n = std::min(kTreeLayers, num_layers - l0);
    for (int l = 0; l < n; ++l) {
      a.cache[l][0] = static_cast<char*>(key_caches[l0 + l]);
      a.cache[l][1] = static_cast<char*>(value_caches[l0 + l]);
      a.c.bt[l] = block_tables[l0 + l];
      a.c.kv_lens[l] = kv_lens[l0 + l];
    }
    const dim3 grid((unsigned)((a.pieces + 127) / 128), (unsigned)num_slots, (unsigned)(2 * n));
    if (w == 16)
      hipLaunchKernelGGL(tree_commit_rows<u32x4>, grid, dim3(128), 0, st, a);
    else if (w == 4)
      hipLaunchKernelGGL(tree_commit_rows<uint32_t>, grid, dim3(128), 0, st, a);
    else
      hipLaunchKernelGGL(tree_commit_rows<uint8_t>, grid, dim3(128), 0, st, a);
    if (int rc = entry_check_launch("tree_commit_rows")) return rc;
  }
  return commit_lens(a.c, num_layers, kv_lens, st);
}

int emx_tree_commit_affine(int num_layers, void* const* arrays, int num_kv_heads, int head_dim, int bits,
                           int group_size, int page_size, int num_blocks, const int32_t* const* block_tables,
                           int num_seqs, int max_blocks_per_seq, int32_t* const* kv_lens, const int32_t* slot_ids,
                           int num_slots, const int32_t* path, const int32_t* accepted,
                           const int32_t* query_start_loc, int num_tokens, void* stream) {
  CommitAffineArgs a{};
  if (int rc = commit_args(num_layers, block_tables, kv_lens, num_seqs, max_blocks_per_seq, page_size, num_blocks,
                           slot_ids, num_slots, path, accepted, query_start_loc, num_tokens, a.c))
    return rc;
  if (bits != 4 && bits != 8) return entry_fail(EMX_ERR_UNSUPPORTED, "bits must be 4 or 8");
  if (num_kv_heads <= 0 || head_dim <= 0 || group_size <= 0 || head_dim % group_size != 0)
    return entry_fail(EMX_ERR_INVALID, "head_dim must be a positive multiple of group_size");
  if ((head_dim * bits) % 32 != 0 || (page_size * bits) % 32 != 0)
    return entry_fail(EMX_ERR_INVALID, "head_dim * bits and page_size * bits must be multiples of 32");
  if (page_size > 256 / bits && page_size % (256 / bits) != 0)
    return entry_fail(EMX_ERR_INVALID, "page_size above 256/bits must be a multiple of 256/bits");
  if (num_layers == 0 || num_slots == 0 || num_tokens == 0) return EMX_OK;
  if (!arrays) return entry_fail(EMX_ERR_INVALID, "null cache pointer");
  for (int k = 0; k < 6 * num_layers; ++k)
    if (!arrays[k]) return entry_fail(EMX_ERR_INVALID, "null cache pointer");
  a.Hkv = num_kv_heads;
  a.D = head_dim;
  a.G = head_dim / group_size;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int l0 = 0; l0 < num_layers; l0 += kTreeLayers) {
    const int n = std::min(kTreeLayers, num_layers - l0);
    for (int l = 0; l < n; ++l) {
      for (int k = 0; k < 6; ++k) a.arr[l][k] = arrays[6 * (l0 + l) + k];
      a.c.bt[l] = block_tables[l0 + l];
      a.c.kv_lens[l] = kv_lens[l0 + l];
    }
    const dim3 grid((unsigned)num_kv_heads, (unsigned)num_slots, (unsigned)n);
    if (bits == 4)
      hipLaunchKernelGGL(tree_commit_affine<4>, grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL(tree_commit_affine<8>, grid, dim3(256), 0, st, a);
    if (int rc = entry_check_launch("tree_commit_affine")) return rc;
  }
  return commit_lens(a.c, num_layers, kv_lens, st);
}

}  // extern "C"
