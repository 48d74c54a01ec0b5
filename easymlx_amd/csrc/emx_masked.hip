// Masked paged attention: the C entry points, and the kernels over unquantized and FP8 caches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/emx_attn.h"
#include "entry.hpp"
#include "masked_generic.hpp"
#include "masked_pick.hpp"

namespace emx {

// Workgroups that the chip holds at once, two to a compute unit; a call of fewer tiles is cut.
constexpr int kMaskedWGs = 512;

constexpr int kMaskedHeads = 128;  // query heads of a kv head: a tile's columns

MaskedShape masked_shape(int T, int S, int Hq, int Hkv, int D, KvKind kind, bool cut) {
  MaskedShape m{};
  const int hg = Hq / Hkv;
  if (hg <= 0 || hg > kMaskedHeads || T <= 0 || S <= 0) return m;
  const bool plain = kind == KvKind::f16 || kind == KvKind::bf16;
  const long cols = (long)T * hg;  // query columns of all sequences, per kv head
  // Sequences of up to 64 columns on average (small trees): two waves to a column, half of the keys each.  Else, where tiles
  // are few, 256 columns: each block of the cache is read half as often (12 trees of 48 to 64 nodes, 64 / 8 heads, up to
  // 32768 keys: 745 us against 896; 8 of 31 to 60, 32 / 8 heads: 73 against 80); where they are many, 128: two workgroups to
  // a compute unit, one begins a tile while the other multiplies (four prompts, window 1024: 252 us against 262).
  m.cw = D <= 128 && hg <= 64 && cols <= 64L * S ? 2 : 4;
  if (plain && D == 128 && m.cw == 4 && cols > 128L * S && cols * Hkv < 256L * kMaskedWGs) m.cw = 8;
  m.tokb = 32 * m.cw / hg;
  // a sequence of q query tokens has at most q / tokb + 1 tiles
  const long least = ((long)T + m.tokb - 1) / m.tokb;
  m.tiles = least + std::min(S, T);
  // (of 512 threads: one to a compute unit)
  const int wgs = D == 256 || m.cw == 8 || (D == 128 && m.cw == 4 && kind == KvKind::affine) ? kMaskedWGs / 2 : kMaskedWGs;
  if (cut && least * Hkv < 2 * wgs) {
    m.wgs = wgs;
    m.desc_bytes = 16 * (size_t)(1 + std::min<long>(m.tiles * Hkv, wgs));
    m.part_bytes = 2 * (size_t)m.wgs * m.cw * (D / 8 + 1) * 1024;
  }
  return m;
}

namespace {

// Where a call's partials start in its workspace: behind the counters, which are zero between calls.
size_t workspace_base() { return (emx_paged_workspace_zeroed_bytes() + 255) & ~(size_t)255; }

bool head_ok(int D) { return D == 64 || D == 128 || D == 256; }

// The call's geometry, and the rule, as the entry points receive them.
struct Call {
  GenericArgs g;
  MaskRule mask;
  void* ws;
  size_t ws_bytes;
  hipStream_t st;
};

int check(const void* queries, int num_tokens, int num_q_heads, int head_dim, int num_kv_heads, int num_blocks,
          int page_size, const int32_t* block_tables, int num_seqs, int max_blocks, const int32_t* kv_lens,
          const int32_t* qsl, float softmax_scale, int sliding_window, int sink_tokens, const int32_t* parents,
          int single_token_decode, void* ws, size_t ws_bytes, void* out, void* stream, Call& c) {
  if (int rc = entry_check_attention(queries, num_tokens, num_q_heads, head_dim, num_kv_heads, num_blocks, page_size,
                                     block_tables, num_seqs, max_blocks, kv_lens, qsl, single_token_decode, out))
    return rc;
  if (!(std::isfinite(softmax_scale) && softmax_scale > 0.f))
    return entry_fail(EMX_ERR_INVALID, "softmax_scale must be positive and finite");
  if (sink_tokens < 0) return entry_fail(EMX_ERR_INVALID, "sink_tokens must be >= 0");
  if ((long long)max_blocks * page_size >= (1LL << 31))
    return entry_fail(EMX_ERR_UNSUPPORTED, "max_blocks_per_seq * page_size must be below 2^31");
  c.g = GenericArgs{queries, out, block_tables, kv_lens, qsl, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim,
                    page_size, num_blocks, max_blocks, softmax_scale * kLog2e, 0, single_token_decode ? 1 : 0};
  c.mask.window = std::max(sliding_window, 0);
  c.mask.sinks = c.mask.window ? sink_tokens : 0;
  c.mask.parents = parents;
  c.ws = ws;
  c.ws_bytes = ws_bytes;
  c.st = reinterpret_cast<hipStream_t>(stream);
  return EMX_OK;
}

template <typename QT, typename KV>
int generic(const Call& c, const KV& kv) {
  const dim3 grid((unsigned)c.g.T, (unsigned)c.g.Hkv, (unsigned)((c.g.Hq / c.g.Hkv + 15) / 16));
  hipLaunchKernelGGL((masked_generic<QT, KV>), grid, dim3(64 * kGenericWaves), 0, c.st, c.g, c.mask, kv);
  return entry_check_launch("masked_generic");
}

// Runs the call on the matrix units where they take its shape; false: nothing launched.
bool mfma(const Call& c, MfmaCall m, int* rc) {
  const GenericArgs& g = c.g;
  m.q = g.q;
  m.out = g.out;
  m.block_tables = g.block_tables;
  m.kv_lens = g.kv_lens;
  m.qsl = g.decode ? nullptr : g.qsl;
  m.T = g.T;
  m.S = g.S;
  m.Hq = g.Hq;
  m.Hkv = g.Hkv;
  m.D = g.D;
  m.bs = g.bs;
  m.nb = g.nb;
  m.max_blocks = g.max_blocks;
  m.scale_log2 = g.scale_log2;
  m.window = c.mask.window;
  if (g.S <= 0 || g.S > kWideSeqs || !mfma_ok(m) || (long long)g.nb * g.bs * (m.kind == KvKind::affine ? g.Hkv : 1) >= (1LL << 31))
    return false;
  const size_t base = workspace_base();
  // rows of one token: the split-K decode (a tile of the kernel below would hold a group's heads alone)
  const size_t rows = g.decode && c.mask.sinks > 0 && !c.mask.parents && g.Hq / g.Hkv <= kMaskedHeads
                          ? decode_mfma_partial_bytes(g.S, g.Hq, g.Hkv, g.D) : 0;
  if (rows && c.ws && c.ws_bytes >= base + rows) {
    launch_masked_rows(m, c.mask.sinks, static_cast<int*>(c.ws),
                       reinterpret_cast<float*>(static_cast<char*>(c.ws) + base), c.st);
    *rc = entry_check_launch("decode_mfma (sinks)");
    return true;
  }
  MaskedShape shape = masked_shape(g.T, g.S, g.Hq, g.Hkv, g.D, m.kind, true);
  if (shape.tokb == 0) return false;
  // (the blocks of a cut launch are counted in 31 bits)
  if (shape.wgs && (!c.ws || c.ws_bytes < base + shape.desc_bytes + shape.part_bytes ||
                    (double)shape.tiles * g.Hkv * ((double)g.max_blocks * g.bs / 32 + 2 + kWideBegin) >= 2147483648.0))
    shape = masked_shape(g.T, g.S, g.Hq, g.Hkv, g.D, m.kind, false);
  if (shape.tiles * g.Hkv >= (1L << 31)) return false;
  MaskedArgs a{};
  a.d.q = static_cast<const h16*>(m.q);
  a.d.kc = static_cast<const uint32_t*>(m.k);
  a.d.vc = static_cast<const uint32_t*>(m.v);
  a.d.kps = m.kps;
  a.d.vps = m.vps;
  a.d.ks = static_cast<const h16*>(m.ks);
  a.d.kb = static_cast<const h16*>(m.kb);
  a.d.vs = static_cast<const h16*>(m.vs);
  a.d.vb = static_cast<const h16*>(m.vb);
  a.d.block_tables = m.block_tables;
  a.d.kv_lens = m.kv_lens;
  a.d.qsl = m.qsl;
  a.d.out = static_cast<h16*>(m.out);
  a.d.S = m.S;
  a.d.Hq = m.Hq;
  a.d.Hkv = m.Hkv;
  a.d.bs = m.bs;
  a.d.nb = m.nb;
  a.d.max_blocks = m.max_blocks;
  a.d.scale_log2 = m.scale_log2;
  a.d.window = m.window;
  a.mask = c.mask;
  a.inv_bs = (uint32_t)(((1ULL << 32) + m.bs - 1) / m.bs);
  a.tokb = shape.tokb;
  a.T = m.T;
  a.tiles = (int)shape.tiles;
  a.wgs = shape.wgs;
  if (a.wgs) {
    char* p = static_cast<char*>(c.ws) + base;
    a.part = reinterpret_cast<float*>(p);
    a.desc = reinterpret_cast<int4*>(p + shape.part_bytes);
  }
  switch (m.kind) {
    case KvKind::f16: launch_masked_kind<KvF16>(a, m.D, shape.cw, c.st); break;
    case KvKind::bf16: launch_masked_kind<KvBF16>(a, m.D, shape.cw, c.st); break;
    case KvKind::fp8: launch_masked_kind<KvFp8>(a, m.D, shape.cw, c.st); break;
    case KvKind::affine: launch_masked_affine(m, a, shape.cw, c.st); break;
  }
  *rc = entry_check_launch("masked_wide");
  return true;
}

}  // namespace
}  // namespace emx

using namespace emx;

extern "C" {

size_t emx_masked_workspace_bytes(int num_tokens, int num_seqs, int num_q_heads, int num_kv_heads, int head_dim) {
  if (num_tokens <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      !head_ok(head_dim))
    return 0;
  size_t part = 0;  // (whatever the cache)
  for (const KvKind kind : {KvKind::f16, KvKind::fp8, KvKind::affine}) {
    const MaskedShape m = masked_shape(num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, kind, true);
    part = std::max(part, m.desc_bytes + m.part_bytes);
  }
  if (num_tokens == num_seqs && num_q_heads / num_kv_heads <= kMaskedHeads)
    part = std::max(part, decode_mfma_partial_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim));
  return part ? workspace_base() + part : 0;
}

int emx_masked_attention_affine(const void* queries, int num_tokens, int num_q_heads, int head_dim,
                                const uint32_t* k_codes, const void* k_scales, const void* k_biases,
                                const uint32_t* v_codes, const void* v_scales, const void* v_biases, int num_blocks,
                                int page_size, int num_kv_heads, int bits, int group_size,
                                const int32_t* block_tables, int num_seqs, int max_blocks_per_seq,
                                const int32_t* kv_lens, const int32_t* query_start_loc, float softmax_scale,
                                int sliding_window, int sink_tokens, const int32_t* tree_parents,
                                int single_token_decode, void* workspace, size_t workspace_bytes, void* out,
                                void* stream) {
  Call c;
  if (int rc = check(queries, num_tokens, num_q_heads, head_dim, num_kv_heads, num_blocks, page_size, block_tables,
                     num_seqs, max_blocks_per_seq, kv_lens, query_start_loc, softmax_scale, sliding_window,
                     sink_tokens, tree_parents, single_token_decode, workspace, workspace_bytes, out, stream, c))
    return rc;
  if (bits != 4 && bits != 8) return entry_fail(EMX_ERR_UNSUPPORTED, "bits must be 4 or 8");
  if (group_size <= 0 || head_dim % group_size != 0)
    return entry_fail(EMX_ERR_INVALID, "head_dim must be a multiple of group_size");
  if ((head_dim * bits) % 32 != 0 || (page_size * bits) % 32 != 0)
    return entry_fail(EMX_ERR_INVALID, "head_dim * bits and page_size * bits must be multiples of 32");
  if (page_size > 256 / bits && page_size % (256 / bits) != 0)
    return entry_fail(EMX_ERR_INVALID, "page_size above 256/bits must be a multiple of 256/bits");
  if (num_tokens == 0) return EMX_OK;
  if (!k_codes || !k_scales || !k_biases || !v_codes || !v_scales || !v_biases)
    return entry_fail(EMX_ERR_INVALID, "null cache pointer");
  MfmaCall m{};
  m.kind = KvKind::affine;
  m.k = k_codes;
  m.v = v_codes;
  m.ks = k_scales;
  m.kb = k_biases;
  m.vs = v_scales;
  m.vb = v_biases;
  m.bits = bits;
  m.gs = group_size;
  int rc = EMX_OK;
  if (mfma(c, m, &rc)) return rc;
  const h16 *ks = static_cast<const h16*>(k_scales), *kb = static_cast<const h16*>(k_biases);
  const h16 *vs = static_cast<const h16*>(v_scales), *vb = static_cast<const h16*>(v_biases);
  if (bits == 4)
    return generic<h16>(c, AffineKV<4>{k_codes, ks, kb, v_codes, vs, vb, num_kv_heads, head_dim, page_size, group_size});
  return generic<h16>(c, AffineKV<8>{k_codes, ks, kb, v_codes, vs, vb, num_kv_heads, head_dim, page_size, group_size});
}

int emx_masked_attention_dense(const void* queries, int num_tokens, int num_q_heads, int head_dim, int dtype,
                               const void* key_cache, const void* value_cache, int num_blocks, int page_size,
                               int num_kv_heads, const int32_t* block_tables, int num_seqs, int max_blocks_per_seq,
                               const int32_t* kv_lens, const int32_t* query_start_loc, float softmax_scale,
                               int sliding_window, int sink_tokens, const int32_t* tree_parents,
                               int single_token_decode, void* workspace, size_t workspace_bytes, void* out,
                               void* stream) {
  Call c;
  if (int rc = check(queries, num_tokens, num_q_heads, head_dim, num_kv_heads, num_blocks, page_size, block_tables,
                     num_seqs, max_blocks_per_seq, kv_lens, query_start_loc, softmax_scale, sliding_window,
                     sink_tokens, tree_parents, single_token_decode, workspace, workspace_bytes, out, stream, c))
    return rc;
  if (dtype != EMX_DTYPE_F16 && dtype != EMX_DTYPE_BF16 && dtype != EMX_DTYPE_F32)
    return entry_fail(EMX_ERR_UNSUPPORTED, "unknown dtype code");
  if (num_tokens == 0) return EMX_OK;
  if (!key_cache || !value_cache) return entry_fail(EMX_ERR_INVALID, "null cache pointer");
  int rc = EMX_OK;
  if (dtype != EMX_DTYPE_F32) {
    MfmaCall m{};
    m.kind = dtype == EMX_DTYPE_F16 ? KvKind::f16 : KvKind::bf16;
    m.k = key_cache;
    m.v = value_cache;
    if (mfma(c, m, &rc)) return rc;
  }
  if (dtype == EMX_DTYPE_F16)
    return generic<h16>(c, DenseKV<F16>{static_cast<const h16*>(key_cache), static_cast<const h16*>(value_cache),
                                        num_kv_heads, head_dim, page_size});
  if (dtype == EMX_DTYPE_BF16)
    return generic<uint16_t>(c, DenseKV<BF16>{static_cast<const uint16_t*>(key_cache),
                                              static_cast<const uint16_t*>(value_cache), num_kv_heads, head_dim,
                                              page_size});
  return generic<float>(c, DenseKV<F32>{static_cast<const float*>(key_cache), static_cast<const float*>(value_cache),
                                        num_kv_heads, head_dim, page_size});
}

int emx_masked_attention_fp8(const void* queries, int num_tokens, int num_q_heads, int head_dim, int dtype,
                             const uint8_t* key_cache, const uint8_t* value_cache, const float* k_scale,
                             const float* v_scale, int num_blocks, int page_size, int num_kv_heads,
                             const int32_t* block_tables, int num_seqs, int max_blocks_per_seq,
                             const int32_t* kv_lens, const int32_t* query_start_loc, float softmax_scale,
                             int sliding_window, int sink_tokens, const int32_t* tree_parents,
                             int single_token_decode, void* workspace, size_t workspace_bytes, void* out,
                             void* stream) {
  Call c;
  if (int rc = check(queries, num_tokens, num_q_heads, head_dim, num_kv_heads, num_blocks, page_size, block_tables,
                     num_seqs, max_blocks_per_seq, kv_lens, query_start_loc, softmax_scale, sliding_window,
                     sink_tokens, tree_parents, single_token_decode, workspace, workspace_bytes, out, stream, c))
    return rc;
  if (dtype != EMX_DTYPE_F16 && dtype != EMX_DTYPE_BF16 && dtype != EMX_DTYPE_F32)
    return entry_fail(EMX_ERR_UNSUPPORTED, "unknown dtype code");
  if (num_tokens == 0) return EMX_OK;
  if (!key_cache || !value_cache || !k_scale || !v_scale)
    return entry_fail(EMX_ERR_INVALID, "null cache or scale pointer");
  int rc = EMX_OK;
  if (dtype == EMX_DTYPE_F16) {
    MfmaCall m{};
    m.kind = KvKind::fp8;
    m.k = key_cache;
    m.v = value_cache;
    m.kps = k_scale;
    m.vps = v_scale;
    if (mfma(c, m, &rc)) return rc;
  }
  const Fp8KV kv{key_cache, value_cache, k_scale, v_scale, num_kv_heads, head_dim, page_size};
  if (dtype == EMX_DTYPE_F16) return generic<h16>(c, kv);
  if (dtype == EMX_DTYPE_BF16) return generic<uint16_t>(c, kv);
  return generic<float>(c, kv);
}

}  // extern "C"
