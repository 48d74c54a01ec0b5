// Masked paged attention (masked_launch.hpp: sliding windows with sinks, drafted trees) on the
// matrix units: head_dim 64, 128 or 256, any GQA ratio up to the columns of a tile, over
// token-major caches [nb, bs, Hkv, D] (fp16 / bf16, FP8 E4M3 with one fp32 scale per page; pages
// of a multiple of 8 tokens) and over affine pages.
//
//   O_i = sum_k p_ik V_k / sum_k p_ik,  p_ik = 2^(scale log2(e) q_i . K_k - m_i) over the keys k
//   that row i sees,
//
// in one pass over the keys with the running reference m_i.
//
// Work: a tile is the 32 CW query columns (token, head), head fastest, of 32 CW / HG tokens of one
// sequence and kv head; its keys go in blocks of NT positions, from the last backwards and then the
// sinks' blocks: those between the sinks and the earliest window are not read.  From the last
// backwards because a drafted node's ancestors then come in the order of its walk to the root: each
// lane keeps one cursor, and a block of drafted keys costs as many steps as it holds ancestors, for
// trees of any size.  Where a launch has tiles enough each is a workgroup's; else the blocks of all
// tiles in a row (and what it costs to begin each, kWideBegin) are cut into equal ranges, one to a
// workgroup, and a tile that is not inside one range leaves its parts' fp32 state to masked_merge,
// which joins them in part order.
//
// A block: K and V are read once per workgroup, a block ahead, into the other of two LDS images of
// 16-bit values, 16-byte chunks turned by the row so that operand reads touch every bank: one barrier
// a block.  fp16 / bf16 rows go there as they are, with no register between (a block's 32 registers
// of a thread were spilled, and each reload waited for the loads themselves: 870 -> 745 us over 12
// trees of 48 to 64 nodes with 64 / 8 heads and up to 32768 keys); FP8 (dec(code) * 2^-8, exact) and
// affine codes (exact sub-normals) through registers.  A wave has 32 columns (KW = 2: and half of the
// block's keys; D = 256: and half of the dims, the two halves of its scores meeting in LDS: a wave's
// state then fits 256 registers, 87 -> 77 us over three prompt chunks on 8-bit pages), on v_mfma
// 32x32x16:
//   S^T : A = K rows, B = queries; a lane ends with half of its tile's scores of ONE column, so that
//         maximum, reference and sum are its own, and lanes meet only where a score passes the
//         reference by 2^kLazyMax;
//   O^T += V^T P^T : A = V^T by the transposing LDS read (affine values lie dim-major already), B = the
//         lane's own probabilities as two 16-bit parts, each the nearest (fp16: 22 bits of the 24; bf16:
//         16, which puts an output off by at most 2^-17 of the largest value it averages: one part would
//         add an error as large as the output's own rounding).
// Bound: matrix instructions, 1.5 times the formula's for the second part, at the 1.27 PFLOP/s that a
// large bf16 product reaches (those 12 trees, 461 GFLOP and 1.04 GB: 543 us of the 746; the matrix units
// are busy in half of the cycles); over affine pages the vector unit and the chain of a block (codes to
// values, scores, softmax: 20 vector instructions to a product).
#pragma once

#include <type_traits>

#include "masked_launch.hpp"
#include "prefill_mfma.hpp"

namespace emx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const h16x8 a, const h16x8 b, const f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(const bf16x8 a, const bf16x8 b, const f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void split_p2(const float (&x)[8], h16x8 (&p)[2]) { split_p(x, p); }
__device__ __forceinline__ void split_p2(const float (&x)[8], bf16x8 (&p)[2]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2v __attribute__((ext_vector_type(2)));
  uint32_t w[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h =
        __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{x[2 * i], x[2 * i + 1]}, bf16x2));
    w[0][i] = h;
    w[1][i] = __builtin_bit_cast(
        uint32_t, __builtin_convertvector(f32x2v{x[2 * i] - __uint_as_float(h << 16),
                                                 x[2 * i + 1] - __uint_as_float(h & 0xFFFF0000u)},
                                          bf16x2));
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) p[k] = __builtin_bit_cast(bf16x8, u32x4{w[k][0], w[k][1], w[k][2], w[k][3]});
}

struct MaskedArgs {
  DecodeArgs d;     // kc / vc: the caches; qsl null: token i is sequence i
  MaskRule mask;
  uint32_t inv_bs;  // ceil(2^32 / bs)
  int tokb;         // query tokens per tile: columns / HG
  int T;            // query rows
  int tiles;        // tiles per kv head, at most
  int wgs;          // > 0: tiles are cut, over at most that many workgroups; 0: a workgroup to a tile
  int4* desc;       // cut: [1 + min(Hkv * tiles, wgs)] {how many of them}, then what masked_merge has to know of a tile
  float* part;      // cut: [2 * wgs][part floats]
};

// What beginning a tile costs (pages, queries, first block; a part written), in blocks: 6 to 9 us against 2 to 3 us a block.
// Ranges are equal with it, else those of short tiles end last (32 trees of 16 nodes on 4-bit pages: 92 us against 99, three
// prompt chunks with 256-wide heads 73 against 76).  A range may be one block: a tree of 25 nodes over 1531 keys takes 19.4
// us against 21.5 with two at least.
constexpr int kWideBegin = 3;
// How many blocks longer than an equal share the longest tile may be before tiles are cut, where there is a workgroup for
// each (parts go to memory and back: 64 KiB each way, and a launch).
constexpr int kWideCutBlocks = 6;
constexpr int kWideParts = 1024;   // more than a tile's parts
constexpr int kWideTreeLds = 512;  // nodes of a tree whose parents are kept in LDS

template <class C, int D, int KW, int CW>
struct WideCfg {
  static constexpr int EB = sizeof(typename C::ET);
  static constexpr int DW = D > 128 ? 2 : 1;        // waves that share a column's dims
  static constexpr int TH = 64 * KW * CW * DW;      // threads
  static constexpr int NT = D > 128 ? 32 * KW : 64; // keys of a block
  static constexpr int KT = NT / KW / 32;           // 32-key tiles of a wave's share of it
  static constexpr int KS = D / 16 / DW;            // QK^T k-slices of a wave
  static constexpr int DT = D / 32 / DW;            // PV dim tiles
  static constexpr int G = 1, GV = 1;               // quantization groups of a key, of a wave's dims
  static constexpr int PR = D * EB / 16;            // 16-byte pieces per row
  static constexpr int NP = NT * PR / TH;           // pieces per thread and block, of K and of V
  static constexpr int VB = NT * D * 2;             // bytes of the V image
  static constexpr int SCB = C::kFp8 ? 2 * 4 * NT : 0;  // of the scales
  static_assert(KT >= 1 && NT * PR % TH == 0, "whole 32-key tiles and pieces");
};
template <int BITS, int GS, int D, int KW, int CW>
struct WideCfg<KvAffine<BITS, GS>, D, KW, CW> {
  static constexpr int DW = D > 128 ? 2 : 1, TH = 64 * KW * CW * DW, NT = D > 128 ? 32 * KW : 64, KT = NT / KW / 32;
  static constexpr int KS = D / 16 / DW, DT = D / 32 / DW, G = D / GS, GV = G / DW;
  static constexpr int RBK = D * BITS / 8;              // bytes of a key's codes
  static constexpr int PR = RBK / 16;                   // 16-byte pieces of them
  static constexpr int NPK = NT * PR;                   // K pieces of a block
  static constexpr int NP = (NPK + TH - 1) / TH;
  static constexpr int UT = 64 / BITS, U = NT / UT;     // V units: 8 bytes, UT tokens of one dim
  static constexpr int NPV = D * U / TH;                // V units per thread
  static constexpr int NPS = 4 * G * NT / 8;            // 16-byte scale pieces of a block
  static constexpr int VB = D * NT * 2;                 // [dim][NT], 16-byte chunks turned by v_turn
  static constexpr int SCB = 3 * 4 * G * NT + 16 * NT;  // ks, vs, vb [group][NT] floats, bias operand rows
  static_assert(NPS <= 64 && D * U % TH == 0, "one scale piece per lane, whole V units per thread");
};

// Where 16-byte chunk c of a row stands in its row, so that the lanes that LDS serves in one cycle touch all 64 banks.
// K: 16 rows at one chunk; token-major V: 4 rows at 4 neighbouring chunks; affine V (a row: NT keys of a dim): 16 rows
// at one chunk.  Each turns with the row alone, so that an operand's address is a lane's, with constant bits flipped.
// (With every row turned by its low three bits alone more than half of the LDS cycles were conflicts.)
template <int D>
__device__ __forceinline__ constexpr int k_turn(const int row, const int c) {
  return c ^ (D == 64 ? (row >> 1) & 7 : row & 15);
}
template <int D>
__device__ __forceinline__ constexpr int v_turn(const int row, const int c) {
  return c ^ (D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2);
}
template <int NT>
__device__ __forceinline__ constexpr int va_turn(const int dim, const int c) {
  return c ^ (NT == 64 ? (dim >> 1) & 7 : (dim >> 2) & 3);
}

// 16 bytes from src + off (each lane its own) to LDS byte `dst` + 16 lane, with no register between.  Nothing waits for it
// but dma_wait: the compiler's own waits count only loads that it knows, which come back in order with these.  (By the
// compiler's builtin every transposing LDS read that follows waits for it, in the block before the one it loads.  A write
// of m0 needs one wait state before a load that goes by it.)
__device__ __forceinline__ void dma16(const char* src, const uint32_t off, const uint32_t dst) {
  const uint64_t a = reinterpret_cast<uint64_t>(src);
  const uint64_t base = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32) |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(m0)
               : "v"(off), "s"(base), "s"(dst)
               : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The same value, as one that the compiler has not seen: what is computed from it inside a loop is computed there, and
// takes no register (or, worse, scratch memory: its reload waits for every load issued before it) all through the loop.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Floats of a part: per column wave DT * 4 + 1 vectors of 4 a lane.
template <int D, int CW>
constexpr int kWidePart = CW * (D / 8 + 1) * 256;

// A tile's blocks: positions backwards from block `hi`, `n` in all, the last `sink` of them the blocks 0 .. sink - 1.
struct MaskedSpan {
  int hi, n, sink;
};

template <int NT>
__device__ __forceinline__ MaskedSpan masked_span(const MaskRule& m, const int past, const int tok_lo,
                                                  const int tok_hi) {
  MaskedSpan r{0, 0, 0};
  const int k_hi = past + tok_hi;
  if (k_hi < 0) return r;
  // the earliest first key of the tile's windows (a node's place is at least its tree's start); a
  // tree's own keys stand at places below their positions, and are all read
  int first = 0;
  if (m.window > 0) first = max(0, (m.parents ? past : past + tok_lo) - m.window + 1);
  if (m.parents) first = min(first, max(past, 0));
  r.hi = k_hi / NT;
  const int lo = min(first, k_hi) / NT;
  r.sink = min((min(m.sinks, k_hi + 1) + NT - 1) / NT, lo);
  r.n = r.hi - lo + 1 + r.sink;
  return r;
}

struct MaskedSeq {
  int s, q0, qlen, past;
};

__device__ __forceinline__ MaskedSeq masked_seq(const MaskedArgs& A, const int s) {
  const DecodeArgs& a = A.d;
  MaskedSeq r;
  r.s = s;
  r.q0 = a.qsl ? a.qsl[s] : s;
  r.qlen = a.qsl ? (r.q0 < 0 ? 0 : max(a.qsl[s + 1] - r.q0, 0)) : 1;
  r.past = min(max(a.kv_lens[s], 0), a.max_blocks * a.bs) - r.qlen;
  return r;
}

// Last token of tile `tile` of the sequence (rows past the call's are no tokens).
__device__ __forceinline__ int masked_tok_hi(const MaskedArgs& A, const MaskedSeq& q, const int tile) {
  return min(min((tile + 1) * A.tokb, q.qlen), A.T - q.q0) - 1;
}

// Blocks of a tile, at least one (an empty one writes its rows' zeros).
template <int NT>
__device__ __forceinline__ int masked_blocks(const MaskedArgs& A, const MaskedSeq& q, const int tile) {
  return max(1, masked_span<NT>(A.mask, q.past, tile * A.tokb, masked_tok_hi(A, q, tile)).n);
}

// The sum over the workgroup of the threads before this one (NW waves; red: NW ints of LDS); total: of all.
template <int NW>
__device__ __forceinline__ int wg_scan(const int mine, int* red, int& total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int x = mine;  // within rows of 16 lanes, then over the rows before
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  __syncthreads();  // (red may still be read)
  if (lane == 63) red[wv] = x;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    base += w < wv ? red[w] : 0;
    total += red[w];
  }
  // (what comes from LDS counts as each lane's own: every address and bound reckoned from it was, in vector registers)
  total = __builtin_amdgcn_readfirstlane(total);
  return base + x - mine;
}

constexpr int kWideSeqs = 1024;   // sequences of a call
constexpr int kWideSeqLds = 256;  // sequences whose place and lengths are kept in LDS

// Sequence s as wide_tiles left it in LDS (a call of more sequences: from memory).
__device__ __forceinline__ MaskedSeq wide_seq(const MaskedArgs& A, const int* seqs, const int s) {
  if (A.d.S > kWideSeqLds) return masked_seq(A, s);
  return MaskedSeq{s, seqs[s], seqs[kWideSeqLds + s], seqs[2 * kWideSeqLds + s]};
}

// tcum[s]: tiles of the sequences before s, tcum[S] of all; seqs: wide_seq's.
template <int NW>
__device__ __forceinline__ void wide_tiles(const MaskedArgs& A, int* tcum, int* seqs, int* red) {
  const int S = A.d.S, ch = (S + 64 * NW - 1) / (64 * NW), s0 = threadIdx.x * ch;
  int mine = 0, total;
  for (int i = 0; i < ch && s0 + i < S; ++i) {
    const MaskedSeq q = masked_seq(A, s0 + i);
    const int n = (q.qlen + A.tokb - 1) / A.tokb;
    tcum[s0 + i] = n;
    mine += n;
    if (S <= kWideSeqLds) {
      seqs[s0 + i] = q.q0;
      seqs[kWideSeqLds + s0 + i] = q.qlen;
      seqs[2 * kWideSeqLds + s0 + i] = q.past;
    }
  }
  int run = wg_scan<NW>(mine, red, total);
  for (int i = 0; i < ch && s0 + i < S; ++i) {
    const int n = tcum[s0 + i];
    tcum[s0 + i] = run;
    run += n;
  }
  if (threadIdx.x == 0) tcum[S] = total;
  __syncthreads();
}

// The sequence of tile t: the largest s with tcum[s] <= t (t < tcum[S]).
__device__ __forceinline__ int wide_seq_of(const int* tcum, const int S, const int t) {
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tcum[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One query row in fp32 on one wave over every key that it sees: rows whose result on the matrix unit is not
// finite are computed again here, dims [d0, d1) of them (there a key that the row does not see still enters its tile's product with p = 0,
// and 0 * inf makes NaN of what these rules leave alone).  64 keys at a time, as attend_row (mfma_common.hpp).
template <class C, int D>
__device__ void attend_masked(const DecodeArgs& a, const MaskRule& mask, const MaskedSeq& sq, const int kvh, const int i,
                              const int hd, const int lane, const int d0 = 0, const int d1 = D) {
  constexpr int N = D / 64;
  typedef typename C::QT QT;
  const auto kv = kv_loader<C>(a, D);
  const int32_t* par = mask.parents ? mask.parents + sq.q0 : nullptr;
  const int depth = par && mask.window > 0 ? node_depth(par, i) : 0;
  const size_t ro = ((size_t)(sq.q0 + i) * a.Hq + (size_t)kvh * (a.Hq / a.Hkv) + hd) * D;
  const QT* q = reinterpret_cast<const QT*>(a.q) + ro;
  float qv[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    qv[n] = to_f32(q[lane + 64 * n]);
    acc[n] = 0.f;
  }
#pragma unroll 1
  for (int base = 0; base <= sq.past + i; base += 64) {
    const int k = base + lane;
    const bool see = k <= sq.past + i && key_visible(mask, par, sq.past, i, depth, k);
    const int blk = see ? a.block_tables[(size_t)sq.s * a.max_blocks + k / a.bs] : -1;
    const bool ok = (unsigned)blk < (unsigned)a.nb;
    const uint64_t okm = __ballot(ok);
    if (!okm) continue;
    float x = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll 1
      for (int d = 0; d < 64; d += 32) {
        float kd[32] = {};
        if (ok) key32(kv, blk, k % a.bs, kvh, 64 * n + d, kd);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          x = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(qv[n]), d + j)), kd[j], x);
      }
    x = ok ? x * a.scale_log2 : -INFINITY;
    const float mn = fmaxf(m, wave_max(x));
    const float p = ok && (mn != -INFINITY || x != x) ? exp2f(x - mn) : 0.f;
    const float al = m == mn ? 1.f : exp2f(m - mn);
    l = l * al + wave_sum(p);
    m = mn;
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] *= al;
#pragma unroll 1
    for (int t = 0; t < 64; t += 8) {
      const uint32_t live = (uint32_t)(okm >> t) & 0xFFu;
      if (!live) continue;
      const int b = __builtin_amdgcn_readlane(blk, t + __builtin_ctz(live));
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float v[8];
        val8(kv, b, (base + t) % a.bs, kvh, lane + 64 * n, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), t + j));
          acc[n] = (live >> j) & 1u ? fmaf(pj, v[j], acc[n]) : acc[n];
        }
      }
    }
  }
  const float li = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (lane + 64 * n >= d0 && lane + 64 * n < d1) from_f32(acc[n] * li, reinterpret_cast<QT*>(a.out) + ro + lane + 64 * n);
}

// Equal ranges of `all` blocks for n workgroups (all >= n): where range w begins, and whose block x is.
struct WideRanges {
  int q, r;
  __device__ __forceinline__ WideRanges(const int all, const int n) : q(all / n), r(all - all / n * n) {}
  __device__ __forceinline__ int begin(const int w) const { return w * q + min(w, r); }
  __device__ __forceinline__ int owner(const int x) const {
    const int big = r * (q + 1);
    return x < big ? x / (q + 1) : r + (x - big) / q;
  }
};

// Column c of a tile: which token and head; token -1 where there is none.
__device__ __forceinline__ void masked_column(const MaskedArgs& A, const MaskedSeq& q, const int tile, const int c,
                                              const int HG, int& tok, int& head) {
  const int t = c / HG;
  tok = tile * A.tokb + t;
  head = c - t * HG;
  if (t >= A.tokb || tok >= q.qlen || (unsigned)(q.q0 + tok) >= (unsigned)A.T) tok = -1;
}

// Four dims from `dim` of a column, normalised and written.  True where a value is not finite.
template <class C, int D>
__device__ __forceinline__ bool masked_write(const DecodeArgs& a, const MaskedSeq& q, const int kvh, const int tok,
                                             const int head, const f32x4 o, const float l, const float inv,
                                             const int dim) {
  typedef typename C::QT QT;
  struct alignas(8) Four {
    QT x[4];
  } v;
  bool bad = not_finite(l);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bad = bad || not_finite(o[r]);
    from_f32(o[r] * inv, &v.x[r]);
  }
  if (tok >= 0)
    *reinterpret_cast<Four*>(reinterpret_cast<QT*>(a.out) +
                             ((size_t)(q.q0 + tok) * a.Hq + (size_t)kvh * (a.Hq / a.Hkv) + head) * D + dim) = v;
  return bad && tok >= 0;
}

// The lowest n of 32 bits (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t below(const int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
}

// (256 registers a wave: two waves to a SIMD)
template <class C, int D, int KW, int CW>
__global__ __launch_bounds__((WideCfg<C, D, KW, CW>::TH), 2) void masked_wide(MaskedArgs A) {
  using P = WideCfg<C, D, KW, CW>;
  typedef typename C::Op Op;
  typedef typename C::QT QT;
  const DecodeArgs& a = A.d;
  constexpr int NT = P::NT, KT = P::KT, KS = P::KS, DT = P::DT, G = P::G, GV = P::GV, TH = P::TH, NW = TH / 64;
  constexpr bool AFF = C::kAffine, FP8 = C::kFp8;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cw = wv % CW, kw = wv / CW % KW;    // this wave's columns, its share of a block's keys
  const int dw = P::DW > 1 ? wv / (CW * KW) : 0;  // ... and of the dims
  const int c32 = lane & 31, half = lane >> 5;

  // ---- LDS: two images of a block (K rows, V, scales; the states of a unit's key waves meet there too), then tables
  constexpr bool DMA = !AFF && !FP8;  // rows go to the images as they are: no register between
  constexpr int oBuf = 0, KB = NT * D * 2, oV = KB, oSc = oV + P::VB;
  constexpr int BUF = (oSc + (DMA ? 0 : P::SCB + 16) + 511) & ~511;
  static_assert(KB % 512 == 0 && P::VB % 512 == 0, "the images' chunks are flipped by address bits");
  constexpr int MEET = KW > 1 ? CW * (4 * DT + 1) * 64 * 16 : 0;
  constexpr int oTc = 2 * BUF > MEET ? 2 * BUF : MEET, oSeq = lds_next(oTc, 4 * (kWideSeqs + 1));
  constexpr int oPar = lds_next(oSeq, 12 * kWideSeqLds), oRed = lds_next(oPar, 4 * kWideTreeLds);
  constexpr int oX = lds_next(oRed, 128);  // two waves to a column's dims: a wave's part of its scores
  constexpr int oEnd = oX + (P::DW > 1 ? TH * KT * 64 : 0);
  static_assert(oEnd <= (TH > 256 ? 163840 : 81920), "256 threads: two workgroups to a compute unit");
  __shared__ __attribute__((aligned(512))) unsigned char lds[oEnd];
  int* tcum = reinterpret_cast<int*>(lds + oTc);
  int* seqs = reinterpret_cast<int*>(lds + oSeq);
  int* lpar = reinterpret_cast<int*>(lds + oPar);
  int* red = reinterpret_cast<int*>(lds + oRed);

  const MaskRule mask = A.mask;
  const int HG = a.Hq / a.Hkv, S = a.S;
  const int row_lo = a.qsl ? a.qsl[0] : 0, row_hi = a.qsl ? a.qsl[S] : A.T;

  bool first_seg = true;
  const bool by_tile = a.Hkv * A.tiles <= A.wgs;
  int4 cut_tile{0, 0, 0, 0};  // for masked_merge: the tile whose first block this range has, and not its last

  // ---- this workgroup's range [at, end) of the units of all tiles, kv head by kv head: kWideBegin to begin a tile, then
  // its blocks
  wide_tiles<NW>(A, tcum, seqs, red);
  if (row_lo > 0 || row_hi < A.T) zero_other_rows<QT>(a, A.T, D, blockIdx.x, gridDim.x);
  // (no more than the launch has room for, whatever query_start_loc holds)
  const int ntiles = min(__builtin_amdgcn_readfirstlane(tcum[S]), A.tiles);
  int kvh, t, u0, todo, w = 0, nwg = 0;  // kv head, tile, unit within it, units left; nwg 0: no tile is cut
  WideRanges ranges(0, 1);
  if (A.wgs == 0) {
    kvh = blockIdx.x % a.Hkv;
    t = ntiles - 1 - (int)blockIdx.x / a.Hkv;  // (the longest of a sequence first)
    u0 = 0;
    todo = 0x7FFFFFFF;
    if (t < 0) return;
  } else {
    const int ch = (ntiles + TH - 1) / TH, t0 = tid * ch;
    int mine = 0, most = 0, per;
    for (int i = 0, s = 0; i < ch && t0 + i < ntiles; ++i) {
      if (i == 0) s = wide_seq_of(tcum, S, t0);
      while (tcum[s + 1] <= t0 + i) ++s;
      const int n = masked_blocks<NT>(A, wide_seq(A, seqs, s), t0 + i - tcum[s]) + kWideBegin;
      mine += n;
      most = max(most, n);
    }
    most = (int)wave_max((float)most);
    if (lane == 0) red[8 + wv] = most;
    const int before = wg_scan<NW>(mine, red, per);
#pragma unroll
    for (int i = 0; i < NW; ++i) most = max(most, red[8 + i]);
    most = __builtin_amdgcn_readfirstlane(most);
    const int all = per * a.Hkv;  // (the host keeps it below 2^31)
    nwg = min(A.wgs, max(1, all));
    if (nwg >= 8) nwg &= ~7;
    const int nt = ntiles * a.Hkv;
    if (nt <= A.wgs && most <= all / nwg + kWideCutBlocks) {  // a tile to a workgroup
      nwg = 0;
      if (blockIdx.x == 0 && tid == 0) A.desc[0] = int4{0, 0, 0, 0};
      if ((int)blockIdx.x >= nt) return;
      kvh = blockIdx.x % a.Hkv;
      t = blockIdx.x / a.Hkv;
      u0 = 0;
      todo = 0x7FFFFFFF;
    } else {
      if ((int)blockIdx.x >= nwg) return;
      // workgroups of one XCD (blockIdx mod 8) take neighbouring ranges: tiles of one sequence and kv head share its L2
      w = nwg >= 8 ? (int)(blockIdx.x % 8) * (nwg / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
      ranges = WideRanges(all, nwg);
      const int at = ranges.begin(w);
      todo = ranges.begin(w + 1) - at;
      kvh = __builtin_amdgcn_readfirstlane(at / per);
      const int r = at - kvh * per;
      if (r >= before && r < before + mine) {  // one thread's tiles hold it
        int x = before, i = 0, s = wide_seq_of(tcum, S, t0);
        for (;; ++i) {
          while (tcum[s + 1] <= t0 + i) ++s;
          const int n = masked_blocks<NT>(A, wide_seq(A, seqs, s), t0 + i - tcum[s]) + kWideBegin;
          if (r < x + n) break;
          x += n;
        }
        red[16] = t0 + i;
        red[17] = r - x;
      }
      if (blockIdx.x == 0 && tid == 0) A.desc[0] = int4{by_tile ? ntiles : nwg, 0, 0, 0};
      __syncthreads();
      t = __builtin_amdgcn_readfirstlane(red[16]);
      u0 = __builtin_amdgcn_readfirstlane(red[17]);
    }
  }

  // ---- lane constants of the operand reads (image-relative bytes; the images start at multiples of 512)
  const int kad = (kw * KT * 32 + c32) * (D * 2) + (k_turn<D>(c32, KS * 2 * dw + half) << 4);  // K: row c32 (+ 32 per tile), chunk 2 w + half
  int vad;  // V: 4 tokens of 16 dims per 16 lanes, chunk 4 d + ..; affine: dim c32 (+ 32 per tile), chunk 4 kt + 2 j + half
  if constexpr (AFF) {
    vad = oV + (dw * DT * 32 + c32) * (NT * 2) + (va_turn<NT>(c32, kw * KT * 4 + half) << 4);
  } else {
    const int i = lane & 15, row = 4 * half + (i >> 2), c = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    vad = oV + (kw * KT * 32 + row) * (D * 2) + (v_turn<D>(row, c + 4 * DT * dw) << 4) + (i & 1) * 8;
  }
  const float sl2 = a.scale_log2;
  const size_t rowb = (size_t)a.Hkv * D * sizeof(typename C::ET);  // token-major
  typedef __attribute__((address_space(3))) unsigned char* lptr;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr)lds;
  uint32_t dma_k = 0, dma_v = 0;  // DMA: a lane's byte among the rows that its wave loads, of K and of V
  if constexpr (DMA) {
    static_assert(TH / P::PR % 16 == 0, "a thread's next rows are turned as its first");
    const int r = tid / P::PR, c = tid % P::PR;
    dma_k = lane / P::PR * (uint32_t)rowb + 16 * k_turn<D>(r, c);
    dma_v = lane / P::PR * (uint32_t)rowb + 16 * v_turn<D>(r, c);
  }

  int sidx = wide_seq_of(tcum, S, t);
  while (u0 + todo > kWideBegin) {  // (a range that ends in what it costs to begin a tile leaves it to the next)
    // ---- a segment: blocks [b0, b1) of tile t
    while (tcum[sidx + 1] <= t) ++sidx;
    MaskedSeq sq = wide_seq(A, seqs, __builtin_amdgcn_readfirstlane(sidx));
    sq.q0 = __builtin_amdgcn_readfirstlane(sq.q0);
    sq.qlen = __builtin_amdgcn_readfirstlane(sq.qlen);
    sq.past = __builtin_amdgcn_readfirstlane(sq.past);
    const int tile = t - __builtin_amdgcn_readfirstlane(tcum[sidx]);
    const int q0 = sq.q0, past = sq.past;
    const int tok_lo = tile * A.tokb, tok_hi = masked_tok_hi(A, sq, tile);
    const MaskedSpan span = masked_span<NT>(mask, past, tok_lo, tok_hi);
    const int nblk = max(1, span.n), u1 = min(nblk + kWideBegin, u0 + min(todo, nblk + kWideBegin - u0));
    const int b0 = max(0, u0 - kWideBegin), b1 = max(0, u1 - kWideBegin);
    const int st_lo = b0, st_hi = min(b1, span.n);  // (an empty tile has a block of nothing)
    const int k_hi = max(past + tok_hi, 0);
    const int32_t* par = mask.parents ? mask.parents + q0 : nullptr;
    const bool tree = par != nullptr, tree_lds = tree && sq.qlen <= kWideTreeLds;
    auto up = [&](const int i) { return tree_lds ? lpar[i] : parent_of(par, i); };
    auto pos_of_block = [&](const int st) {
      const int lo = span.n - span.sink;
      return (st < lo ? span.hi - st : span.sink - 1 - (st - lo)) * NT;
    };

    // ---- pages: lane l holds the page id of key l of a block (positions past the tile's last key repeat it)
    const char* kbase = reinterpret_cast<const char*>(a.kc) + (AFF ? 0 : (size_t)kvh * (D * sizeof(typename C::ET)));
    const char* vbase = reinterpret_cast<const char*>(a.vc) + (AFF ? 0 : (size_t)kvh * (D * sizeof(typename C::ET)));
    const int32_t* bt = a.block_tables + (size_t)sq.s * a.max_blocks;
    auto page_id = [&](const int st) {
      return bt[page_of(min(pos_of_block(st) + (lane & (NT - 1)), k_hi), A.inv_bs)];
    };
    u32x4 rk[P::NP], rv[AFF ? 1 : P::NP];  // the next block's pieces (DMA: not used)
    u32x2 ru[AFF ? 16 : 1];                // affine: its V units
    u32x4 rs;                              // affine, wave 0: scale piece `lane`
    uint64_t okn = 0;                      // keys of that block on a valid page
    float psk = 0.f, psv = 0.f;            // FP8: page scales of key `lane` of that block
    auto load_block = [&](const int st, const int blk, const int buf) {
      const unsigned tid = anew(threadIdx.x), lane = tid & 63;
      const bool ok = (unsigned)blk < (unsigned)a.nb;
      okn = __ballot(ok);
      if constexpr (DMA) {
        // A wave's 64 pieces, DR rows of one page (its tokens are a multiple of 8), stand in a row in the image: each lane
        // takes the chunk that belongs there.  What is the wave's is reckoned by the scalar unit
        constexpr int DR = 64 / P::PR;
#pragma unroll
        for (int n = 0; n < P::NP; ++n) {
          const int r0 = (wv + n * (TH / 64)) * DR, s = min(pos_of_block(st) + r0, k_hi);
          const int id = __builtin_amdgcn_readlane(blk, r0), b = (unsigned)id < (unsigned)a.nb ? id : 0;
          const size_t o = (size_t)(b * a.bs + s - page_of(s, A.inv_bs) * a.bs) * rowb;
          const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + oBuf + buf * BUF + (wv + n * (TH / 64)) * 1024);
          uint32_t back = 0;  // rows past the tile's last key repeat it
          if (s + DR - 1 > k_hi) back = (uint32_t)max((int)(lane / P::PR) - (k_hi - s), 0) * (uint32_t)rowb;
          dma16(kbase + o, dma_k - back, dst);
          dma16(vbase + o, dma_v - back, dst + oV);
        }
        return;
      }
      const int pos = min(pos_of_block(st) + (lane & (NT - 1)), k_hi);
      const int b = ok ? blk : 0;
      const int off = pos - page_of(pos, A.inv_bs) * a.bs;
      if constexpr (AFF) {
        constexpr int B = C::kBits;
        const int row = (b * a.Hkv + kvh) * a.bs + off;
        if (wv == 0) {
          const int pc = min((int)lane, P::NPS - 1), seg = pc / (NT / 8), arr = seg / G, g = seg % G;
          const int r8 = __shfl(row, 8 * (pc % (NT / 8)), 64), o8 = __shfl(off, 8 * (pc % (NT / 8)), 64);
          const h16 *b_ks = a.ks, *b_kb = a.kb, *b_vs = a.vs, *b_vb = a.vb;
          asm("" : "+s"(b_ks), "+s"(b_kb), "+s"(b_vs), "+s"(b_vb));  // picked from registers, not by a vector load
          const h16* base = arr == 0 ? b_ks : arr == 1 ? b_kb : arr == 2 ? b_vs : b_vb;
          typedef const __attribute__((address_space(1))) u32x4* gu32x4;
          // (past the tile's last key the group's first token may repeat it: aligned down, inside the page)
          rs = *(gu32x4)(base + (size_t)G * (r8 - o8) + (size_t)g * a.bs + (o8 & ~7));
        }
#pragma unroll
        for (int n = 0; n < P::NP; ++n) {  // (fewer pieces than threads: the others repeat them)
          const int r = __shfl(row, (tid / P::PR + n * (TH / P::PR)) & (NT - 1), 64);
          rk[n] = *reinterpret_cast<const u32x4*>(kbase + (size_t)r * P::RBK + 16 * (tid % P::PR));
        }
        const int T = min(a.bs, 256 / B);  // tokens of a value tile (a power of two)
        const int r = __shfl(row, tid % P::U * P::UT, 64), o = (r & (T - 1)) & ~(P::UT - 1);
        const uint32_t* vu = reinterpret_cast<const uint32_t*>(vbase) + (size_t)(r & ~(T - 1)) * (D * B / 32) +
                             ((int)(tid / P::U) * T + o) * B / 32;
#pragma unroll
        for (int n = 0; n < P::NPV; ++n) ru[n] = *reinterpret_cast<const u32x2*>(vu + n * (TH / P::U) * T * B / 32);
      } else {
        const int row = b * a.bs + off;
        if constexpr (FP8) {
          psk = a.kps[b];
          psv = a.vps[b];
        }
#pragma unroll
        for (int n = 0; n < P::NP; ++n) {
          const int r = tid / P::PR + n * (TH / P::PR), c = (int)(tid % P::PR);
          const size_t o = (size_t)__shfl(row, r, 64) * rowb;
          rk[n] = *reinterpret_cast<const u32x4*>(kbase + o + 16 * c);
          rv[n] = *reinterpret_cast<const u32x4*>(vbase + o + 16 * c);
        }
      }
    };
    // ... and their way to image `buf`, once they are here.  vex: the exponent that the value scales of the images carry
    int vex = 0;
    auto store_block = [&](const int st, const int buf) {
      const unsigned tid = anew(threadIdx.x), lane = tid & 63;
      unsigned char* img = lds + oBuf + buf * BUF;
      if constexpr (AFF) {
        constexpr int B = C::kBits;
        // (chunk numbers are multiples of the chunks of a piece or unit: the next ones stand at flipped address bits; the
        // rows of a thread's next piece or unit are turned as its first's)
        static_assert(TH / P::PR % 16 == 0 && TH / P::U % 16 == 0, "turned alike");
        const int kr0 = (tid / P::PR) & (NT - 1), ka0 = kr0 * (D * 2) + (k_turn<D>(kr0, tid % P::PR * (16 / B)) << 4);
#pragma unroll
        for (int n = 0; n < P::NP; ++n) {
          unsigned char* kr = img + n * (TH / P::PR) * (D * 2);
          if (P::NPK >= TH || tid < P::NPK) {
            if constexpr (B == 4) {
#pragma unroll
              for (int i = 0; i < 4; ++i) *reinterpret_cast<h16x8*>(kr + (ka0 ^ (i << 4))) = unpack4_high(rk[n][i]);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i)
                *reinterpret_cast<h16x8*>(kr + (ka0 ^ (i << 4))) = unpack8(rk[n][2 * i], rk[n][2 * i + 1]);
            }
          }
        }
        // values: a dim's 16 tokens stand as 0-3, 8-11 and 4-7, 12-15: one read has a lane's eight
        const int dim = tid / P::U, uu = tid % P::U;
        const int va0 = dim * (NT * 2) + (va_turn<NT>(dim, B == 4 ? 2 * uu : uu & ~1) << 4) + (B == 4 ? 0 : 8 * (uu & 1));
#pragma unroll
        for (int n = 0; n < P::NPV; ++n) {
          unsigned char* vr = img + oV + n * (TH / P::U) * (NT * 2);
          if constexpr (B == 4) {
            const u32x4 x = __builtin_bit_cast(u32x4, unpack4_high(ru[n][0]));
            const u32x4 y = __builtin_bit_cast(u32x4, unpack4_high(ru[n][1]));
            *reinterpret_cast<u32x4*>(vr + va0) = u32x4{x[0], x[1], y[0], y[1]};
            *reinterpret_cast<u32x4*>(vr + (va0 ^ 16)) = u32x4{x[2], x[3], y[2], y[3]};
          } else {  // (a unit is the first or the second half of its 16)
            const u32x4 x = __builtin_bit_cast(u32x4, unpack8(ru[n][0], ru[n][1]));
            *reinterpret_cast<u32x2*>(vr + va0) = u32x2{x[0], x[1]};
            *reinterpret_cast<u32x2*>(vr + (va0 ^ 16)) = u32x2{x[2], x[3]};
          }
        }
        if (wv == 0) {
          float* ksf = reinterpret_cast<float*>(img + oSc);
          float *vsf = ksf + G * NT, *vbf = vsf + G * NT;
          h16* kbe = reinterpret_cast<h16*>(vbf + G * NT);
          // scales of keys past the tile's last one or on an invalid page (which may hold anything) as zeros
          const int pc = min((int)lane, P::NPS - 1), t8 = 8 * (pc % (NT / 8)), seg = pc / (NT / 8), arr = seg / G,
                    g = seg % G;
          const int live = k_hi + 1 - pos_of_block(st) - t8;
          u32x4 x = rs;
          if (live < 8 || !((okn >> t8) & 1)) {
            const int n = (okn >> t8) & 1 ? live : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= (2 * e < n ? 0x0000FFFFu : 0u) | (2 * e + 1 < n ? 0xFFFF0000u : 0u);
          }
          int vm = 0;  // largest |v_scale|, as fp16 bits
          if (arr == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vm = max(vm, (int)max(x[e] & 0x7FFFu, (x[e] >> 16) & 0x7FFFu));
          }
          // the accumulator's exponent follows the value scales' (exact powers of two; 6 binades of slack)
          const int ex = ((int)wave_max((float)vm) >> 10) - 15;
          if (ex > vex || ex < vex - 6) vex = ex;
          if (lane == 0) *reinterpret_cast<int*>(img + oSc + P::SCB) = vex;
          if (lane < P::NPS) {
            const float f = arr == 0   ? (float)(1 << C::kCodeExp)
                            : arr == 2 ? __uint_as_float((uint32_t)(127 - vex) << 23)
                                       : 1.f;
            const h16x8 hv = __builtin_bit_cast(h16x8, x);
            if (arr == 1) {
#pragma unroll
              for (int e = 0; e < 8; ++e) *reinterpret_cast<h16x2*>(kbe + 8 * (t8 + e) + 2 * g) = h16x2{hv[e], hv[e]};
            } else {
              float* dst = (arr == 0 ? ksf : arr == 2 ? vsf : vbf) + g * NT + t8;
#pragma unroll
              for (int q = 0; q < 2; ++q)
                *reinterpret_cast<f32x4*>(dst + 4 * q) = f32x4{(float)hv[4 * q] * f, (float)hv[4 * q + 1] * f,
                                                               (float)hv[4 * q + 2] * f, (float)hv[4 * q + 3] * f};
            }
          }
        }
      } else if constexpr (DMA) {
        dma_wait();
      } else {
        static_assert(TH / P::PR % 16 == 0, "a thread's next rows are turned as its first");
        const int row = tid / P::PR, c = tid % P::PR * 2;
        const int ka0 = row * (D * 2) + (k_turn<D>(row, c) << 4), va0 = oV + row * (D * 2) + (v_turn<D>(row, c) << 4);
#pragma unroll
        for (int n = 0; n < P::NP; ++n) {
          unsigned char* rows = img + n * (TH / P::PR) * (D * 2);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            auto wide8 = [&](const u32x4 x) {
              return as_h8(e4m3x2_to_h16x2(__builtin_amdgcn_perm(0u, x[2 * e], 0x0C010C00u)),
                           e4m3x2_to_h16x2(__builtin_amdgcn_perm(0u, x[2 * e], 0x0C030C02u)),
                           e4m3x2_to_h16x2(__builtin_amdgcn_perm(0u, x[2 * e + 1], 0x0C010C00u)),
                           e4m3x2_to_h16x2(__builtin_amdgcn_perm(0u, x[2 * e + 1], 0x0C030C02u)));
            };
            *reinterpret_cast<h16x8*>(rows + (ka0 ^ (e << 4))) = wide8(rk[n]);
            *reinterpret_cast<h16x8*>(rows + (va0 ^ (e << 4))) = wide8(rv[n]);
          }
        }
        if (wv == 0) {
          // value scales enter with the probabilities, brought near 1 by a power of two that the accumulator carries
          const float vmax = wave_max(psv);
          const int ex = min(max((int)((__float_as_uint(vmax) >> 23) & 0xFFu) - 127, -60), 60);
          if (ex > vex || ex < vex - 6) vex = ex;
          if (lane == 0) *reinterpret_cast<int*>(img + oSc + P::SCB) = vex;
          float* ksf = reinterpret_cast<float*>(img + oSc);
          if (lane < NT) {
            ksf[lane] = psk * 256.f;
            ksf[NT + lane] = psv * __uint_as_float((uint32_t)(127 - vex) << 23);
          }
        }
      }
    };

    int blk0 = 0, blk1 = 0;
    if (st_lo < st_hi) {
      blk0 = page_id(st_lo);
      blk1 = page_id(min(st_lo + 1, st_hi - 1));
    }
    __syncthreads();  // (the last segment's LDS is free)
    if (tree_lds) {
      for (int i = tid; i <= tok_hi; i += TH) lpar[i] = parent_of(par, i);
      __syncthreads();
    }
    if (st_lo < st_hi) load_block(st_lo, blk0, 0);

    // ---- this lane's column
    int tok, head;
    masked_column(A, sq, tile, cw * 32 + c32, HG, tok, head);
    const bool busy = P::DW > 1 || __any(tok >= 0);  // (waves that meet in a block all take part)
    int cur = tree ? tok : -1, back = 0;  // tree: the cursor, and how many steps above the column's node it is
    int depth = 0;
    if (tree && mask.window > 0)
      for (int i = tok; i >= 0 && (i = up(i)) >= 0;) ++depth;
    const int place = past + (tree ? depth : tok);
    const int limit = tok < 0 ? -1 : tree ? past - 1 : place;  // last key of those outside the tree
    const int start = mask.window > 0 ? max(0, place - mask.window + 1) : 0;
    int lim_lo = tok >= 0 ? limit : 0x7FFFFFFF, start_hi = tok >= 0 ? start : 0;  // over the wave's columns
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, 64));
      start_hi = max(start_hi, __shfl_xor(start_hi, o, 64));
    }
    lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
    start_hi = __builtin_amdgcn_readfirstlane(start_hi);

    // ---- query operands (zeros for absent columns)
    Op qB[KS];
    Op qbias = Op{};  // affine: the query's sum over each group as fp16 hi + lo at 2 g, 2 g + 1 (lanes of half 0)
    {
      const bool ok = tok >= 0;
      const QT* qp = reinterpret_cast<const QT*>(a.q) +
                     ((size_t)(ok ? q0 + tok : 0) * a.Hq + (size_t)kvh * HG + (ok ? head : 0)) * D + 16 * KS * dw + 8 * half;
      float gsum[GV] = {};
#pragma unroll
      for (int w2 = 0; w2 < KS; ++w2) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 16 * w2);
        const Op v = __builtin_bit_cast(Op, ok ? x : u32x4{0u, 0u, 0u, 0u});
        if constexpr (AFF) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            qB[w2][i] = v[slot_perm<C::kBits>(i)];  // the unpacked codes' order
            gsum[w2 * GV / KS] += (float)v[i];
          }
        } else {
          qB[w2] = v;
        }
      }
      if constexpr (AFF) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float x = gsum[g % GV] + __shfl_xor(gsum[g % GV], 32, 64);
          const h16 hi = (h16)x;
          if (half == 0 && g / GV == dw) {
            qbias[2 * g] = hi;
            qbias[2 * g + 1] = (h16)(x - (float)hi);
          }
        }
      }
    }

    float m_run = -INFINITY, l_part = 0.f;
    f32x16 acc[DT];
    float pb[GV] = {};  // affine: sum p * v_bias
    int vexp = 0;      // FP8, affine: acc holds the sum / 2^vexp
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    if constexpr (AFF) {  // the bias operand's unused halves stay zero
      for (int i = tid; i < 2 * NT; i += TH)
        *reinterpret_cast<u32x4*>(lds + oBuf + (i / NT) * BUF + oSc + 12 * G * NT + 16 * (i % NT)) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    if (st_lo < st_hi) store_block(st_lo, 0);
    __syncthreads();

    for (int st = st_lo; st < st_hi; ++st) {
      const int buf = (st - st_lo) & 1;
      const uint64_t okm = okn;
      if (st + 1 < st_hi) {
        load_block(st + 1, blk1, buf ^ 1);
        blk1 = page_id(min(st + 2, st_hi - 1));
      }
      const unsigned char* img = lds + oBuf + buf * BUF;
      if (busy) {
        const float* ksf = reinterpret_cast<const float*>(img + oSc);
        if constexpr (AFF || FP8) {
          const int ex = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(img + oSc + P::SCB));
          if (ex != vexp) {
            const float f = __uint_as_float((uint32_t)(127 + min(max(vexp - ex, -126), 127)) << 23);
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
            vexp = ex;
          }
        }
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const int ki = oBuf + buf * BUF + kad, vi = oBuf + buf * BUF + vad;
        auto read_k = [&](const int kt, const int w2) {
          return *reinterpret_cast<const Op*>(lds + (ki ^ (w2 << 5)) + kt * 64 * D);
        };
        auto read_v = [&](const int kt, const int j, const int d) {
          if constexpr (AFF) {
            return *reinterpret_cast<const Op*>(lds + (vi ^ ((4 * kt + 2 * j) << 4)) + d * 64 * NT);
          } else {
            const unsigned char* p = lds + (vi ^ (d << 6)) + (32 * kt + 16 * j) * (D * 2);
            const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p)));
            const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 8 * (D * 2))));
            return __builtin_bit_cast(Op, u32x4{v0[0], v0[1], v1[0], v1[1]});
          }
        };
        // ---- S^T, 32 keys at a time, from the last backwards as the cursors go: element i is key 8 (i / 4) + 4 half + i % 4.
        // Operands are read ahead of the products that take them, held in that order by the barriers (the compiler
        // put each read right before its use: a wait of the whole LDS latency per product)
        constexpr int KA = KS < 4 ? KS : 4;  // K operands read ahead
        Op ka[KA];
#pragma unroll
        for (int i = 0; i < KA; ++i) ka[i] = read_k(KT - 1, i);
        f32x16 sc[KT];
#pragma unroll
        for (int kt = KT - 1; kt >= 0; --kt) {
          __builtin_amdgcn_sched_barrier(0);
          const int k0 = (kw * KT + kt) * 32;
          f32x16 c;
          auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < 16; ++i) c[i] = 0.f;
          };
          auto product = [&](const int w2) {
            c = mfma32(ka[w2 % KA], qB[w2], c);
            if (w2 + KA < KS) ka[w2 % KA] = read_k(kt, w2 + KA);
            else if (kt > 0) ka[w2 % KA] = read_k(kt - 1, w2 + KA - KS);
          };
          clear();
          if constexpr (AFF) {
            const h16* kbe = reinterpret_cast<const h16*>(ksf + 3 * G * NT);
            sc[kt] = mfma32(*reinterpret_cast<const Op*>(kbe + 8 * (k0 + c32)), qbias, c);
#pragma unroll
            for (int g = 0; g < GV; ++g) {
              clear();
#pragma unroll
              for (int w2 = g * KS / GV; w2 < (g + 1) * KS / GV; ++w2) product(w2);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const f32x4 ks4 = *reinterpret_cast<const f32x4*>(ksf + (GV * dw + g) * NT + k0 + 8 * j + 4 * half);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[kt][4 * j + r] = fmaf(c[4 * j + r], ks4[r], sc[kt][4 * j + r]);
              }
              __builtin_amdgcn_sched_barrier(0);  // (the scales' reads stay with their group)
            }
          } else {
#pragma unroll
            for (int w2 = 0; w2 < KS; ++w2) product(w2);
            sc[kt] = c;
            if constexpr (FP8) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const f32x4 ks4 = *reinterpret_cast<const f32x4*>(ksf + k0 + 8 * j + 4 * half);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[kt][4 * j + r] *= ks4[r];
              }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (P::DW > 1) {  // the other half of the dims
          f32x4* mine = reinterpret_cast<f32x4*>(lds + oX) + wv * (KT * 256) + lane;
          const f32x4* other = reinterpret_cast<f32x4*>(lds + oX) + (wv ^ (CW * KW)) * (KT * 256) + lane;
#pragma unroll
          for (int i = 0; i < 4 * KT; ++i) {
            const f32x16& x = sc[i / 4];
            mine[i * 64] = f32x4{x[i % 4 * 4], x[i % 4 * 4 + 1], x[i % 4 * 4 + 2], x[i % 4 * 4 + 3]};
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 4 * KT; ++i) {
            const f32x4 y = other[i * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[i / 4][i % 4 * 4 + r] += y[r];
          }
        }

        // ---- mask, where some key is not visible to every column of the wave
        const int kp = pos_of_block(st) + kw * KT * 32;
        const uint64_t okw = okm >> (kw * KT * 32);
        constexpr uint64_t kAll = KT == 2 ? ~0ull : 0xFFFFFFFFull;
        const bool drafted = tree && kp + 32 * KT > past;
        const bool full = !drafted && kp + 32 * KT - 1 <= lim_lo && (kp >= start_hi || kp + 32 * KT <= mask.sinks) &&
                          (okw & kAll) == kAll;
        if (!full) {
#pragma unroll
          for (int kt = KT - 1; kt >= 0; --kt) {
            // bit k: the column sees key k1 + k
            const int k1 = kp + 32 * kt;
            uint32_t see = below(limit + 1 - k1) & (~below(start - k1) | below(mask.sinks - k1));
            if (drafted) {
              while (cur >= 0 && past + cur >= k1) {
                const int b = past + cur - k1;
                if (b < 32 && (mask.window <= 0 || back < mask.window || place - back < mask.sinks)) see |= 1u << b;
                cur = up(cur);
                ++back;
              }
            }
            see = (see & (uint32_t)(okw >> (32 * kt))) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kt][i] = (see >> (8 * (i / 4) + i % 4)) & 1u ? sc[kt][i] : -INFINITY;
          }
        }

        // ---- online softmax: the lane's own scores of its column
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, sc[kt][i]), sc[kt][i + 1]);
        if (__any(top * sl2 > m_run + kLazyMax)) {
          const float m_new = fmaxf(m_run, fmaxf(top, __shfl_xor(top, 32, 64)) * sl2);
          const bool rise = m_new > m_run + kLazyMax;  // also the first finite maximum
          const float al = rise ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
          l_part *= al;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] *= al;
          if constexpr (AFF) {
#pragma unroll
            for (int g = 0; g < GV; ++g) pb[g] *= al;
          }
          if (rise) m_run = m_new;
        }
        // p <= 2^(kLazyMax + 6), times a value scale below 2: inside fp16, and small p stay clear of its sub-normals
        const float m_sub = fmaxf(m_run, -3.0e38f) - 6.f;

        // ---- O^T += V^T P^T in steps of 16 keys (and one group); a step's operands are made while the products of the step
        // before it run
        constexpr int DG = DT / GV, US = KT * 2 * GV;  // dim tiles of a group, steps
        Op va[2][DG], pB[2][2];
        auto make = [&](const int u) {
          const int kt = KT - 1 - u / (2 * GV), j = u / GV % 2, g = u % GV, k0 = (kw * KT + kt) * 32 + 16 * j + 4 * half;
#pragma unroll
          for (int d = 0; d < DG; ++d) va[u & 1][d] = read_v(kt, j, g * DG + d);
          if (g == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sc[kt][8 * j + e] = __builtin_amdgcn_exp2f(fmaf(sc[kt][8 * j + e], sl2, -m_sub));
              l_part += sc[kt][8 * j + e];
            }
          }
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = sc[kt][8 * j + e];
          if constexpr (AFF || FP8) {
            const float *vsf = ksf + (FP8 ? 1 : G + GV * dw + g) * NT + k0, *vbf = vsf + G * NT;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const f32x4 vs4 = *reinterpret_cast<const f32x4*>(vsf + 8 * e);
              if constexpr (AFF) {
                const f32x4 vb4 = *reinterpret_cast<const f32x4*>(vbf + 8 * e);
#pragma unroll
                for (int r = 0; r < 4; ++r) pb[g] = fmaf(x[4 * e + r], vb4[r], pb[g]);
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) x[4 * e + r] *= vs4[r];
            }
          }
          split_p2(x, pB[u & 1]);
        };
        make(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < US; ++u) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < DG; ++d)
              acc[u % GV * DG + d] = mfma32(va[u & 1][d], pB[u & 1][k], acc[u % GV * DG + d]);
          if (u + 1 < US) make(u + 1);
#pragma unroll
          for (int i = 0; i < 2 * DG; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x2, 8, 0);    // what the vector unit does meanwhile
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (st + 1 < st_hi) store_block(st + 1, buf ^ 1);
      __syncthreads();
    }

    if constexpr (AFF) {  // codes entered as code * 2^-kCodeExp; the bias term joins its group's dims
      const float f = __uint_as_float((uint32_t)(127 + vexp + C::kCodeExp) << 23);
#pragma unroll
      for (int g = 0; g < GV; ++g) {
        const float bias = pb[g] + __shfl_xor(pb[g], 32, 64);
#pragma unroll
        for (int d = g * DT / GV; d < (g + 1) * DT / GV; ++d) acc[d] = acc[d] * f + bias;
      }
    }
    if constexpr (FP8) {  // the codes entered as value * 2^-8
      const float f = __uint_as_float((uint32_t)(127 + vexp + 8) << 23);
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= f;
    }
    float l = l_part + __shfl_xor(l_part, 32, 64);

    // ---- KW = 2: the second key wave's state joins the first's
    if constexpr (KW > 1) {
      f32x4* meet = reinterpret_cast<f32x4*>(lds + oBuf) + (size_t)cw * (4 * DT + 1) * 64 + lane;
      if (kw == 1) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            meet[(4 * d + j) * 64] = f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
        meet[4 * DT * 64] = f32x4{m_run, l, 0.f, 0.f};
      }
      __syncthreads();
      if (kw == 0) {
        const f32x4 o = meet[4 * DT * 64];
        const float M = fmaxf(m_run, o[0]);
        // (a wave without a live key has m = -inf and zeros, one of NaN scores only a sum that is NaN)
        const float f0 = m_run == -INFINITY ? (l == 0.f ? 0.f : l) : __builtin_amdgcn_exp2f(m_run - M);
        const float f1 = o[0] == -INFINITY ? (o[1] == 0.f ? 0.f : o[1]) : __builtin_amdgcn_exp2f(o[0] - M);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 y = meet[(4 * d + j) * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[d][4 * j + r] = acc[d][4 * j + r] * f0 + y[r] * f1;
          }
        l = l * f0 + o[1] * f1;
        m_run = M;
      }
    }

    const bool whole = b0 == 0 && b1 == nblk;
    if (nwg > 0 && b0 == 0) {
      const int g0 = ranges.begin(w + 1) - todo - u0;  // the tile's first unit in the launch
      if (!whole)
        cut_tile = int4{sq.s, tile, kvh * kWideParts + ranges.owner(g0 + kWideBegin + nblk - 1) - w + 1,
                        2 * w + (first_seg ? 0 : 1)};
      if (by_tile && tid == 0) A.desc[1 + kvh * A.tiles + t] = cut_tile;
    }
    if (kw == 0) {
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        bool bad = false;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            bad |= masked_write<C, D>(a, sq, kvh, tok, head,
                                      f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]}, l,
                                      inv, 32 * (dw * DT + d) + 8 * j + 4 * half);
        uint64_t again = __ballot(bad);
        again = (again | (again >> 32)) & 0xFFFFFFFFull;
        if (again) {
          __builtin_amdgcn_s_waitcnt(0);  // (the rows' first results are out before their second)
          for (; again; again &= again - 1) {
            const int c = __builtin_ctzll(again);
            attend_masked<C, D>(a, mask, sq, kvh, __builtin_amdgcn_readlane(tok, c), __builtin_amdgcn_readlane(head, c),
                                lane, dw * DT * 32, (dw + 1) * DT * 32);
          }
        }
      } else {
        f32x4* st = reinterpret_cast<f32x4*>(A.part + (size_t)(2 * w + (first_seg ? 0 : 1)) * kWidePart<D, CW>) +
                    (size_t)cw * (D / 8 + 1) * 64 + lane;
        if (tok >= 0) {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              st[(4 * (dw * DT + d) + j) * 64] = f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
        }
        if (dw == 0) st[(D / 8) * 64] = f32x4{m_run, l, 0.f, 0.f};
      }
    }
    first_seg = false;
    if (nwg == 0) return;
    todo -= u1 - u0;
    u0 = 0;
    if (++t == ntiles) {
      t = 0;
      ++kvh;
      sidx = 0;
    }
  }
  if (!by_tile && tid == 0) A.desc[1 + w] = cut_tile;
}

// Joins the parts of cut tiles, in part order.  Grid (descriptors, column waves, dims / 32 NV): a wave has 32 columns and 8 NV
// dims of one tile, its workgroup 32 NV.  Bound by the parts' way to memory and back (256 columns: 131 KB each): NV = 4, 192
// tiles in two or three parts 17 us (NV = 1 with eight loads a round however few the parts: 34), but NV = 1 where
// descriptors are few and their parts many: a tree of 25 nodes in 24 parts 5.4 us against 7.8.
template <class C, int D, int CW, int NV>
__global__ __launch_bounds__(NV * 32 > D ? 8 * D / NV : 256) void masked_merge(MaskedArgs A) {
  const DecodeArgs& a = A.d;
  const int lane = threadIdx.x & 63, cw = blockIdx.y;
  const int v0 = (blockIdx.z * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * NV;  // dims 8 v0 ..
  const bool by_tile = a.Hkv * A.tiles <= A.wgs;
  // (descriptors in the order of the workgroups that wrote the parts, XCD by XCD)
  const int n = gridDim.x, id = n % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * (n / 8) + (int)blockIdx.x / 8;
  const int4 de = A.desc[1 + id];
  if ((by_tile ? id % A.tiles : id) >= A.desc[0].x) return;
  const int np = de.z % kWideParts, kvh = de.z / kWideParts;
  if (np == 0) return;
  const int c32 = lane & 31, half = lane >> 5;
  const f32x4* base = reinterpret_cast<const f32x4*>(A.part) + (size_t)cw * (D / 8 + 1) * 64 + lane;
  // the first part's slot, then the first slots of the workgroups that follow
  const int slot0 = de.w, next0 = (de.w | 1) + 1;
  auto slot = [&](const int q) { return (size_t)(q == 0 ? slot0 : next0 + 2 * (q - 1)) * (kWidePart<D, CW> / 4); };
  const MaskedSeq sq = masked_seq(A, de.x);
  int tok, head;
  masked_column(A, sq, de.y, cw * 32 + c32, a.Hq / a.Hkv, tok, head);
  if (!__any(tok >= 0)) return;
  float m = -INFINITY, l = 0.f;
  f32x4 o[NV] = {};
  auto join = [&](auto parts) {
    constexpr int U = decltype(parts)::value;
    for (int q0 = 0; q0 < np; q0 += U) {
      f32x4 x[U][NV];
      f32x2 ml[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        ml[k] = f32x2{-INFINITY, 0.f};
        if (q0 + k < np) {
          const f32x4* st = base + slot(q0 + k);
          ml[k] = *reinterpret_cast<const f32x2*>(st + (D / 8) * 64);
#pragma unroll
          for (int j = 0; j < NV; ++j) x[k][j] = st[(v0 + j) * 64];  // (a column that is none holds anything)
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < U; ++k) top = fmaxf(top, ml[k][0]);
      // (a part without a live key has m = -inf and zeros, one of NaN scores only a sum that is NaN)
      auto weight = [&](const float m1, const float l1) {
        return m1 == -INFINITY ? (l1 == 0.f ? 0.f : l1) : __builtin_amdgcn_exp2f(m1 - top);
      };
      const float f0 = weight(m, l);
      l *= f0;
#pragma unroll
      for (int j = 0; j < NV; ++j) o[j] *= f0;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (q0 + k < np) {
          const float f = weight(ml[k][0], ml[k][1]);
          l = fmaf(ml[k][1], f, l);
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][r] = fmaf(x[k][j][r], f, o[j][r]);
        }
      }
      m = top;
    }
  };
  np <= 3 ? join(std::integral_constant<int, 3>{}) : join(std::integral_constant<int, 8>{});
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < NV; ++j) bad |= masked_write<C, D>(a, sq, kvh, tok, head, o[j], l, inv, 8 * (v0 + j) + 4 * half);
  // rows that are not finite here: these dims again in fp32
  uint64_t again = __ballot(bad);
  again = (again | (again >> 32)) & 0xFFFFFFFFull;
  if (again) {
    __builtin_amdgcn_s_waitcnt(0);  // (the rows' first results are out before their second)
    for (; again; again &= again - 1) {
      const int c = __builtin_ctzll(again);
      attend_masked<C, D>(a, A.mask, sq, kvh, __builtin_amdgcn_readlane(tok, c), __builtin_amdgcn_readlane(head, c), lane,
                          8 * v0, 8 * (v0 + NV));
    }
  }
}

}  // namespace emx
