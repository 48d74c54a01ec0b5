// Masked paged attention (masked_launch.hpp: sliding windows with sinks, drafted trees) on the
// matrix units: head_dim 64, 128 or 256, any GQA ratio up to the columns of a tile, over
// token-major caches [nb, bs, Hkv, D] (fp16 / bf16, FP8 E4M3 with one fp32 scale per page; pages
// of a multiple of 8 tokens) and over affine pages.
//
//   O_i = sum_k p_ik V_k / sum_k p_ik,  p_ik = 2^(scale log2(e) q_i . K_k - m_i) over the keys k
//   that row i sees,
//
// in one pass over the keys with the running maximum m_i.
//
// Work: a tile is the 64 CT query columns (token, head), head fastest, of COLS / HG tokens of one
// sequence and kv head; its keys go in blocks of NT positions, from the last backwards and then the
// sinks' blocks: those between the sinks and the earliest window are not read.  From the last
// backwards because a drafted node's ancestors then come in the order of its walk to the root: each
// lane keeps one cursor per column, and a block of drafted keys costs as many steps as it holds
// ancestors, for trees of any size.  One workgroup (4 waves) takes one unit, a tile or one of the
// equal parts of its blocks: masked_plan counts the launch's blocks on the device and cuts the tiles
// of a sequence so that no part is much longer than an even share of the grid.  Parts leave their
// fp32 state (accumulator, maximum, sum) and masked_merge joins them in part order.
//
// A block, as in prefill_mfma.hpp: K and V rows are loaded once per workgroup a block ahead, go to
// LDS as 16-bit values (FP8: dec(code) * 2^-8, exact; affine codes as exact sub-normals, scale and
// bias applied in fp32), and each wave takes S^T = K Q^T, the softmax of its columns and
// O^T += V^T P^T on v_mfma 16x16x32, the probabilities entering as the sum of two 16-bit parts
// (fp16: 22 bits of the 24; bf16: 16, which puts an output off by at most 2^-17 of the largest value it
// averages, a five-hundredth of the output's own rounding).  Waves without a column skip the products.
#pragma once

#include "masked_launch.hpp"
#include "prefill_mfma.hpp"

namespace emx {

// Probabilities as two 16-bit parts (mfma_common.hpp has three for bf16), each the nearest.
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
  int tiles;        // tiles per kv head the grid has room for
  int share_of;     // units per kv head the launch's blocks are spread over, 0: tiles are not cut
  int units;        // units per kv head the grid has room for
  float* part;      // [units * Hkv][part bytes]
};

// Fewest blocks of a part: cutting costs a part's state out and back (64 KiB each way at D 128,
// as much as two blocks' K and V).
constexpr int kMaskedPartBlocks = 8;

// A tile's blocks: positions [hi NT - .., ..] backwards from block `hi`, `n` in all, the last `sink` of
// them the blocks 0 .. sink - 1.
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

struct MaskedUnit {
  int s, q0, qlen, past;  // the sequence
  int tile, part, nparts; // nparts: the sequence's; a tile of few blocks has fewer
  int first;              // unit of the tile's part 0
  int live;               // 0: no such unit (past the launch's last)
  int units;              // of the launch, per kv head
};

// Unit `u` of the launch (`by_tile`: the unit of part 0 of the launch's tile `u`).  The workgroup counts it: a thread
// has ch sequences in order.  wred: 16 ints of LDS.
template <int NT>
__device__ __forceinline__ MaskedUnit masked_plan(const MaskedArgs& A, const int u, const bool by_tile, int* wred) {
  const DecodeArgs& a = A.d;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int ch = (a.S + 255) / 256, s0 = tid * ch;
  auto seq = [&](const int s, int& q0, int& qlen, int& past, int& tiles) {
    q0 = a.qsl ? a.qsl[s] : s;
    qlen = a.qsl ? (q0 < 0 ? 0 : max(a.qsl[s + 1] - q0, 0)) : 1;
    past = min(max(a.kv_lens[s], 0), a.max_blocks * a.bs) - qlen;
    tiles = (qlen + A.tokb - 1) / A.tokb;
  };
  // blocks of a sequence's last tile (the longest), and of all tiles: about the mean of the first and the last
  auto longest = [&](const int qlen, const int past, const int tiles) {
    return tiles > 0 ? masked_span<NT>(A.mask, past, (tiles - 1) * A.tokb, qlen - 1).n : 0;
  };
  int share = 0;
  if (A.share_of > 0) {
    float sum = 0.f;
    for (int i = 0; i < ch && s0 + i < a.S; ++i) {
      int q0, qlen, past, tiles;
      seq(s0 + i, q0, qlen, past, tiles);
      if (tiles > 0)
        sum += 0.5f * tiles *
               (longest(qlen, past, tiles) + masked_span<NT>(A.mask, past, 0, min(A.tokb, qlen) - 1).n);
    }
    sum = wave_sum(sum);
    if (lane == 0) wred[wv] = __float_as_int(sum);
    __syncthreads();
    sum = __int_as_float(wred[0]) + __int_as_float(wred[1]) + __int_as_float(wred[2]) + __int_as_float(wred[3]);
    share = max(kMaskedPartBlocks, (int)ceilf(sum / (float)A.share_of));
  }
  auto parts_of = [&](const int n) { return share > 0 ? max(1, (n + share - 1) / share) : 1; };
  int mine = 0, tmine = 0;
  for (int i = 0; i < ch && s0 + i < a.S; ++i) {
    int q0, qlen, past, tiles;
    seq(s0 + i, q0, qlen, past, tiles);
    mine += tiles * parts_of(longest(qlen, past, tiles));
    tmine += tiles;
  }
  int x = mine, y = tmine;  // inclusive scans: units, tiles
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x1 = __shfl_up(x, o, 64), y1 = __shfl_up(y, o, 64);
    if (lane >= o) {
      x += x1;
      y += y1;
    }
  }
  if (lane == 63) {
    wred[4 + wv] = x;
    wred[8 + wv] = y;
  }
  __syncthreads();
  int xb = 0, yb = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wv) {
      xb += wred[4 + w];
      yb += wred[8 + w];
    }
    total += wred[4 + w];
  }
  int run = xb + x - mine, trun = yb + y - tmine;
  __shared__ MaskedUnit found;
  if (tid == 0) found.live = 0;
  __syncthreads();
  const int at = by_tile ? trun : run, have = by_tile ? tmine : mine;
  if (u >= at && u < at + have) {
    for (int i = 0; i < ch && s0 + i < a.S; ++i) {
      MaskedUnit f;
      int tiles;
      seq(s0 + i, f.q0, f.qlen, f.past, tiles);
      f.nparts = parts_of(longest(f.qlen, f.past, tiles));
      const int o = by_tile ? (u - trun) * f.nparts : u - run;
      if (o < tiles * f.nparts) {
        f.s = s0 + i;
        f.tile = tiles - 1 - o / f.nparts;  // the longest first
        f.part = o % f.nparts;
        f.first = run + o - f.part;
        f.live = 1;
        found = f;
        break;
      }
      run += tiles * f.nparts;
      trun += tiles;
    }
  }
  __syncthreads();
  MaskedUnit r = found;
  int* w = reinterpret_cast<int*>(&r);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(MaskedUnit) / 4); ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
  r.units = total;
  return r;
}

// Parts a tile of n blocks has, of the most a tile of its sequence has.
__device__ __forceinline__ int masked_parts(const int n, const int most) {
  return min(most, max(1, (n + kMaskedPartBlocks - 1) / kMaskedPartBlocks));
}

// One query row in fp32 on one wave over every key that it sees: rows whose result on the matrix unit is not
// finite are computed again here (there a key that the row does not see still enters its tile's product with p = 0,
// and 0 * inf makes NaN of what these rules leave alone).  64 keys at a time, as attend_row (mfma_common.hpp).
template <class C, int D>
__device__ void attend_masked(const DecodeArgs& a, const MaskRule& mask, const int32_t* par, const int s, const int kvh,
                              const typename C::QT* q, const int past, const int i, float& l, float (&acc)[D / 64],
                              const int lane) {
  constexpr int N = D / 64;
  const auto kv = kv_loader<C>(a, D);
  const int depth = par && mask.window > 0 ? node_depth(par, i) : 0;
  float qv[N], m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    qv[n] = to_f32(q[lane + 64 * n]);
    acc[n] = 0.f;
  }
#pragma unroll 1
  for (int base = 0; base <= past + i; base += 64) {
    const int k = base + lane;
    const bool see = k <= past + i && key_visible(mask, par, past, i, depth, k);
    const int blk = see ? a.block_tables[(size_t)s * a.max_blocks + k / a.bs] : -1;
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
}

// The tile's columns that are not finite, again in fp32: `bad` holds for a lane of a column (token ctok, head chead).
template <class C, int D>
__device__ __forceinline__ void masked_again(const DecodeArgs& a, const MaskRule& mask, const int32_t* par,
                                             const MaskedUnit& u, const int kvh, const bool bad, const int ctok,
                                             const int chead, const int lane) {
  typedef typename C::QT QT;
  const int HG = a.Hq / a.Hkv;
  uint64_t todo = __ballot(bad && ctok >= 0);
  todo = (todo | (todo >> 16) | (todo >> 32) | (todo >> 48)) & 0xFFFFu;
  while (todo) {
    const int c = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int t = __builtin_amdgcn_readlane(ctok, c), hh = __builtin_amdgcn_readlane(chead, c);
    const size_t ro = ((size_t)(u.q0 + t) * a.Hq + (size_t)kvh * HG + hh) * D;
    float lr, x[D / 64];
    attend_masked<C, D>(a, mask, par, u.s, kvh, reinterpret_cast<const QT*>(a.q) + ro, u.past, t, lr, x, lane);
    const float li = lr > 0.f || lr != lr ? 1.f / lr : 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) from_f32(x[i] * li, reinterpret_cast<QT*>(a.out) + ro + lane + 64 * i);
  }
}

// Column c of a tile: which token and head, -1 where there is none.
__device__ __forceinline__ void masked_column(const MaskedArgs& A, const MaskedUnit& u, const int c, const int HG,
                                              int& ctok, int& chead) {
  const int t = c / HG;
  ctok = u.tile * A.tokb + t;
  chead = c - t * HG;
  if (t >= A.tokb || ctok >= u.qlen || (unsigned)(u.q0 + ctok) >= (unsigned)A.T) ctok = -1;
}

// Bytes of one part's state: per wave CT (D / 16) + 1 vectors of 16 bytes a lane.
template <int D, int CT>
constexpr int kMaskedPartBytes = 4 * (CT * (D / 16) + 1) * 64 * 16;

// Lane (col, jj) of a wave holds dims 16 b + 4 jj + r of its columns: normalised and written.  True where a value is
// not finite.
template <class C, int D>
__device__ __forceinline__ bool masked_write(const DecodeArgs& a, const MaskedUnit& u, const int kvh, const int ctok,
                                             const int chead, const f32x4 o, const float l, const int dim) {
  typedef typename C::QT QT;
  struct alignas(8) Four {
    QT x[4];
  } v;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bool bad = not_finite(l);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bad = bad || not_finite(o[r]);
    from_f32(o[r] * inv, &v.x[r]);
  }
  if (ctok >= 0)
    *reinterpret_cast<Four*>(reinterpret_cast<QT*>(a.out) +
                             ((size_t)(u.q0 + ctok) * a.Hq + (size_t)kvh * (a.Hq / a.Hkv) + chead) * D + dim) = v;
  return bad;
}

constexpr int kMaskedTreeLds = 1024;  // nodes of a tree whose parents are kept in LDS

template <class C, int D, int CT>
__global__ __launch_bounds__(256, 2) void masked_mfma(MaskedArgs A) {
  using P = PrefillMfmaCfg<C, D, CT>;
  typedef typename C::Op Op;
  typedef typename C::QT QT;
  const DecodeArgs& a = A.d;
  constexpr int NT = P::NT;
  constexpr int PARTB = kMaskedPartBytes<D, CT>;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, jj = lane >> 4;

  // LDS: one array of the size needed (not the shared arena: three workgroups fit a compute unit)
  constexpr bool AFF = C::kAffine;
  constexpr int G = [] {
    if constexpr (C::kAffine) return P::G;
    return 1;
  }();
  constexpr int oPar = 0, oWred = lds_next(oPar, 4 * kMaskedTreeLds), oKe = lds_next(oWred, 64);
  constexpr int oVe = lds_next(oKe, 2 * NT * P::KSTR), oKsf = lds_next(oVe, 2 * (AFF ? D : NT) * P::VSTR);
  constexpr int oVsf = lds_next(oKsf, 4 * G * NT), oVbf = lds_next(oVsf, 4 * G * NT);
  constexpr int oKbe = lds_next(oVbf, AFF ? 4 * G * NT : 0), oEnd = lds_next(oKbe, AFF ? 16 * NT : 0);
  __shared__ __attribute__((aligned(16))) unsigned char lds[oEnd];
  int* lpar = reinterpret_cast<int*>(lds + oPar);
  int* wred = reinterpret_cast<int*>(lds + oWred);
  uint16_t* ke = reinterpret_cast<uint16_t*>(lds + oKe);  // [key][KSTR]
  uint16_t* ve = reinterpret_cast<uint16_t*>(lds + oVe);  // [key][VSTR]; affine: [dim][VSTR]
  float* ksf = reinterpret_cast<float*>(lds + oKsf);      // key scale of each key; affine: [group][NT], * 2^kCodeExp
  float* vsf = reinterpret_cast<float*>(lds + oVsf);      // value scales / 2^vexp
  float* vbf = reinterpret_cast<float*>(lds + oVbf);      // affine: value biases
  h16* kbe = reinterpret_cast<h16*>(lds + oKbe);          // affine: bias operand rows, key bias of group g at 2 g, 2 g + 1

  const int kvh = blockIdx.x % a.Hkv, bid = blockIdx.x / a.Hkv;
  const MaskedUnit u = masked_plan<NT>(A, bid, false, wred);
  if (!u.live) {
    if (a.qsl) zero_other_rows<QT>(a, A.T, D, blockIdx.x - u.units * a.Hkv, (A.units - u.units) * a.Hkv);
    return;
  }
  const int s = u.s, q0 = u.q0, past = u.past;
  const int HG = a.Hq / a.Hkv;
  const MaskRule mask = A.mask;
  const int32_t* par = mask.parents ? mask.parents + q0 : nullptr;
  const int tok_lo = u.tile * A.tokb, tok_hi = min(min(tok_lo + A.tokb, u.qlen), A.T - q0) - 1;
  const MaskedSpan span = masked_span<NT>(mask, past, tok_lo, tok_hi);
  const int nparts = masked_parts(span.n, u.nparts);
  if (u.part >= nparts) return;
  const int st_lo = u.part * span.n / nparts, st_hi = (u.part + 1) * span.n / nparts;  // blocks [st_lo, st_hi)
  const int k_hi = past + tok_hi;
  auto block_of = [&](const int st) {
    const int lo = span.n - span.sink;
    return st < lo ? span.hi - st : span.sink - 1 - (st - lo);
  };

  // ---- a tree's parents to LDS (trees of up to kMaskedTreeLds nodes)
  const bool tree = par != nullptr, tree_lds = tree && u.qlen <= kMaskedTreeLds;
  if (tree_lds) {
    for (int i = tid; i <= tok_hi; i += 256) lpar[i] = parent_of(par, i);
    __syncthreads();
  }
  auto up = [&](const int i) { return tree_lds ? lpar[i] : parent_of(par, i); };

  // ---- this lane's query columns
  int ctok[CT], chead[CT], limit[CT], start[CT], place[CT];
  int cur[CT], back[CT];  // tree: the cursor, and how many steps above the column's node it is
  bool any = false;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    masked_column(A, u, (ct * 4 + wv) * 16 + col, HG, ctok[ct], chead[ct]);
    any = any || ctok[ct] >= 0;
    cur[ct] = tree ? ctok[ct] : -1;
    back[ct] = 0;
    int depth = 0;
    if (tree && mask.window > 0)
      for (int i = ctok[ct]; i >= 0 && (i = up(i)) >= 0;) ++depth;
    place[ct] = past + (tree ? depth : ctok[ct]);
    limit[ct] = ctok[ct] < 0 ? -1 : tree ? past - 1 : place[ct];  // last key of those outside the tree
    start[ct] = mask.window > 0 ? max(0, place[ct] - mask.window + 1) : 0;
  }
  const bool busy = __any(any);

  // ---- query operands (zeros for absent columns)
  Op qB[CT][P::KS];
  Op qbias[CT];  // affine, lane group 0: the query's sum over each group as fp16 hi + lo at 2 g, 2 g + 1
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const bool ok = ctok[ct] >= 0;
    const QT* qp = reinterpret_cast<const QT*>(a.q) +
                   ((size_t)(ok ? q0 + ctok[ct] : 0) * a.Hq + (size_t)kvh * HG + (ok ? chead[ct] : 0)) * D + 8 * jj;
    float gsum[G] = {};
#pragma unroll
    for (int w = 0; w < P::KS; ++w) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 32 * w);
      const Op v = __builtin_bit_cast(Op, ok ? x : u32x4{0u, 0u, 0u, 0u});
      if constexpr (AFF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          qB[ct][w][i] = v[slot_perm<C::kBits>(i)];  // the unpacked codes' order
          gsum[32 * w / C::kGS] += (float)v[i];
        }
      } else {
        qB[ct][w] = v;
      }
    }
    if constexpr (AFF) {
      qbias[ct] = Op{};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float x = rows4_sum(gsum[g]);
        const h16 hi = (h16)x;
        if (jj == 0) {
          qbias[ct][2 * g] = hi;
          qbias[ct][2 * g + 1] = (h16)(x - (float)hi);
        }
      }
    }
  }

  // ---- pages: lane l holds the page id of key l of a block (positions past the tile's last key repeat it)
  const size_t rowb = (size_t)a.Hkv * D * sizeof(typename C::ET);  // token-major
  const char* kbase = reinterpret_cast<const char*>(a.kc) + (AFF ? 0 : (size_t)kvh * (D * sizeof(typename C::ET)));
  const char* vbase = reinterpret_cast<const char*>(a.vc) + (AFF ? 0 : (size_t)kvh * (D * sizeof(typename C::ET)));
  const int32_t* bt = a.block_tables + (size_t)s * a.max_blocks;
  auto page_id = [&](const int st) {
    return bt[page_of(min(block_of(st) * NT + (lane & (NT - 1)), k_hi), A.inv_bs)];
  };
  u32x4 rk[P::NP], rv[P::NP];  // the next block's pieces
  u32x2 ru[AFF ? 8 : 1];       // affine: its V units
  u32x4 rs;                    // affine: scale piece `lane` (every wave loads them: the largest scale is a wave's business)
  uint64_t okn = 0;            // keys of that block on a valid page
  float psk = 0.f, psv = 0.f;  // FP8: page scales of key `lane` of that block
  auto load_step = [&](const int st, const int blk) {
    const int pos = min(block_of(st) * NT + (lane & (NT - 1)), k_hi);
    const bool ok = (unsigned)blk < (unsigned)a.nb;
    okn = __ballot(ok);
    const int b = ok ? blk : 0;
    const int off = pos - page_of(pos, A.inv_bs) * a.bs;
    if constexpr (AFF) {
      constexpr int B = C::kBits;
      const int row = (b * a.Hkv + kvh) * a.bs + off;
      {
        const int pc = min(lane, P::NPS - 1), seg = pc / (NT / 8), arr = seg / G, g = seg % G;
        const int r8 = __shfl(row, 8 * (pc % (NT / 8)), 64), o8 = __shfl(off, 8 * (pc % (NT / 8)), 64);
        const h16 *b_ks = a.ks, *b_kb = a.kb, *b_vs = a.vs, *b_vb = a.vb;
        asm("" : "+s"(b_ks), "+s"(b_kb), "+s"(b_vs), "+s"(b_vb));  // picked from registers, not by a vector load
        const h16* base = arr == 0 ? b_ks : arr == 1 ? b_kb : arr == 2 ? b_vs : b_vb;
        typedef const __attribute__((address_space(1))) u32x4* gu32x4;
        // (past the tile's last key the group's first token may repeat it: aligned down, inside the page)
        rs = *(gu32x4)(base + (size_t)G * (r8 - o8) + (size_t)g * a.bs + (o8 & ~7));
      }
#pragma unroll
      for (int n = 0; n < P::NP; ++n) {
        const int e = tid + 256 * n;  // (fewer than 256 pieces: the others repeat them)
        const int r = __shfl(row, (e / P::PR) & (NT - 1), 64);
        rk[n] = *reinterpret_cast<const u32x4*>(kbase + (size_t)r * P::RBK + 16 * (e % P::PR));
      }
      const int T = min(a.bs, 256 / B);  // tokens of a value tile (a power of two)
#pragma unroll
      for (int n = 0; n < P::NPV; ++n) {
        const int e = tid + 256 * n, uu = e % P::U, dim = e / P::U;
        const int r = __shfl(row, uu * P::UT, 64);
        const int o = (r & (T - 1)) & ~(P::UT - 1);
        ru[n] = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint32_t*>(vbase) +
                                                (size_t)(r & ~(T - 1)) * (D * B / 32) + (dim * T + o) * B / 32);
      }
    } else {
      const int row = b * a.bs + off;
      if constexpr (C::kFp8) {
        psk = a.kps[b];
        psv = a.vps[b];
      }
#pragma unroll
      for (int n = 0; n < P::NP; ++n) {
        const size_t o = (size_t)__shfl(row, tid / P::PR + n * P::RP, 64) * rowb + 16 * (tid % P::PR);
        rk[n] = *reinterpret_cast<const u32x4*>(kbase + o);
        rv[n] = *reinterpret_cast<const u32x4*>(vbase + o);
      }
    }
  };

  float m_run[CT], l_part[CT];
  f32x4 acc[CT][P::SB];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m_run[ct] = -INFINITY;
    l_part[ct] = 0.f;
#pragma unroll
    for (int b = 0; b < P::SB; ++b) acc[ct][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sl2 = a.scale_log2;
  int vexp = 0;          // FP8, affine: acc holds the sum / 2^vexp
  float pb[CT][G] = {};  // affine: sum p * v_bias
  if constexpr (AFF) {   // the bias operand's unused halves stay zero
    for (int i = tid; i < NT; i += 256) *reinterpret_cast<u32x4*>(kbe + 8 * i) = u32x4{0u, 0u, 0u, 0u};
  }

  int blk1 = 0;
  if (st_lo < st_hi) {
    load_step(st_lo, page_id(st_lo));
    blk1 = page_id(min(st_lo + 1, st_hi - 1));
  }
  for (int st = st_lo; st < st_hi; ++st) {
    const int pos0 = block_of(st) * NT;
    __syncthreads();  // the previous block's tiles are no longer read
    if constexpr (AFF) {
      constexpr int B = C::kBits;
#pragma unroll
      for (int n = 0; n < P::NP; ++n) {
        const int e = tid + 256 * n;
        uint16_t* kr = ke + affine_pos((e / P::PR) & (NT - 1)) * P::KSTR + (e % P::PR) * (128 / B);
        if (e < P::NPK) {
          if constexpr (B == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<h16x8*>(kr + 8 * i) = unpack4_high(rk[n][i]);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<h16x8*>(kr + 8 * i) = unpack8(rk[n][2 * i], rk[n][2 * i + 1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < P::NPV; ++n) {
        const int e = tid + 256 * n;
        uint16_t* vr = ve + (e / P::U) * P::VSTR + (e % P::U) * P::UT;
        if constexpr (B == 4) {
          *reinterpret_cast<h16x8*>(vr) = unpack4_high(ru[n][0]);
          *reinterpret_cast<h16x8*>(vr + 8) = unpack4_high(ru[n][1]);
        } else {
          *reinterpret_cast<h16x8*>(vr) = unpack8(ru[n][0], ru[n][1]);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < P::NP; ++n) {
        const int r = tid / P::PR + n * P::RP, c = (tid % P::PR) * (16 / P::EB);
        put_piece<C>(ke + r * P::KSTR + c, rk[n]);
        put_piece<C>(ve + r * P::VSTR + c, rv[n]);
      }
    }
    const uint64_t okm = okn;
    if constexpr (AFF) {
      // scales of keys past the tile's last one or on an invalid page (which may hold anything) as zeros
      const int pc = min(lane, P::NPS - 1), t8 = 8 * (pc % (NT / 8)), seg = pc / (NT / 8), arr = seg / G, g = seg % G;
      const int live = k_hi + 1 - pos0 - t8;
      u32x4 x = rs;
      if (live < 8 || !((okm >> t8) & 1)) {
        const int n = (okm >> t8) & 1 ? live : 0;
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
      if (ex > vexp || ex < vexp - 6) {
        const float f = __uint_as_float((uint32_t)(127 + vexp - ex) << 23);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int b = 0; b < P::SB; ++b) acc[ct][b] *= f;
        vexp = ex;
      }
      if (wv == 0 && lane < P::NPS) {
        const float down = __uint_as_float((uint32_t)(127 - vexp) << 23);
        const float f = arr == 0 ? (float)(1 << C::kCodeExp) : arr == 2 ? down : 1.f;
        const h16x8 hv = __builtin_bit_cast(h16x8, x);
        if (arr == 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<h16x2*>(kbe + 8 * affine_pos(t8 + e) + 2 * g) = h16x2{hv[e], hv[e]};
        } else {
          float* dst = (arr == 0 ? ksf : arr == 2 ? vsf : vbf) + g * NT;
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<f32x4*>(dst + affine_pos(t8 + 4 * q)) =
                f32x4{(float)hv[4 * q] * f, (float)hv[4 * q + 1] * f, (float)hv[4 * q + 2] * f, (float)hv[4 * q + 3] * f};
        }
      }
    }
    if constexpr (C::kFp8) {
      // value scales enter with the probabilities, brought near 1 by a power of two that the
      // accumulator carries (exact; rescaled when the block's largest scale has another exponent)
      const float vmax = wave_max(psv);
      const int ex = min(max((int)((__float_as_uint(vmax) >> 23) & 0xFFu) - 127, -60), 60);
      if (ex != vexp) {
        const float f = __uint_as_float((uint32_t)(127 + min(max(vexp - ex, -126), 127)) << 23);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int b = 0; b < P::SB; ++b) acc[ct][b] *= f;
        vexp = ex;
      }
      const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
      if (tid < NT) {
        ksf[tid] = psk * 256.f;
        vsf[tid] = psv * down;
      }
    }
    __syncthreads();
    if (st + 1 < st_hi) {
      load_step(st + 1, blk1);
      blk1 = page_id(min(st + 2, st_hi - 1));
    }
    if (!busy) continue;

#pragma unroll
    for (int hh = 0; hh < NT / 32; ++hh) {
      const int h = NT / 32 - 1 - hh;  // backwards, as the cursors go
      const int kp = pos0 + 32 * h;
      // ---- tree: the drafted keys of the half that each column sees
      uint32_t bits[CT];
      const bool drafted = tree && kp + 31 >= past;
      if (drafted) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          bits[ct] = 0;
          while (cur[ct] >= 0 && past + cur[ct] >= kp) {
            const int b = past + cur[ct] - kp;
            if (b < 32 && (mask.window <= 0 || back[ct] < mask.window || place[ct] - back[ct] < mask.sinks))
              bits[ct] |= 1u << b;
            cur[ct] = up(cur[ct]);
            ++back[ct];
          }
        }
      }
      // ---- S^T: lane (col, jj) gets keys 32 h + 16 t + 4 jj + r of its columns
      float sc[CT][8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* kr = ke + (32 * h + 16 * t + col) * P::KSTR + 8 * jj;
        f32x4 c[CT][G];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int g = 0; g < G; ++g) c[ct][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < P::KS; ++w) {
          const Op K = *reinterpret_cast<const Op*>(kr + 32 * w);
          const int g = w * G / P::KS;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) c[ct][g] = mfma_op(K, qB[ct][w], c[ct][g]);
        }
        if constexpr (AFF) {
          // (the bias operand is zero outside lane group 0)
          const Op KB = *reinterpret_cast<const Op*>(kbe + 8 * (32 * h + 16 * t + col));
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            f32x4 v = mfma_op(KB, qbias[ct], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const f32x4 ks4 = *reinterpret_cast<const f32x4*>(ksf + g * NT + 32 * h + 16 * t + 4 * jj);
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] = fmaf(c[ct][g][r], ks4[r], v[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[ct][4 * t + r] = v[r];
          }
        } else {
          f32x4 ks4 = {1.f, 1.f, 1.f, 1.f};
          if constexpr (C::kFp8) ks4 = *reinterpret_cast<const f32x4*>(ksf + 32 * h + 16 * t + 4 * jj);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[ct][4 * t + r] = C::kFp8 ? c[ct][0][r] * ks4[r] : c[ct][0][r];
        }
      }

      // ---- mask where a key of the half is not visible to every column
      const uint32_t okh = (uint32_t)(okm >> (32 * h));
      bool full = okh == 0xFFFFFFFFu && !drafted;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        full = full && kp + 31 <= limit[ct] && (kp >= start[ct] || kp + 31 < mask.sinks);
      if (!full) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = AFF ? 8 * jj + e : 16 * (e >> 2) + 4 * jj + (e & 3);
            bool see = kp + k <= limit[ct] && (kp + k >= start[ct] || kp + k < mask.sinks);
            if (drafted) see = see || ((bits[ct] >> k) & 1u);
            if (!see || !((okh >> k) & 1u)) sc[ct][e] = -INFINITY;
          }
      }

      // ---- online softmax
      float m_new[CT];
      bool grow = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float tmax = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) tmax = fmaxf(tmax, sc[ct][e]);
        m_new[ct] = fmaxf(m_run[ct], rows4_max(tmax) * sl2);
        grow = grow || m_new[ct] > m_run[ct] + kLazyMax;
      }
      if (__any(grow)) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bool rise = m_new[ct] > m_run[ct] + kLazyMax;  // also the first finite maximum
          const float al = rise ? __builtin_amdgcn_exp2f(m_run[ct] - m_new[ct]) : 1.f;
          l_part[ct] *= al;
#pragma unroll
          for (int b = 0; b < P::SB; ++b) acc[ct][b] *= al;
          if constexpr (AFF) {
#pragma unroll
            for (int g = 0; g < G; ++g) pb[ct][g] *= al;
          }
          if (rise) m_run[ct] = m_new[ct];
        }
      }
      Op pB[CT][2];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        // p <= 2^(kLazyMax + 6), times a value scale below 2: inside fp16, and small p stay
        // clear of its sub-normals
        const float m_sub = fmaxf(m_run[ct], -3.0e38f) - 6.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sc[ct][e] = __builtin_amdgcn_exp2f(fmaf(sc[ct][e], sl2, -m_sub));
          l_part[ct] += sc[ct][e];
        }
        if constexpr (C::kFp8) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const f32x4 vs4 = *reinterpret_cast<const f32x4*>(vsf + 32 * h + 16 * t + 4 * jj);
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[ct][4 * t + r] *= vs4[r];
          }
        }
        if constexpr (!AFF) split_p2(sc[ct], pB[ct]);
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if constexpr (AFF) {  // this group's operand: p * v_scale; the bias term in fp32
          f32x4 vs4[2], vb4[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            vs4[t] = *reinterpret_cast<const f32x4*>(vsf + g * NT + 32 * h + 16 * t + 4 * jj);
            vb4[t] = *reinterpret_cast<const f32x4*>(vbf + g * NT + 32 * h + 16 * t + 4 * jj);
          }
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] = sc[ct][e] * vs4[e >> 2][e & 3];
              pb[ct][g] = fmaf(sc[ct][e], vb4[e >> 2][e & 3], pb[ct][g]);
            }
            split_p2(x, pB[ct]);
          }
        }
#pragma unroll
        for (int b = g * P::SB / G; b < (g + 1) * P::SB / G; ++b) {
          Op V;
          if constexpr (AFF) {
            V = *reinterpret_cast<const Op*>(ve + (16 * b + col) * P::VSTR + 32 * h + 8 * jj);
          } else {
            const u32x2 v0 = read_tr(ve, P::VSTR, 32 * h, 16 * b, col, jj);
            const u32x2 v1 = read_tr(ve, P::VSTR, 32 * h + 16, 16 * b, col, jj);
            V = __builtin_bit_cast(Op, u32x4{v0[0], v0[1], v1[0], v1[1]});
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) acc[ct][b] = mfma_op(V, pB[ct][k], acc[ct][b]);
        }
      }
    }
  }
  if constexpr (AFF) {  // codes entered as code * 2^-kCodeExp; the bias term joins its group's dims
    const float f = __uint_as_float((uint32_t)(127 + vexp + C::kCodeExp) << 23);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int b = 0; b < P::SB; ++b) {
        const float bias = rows4_sum(pb[ct][b * G / P::SB]);
        acc[ct][b] = acc[ct][b] * f + bias;
      }
  }
  if constexpr (C::kFp8) {  // the codes entered as value * 2^-8
    const float f = __uint_as_float((uint32_t)(127 + vexp + 8) << 23);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int b = 0; b < P::SB; ++b) acc[ct][b] *= f;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) l_part[ct] = rows4_sum(l_part[ct]);

  // ---- a part: its columns' state for masked_merge
  if (nparts > 1) {
    float* st = A.part + ((size_t)(u.first + u.part) * a.Hkv + kvh) * (PARTB / 4);
    constexpr int NV = CT * P::SB;
    float* mine = st + (size_t)wv * (NV + 1) * 256 + lane * 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      if (ctok[ct] >= 0)
#pragma unroll
        for (int b = 0; b < P::SB; ++b) *reinterpret_cast<f32x4*>(mine + (P::SB * ct + b) * 256) = acc[ct][b];
    *reinterpret_cast<f32x4*>(mine + NV * 256) = f32x4{m_run[0], m_run[CT - 1], l_part[0], l_part[CT - 1]};
    return;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < P::SB; ++b)
      bad |= masked_write<C, D>(a, u, kvh, ctok[ct], chead[ct], acc[ct][b], l_part[ct], 16 * b + 4 * jj);
    if (__any(bad && ctok[ct] >= 0)) {
      __builtin_amdgcn_s_waitcnt(0);  // (the row's first result is out before its second)
      masked_again<C, D>(a, mask, par, u, kvh, bad, ctok[ct], chead[ct], lane);
    }
  }
}

// Joins the parts of cut tiles, in part order.  Grid (tiles, Hkv, CT): a workgroup has the columns
// [64 ct, 64 ct + 64) of one tile, a wave 16 of them.
template <class C, int D, int CT>
__global__ __launch_bounds__(256) void masked_merge(MaskedArgs A) {
  using P = PrefillMfmaCfg<C, D, CT>;
  const DecodeArgs& a = A.d;
  __shared__ int wred[16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, jj = lane >> 4, kvh = blockIdx.y, ct = blockIdx.z;
  const MaskedUnit u = masked_plan<P::NT>(A, blockIdx.x, true, wred);
  if (!u.live) return;
  const int tok_lo = u.tile * A.tokb, tok_hi = min(min(tok_lo + A.tokb, u.qlen), A.T - u.q0) - 1;
  const int np = masked_parts(masked_span<P::NT>(A.mask, u.past, tok_lo, tok_hi).n, u.nparts);
  if (np <= 1) return;
  int ctok, chead;
  masked_column(A, u, (ct * 4 + wv) * 16 + col, a.Hq / a.Hkv, ctok, chead);
  if (!__any(ctok >= 0)) return;
  constexpr int PARTB = kMaskedPartBytes<D, CT>, NV = CT * P::SB;
  const float* mine = A.part + ((size_t)u.first * a.Hkv + kvh) * (PARTB / 4) + (size_t)wv * (NV + 1) * 256 + lane * 4;
  const size_t next = (size_t)a.Hkv * (PARTB / 4);
  float m = -INFINITY;
  for (int q = 0; q < np; ++q) m = fmaxf(m, mine[q * next + NV * 256 + (ct == 0 ? 0 : 1)]);
  float l = 0.f;
  f32x4 o[P::SB];
#pragma unroll
  for (int b = 0; b < P::SB; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int q = 0; q < np; ++q) {
    const float* st = mine + q * next;
    const float m1 = st[NV * 256 + (ct == 0 ? 0 : 1)], l1 = st[NV * 256 + (ct == 0 ? 2 : 3)];
    // (a part without a live key has m1 = -inf and zeros, one of NaN scores only a sum that is NaN)
    const float f = m1 == -INFINITY ? (l1 == 0.f ? 0.f : l1) : __builtin_amdgcn_exp2f(m1 - m);
    l = fmaf(l1, f, l);
    if (ctok >= 0)
#pragma unroll
      for (int b = 0; b < P::SB; ++b) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(st + (P::SB * ct + b) * 256);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[b][r] = fmaf(x[r], f, o[b][r]);
      }
  }
  bool bad = false;
#pragma unroll
  for (int b = 0; b < P::SB; ++b) bad |= masked_write<C, D>(a, u, kvh, ctok, chead, o[b], l, 16 * b + 4 * jj);
  if (__any(bad && ctok >= 0)) {
    __builtin_amdgcn_s_waitcnt(0);
    masked_again<C, D>(a, A.mask, A.mask.parents ? A.mask.parents + u.q0 : nullptr, u, kvh, bad, ctok, chead, lane);
  }
}

}  // namespace emx
