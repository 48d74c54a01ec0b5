"""Attention with sinks and of drafted trees over every cache type vs the float64 oracle.

Bound of a result: half a step of the 16-bit output (2^-11 / 2^-8 of the value) plus the fp32 arithmetic (scores
are fp32 sums of up to 256 products, |s| <= ~16, so a probability is off by at most ~2^-18 of itself and an output by
2^-16 of the largest value it averages) plus, in bf16, the probabilities' second half step (2^-17 of the same).
fp32: 2^-15 of the largest value (sums of up to 1100 terms rounded one by one, 2^-24 each, twice) and its own half step.
"""

import numpy as np
import pytest
import torch

from easymlx_amd import paged_attention, tree_attention
from oracle import masked
from tests.test_gpu_mfma import batch

pytestmark = pytest.mark.gpu

KINDS = ["f16", "bf16", "fp8", "q4", "q8"]


def cache_args(b, dev):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    sc = b["scales"]
    if isinstance(sc, dict):
        return {k: x.to(dev) if isinstance(x, torch.Tensor) else x for k, x in sc.items()}
    return dict(k_scale=t(sc[0]), v_scale=t(sc[1])) if sc is not None else {}


def run(b, dev, window=0, sinks=0, parents=None, decode=False, **kw):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    args = (b["q"].to(dev), b["cache"][0].to(dev), b["cache"][1].to(dev), t(b["tables"]), t(b["kvl"]), t(b["qsl"]))
    rule = dict(sliding_window=window, sink_tokens=sinks, **cache_args(b, dev), **kw)
    if parents is None:
        out = paged_attention(*args, single_token_decode=decode, **rule)
    else:
        out = tree_attention(*args, t(np.asarray(parents, np.int32)), **rule)
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


def expected(b, window=0, sinks=0, parents=None):
    return masked.masked_attention(b["q"].double().numpy(), b["exact"][0], b["exact"][1], b["tables"], b["kvl"],
                                   b["qsl"], window=window, sinks=sinks, parents=parents)


def check(b, got, exp):
    ulp, arith = {torch.bfloat16: (2.0 ** -8, 2.0 ** -16 + 2.0 ** -17), torch.float16: (2.0 ** -11, 2.0 ** -16),
                  torch.float32: (2.0 ** -24, 2.0 ** -15)}[b["q"].dtype]
    bound = ulp * np.abs(exp) + arith * np.abs(b["exact"][1]).max() + 2.0 ** -24
    err = np.abs(got - exp)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"{int((err > bound).sum())} of {err.size}, worst {(err / bound).max():.2f} of the bound"


def tree(rng, n, wild=False):
    """Parents of n nodes below random earlier ones; wild: entries among them that are no earlier node."""
    p = [-1] + [int(rng.integers(max(0, i // 3 - 1), i)) for i in range(1, n)]
    for i in range(n):
        if wild and rng.random() < 0.15:
            p[i] = int(rng.choice([-5, i, i + 3, 1 << 30]))
    return p[:n]


def trees(b, seed, wild=False):
    rng = np.random.default_rng(seed)
    return np.concatenate([tree(rng, int(n), wild) for n in np.diff(b["qsl"])] + [[]]).astype(np.int32)


SHAPES = [(64, 16, 8, 2, 64), (128, 16, 6, 2, 64), (128, 128, 32, 8, 128), (256, 64, 4, 4, 64), (256, 32, 16, 1, 128)]
CONTEXTS = [1, 3, 31, 32, 33, 64, 65, 129, 0, 300, 1000, 5]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,page,hq,hkv,gs", SHAPES)
def test_decode_with_sinks(cuda, kind, d, page, hq, hkv, gs):
    print(f"[sinks decode {kind} d{d} page{page} {hq}/{hkv}]", flush=True)
    b = batch(kind, [1] * len(CONTEXTS), CONTEXTS, hq, hkv, d, page, seed=d + page + hq, gs=gs,
              invalid=[(5, 1), (9, 0), (10, 2)] if page < 64 else [])
    for window, sinks in ((1, 1), (64, 4), (100, 70), (33, 500)):
        check(b, run(b, cuda, window, sinks, decode=True), expected(b, window, sinks))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,page,hq,hkv,gs", SHAPES)
def test_ragged_with_sinks(cuda, kind, d, page, hq, hkv, gs):
    """Prompts with and without cached tokens before them, rows of one token, an empty one, more queries than keys."""
    print(f"[sinks ragged {kind} d{d} page{page} {hq}/{hkv}]", flush=True)
    qlens, kvl = [5, 1, 0, 130, 33, 1, 20, 64], [5, 700, 40, 130, 500, 1, 12, 0]
    b = batch(kind, qlens, kvl, hq, hkv, d, page, seed=d + page + hq + 1, gs=gs,
              invalid=[(1, 2), (4, 0)] if page < 64 else [])
    for window, sinks in ((1, 1), (40, 4), (100, 130)):
        check(b, run(b, cuda, window, sinks), expected(b, window, sinks))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,page,hq,hkv,gs", SHAPES)
def test_tree(cuda, kind, d, page, hq, hkv, gs):
    """Trees of one node to more than a tile's, at block edges, deeper than the window, longer than their cache."""
    print(f"[tree {kind} d{d} page{page} {hq}/{hkv}]", flush=True)
    qlens, kvl = [1, 7, 0, 25, 64, 70, 130, 16, 9, 3], [1, 7, 30, 300, 64, 135, 700, 12, 1000, 0]
    b = batch(kind, qlens, kvl, hq, hkv, d, page, seed=d + page + hq + 2, gs=gs,
              invalid=[(3, 2), (8, 0)] if page < 64 else [])
    for window, sinks, wild in ((0, 0, False), (0, 3, True), (5, 2, False), (2, 0, True), (80, 40, False)):
        p = trees(b, window + sinks, wild)
        check(b, run(b, cuda, window, sinks, p), expected(b, window, sinks if window else 0, p))


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_chain_is_a_causal_run(cuda, kind):
    """Chains beside trees: parents[i] = i - 1 is an ordinary prompt, of more nodes than are kept in LDS."""
    b = batch(kind, [1100, 40, 1], [1300, 900, 77], 4, 1, 128, 32, seed=5)
    p = np.concatenate([np.arange(1100) - 1, tree(np.random.default_rng(1), 40), [-1]])
    for window, sinks in ((0, 0), (200, 5)):
        exp = expected(b, window, sinks, p)
        causal = expected(b, window, sinks)
        np.testing.assert_allclose(exp[:1100], causal[:1100], atol=1e-12)
        check(b, run(b, cuda, window, sinks, p), exp)


@pytest.mark.parametrize("kind", ["f16", "bf16", "fp8", "q4"])
def test_long_context_is_cut(cuda, kind):
    """A few nodes over a long context: tiles in many parts, the same bits every time, and uncut without a workspace."""
    b = batch(kind, [3, 1], [30_011, 4001], 8, 2, 128, 16, seed=3)
    p = [-1, 0, 0, -1]
    exp = expected(b, 0, 0, p)
    first = run(b, cuda, 0, 0, p)
    check(b, first, exp)
    assert np.array_equal(first, run(b, cuda, 0, 0, p))
    check(b, run(b, cuda, 0, 0, p, workspace=torch.empty(0, dtype=torch.uint8, device=cuda)), exp)
    check(b, run(b, cuda, 9000, 4, None), expected(b, 9000, 4))


@pytest.mark.parametrize("kind,d,page,hq,hkv,gs", [("f16", 96, 16, 4, 2, 64), ("bf16", 128, 12, 6, 3, 64),
                                                   ("f16", 128, 16, 200, 1, 64), ("fp8", 40, 5, 4, 4, 64),
                                                   ("q8", 64, 4, 4, 2, 32), ("q4", 128, 16, 20, 1, 32)])
def test_other_shapes(cuda, kind, d, page, hq, hkv, gs):
    """Head sizes, pages, groups and head counts outside the matrix units' shapes."""
    b = batch(kind, [1, 40, 0, 9], [70, 300, 4, 7], hq, hkv, d, page, seed=d + hq, gs=gs, invalid=[(1, 3)])
    p = trees(b, 1)
    for window, sinks in ((0, 0), (30, 5), (3, 100)):
        check(b, run(b, cuda, window, sinks, p), expected(b, window, sinks, p))
        if window:
            check(b, run(b, cuda, window, sinks), expected(b, window, sinks))


def test_fp32_and_wide_queries(cuda):
    """fp32 over an fp32 cache, and bf16 / fp32 queries over FP8 pages."""
    b = batch("f16", [30, 1], [200, 90], 4, 2, 64, 16, seed=8)
    p = trees(b, 2)
    b.update(q=b["q"].float(), cache=[c.float() for c in b["cache"]])
    check(b, run(b, cuda, 0, 0, p), expected(b, 0, 0, p))
    check(b, run(b, cuda, 17, 3), expected(b, 17, 3))
    b = batch("fp8", [30, 1], [200, 90], 4, 2, 64, 16, seed=8)
    for dt in (torch.bfloat16, torch.float32):
        b["q"] = b["q"].to(dt)
        check(b, run(b, cuda, 0, 0, p), expected(b, 0, 0, p))


def where(b, s, pos):
    page = b["cache"][0].shape[1]
    return int(b["tables"][s, pos // page]), pos % page


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(128, 16), (96, 16)])
def test_unseen_keys_may_hold_anything(cuda, kind, shape):
    """Infinities and NaN in a sibling's row, between sinks and window and behind the sequence; an infinity in a row's own."""
    d, page = shape
    b = batch(kind, [6], [90], 4, 2, d, page, seed=9)
    p = [-1, 0, 0, 1, 2, 0]
    exp = expected(b, 0, 0, p)
    k, v = b["cache"]
    blk, off = where(b, 0, 84 + 3)  # node 3: seen by itself alone
    k[blk, off, 0], v[blk, off, 1] = float("nan"), float("inf")
    blk, off = where(b, 0, 90)  # behind the sequence
    k[blk, off], v[blk, off] = float("inf"), float("nan")
    got = run(b, cuda, 0, 0, p)
    rows = [0, 1, 2, 4, 5]
    one = dict(b, q=b["q"][rows])
    check(one, got[rows], exp[rows])
    assert np.isnan(got[3, :2]).all()  # a key of NaN in kv head 0
    assert (np.isinf(got[3, 2:]) & (got[3, 2:] > 0)).all()  # a value of infinity in kv head 1
    # between sinks and window
    b = batch(kind, [1, 3], [300, 400], 4, 2, d, page, seed=10)
    exp = expected(b, 20, 4)
    for s, n in ((0, 300), (1, 400)):
        for pos in range(4, n - 30):
            blk, off = where(b, s, pos)
            b["cache"][0][blk, off], b["cache"][1][blk, off] = float("nan"), float("inf")
    check(b, run(b, cuda, 20, 4), exp)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_decode_rows_beside_anything(cuda, kind):
    """Rows of one token: junk between sinks and window, and an infinite value among the sinks or in the window."""
    lens = [700, 40, 1500, 3000]
    b = batch(kind, [1] * 4, lens, 8, 2, 128, 16, seed=10)
    exp = expected(b, 600, 70)
    for s, n in enumerate(lens):
        for pos in range(70, n - 600):
            blk, off = where(b, s, pos)
            b["cache"][0][blk, off], b["cache"][1][blk, off] = float("nan"), float("inf")
    check(b, run(b, cuda, 600, 70, decode=True), exp)
    for s, pos in ((2, 69), (3, 2400)):
        blk, off = where(b, s, pos)
        b["cache"][1][blk, off, 1, 5] = -float("inf")
    got = run(b, cuda, 600, 70, decode=True)
    assert (got[2:, 4:, 5] == -np.inf).all()
    keep = np.ones_like(exp, bool)
    keep[2:, 4:, 5] = False
    check(b, np.where(keep, got, 0), np.where(keep, exp, 0))


def test_infinite_value_in_a_cut_tile(cuda):
    """A seen value of infinity among many parts: that dim alone, for the rows that see it."""
    b = batch("f16", [3], [20_000], 4, 1, 128, 16, seed=12)
    p = [-1, 0, 0]
    exp = expected(b, 0, 0, p)
    blk, off = where(b, 0, 19_998)  # node 1
    b["cache"][1][blk, off, 0, 7] = float("inf")
    got = run(b, cuda, 0, 0, p)
    assert (got[1, :, 7] == np.inf).all()
    keep = np.ones_like(exp, bool)
    keep[1, :, 7] = False
    check(b, np.where(keep, got, 0), np.where(keep, exp, 0))


@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_rows_of_no_sequence(cuda, kind):
    """Rows before the first sequence and behind the last (a padded call) are zeros."""
    b = batch(kind, [4, 37, 9], [40, 200, 9], 8, 2, 128, 16, seed=4)
    b["qsl"] = np.asarray([4, 41, 41, 45], np.int32)
    p = np.full(50, -1, np.int32)
    p[4:45] = np.concatenate([tree(np.random.default_rng(0), 37), tree(np.random.default_rng(1), 4)])
    for w, s, pp in ((0, 0, p), (25, 3, None)):
        exp = expected(b, w, s, pp)
        assert (exp[:4] == 0).all() and (exp[45:] == 0).all()
        got = run(b, cuda, w, s, pp, out=torch.full_like(b["q"], 7.0).to(cuda))
        check(b, got, exp)
        assert (got[:4] == 0).all() and (got[45:] == 0).all()


def test_strides_types_and_streams(cuda):
    """Strided queries, 64-bit and host integers, a call on another stream, views of a larger pool."""
    b = batch("f16", [9, 1, 30], [100, 40, 300], 8, 2, 64, 16, seed=6)
    p = trees(b, 4)
    exp = expected(b, 60, 4, p)
    wide = torch.randn(40, 8, 128, dtype=torch.float16)
    wide[:, :, 32:96] = b["q"]
    q = wide.to(cuda)[:, :, 32:96]
    k, v = (c.to(cuda) for c in b["cache"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree_attention(q, k, v, torch.from_numpy(b["tables"]).long(), b["kvl"].tolist(),
                             torch.from_numpy(b["qsl"]).long().to(cuda), p.tolist(), sliding_window=60, sink_tokens=4)
    side.synchronize()
    check(b, got.double().cpu().numpy(), exp)
    with pytest.raises(ValueError, match="out must be"):
        tree_attention(q, k, v, b["tables"], b["kvl"], b["qsl"], p, out=torch.empty(40, 8, 128, device=cuda)[..., :64])
    with pytest.raises(ValueError, match="device"):
        tree_attention(q, k.cpu(), v, b["tables"], b["kvl"], b["qsl"], p)
    with pytest.raises(NotImplementedError, match="queries' dtype"):
        tree_attention(q.bfloat16(), k, v, b["tables"], b["kvl"], b["qsl"], p)


def test_sinks_without_a_window_are_the_plain_call(cuda):
    b = batch("bf16", [9, 1], [100, 40], 8, 2, 64, 16, seed=6)
    assert np.array_equal(run(b, cuda, 0, 5), run(b, cuda, 0, 0))


def test_captured_calls(cuda):
    """Two graphs of one stream, replayed on two streams at once with eager calls between, over changed inputs."""
    a = batch("bf16", [5, 5, 5], [3000, 900, 40], 8, 2, 128, 16, seed=1)
    w = batch("q4", [1, 1], [5000, 70], 8, 2, 128, 128, seed=2)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731
    pa = trees(a, 1)
    ia = [a["q"].to(cuda), a["cache"][0].to(cuda), a["cache"][1].to(cuda), t(a["tables"]), t(a["kvl"]), t(a["qsl"]), t(pa)]
    iw = [w["q"].to(cuda), w["cache"][0].to(cuda), w["cache"][1].to(cuda), t(w["tables"]), t(w["kvl"]), t(w["qsl"])]
    kw = dict(sliding_window=2000, sink_tokens=4, single_token_decode=True, **cache_args(w, cuda))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        for call in (lambda: tree_attention(*ia), lambda: paged_attention(*iw, **kw)):
            call()
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = call()
            graphs.append((g, out))
    side = torch.cuda.Stream()
    for i, lens in enumerate(([3000, 900, 40], [17, 2999, 5], [2000, 5, 600])):
        lens = np.minimum(lens, (a["tables"] >= 0).sum(1) * 16).astype(np.int32)
        pa = trees(a, 7 + i)
        ia[4].copy_(t(lens))
        ia[6].copy_(t(pa))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        eager = tree_attention(*ia)
        torch.cuda.synchronize()
        got = graphs[0][1].double().cpu().numpy()
        check(a, got, expected(dict(a, kvl=lens), 0, 0, pa))
        assert np.array_equal(got, eager.double().cpu().numpy())
        check(w, graphs[1][1].double().cpu().numpy(), expected(w, 2000, 4))


@pytest.mark.parametrize("count", [300, 1100])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_many_sequences(cuda, kind, count):
    """More sequences than the kernel keeps in LDS, and more than it takes (the general kernel's): none to three tokens."""
    print(f"[{count} sequences {kind}]", flush=True)
    rng = np.random.default_rng(count)
    qlens = [int(x) for x in rng.integers(0, 4, count)]
    kvl = [q + int(x) for q, x in zip(qlens, rng.integers(0, 90, count))]
    b = batch(kind, qlens, kvl, 8, 2, 64, 16, seed=count, gs=64)
    for window, sinks in ((17, 3), (40, 20)):
        check(b, run(b, cuda, window, sinks), expected(b, window, sinks))
    p = trees(b, count)
    check(b, run(b, cuda, 0, 0, p), expected(b, 0, 0, p))


@pytest.mark.parametrize("kind", KINDS)
def test_more_tiles_than_workgroups(cuda, kind):
    """Long prompts and trees of many heads: a workgroup to a tile, none of them cut."""
    print(f"[many tiles {kind}]", flush=True)
    b = batch(kind, [700, 33, 700, 700], [700, 400, 731, 705], 64, 8, 128, 32, seed=3, gs=64)
    check(b, run(b, cuda, 24, 2), expected(b, 24, 2))
    p = trees(b, 7)
    check(b, run(b, cuda, 30, 5, p), expected(b, 30, 5, p))
