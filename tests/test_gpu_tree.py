"""Drafted trees around the attention: acceptance, commit of the accepted path, and whole steps with both."""

import numpy as np
import pytest
import torch

from easymlx_amd import (
    AffinePageCacheView,
    Fp8PageCacheView,
    OperationRegistry,
    PageCache,
    PageCacheView,
    PageMetadata,
    RotaryEmbedding,
    commit_tree,
    tree_accept,
)
from oracle import masked
from tests.test_gpu_masked import tree

pytestmark = pytest.mark.gpu


def drafted(rng, sizes, vocab=5, dtype=np.int64):
    """Trees whose tokens and targets come from a small vocabulary: several children agree, paths are long."""
    parents = np.concatenate([tree(rng, n) for n in sizes] + [[]]).astype(np.int32)
    tokens = rng.integers(0, vocab, parents.size).astype(dtype)
    targets = rng.integers(0, vocab, parents.size).astype(dtype)
    return tokens, targets, parents, np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_accept(cuda, dtype):
    """Empty trees, one node, sizes around a wave and above, a chain of 300 that is accepted whole."""
    rng = np.random.default_rng(4)
    sizes = [0, 1, 2, 7, 63, 64, 65, 130, 300, 25, 0]
    for vocab in (2, 5, 1 << 30):
        tokens, targets, parents, qsl = drafted(rng, sizes, vocab, dtype)
        at = qsl[8]
        parents[at:at + 300] = np.arange(300) - 1
        targets[at:at + 299] = tokens[at + 1:at + 300]
        exp = masked.tree_accept(tokens, targets, parents, qsl)
        got = tree_accept(torch.from_numpy(tokens).to(cuda), torch.from_numpy(targets).to(cuda), parents, qsl)
        assert got.next_tokens.dtype == torch.from_numpy(tokens).dtype
        for g, e in zip(got, exp):
            np.testing.assert_array_equal(g.cpu().numpy(), e)
        assert exp[1][8] == 300


def test_accept_large_tokens_and_padded_rows(cuda):
    """Tokens that differ above 32 bits only, and rows of no sequence."""
    tokens = np.array([7, 5, 1 << 40, 0, 9, 9], np.int64)
    targets = np.array([0, 0, 3, 0, 9, 9], np.int64)
    parents = np.array([0, -1, 0, 0, -1, 0], np.int32)
    qsl = np.array([1, 4], np.int32)
    got = tree_accept(*(torch.from_numpy(x).to(cuda) for x in (tokens, targets, parents, qsl)))
    assert got.path.tolist() == [-1, 0, 2, -1, -1, -1] and got.accepted.tolist() == [2]
    assert got.next_tokens.tolist() == [0]
    none = tree_accept(*(torch.zeros(0, dtype=torch.int64, device=cuda) for _ in range(3)), [0])
    assert none.path.numel() == none.accepted.numel() == 0


def view_of(kind, dev, num_seqs=5, max_len=96, hkv=3, d=64, page=16, gs=64, seed=0):
    """A cache of random contents, its pages in random order."""
    kw = dict(num_seqs=num_seqs, max_seq_len=max_len, num_kv_heads=hkv, head_dim=d, block_size=page, device=dev)
    if kind in ("q4", "q8"):
        v = AffinePageCacheView.init(bits=int(kind[1]), group_size=gs, **kw)
    elif kind == "fp8":
        v = Fp8PageCacheView.init(**kw)
    else:
        v = PageCacheView.init(dtype={"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[kind], **kw)
    rng = np.random.default_rng(seed)
    for t in v.page_arrays():
        raw = rng.integers(0, 256, t.numel() * t.element_size()).astype(np.uint8)
        if t.is_floating_point():
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape), dtype=np.float32)).to(t.dtype))
        else:
            t.copy_(torch.from_numpy(raw).view(t.dtype).reshape(t.shape))
    perm = torch.from_numpy(rng.permutation(v.num_blocks).astype(np.int32)).to(dev)
    v.block_tables = perm[:v.block_tables.numel()].reshape(v.block_tables.shape).contiguous()
    return v


def rows_of(v):
    """What the cache holds per token, as [nb, page, n] arrays: caches, or codes and their scales."""
    if v.is_affine:
        return [x.cpu().numpy() for x in v.to_logical().values()]
    rows = [v.key_cache, v.value_cache]
    return [x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]).cpu().numpy() for x in rows]


SIZES, LENS = [25, 1, 40, 0, 9], [60, 1, 96, 30, 9]


def paths(rng, sizes, qsl):
    """Ascending paths of random nodes, -1 behind them."""
    path, count = np.full(qsl[-1], -1, np.int32), []
    for lo, n in zip(qsl, sizes):
        k = int(rng.integers(1, n + 1)) if n else 0
        path[lo:lo + k] = np.concatenate([[0], 1 + np.sort(rng.permutation(n - 1)[:k - 1])])[:k] if k else []
        count.append(k)
    return path, np.asarray(count, np.int32)


@pytest.mark.parametrize("kind,page,gs,d,hkv", [("f16", 16, 64, 64, 3), ("bf16", 7, 64, 64, 3), ("f32", 16, 64, 6, 1),
                                                ("fp8", 16, 64, 64, 3), ("fp8", 4, 64, 7, 3), ("q4", 16, 64, 64, 3),
                                                ("q4", 128, 64, 128, 2), ("q8", 32, 128, 256, 1), ("q8", 8, 32, 96, 2),
                                                ("q4", 8, 64, 64, 2)])
def test_commit(cuda, kind, page, gs, d, hkv):
    """Every array of two layers, with their own tables and lengths; the rest of the cache as it was."""
    print(f"[commit {kind} page{page} d{d}]", flush=True)
    rng = np.random.default_rng(page + d)
    qsl = np.concatenate([[0], np.cumsum(SIZES)]).astype(np.int32)
    path, count = paths(rng, SIZES, qsl)
    views = [view_of(kind, cuda, hkv=hkv, d=d, page=page, gs=gs, seed=s) for s in (1, 2)]
    scales = [x.clone() for v in views for x in v.page_arrays()[2:]] if kind == "fp8" else []
    exp = []
    for v in views:
        v.kv_lens.copy_(torch.tensor(LENS, dtype=torch.int32))
        r = [masked.tree_commit(x, v.block_tables.cpu().numpy(), LENS, path, count, qsl) for x in rows_of(v)]
        exp.append(r)
    PageCache(views).commit_tree(torch.from_numpy(path).to(cuda), torch.from_numpy(count).to(cuda), qsl)
    for v, r in zip(views, exp):
        for got, (rows, lens) in zip(rows_of(v), r):
            np.testing.assert_array_equal(got, rows)
            np.testing.assert_array_equal(v.kv_lens.cpu().numpy(), lens)
    for a, b in zip(scales, [x for v in views for x in v.page_arrays()[2:]] if scales else []):
        assert torch.equal(a, b)


def test_commit_slots_shared_lengths_many_layers(cuda):
    """Trees of some sequences in another order, 70 layers that share tables and lengths, in more than one launch."""
    rng = np.random.default_rng(3)
    sizes, slots = [12, 30, 5], [4, 0, 2]
    qsl = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    path, count = paths(rng, sizes, qsl)
    views = [view_of("f16", cuda, seed=s, hkv=1) for s in range(70)]
    lens = [96, 7, 5, 50, 33]
    for v in views:
        v.block_tables = views[0].block_tables
        v.kv_lens = views[0].kv_lens
    views[0].kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    bt = views[0].block_tables.cpu().numpy()
    exp = [[masked.tree_commit(x, bt, lens, path, count, qsl, slots) for x in rows_of(v)] for v in views]
    commit_tree(views, path, count, qsl, slot_ids=slots)
    for v, r in zip(views, exp):
        for got, (rows, after) in zip(rows_of(v), r):
            np.testing.assert_array_equal(got, rows)
    np.testing.assert_array_equal(views[0].kv_lens.cpu().numpy(), exp[0][0][1])


def test_commit_follows_replaced_tensors(cuda):
    """A cache whose tensors, or views, are replaced between two commits: the new ones change."""
    path, qsl = torch.tensor([0, 2, -1], dtype=torch.int32, device=cuda), [0, 3]
    count = torch.tensor([2], dtype=torch.int32, device=cuda)
    cache = PageCache([view_of("f16", cuda, seed=s) for s in (1, 2)])
    for change in (lambda: None, lambda: setattr(cache[0], "key_cache", cache[0].key_cache.clone()),
                   lambda: setattr(cache[1], "kv_lens", torch.zeros_like(cache[1].kv_lens)),
                   lambda: cache.__setitem__(0, view_of("q8", cuda, seed=4)), lambda: cache.views.pop()):
        change()
        exp = []
        for v in cache:
            v.kv_lens.copy_(torch.tensor([40, 0, 0, 0, 0], dtype=torch.int32))
            exp.append([masked.tree_commit(x, v.block_tables.cpu().numpy(), [40, 0, 0, 0, 0], [0, 2, -1], [2], qsl)
                        for x in rows_of(v)])
        cache.commit_tree(path, count, qsl)
        for v, r in zip(cache, exp):
            for got, (rows, lens) in zip(rows_of(v), r):
                np.testing.assert_array_equal(got, rows)
                np.testing.assert_array_equal(v.kv_lens.cpu().numpy(), lens)


def test_commit_bad_pages_and_paths(cuda):
    """Pages outside the pool, a tree that starts before its sequence, entries that do not ascend: left alone."""
    v = view_of("q8", cuda, page=8)
    v.block_tables[0, 3], v.block_tables[1, 2] = -1, v.num_blocks + 4
    lens = [40, 30, 5, 96, 20]
    v.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    sizes = [20, 20, 10, 10, 10]
    qsl = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    path = np.concatenate([np.arange(20), np.arange(20), np.arange(10), [0, 0, 5, 2, 11, 1 << 30, -7, 9, 9, 9],
                           np.arange(10)]).astype(np.int32)
    path[1:15] += 5
    path[21:35] += 4
    path[41:45] += 3
    count = np.asarray([15, 15, 5, 10, -3], np.int32)
    bt = v.block_tables.cpu().numpy()
    exp = [masked.tree_commit(x, bt, lens, path, count, qsl) for x in rows_of(v)]
    v.commit_tree(path, count, qsl)
    for got, (rows, after) in zip(rows_of(v), exp):
        np.testing.assert_array_equal(got, rows)
    np.testing.assert_array_equal(v.kv_lens.cpu().numpy(), exp[0][1])


# ---------------------------------------------------------------- whole steps
@pytest.mark.parametrize("kind", ["f16", "bf16", "fp8", "q4", "q8"])
def test_step_leaves_what_plain_decoding_writes(cuda, kind):
    """Prompt, drafted trees written with rotation, attention, acceptance, commit: the cache then holds, and the next
    token's attention gives, what writing the accepted tokens one after the other would have."""
    op = OperationRegistry.create("unified_attention")
    hq, hkv, d, page = 8, 2, 64, 16
    dt = torch.bfloat16 if kind == "bf16" else torch.float16
    rope = RotaryEmbedding(d, base=10000.0)
    g = torch.Generator().manual_seed(11)
    make = lambda n: tuple(torch.randn(n, h, d, generator=g).to(dt).to(cuda) for h in (hq, hkv, hkv))  # noqa: E731

    def fresh():
        kw = dict(num_seqs=3, max_seq_len=192, num_kv_heads=hkv, head_dim=d, block_size=page, device=cuda)
        if kind in ("q4", "q8"):
            return AffinePageCacheView.init(bits=int(kind[1]), group_size=64, **kw)
        return Fp8PageCacheView.init(**kw) if kind == "fp8" else PageCacheView.init(dtype=dt, **kw)

    def step(view, qkv, lens, **rule):
        q, kc, vc, md = view.concatenate_to_cache(
            *qkv, cache_metadata=PageMetadata(query_start_loc=None, slot_ids=(0, 1, 2), **rule), rope=rope,
            slot_ids=(0, 1, 2), query_lens=lens)
        md.query_start_loc = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32, device=cuda)
        return op(query=q, key=kc, value=vc, cache_metadata=md, cache_view=view).attention_outputs

    prompt, sizes = make(60), (9, 1, 25)
    a, b = fresh(), fresh()
    for v in (a, b):
        step(v, prompt, (30, 13, 17))
    tokens, targets, parents, qsl = drafted(np.random.default_rng(2), sizes, 3)
    rows = make(35)
    out = step(a, rows, sizes, tree_parents=torch.from_numpy(parents).to(cuda))
    took = tree_accept(torch.from_numpy(tokens).to(cuda), torch.from_numpy(targets).to(cuda), parents, qsl)
    a.commit_tree(took.path, took.accepted, qsl)
    count = took.accepted.tolist()
    assert max(count) > 2
    # the accepted tokens of every sequence as one causal run
    nodes = [qsl[s] + int(n) for s in range(3) for n in took.path.tolist()[qsl[s]:qsl[s] + count[s]]]
    run = tuple(x[nodes] for x in rows)
    exp = step(b, run, tuple(count))
    assert a.kv_lens.tolist() == b.kv_lens.tolist() == [30 + count[0], 13 + count[1], 17 + count[2]]
    if kind != "fp8":  # (FP8: the two writes have other maxima, so other scales)
        cu = torch.tensor([0, *np.cumsum(a.kv_lens.tolist())])
        for x, y in zip(a.gather_kv_cache(a.block_tables, cu), b.gather_kv_cache(b.block_tables, cu)):
            assert torch.equal(x, y)
        # the nodes of the path saw the same keys: the two outputs differ by the order of their sums
        err = (out[nodes].double() - exp.double()).abs()
        assert (err <= 2 * torch.finfo(dt).eps / 2 * exp.double().abs() + 2.0 ** -14).all()
        x, y = step(a, nxt := make(3), (1, 1, 1)), step(b, nxt, (1, 1, 1))
        assert torch.equal(x, y)


def test_positions_of_other_rotations(cuda):
    """A callable that is no RotaryEmbedding gets every node's own position."""
    rope = RotaryEmbedding(64, base=500.0)
    turned = lambda x, offset=0: rope(x, offset=offset)  # noqa: E731
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(8, h, 64, generator=g).half().to(cuda) for h in (4, 2, 2)]
    parents = torch.tensor([-1, 0, 0, 1, -1, 0, 1, 0], dtype=torch.int32, device=cuda)
    md = PageMetadata(query_start_loc=None, slot_ids=(1, 0), tree_parents=parents)
    out = []
    for r in (turned, rope):
        v = PageCacheView.init(num_seqs=2, max_seq_len=64, num_kv_heads=2, head_dim=64, device=cuda)
        v.kv_lens.copy_(torch.tensor([5, 9], dtype=torch.int32))
        q, *_ = v.concatenate_to_cache(*x, cache_metadata=md, rope=r, query_lens=(4, 4))
        out.append((q, v.key_cache))
    pos = torch.tensor([9, 10, 10, 11, 5, 6, 7, 6], device=cuda)
    exp = rope.rotate(x[0].transpose(0, 1), pos).transpose(0, 1)
    for q, _ in out:
        # one fp16 rounding on either side and fp32 sines of angles up to 11
        assert ((q - exp).abs().float() <= 2.0 ** -10 * exp.abs().float() + 2.0 ** -18).all()
    assert ((out[0][1] - out[1][1]).abs().float() <= 2.0 ** -10 * out[1][1].abs().float() + 2.0 ** -18).all()


def test_captured_verification(cuda):
    """Acceptance and commit of a whole cache in one graph, replayed over changed trees with eager work between."""
    views = [view_of("f16", cuda, seed=s) for s in range(3)]
    cache = PageCache(views)
    sizes, lens = [25, 1, 40, 7, 9], [60, 1, 96, 30, 9]
    rng = np.random.default_rng(5)
    tokens, targets, parents, qsl = (torch.from_numpy(x).to(cuda) for x in drafted(rng, sizes, 3))
    before = [[t.clone() for t in v.page_arrays()] for v in views]

    def reset():
        for v, old in zip(views, before):
            v.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32, device=cuda))
            for t, o in zip(v.page_arrays(), old):
                t.copy_(o)

    def step():
        took = tree_accept(tokens, targets, parents, qsl)
        cache.commit_tree(took.path, took.accepted, qsl)
        return took

    reset()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            took = step()
    for i in range(3):
        tk, tg, pr, q = drafted(np.random.default_rng(20 + i), sizes, 3)
        for dst, src in ((tokens, tk), (targets, tg), (parents, pr)):
            dst.copy_(torch.from_numpy(src).to(cuda))
        reset()
        torch.cuda.synchronize()
        exp = masked.tree_accept(tk, tg, pr, q)
        rows = [[masked.tree_commit(x, v.block_tables.cpu().numpy(), lens, exp[0], exp[1], q) for x in rows_of(v)]
                for v in views]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(took, exp):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
        for v, r in zip(views, rows):
            for got, (x, after) in zip(rows_of(v), r):
                np.testing.assert_array_equal(got, x)
                np.testing.assert_array_equal(v.kv_lens.cpu().numpy(), after)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_captured_decode_with_sinks(cuda, kind):
    """A decode step with sinks in the metadata, through the compiled proxy and the operator in one graph: every replay
    gives what the eager views give."""
    from easymlx_amd import CompiledPagedCacheProxy

    op = OperationRegistry.create("unified_attention")
    S, hq, hkv, d, page = 5, 8, 2, 64, 16
    g = torch.Generator().manual_seed(4)
    make = lambda n: tuple(torch.randn(n, h, d, generator=g).half().to(cuda) for h in (hq, hkv, hkv))  # noqa: E731
    kw = dict(num_seqs=S, max_seq_len=192, num_kv_heads=hkv, head_dim=d, block_size=page, device=cuda)
    a, b = (AffinePageCacheView.init(bits=4, group_size=64, **kw) if kind == "q4"
            else PageCacheView.init(dtype=torch.float16, **kw) for _ in range(2))
    slots, lens = tuple(range(S)), (60, 1, 100, 33, 7)
    prompt = make(sum(lens))
    for v in (a, b):
        v.concatenate_to_cache(*prompt, cache_metadata=PageMetadata(query_start_loc=None, slot_ids=slots),
                               slot_ids=slots, query_lens=lens)
    md = PageMetadata(query_start_loc=torch.arange(S + 1, dtype=torch.int32, device=cuda), slot_ids=slots,
                      sliding_window=20, sink_tokens=3, is_single_token_decode=True)
    proxy, buf, out = CompiledPagedCacheProxy(a), make(S), torch.zeros(S, hq, d, dtype=torch.float16, device=cuda)

    def step():
        q, kc, vc, m = proxy.concatenate_to_cache(*buf, cache_metadata=md)
        out.copy_(op(query=q, key=kc, value=vc, cache_metadata=m, cache_view=a).attention_outputs)

    def eager():
        q, kc, vc, m = b.concatenate_to_cache(*buf, cache_metadata=md, slot_ids=slots, query_lens=(1,) * S)
        return op(query=q, key=kc, value=vc, cache_metadata=m, cache_view=b).attention_outputs

    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    first = eager()
    assert torch.equal(out, first) and bool(first.abs().sum() > 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(4):
        for x, y in zip(buf, make(S)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager()) and torch.equal(a.kv_lens, b.kv_lens)
        # without its sinks the step gives something else
        plain = op(query=buf[0], key=b.key_cache, value=b.value_cache, cache_view=b,
                   cache_metadata=PageMetadata(query_start_loc=md.query_start_loc, block_tables=b.block_tables,
                                               kv_lens=b.kv_lens, block_size=page, sliding_window=20,
                                               is_single_token_decode=True)).attention_outputs
        assert not torch.equal(out, plain)
