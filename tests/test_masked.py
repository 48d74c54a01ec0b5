"""Masked attention, drafted trees and their commit on the CPU: the oracle against known answers, refusals of the
Python entry points and argument errors of the C ones (no kernel is launched here)."""

import ctypes

import numpy as np
import pytest
import torch

from easymlx_amd import PageCache, PageCacheView, PageMetadata, commit_tree, paged_attention, tree_accept, tree_attention
from oracle import masked
from oracle.paged_attention import paged_attention as oracle_attention

TREE = [-1, 0, 0, 1, 2, 2, 4]  # 0 - (1 - 3, 2 - (4 - 6, 5))


def _cache(rng, nb, bs, hkv, d):
    return rng.standard_normal((nb, bs, hkv, d)), rng.standard_normal((nb, bs, hkv, d))


# ---------------------------------------------------------------- the oracle
def test_ancestors_known_answer():
    see, depth = masked.ancestors(TREE)
    assert [np.flatnonzero(r).tolist() for r in see] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 5],
                                                         [0, 2, 4, 6]]
    assert depth.tolist() == [0, 1, 1, 2, 2, 2, 3]
    # entries that are no earlier node make roots
    see, depth = masked.ancestors([5, 1, 0, 7, -3])
    assert depth.tolist() == [0, 0, 1, 0, 0] and see.sum() == 6


def test_visible_known_answers():
    s = lambda m: ["".join(".x"[int(v)] for v in r) for r in m]  # noqa: E731
    assert s(masked.visible(2, 6, 2, 1)) == ["x..xx.", "x...xx"]
    assert s(masked.visible(1, 4, 2, 3)) == ["xxxx"]  # sinks that reach the window
    assert s(masked.visible(3, 5, 0, 0, [-1, 0, 0])) == ["xxx..", "xxxx.", "xxx.x"]
    # places: node 2 stands at 3, as node 1 does: a window of 2 reaches back to the root
    assert s(masked.visible(3, 5, 2, 1, [-1, 0, 0])) == ["xxx..", "x.xx.", "x.x.x"]
    assert s(masked.visible(4, 2, 0, 0, [-1, 0, 1, 0])) == ["..", "..", "x.", ".x"]  # a tree longer than its cache


@pytest.mark.parametrize("window", [0, 1, 5])
def test_oracle_is_the_paged_one_without_sinks(window):
    rng = np.random.default_rng(3)
    k, v = _cache(rng, 9, 4, 2, 8)
    tables = np.array([[0, 5, 7, -1], [1, 2, 3, 8]], np.int32)
    q = rng.standard_normal((6, 4, 8))
    lens, qsl = np.array([9, 14], np.int32), np.array([0, 2, 6], np.int32)
    exp = oracle_attention(q, k, v, tables, lens, qsl, sliding_window=window, compute_dtype=np.float64,
                           out_dtype=np.float64)
    for parents in (None, np.array([-1, 0, -1, 0, 1, 2])):  # chains are causal runs
        got = masked.masked_attention(q, k, v, tables, lens, qsl, window=window, parents=parents)
        np.testing.assert_allclose(got, exp, rtol=0, atol=1e-12)


def test_oracle_accept_and_commit_known_answers():
    tokens = np.array([9, 1, 2, 3, 4, 4, 6, 50, 60], np.int64)
    targets = np.array([2, 3, 4, 0, 6, 0, 77, 60, 8], np.int64)
    parents = np.array(TREE + [-1, 0], np.int32)
    path, accepted, following = masked.tree_accept(tokens, targets, parents, [0, 7, 7, 9])
    assert path.tolist() == [0, 2, 4, 6, -1, -1, -1, 0, 1]
    assert accepted.tolist() == [4, 0, 2] and following.tolist() == [77, -1, 8]
    rows = np.arange(24).reshape(6, 4)
    tables = np.array([[5, 0, 1], [2, 3, 4], [2, 3, 4]], np.int32)
    new, lens = masked.tree_commit(rows, tables, [9, 5, 4], path, accepted, [0, 7, 7, 9])
    # sequence 0's tree starts at position 2: rows 2 3 | 4 5 6 7 | 8 in pages 5, 0, 1
    assert new[5].tolist() == [20, 21, 22, 0] and new[0].tolist() == [2, 4, 2, 3]
    assert lens.tolist() == [6, 5, 4] and (new[1:5] == rows[1:5]).all()


# ---------------------------------------------------------------- refusals
def _dense(T=3, hq=4, hkv=2, d=8, nb=3, bs=4, S=1):
    return (torch.zeros(T, hq, d), torch.zeros(nb, bs, hkv, d), torch.zeros(nb, bs, hkv, d),
            torch.zeros(S, 2, dtype=torch.int32), torch.full((S,), 5, dtype=torch.int32),
            torch.tensor([0, T], dtype=torch.int32))


def test_attention_refusals():
    a = _dense()
    with pytest.raises(ValueError, match="sink_tokens must be >= 0"):
        paged_attention(*a, sliding_window=4, sink_tokens=-1)
    with pytest.raises(ValueError, match="requires tree_parents"):
        tree_attention(*a, None)
    with pytest.raises(ValueError, match="tree_parents must be rank-1"):
        tree_attention(*a, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="tree_parents must be rank-1"):
        tree_attention(*a, torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="must be integers"):
        tree_attention(*a, torch.zeros(3))
    with pytest.raises(RuntimeError, match="GPU only"):
        tree_attention(*a, [-1, 0, 0])
    with pytest.raises(RuntimeError, match="GPU only"):
        paged_attention(*a, sliding_window=4, sink_tokens=1)
    out = tree_attention(torch.ones(0, 4, 8), *a[1:5], torch.zeros(2, dtype=torch.int32), [])
    assert out.shape == (0, 4, 8)


def test_accept_refusals():
    t = torch.zeros(3, dtype=torch.int64)
    qsl = [0, 3]
    with pytest.raises(ValueError, match="one length"):
        tree_accept(t, t[:2], [-1, 0, 0], qsl)
    with pytest.raises(ValueError, match="int32 or int64"):
        tree_accept(t, t.int(), [-1, 0, 0], qsl)
    with pytest.raises(ValueError, match="int32 or int64"):
        tree_accept(t.float(), t.float(), [-1, 0, 0], qsl)
    with pytest.raises(ValueError, match="tree_parents"):
        tree_accept(t, t, [-1, 0], qsl)
    with pytest.raises(ValueError, match="query_start_loc"):
        tree_accept(t, t, [-1, 0, 0], torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="GPU only"):
        tree_accept(t, t, [-1, 0, 0], qsl)


def test_commit_refusals():
    view = PageCacheView.init(num_seqs=2, max_seq_len=16, num_kv_heads=1, head_dim=8, block_size=4, device="cpu")
    path = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="one entry more"):
        view.commit_tree(path, [1], [0])
    with pytest.raises(ValueError, match="more trees than sequences"):
        view.commit_tree(path, [1, 1, 1], [0, 1, 2, 3])
    with pytest.raises(ValueError, match="only once"):
        view.commit_tree(path, [1, 1], [0, 1, 3], slot_ids=[1, 1])
    with pytest.raises(ValueError, match="one sequence per tree"):
        view.commit_tree(path, [1, 1], [0, 1, 3], slot_ids=[1])
    with pytest.raises(ValueError, match="path must be rank-1"):
        view.commit_tree(path[None], [1], [0, 3])
    with pytest.raises(RuntimeError, match="GPU only"):
        PageCache([view]).commit_tree(path, [1], [0, 3])
    other = PageCacheView.init(num_seqs=2, max_seq_len=16, num_kv_heads=2, head_dim=8, block_size=4, device="cpu")
    other.key_cache = other.key_cache[:, :, :1]
    with pytest.raises(ValueError, match="contiguous"):
        commit_tree([other], path, [1], [0, 3])
    commit_tree([], path, [1], [0, 3])


def test_metadata_carries_the_rule():
    md = PageMetadata(query_start_loc=[0, 1], sliding_window=8, sink_tokens=4, tree_parents=[-1])
    md = md.with_cache_state(block_tables=0, kv_lens=0, block_size=16).with_sliding_window(9)
    assert md.sink_tokens == 4 and md.tree_parents == [-1] and md.sliding_window == 9


def test_write_refuses_parents_of_another_length():
    view = PageCacheView.init(num_seqs=1, max_seq_len=16, num_kv_heads=1, head_dim=8, block_size=4, device="cpu")
    x = torch.zeros(2, 1, 8)
    for parents in ([-1], [[-1, 0]], [-1.0, 0.0]):
        md = PageMetadata(query_start_loc=[0, 2], slot_ids=(0,), tree_parents=torch.tensor(parents))
        with pytest.raises(ValueError, match="tree_parents"):
            view.concatenate_to_cache(x, x, x, cache_metadata=md)


@pytest.fixture(scope="module")
def lib():
    import os

    from easymlx_amd import _native

    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libemx_attn.so not built (run __graft_entry__.build())")
    return _native.load()


def test_abi_argument_errors(lib):
    from easymlx_amd import _native

    invalid, unsupported, ok = _native.EMX_ERR_INVALID, _native.EMX_ERR_UNSUPPORTED, _native.EMX_OK
    one = ctypes.c_int64(0)
    p = ctypes.addressof(one)

    def dense(T=1, hq=4, d=64, dtype=0, k=p, nb=1, bs=16, hkv=2, S=1, mb=1, scale=1.0, window=4, sinks=1):
        return lib.emx_masked_attention_dense(p, T, hq, d, dtype, k, k, nb, bs, hkv, p, S, mb, p, p, scale, window,
                                              sinks, None, 0, None, 0, p, None)

    assert dense(hq=3) == invalid and b"GQA" in lib.emx_last_error()
    assert dense(scale=0.0) == invalid and b"softmax_scale" in lib.emx_last_error()
    assert dense(scale=float("nan")) == invalid and dense(scale=-1.0) == invalid
    assert dense(sinks=-1) == invalid and b"sink_tokens" in lib.emx_last_error()
    assert dense(d=320) == unsupported and dense(dtype=7) == unsupported
    assert dense(mb=1 << 28) == unsupported and b"2^31" in lib.emx_last_error()
    assert dense(k=None) == invalid
    assert dense(T=0) == ok

    def affine(bits=4, gs=64, bs=16, k=p):
        return lib.emx_masked_attention_affine(p, 1, 4, 64, k, k, k, k, k, k, 1, bs, 2, bits, gs, p, 1, 1, p, p, 1.0, 4,
                                               1, None, 0, None, 0, p, None)

    assert affine(bits=3) == unsupported and affine(gs=48) == invalid and affine(bs=12) == invalid
    assert affine(bs=72) == invalid and affine(k=None) == invalid
    assert lib.emx_masked_attention_fp8(p, 1, 4, 64, 0, p, p, None, p, 1, 16, 2, p, 1, 1, p, p, 1.0, 4, 1, None, 0,
                                        None, 0, p, None) == invalid

    assert lib.emx_tree_positions(None, p, 1, 1, p, None) == invalid
    assert lib.emx_tree_positions(None, None, 0, 0, None, None) == ok
    assert lib.emx_tree_accept(p, p, 2, p, p, 1, 1, p, p, p, None) == unsupported
    assert lib.emx_tree_accept(p, p, 4, p, p, -1, 1, p, p, p, None) == invalid
    assert lib.emx_tree_accept(p, p, 4, None, p, 1, 1, p, p, p, None) == invalid
    ptr = (ctypes.c_void_p * 6)(*[p] * 6)
    rows = lambda n=1, k=ptr, row=64, bs=16, nb=1, S=1, slots=None, trees=1, path=p: lib.emx_tree_commit_rows(  # noqa: E731
        n, k, ptr, row, bs, nb, ptr, S, 1, ptr, slots, trees, path, p, p, 1, None)
    assert rows(n=-1) == invalid and rows(row=0) == invalid and rows(bs=0) == invalid and rows(path=None) == invalid
    assert rows(trees=2) == invalid and b"more trees" in lib.emx_last_error()
    assert rows(nb=1 << 28) == unsupported and rows(S=1 << 20, trees=70000) == unsupported
    assert rows(k=(ctypes.c_void_p * 1)(None)) == invalid and rows(k=None) == invalid
    assert rows(n=0) == ok and rows(trees=0) == ok
    aff = lambda bits=4, d=64, gs=64, arr=ptr: lib.emx_tree_commit_affine(  # noqa: E731
        1, arr, 2, d, bits, gs, 16, 1, ptr, 1, 1, ptr, None, 1, p, p, p, 1, None)
    assert aff(bits=2) == unsupported and aff(d=60) == invalid and aff(arr=None) == invalid


def test_masked_workspace_bytes(lib):
    """Room for the parts of cut tiles where a call has few tiles; none where its tiles fill the GPU."""
    head = lib.emx_paged_workspace_zeroed_bytes()
    assert lib.emx_masked_workspace_bytes(25, 1, 32, 8, 128) > head
    assert lib.emx_masked_workspace_bytes(1, 1, 32, 8, 96) == 0
    assert lib.emx_masked_workspace_bytes(16384, 4, 32, 8, 128) == 0
    assert lib.emx_masked_workspace_bytes(1, 1, 200, 1, 128) == 0  # more heads than a tile's columns
    assert lib.emx_masked_workspace_bytes(0, 1, 32, 8, 128) == 0
