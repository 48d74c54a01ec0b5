"""Verification of drafted token trees over a paged cache.

A step of speculative decoding with a tree, for every sequence of a batch:

1. the drafted tokens' rows are written behind the sequence (``concatenate_to_cache`` with
   ``PageMetadata.tree_parents``: a node is rotated at the position that it has if its path is taken);
2. :func:`tree_attention` in every layer: a node sees the tokens before the tree, itself and its ancestors;
3. :func:`tree_accept`: the path of nodes that the model agrees with, and its next token;
4. ``PageCache.commit_tree``: that path's rows move to the front of the tree's place in every layer.

``tree_parents [total_tokens]`` holds, for every row of the call, the index of its parent within its own sequence's
rows (an earlier row; ``-1``, as any other value, makes a root).  A chain (``parents[i] = i - 1``) is an ordinary
causal run of tokens.  The reference has no counterpart.
"""

from __future__ import annotations

import typing as tp

import torch

from .. import _native
from .unified_attention import _i32, paged_attention


class TreeAccept(tp.NamedTuple):
    """What :func:`tree_accept` returns."""

    path: torch.Tensor  # int32 [total_tokens]: row query_start_loc[s] + k is the path's k-th node, -1 behind the path
    accepted: torch.Tensor  # int32 [num_seqs]: nodes of the path
    next_tokens: torch.Tensor  # [num_seqs] in the tokens' dtype: the model's choice after the path, -1 for no tree


def tree_attention(
    queries: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables,
    kv_lens,
    query_start_loc,
    tree_parents,
    *,
    softmax_scale: float | None = None,
    sliding_window: int | None = None,
    sink_tokens: int | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    k_biases: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    v_biases: torch.Tensor | None = None,
    bits: int | None = None,
    group_size: int | None = None,
    workspace: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of drafted trees over a paged cache that already holds their keys and values.

    ``queries [total_tokens, Hq, D]``; rows ``query_start_loc[s] .. query_start_loc[s + 1]`` are the nodes of
    sequence ``s``, whose keys and values are the last ones of its ``kv_lens[s]`` tokens.  Node ``i`` sees every key
    before the tree and, in it, its own and its ancestors'.  ``sliding_window`` and ``sink_tokens`` go by places, a
    node's being the tree's start plus its depth.  Caches as in
    :func:`~easymlx_amd.operations.unified_attention.paged_attention`.  Trees may have any number of nodes.

    Returns ``[total_tokens, Hq, D]`` in the queries' dtype.
    """
    if tree_parents is None:
        raise ValueError("tree_attention requires tree_parents")
    return paged_attention(
        queries, key_cache, value_cache, block_tables, kv_lens, query_start_loc, softmax_scale=softmax_scale,
        sliding_window=sliding_window, sink_tokens=sink_tokens, tree_parents=tree_parents, k_scale=k_scale,
        v_scale=v_scale, k_scales=k_scales, k_biases=k_biases, v_scales=v_scales, v_biases=v_biases, bits=bits,
        group_size=group_size, workspace=workspace, out=out)


def tree_accept(tokens: torch.Tensor, targets: torch.Tensor, tree_parents, query_start_loc) -> TreeAccept:
    """The path of every drafted tree that the model agrees with.

    ``tokens [total_tokens]``: the nodes' tokens; ``targets [total_tokens]``: the token that the model chooses after
    each node (greedy, or drawn: a path of drawn tokens follows the model's distribution).  Node 0, the token that
    the last step chose, is always taken; then, of the last taken node's children, the first whose token is the
    target after that node, until there is none.  int32 or int64, on the device; nothing is read back to the host.
    """
    if tokens.ndim != 1 or targets.shape != tokens.shape:
        raise ValueError("tokens and targets must be rank-1 of one length: [total_tokens]")
    if tokens.dtype not in (torch.int32, torch.int64) or targets.dtype != tokens.dtype:
        raise ValueError("tokens and targets must be int32 or int64, both the same")
    if not isinstance(tree_parents, torch.Tensor):
        tree_parents = torch.as_tensor(tree_parents)
    if not isinstance(query_start_loc, torch.Tensor):
        query_start_loc = torch.as_tensor(query_start_loc)
    if tree_parents.shape != tokens.shape or tree_parents.is_floating_point():
        raise ValueError("tree_parents must be rank-1 integers: [total_tokens]")
    if query_start_loc.ndim != 1 or query_start_loc.shape[0] < 1:
        raise ValueError("query_start_loc must be rank-1: [num_seqs + 1]")
    dev = tokens.device
    if dev.type != "cuda":
        raise RuntimeError("tree_accept runs on the GPU only; tokens are on " + str(dev))
    if targets.device != dev:
        raise ValueError(f"targets must be on the tokens' device {dev}")
    tokens, targets = tokens.contiguous(), targets.contiguous()
    parents, qsl = _i32(tree_parents, dev), _i32(query_start_loc, dev)
    n, total = int(qsl.shape[0]) - 1, int(tokens.shape[0])
    path = torch.empty((total,), dtype=torch.int32, device=dev)
    accepted = torch.empty((n,), dtype=torch.int32, device=dev)
    following = torch.empty((n,), dtype=tokens.dtype, device=dev)
    with _native.on_device(dev):
        _native.check(_native.load().emx_tree_accept(
            tokens.data_ptr(), targets.data_ptr(), tokens.element_size(), parents.data_ptr(), qsl.data_ptr(), n, total,
            path.data_ptr(), accepted.data_ptr(), following.data_ptr(), _native.stream_ptr(dev)))
    return TreeAccept(path, accepted, following)


__all__ = ("TreeAccept", "tree_accept", "tree_attention")
