"""Keeping the accepted path of a drafted tree in the cache.

The rows of a tree's nodes stand behind their sequence in the order of the call.  Once a path through the tree is
accepted (:func:`~easymlx_amd.operations.tree_attention.tree_accept`), its rows move to the front of the tree's place,
where they have the positions that they were rotated for, and the sequence's length drops to the path's end.  The
reference has no counterpart; its ``PageCacheView.copy_blocks`` (``lib/python/easymlx/caching/paged/cache.py:944-972``)
moves whole pages.
"""

from __future__ import annotations

import ctypes
import typing as tp

import torch

from .. import _native


def _shape_of(view) -> tuple:
    """What the layers of one launch have alike."""
    return (type(view).page_arrays, view.num_seqs, view.blocks_per_seq, view.num_blocks, view.block_size,
            view.num_kv_heads, view.head_dim, view.key_cache.dtype, getattr(view, "bits", None),
            getattr(view, "group_size", None), view.key_cache.device)


def _index(name: str, x, device) -> torch.Tensor:
    x = torch.as_tensor(x)
    if x.ndim != 1 or x.is_floating_point() or x.is_complex():
        raise ValueError(f"{name} must be rank-1 integers")
    return x.to(device=device, dtype=torch.int32).contiguous()


def commit_tree(views: tp.Sequence[tp.Any], path, accepted, query_start_loc, *, slot_ids=None) -> None:
    """Keep the accepted path of every drafted tree in the caches of ``views`` (one per layer).

    Tree ``i`` is the last ``q = query_start_loc[i + 1] - query_start_loc[i]`` tokens of sequence ``slot_ids[i]``
    (``i`` without ``slot_ids``).  The row of node ``path[query_start_loc[i] + k]``, ``k < accepted[i]``, moves to
    position ``kv_len - q + k`` and the sequence's ``kv_lens`` entry becomes ``kv_len - q + accepted[i]``, in every
    layer; layers that share their ``kv_lens`` tensor see it change once.  ``path`` ascends inside a tree, as
    :func:`~easymlx_amd.operations.tree_attention.tree_accept` returns it.  Affine pages move codes, scales and biases
    as they are, FP8 pages codes: a tree's rows are written with one scale.  A sequence may appear once.
    Everything stays on the device: a step with this call can be captured in a graph.
    """
    views = list(views)
    if not views:
        return
    dev = views[0].key_cache.device
    path, accepted = _index("path", path, dev), _index("accepted", accepted, dev)
    qsl = _index("query_start_loc", query_start_loc, dev)
    n = int(accepted.shape[0])
    if int(qsl.shape[0]) != n + 1:
        raise ValueError("query_start_loc must have one entry more than accepted")
    if slot_ids is None:
        if any(n > v.num_seqs for v in views):
            raise ValueError("more trees than sequences")
    else:
        if not isinstance(slot_ids, torch.Tensor):
            slot_ids = tuple(int(s) for s in slot_ids)
            if len(set(slot_ids)) != len(slot_ids):
                raise ValueError("a sequence may appear only once in slot_ids")
        elif slot_ids.ndim != 1:
            raise ValueError("slot_ids must be rank-1")
        if len(slot_ids) != n:
            raise ValueError("slot_ids must hold one sequence per tree")
    for v in views:
        if v.block_tables.dtype != torch.int32 or v.kv_lens.dtype != torch.int32:
            raise ValueError("block_tables and kv_lens must be int32")
        if not v.kv_lens.is_contiguous() or any(not t.is_contiguous() for t in v.page_arrays()):
            raise ValueError("commit_tree changes caches and kv_lens in place: they must be contiguous")
        if v.key_cache.device != dev or v.block_tables.device != dev or v.kv_lens.device != dev:
            raise ValueError("the layers' caches, tables and lengths must be on one device")
    if dev.type != "cuda":
        raise RuntimeError("commit_tree runs on the GPU only; the cache is on " + str(dev))
    if n == 0 or int(path.shape[0]) == 0:
        return
    if slot_ids is not None:
        slot_ids = (views[0]._slot_ids_device(slot_ids) if isinstance(slot_ids, tuple)
                    else slot_ids.to(device=dev, dtype=torch.int32).contiguous())
    # runs of layers of one shape; a run that shares its lengths with another would see them change between the two
    runs: list[list] = []
    for v in views:
        if runs and _shape_of(runs[-1][0]) == _shape_of(v):
            runs[-1].append(v)
        else:
            runs.append([v])
    if len(runs) > 1:
        seen: dict[int, int] = {}
        for i, run in enumerate(runs):
            for v in run:
                if seen.setdefault(v.kv_lens.data_ptr(), i) != i:
                    raise ValueError("layers of different shapes cannot share kv_lens")
    with torch.cuda.device(dev):
        stream = _native.stream_ptr(dev)
        for run in runs:
            _commit(run, path, accepted, qsl, slot_ids, n, stream)


def _commit(views, path, accepted, qsl, slot_ids, n, stream) -> None:
    lib, v0, m = _native.load(), views[0], len(views)
    tables = [v.block_tables.contiguous() for v in views]
    pointers = lambda ts: (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])  # noqa: E731
    tree = (pointers(tables), v0.num_seqs, v0.blocks_per_seq, pointers([v.kv_lens for v in views]),
            None if slot_ids is None else slot_ids.data_ptr(), n, path.data_ptr(), accepted.data_ptr(), qsl.data_ptr(),
            int(path.shape[0]), stream)
    if v0.is_affine:
        rc = lib.emx_tree_commit_affine(m, pointers([t for v in views for t in v.page_arrays()]), v0.num_kv_heads,
                                        v0.head_dim, v0.bits, v0.group_size, v0.block_size, v0.num_blocks, *tree)
    else:
        rc = lib.emx_tree_commit_rows(m, pointers([v.key_cache for v in views]),
                                      pointers([v.value_cache for v in views]),
                                      v0.num_kv_heads * v0.head_dim * v0.key_cache.element_size(), v0.block_size,
                                      v0.num_blocks, *tree)
    _native.check(rc)


__all__ = ("commit_tree",)
