"""Keeping the accepted path of a drafted tree in the cache.

The rows of a tree's nodes stand behind their sequence in the order of the call.  Once a path through the tree is
accepted (:func:`~easymlx_amd.operations.tree_attention.tree_accept`), its rows move to the front of the tree's place,
where they have the positions that they were rotated for, and the sequence's length drops to the path's end.  The
reference has no counterpart; its ``PageCacheView.copy_blocks`` (``lib/python/easymlx/caching/paged/cache.py:944-972``)
moves whole pages.
"""

from __future__ import annotations

import ctypes
import operator
import typing as tp

import torch

from .. import _native


def _shape_of(view) -> tuple:
    """What the layers of one launch have alike."""
    return (type(view).page_arrays, view.block_tables.shape, view.key_cache.shape, view.value_cache.shape,
            view.block_size, view.num_kv_heads, view.head_dim, view.key_cache.dtype, getattr(view, "bits", None),
            getattr(view, "group_size", None))


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


class CommitPlan:
    """The arrays of several layers, checked and laid out for the launches of :func:`commit_tree`.

    A :class:`~easymlx_amd.caching.pagecache.PageCache` keeps one for its views: checking the arrays of 32 layers and
    listing their addresses takes longer than moving the rows.  :meth:`fits` tells whether the views still hold
    those very tensors at those addresses.
    """

    def __init__(self, views: tp.Sequence[tp.Any]):
        self.views = list(views)
        dev = self.device = self.views[0].key_cache.device
        self.num_seqs = min(v.num_seqs for v in self.views)
        for v in self.views:
            if v.block_tables.dtype != torch.int32 or v.kv_lens.dtype != torch.int32:
                raise ValueError("block_tables and kv_lens must be int32")
            arrays = [*v.page_arrays(), v.block_tables, v.kv_lens]
            if any(not t.is_contiguous() for t in arrays):
                raise ValueError("commit_tree changes caches in place: they, tables and lengths must be contiguous")
            if any(t.device != dev for t in arrays):
                raise ValueError("the layers' caches, tables and lengths must be on one device")
        self.tensors = self._tensors(self.views)
        self.addresses = [t.data_ptr() for t in self.tensors]
        # runs of layers of one shape; a run that shared its lengths with another would see them change between the two
        runs: list[list] = []
        for v in self.views:
            if runs and _shape_of(runs[-1][0]) == _shape_of(v):
                runs[-1].append(v)
            else:
                runs.append([v])
        seen: dict[int, int] = {}
        for i, run in enumerate(runs):
            for v in run:
                if seen.setdefault(v.kv_lens.data_ptr(), i) != i:
                    raise ValueError("layers of different shapes cannot share kv_lens")
        self.runs = [self._run(r) for r in runs]

    @staticmethod
    def _tensors(views) -> list[torch.Tensor]:
        return [t for v in views for t in (*v.page_arrays(), v.block_tables, v.kv_lens)]

    @staticmethod
    def _run(views) -> tuple:
        """(affine, arguments before the trees, the sequences' arguments) of a run's C call."""
        v = views[0]
        seqs = (_pointers([x.block_tables for x in views]), v.num_seqs, v.blocks_per_seq,
                _pointers([x.kv_lens for x in views]))
        if v.is_affine:
            return True, (len(views), _pointers([t for x in views for t in x.page_arrays()]), v.num_kv_heads,
                          v.head_dim, v.bits, v.group_size, v.block_size, v.num_blocks), seqs
        row = v.num_kv_heads * v.head_dim * v.key_cache.element_size()
        return False, (len(views), _pointers([x.key_cache for x in views]), _pointers([x.value_cache for x in views]),
                       row, v.block_size, v.num_blocks), seqs

    def fits(self, views) -> bool:
        if len(views) != len(self.views) or not all(map(operator.is_, views, self.views)):
            return False
        now = self._tensors(views)
        return (len(now) == len(self.tensors) and all(map(operator.is_, now, self.tensors))
                and [t.data_ptr() for t in now] == self.addresses)


def _index(name: str, x, device) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x)
    if x.ndim != 1 or x.is_floating_point() or x.is_complex():
        raise ValueError(f"{name} must be rank-1 integers")
    if x.dtype == torch.int32 and x.device == device and x.is_contiguous():
        return x
    return x.to(device=device, dtype=torch.int32).contiguous()


def commit_tree(views: tp.Sequence[tp.Any], path, accepted, query_start_loc, *, slot_ids=None,
                plan: CommitPlan | None = None) -> None:
    """Keep the accepted path of every drafted tree in the caches of ``views`` (one per layer).

    Tree ``i`` is the last ``q = query_start_loc[i + 1] - query_start_loc[i]`` tokens of sequence ``slot_ids[i]``
    (``i`` without ``slot_ids``).  The row of node ``path[query_start_loc[i] + k]``, ``k < accepted[i]``, moves to
    position ``kv_len - q + k`` and the sequence's ``kv_lens`` entry becomes ``kv_len - q + accepted[i]``, in every
    layer; layers that share their ``kv_lens`` tensor see it change once.  ``path`` ascends inside a tree, as
    :func:`~easymlx_amd.operations.tree_attention.tree_accept` returns it.  Affine pages move codes, scales and biases
    as they are, FP8 pages codes: a tree's rows are written with one scale.  A sequence may appear once.
    Everything stays on the device: a step with this call can be captured in a graph.  ``plan``: the views'
    :class:`CommitPlan`, made for the call without it.
    """
    if not views:
        return
    if plan is None:
        plan = CommitPlan(views)
    dev = plan.device
    path, accepted = _index("path", path, dev), _index("accepted", accepted, dev)
    qsl = _index("query_start_loc", query_start_loc, dev)
    n = int(accepted.shape[0])
    if int(qsl.shape[0]) != n + 1:
        raise ValueError("query_start_loc must have one entry more than accepted")
    if slot_ids is None:
        if n > plan.num_seqs:
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
    if dev.type != "cuda":
        raise RuntimeError("commit_tree runs on the GPU only; the cache is on " + str(dev))
    total = int(path.shape[0])
    if n == 0 or total == 0:
        return
    slots = None
    if slot_ids is not None:
        slot_ids = (plan.views[0]._slot_ids_device(slot_ids) if isinstance(slot_ids, tuple)
                    else _index("slot_ids", slot_ids, dev))
        slots = slot_ids.data_ptr()
    lib = _native.load()
    with _native.on_device(dev):
        trees = (slots, n, path.data_ptr(), accepted.data_ptr(), qsl.data_ptr(), total, _native.stream_ptr(dev))
        for affine, arrays, seqs in plan.runs:
            call = lib.emx_tree_commit_affine if affine else lib.emx_tree_commit_rows
            _native.check(call(*arrays, *seqs, *trees))


__all__ = ("CommitPlan", "commit_tree")
