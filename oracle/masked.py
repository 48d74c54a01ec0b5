"""Masked paged attention, drafted trees and their commit, from their definitions (TEST INFRASTRUCTURE ONLY).

No counterpart in the reference: sequences, positions and empty rows follow :mod:`oracle.paged_attention`; what a row
sees is written out key by key.  Pinned by tests/test_masked.py: with no sinks and no tree the result is that of
:func:`oracle.paged_attention.paged_attention`, a chain is a causal run, and small trees have known answers.
"""

from __future__ import annotations

import numpy as np

from .paged_attention import gather_sequence


def ancestors(parents) -> tuple[np.ndarray, np.ndarray]:
    """(bool [n, n]: whether node j is node i or above it, depth [n]); an entry that is no earlier node makes a root."""
    n = len(parents)
    see, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i, p in enumerate(int(x) for x in parents):
        if 0 <= p < i:
            see[i] = see[p]
            depth[i] = depth[p] + 1
        see[i, i] = True
    return see, depth


def visible(q_len: int, kv_len: int, window: int, sinks: int, parents=None) -> np.ndarray:
    """bool [q_len, kv_len]: the keys that each query of a sequence sees."""
    past = kv_len - q_len
    key = np.arange(kv_len)
    if parents is None:
        at, place = past + np.arange(q_len), key
        see = key[None] <= at[:, None]
    else:
        up, depth = ancestors(parents)
        at = past + depth
        first = max(past, 0)
        see = np.ones((q_len, kv_len), bool)
        see[:, first:] = up[:, first - past:]
        place = key.copy()
        place[first:] = at[first - past:]
    if window > 0:
        see &= (place[None] > at[:, None] - window) | (place[None] < sinks)
    return see


def masked_attention(queries, key_cache, value_cache, block_tables, kv_lens, query_start_loc, *, window=0, sinks=0,
                     parents=None, softmax_scale=None) -> np.ndarray:
    """float64 ``[T, Hq, D]`` over a logical ``[nb, bs, Hkv, D]`` cache; rows of no sequence are zeros."""
    q = np.asarray(queries, np.float64)
    T, hq, d = q.shape
    hkv = key_cache.shape[2]
    scale = 1.0 / np.sqrt(d) if softmax_scale is None else softmax_scale
    out = np.zeros(q.shape)
    cap = block_tables.shape[1] * key_cache.shape[1]
    for s in range(len(kv_lens)):
        lo, hi = int(query_start_loc[s]), int(query_start_loc[s + 1])
        n = min(max(int(kv_lens[s]), 0), cap)
        if hi <= lo or n == 0:
            continue
        k, ok = gather_sequence(key_cache, block_tables[s], n)
        v, _ = gather_sequence(value_cache, block_tables[s], n)
        see = visible(hi - lo, n, window, sinks, None if parents is None else parents[lo:hi]) & ok[None]
        for h in range(hq):
            x = scale * (q[lo:hi, h] @ k[:, h // (hq // hkv)].astype(np.float64).T)
            x = np.where(see, x, -np.inf)
            top = x.max(axis=1, keepdims=True)
            p = np.where(see, np.exp(x - np.where(np.isfinite(top), top, 0)), 0)
            total = p.sum(axis=1, keepdims=True)
            o = p @ v[:, h // (hq // hkv)].astype(np.float64)
            out[lo:hi, h] = np.where(total > 0, o / np.where(total > 0, total, 1), 0)
    return out


def tree_accept(tokens, targets, parents, query_start_loc):
    """(path [T], accepted [S], next [S])."""
    path = np.full(len(tokens), -1, np.int32)
    accepted, following = [], []
    for lo, hi in zip(query_start_loc[:-1], query_start_loc[1:]):
        took = [0] if hi > lo else []
        while took:
            c = took[-1]
            hit = [j for j in range(c + 1, hi - lo) if parents[lo + j] == c and tokens[lo + j] == targets[lo + c]]
            if not hit:
                break
            took.append(hit[0])
        path[lo:lo + len(took)] = took
        accepted.append(len(took))
        following.append(targets[lo + took[-1]] if took else -1)
    return path, np.asarray(accepted, np.int32), np.asarray(following)


def tree_commit(rows, block_tables, kv_lens, path, accepted, query_start_loc, slot_ids=None):
    """``(rows, kv_lens)`` after the commit; ``rows [nb, bs, ...]``: anything that a cache holds per token."""
    rows, lens = rows.copy(), np.array(kv_lens)
    nb, bs = rows.shape[:2]
    for i, count in enumerate(accepted):
        s = i if slot_ids is None else int(slot_ids[i])
        lo, n = int(query_start_loc[i]), int(query_start_loc[i + 1] - query_start_loc[i])
        if not 0 <= s < len(lens) or n <= 0:
            continue
        first = int(lens[s]) - n
        for k in range(min(max(int(count), 0), n)):
            src, dst = first + int(path[lo + k]), first + k
            if not k < int(path[lo + k]) < n or dst < 0 or src // bs >= block_tables.shape[1]:
                continue
            a, b = block_tables[s, src // bs], block_tables[s, dst // bs]
            if 0 <= a < nb and 0 <= b < nb:
                rows[b, dst % bs] = rows[a, src % bs]
        lens[s] = first + min(max(int(count), 0), n)
    return rows, lens
