"""Attention with sinks, attention of a drafted tree, and the commit of its accepted path: what is timed and compared.

A case is one call as a serving loop makes it, over a paged cache:

* ``window`` -- ``paged_attention`` with a sliding window and a few first tokens that stay visible (sinks):
  a query at position ``p`` sees the keys ``k <= p`` with ``k > p - window`` or ``k < sinks``.  Decode batches
  (one query token per sequence) and ragged ones (prompt chunks, rows of one token beside them);
* ``tree``   -- ``tree_attention``: every sequence's last tokens in the cache are a tree of drafted tokens; a
  node sees the tokens before the tree and, inside it, itself and its ancestors;
* ``commit`` -- ``tree_accept`` and ``PageCache.commit_tree``: the path of drafted tokens that the target model
  agrees with, whose rows move to the front of the tree's place in the cache of every layer.

Caches: unquantized fp16 / bf16 ``[num_blocks, page, Hkv, D]``, FP8 (E4M3) codes in that layout with a scale per
page, affine 4-bit and 8-bit pages (key codes token-major, value codes dim-major in tiles, fp16 scale and bias per
token and group).  Lengths are spread over a case's range and the pages of a sequence lie anywhere in the pool.

``own`` false: plain torch in 32 bits.  ``own`` true: the calls a user makes.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"

# ---------------------------------------------------------------- cases


def _window(name, cache, seqs, ctx, q, hq, hkv, d, page, window, sinks, group=64, rows=0):
    return dict(name=name, kind="window", cache=cache, seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], q_lo=q[0], q_hi=q[1],
                hq=hq, hkv=hkv, d=d, page=page, group=group, window=window, sinks=sinks, rows=rows)


def _tree(name, cache, seqs, ctx, n, hq, hkv, d, page, group=64, window=0, sinks=0):
    return dict(name=name, kind="tree", cache=cache, seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], q_lo=n[0], q_hi=n[1],
                hq=hq, hkv=hkv, d=d, page=page, group=group, window=window, sinks=sinks, rows=0)


def _commit(name, cache, seqs, ctx, n, hkv, d, page, layers):
    return dict(name=name, kind="commit", cache=cache, seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], q_lo=n[0], q_hi=n[1],
                hkv=hkv, d=d, page=page, layers=layers)


def listed():
    return [
        # one user, one token, a short window: the latency of a call
        _window("window_one_f16", "f16", 1, (700, 700), (1, 1), 8, 2, 64, 16, 256, 4),
        # a serving batch over 4-bit pages, streams far longer than the window
        _window("window_batch_q4", "q4", 32, (2048, 16384), (1, 1), 32, 8, 128, 128, 4096, 4),
        # the same kind of batch over the default cache and page, odd lengths
        _window("window_batch_bf16", "bf16", 48, (3001, 20011), (1, 1), 32, 8, 128, 16, 4096, 64),
        # four prompts with a window much shorter than they are: the compute-bound call
        _window("window_prompts_bf16", "bf16", 4, (1500, 8500), (1500, 2500), 32, 8, 128, 16, 1024, 4),
        # continuous batching: three prompt chunks beside twelve decoding sequences, FP8 pages
        _window("window_mixed_fp8", "fp8", 15, (300, 9000), (203, 700), 32, 8, 128, 64, 2000, 16, rows=12),
        # head size 256 over 8-bit pages, a sink that is longer than a page
        _window("window_chunk_q8_d256", "q8", 3, (333, 5000), (33, 450), 16, 4, 256, 32, 700, 40),
        # one user drafting a small tree: the latency of a verification step
        _tree("tree_one_f16", "f16", 1, (1531, 1531), (25, 25), 32, 8, 128, 16),
        # a serving batch over 4-bit pages, trees of 16 nodes
        _tree("tree_batch_q4", "q4", 32, (512, 4096), (16, 16), 32, 8, 128, 128),
        # a smaller batch with large trees of different sizes over the default cache
        _tree("tree_wide_bf16", "bf16", 8, (500, 8000), (31, 60), 32, 8, 128, 16),
        # long documents: most of the call's time is reading the cache
        _tree("tree_long_bf16", "bf16", 12, (8000, 32768), (48, 64), 64, 8, 128, 64),
        # one user's accepted path moved in a small model's cache
        _commit("commit_one_f16", "f16", 1, (1531, 1531), (25, 25), 2, 64, 16, 16),
        # a serving batch's accepted paths moved in the 32 layers of a larger one
        _commit("commit_batch_bf16", "bf16", 32, (64, 600), (16, 60), 8, 128, 16, 32),
    ]


def draw(rng: random.Random):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("window", "window", "tree", "tree", "commit"))
        cache = rng.choice(("f16", "bf16") if kind == "commit" else ("f16", "bf16", "fp8", "q4", "q8"))
        hq, hkv = rng.choice(((32, 8), (16, 2), (8, 8), (28, 4), (64, 8), (16, 4), (12, 4)))
        d = rng.choice((64, 128, 128, 256))
        page = rng.choice((16, 32, 64, 128))
        seqs = log(1, 48)
        lo = log(1, 8000)
        hi = lo + log(1, 12000)
        if kind == "commit":
            n = log(2, 64)
            c = _commit("", cache, seqs, (lo % 600 + n, lo % 600 + n + hi % 300), (max(1, n // 2), n), hkv, d, page,
                        log(1, 32))
        elif kind == "tree":
            n = log(2, 64)
            c = _tree("", cache, seqs, (lo + n, hi + n), (max(1, n // 2), n), hq, hkv, d, page,
                      group=rng.choice((64, 128)) if d > 64 else 64)
            if rng.random() < 0.3:
                c.update(window=log(64, 4096), sinks=rng.choice((0, 1, 4, 64)))
        else:
            q = 1 if rng.random() < 0.5 else log(2, 2500)
            c = _window("", cache, seqs, (lo + q, hi + q), (max(1, q // 2), q), hq, hkv, d, page, log(16, 8192),
                        rng.choice((1, 4, 4, 16, 64, 129)), group=rng.choice((64, 128)) if d > 64 else 64)
            if q > 1 and seqs > 2:
                c["rows"] = rng.randrange(seqs)
        del c["name"]
        padded = c["seqs"] * c["ctx_hi"]  # what the plain form lays out: keys and scores
        if _cost(c) <= most and padded * hkv * d <= 1.2e9 and padded * c["q_hi"] * hq <= 3e9:
            return c


def _lens(case):
    """(query tokens, cached tokens) of every sequence, spread over the case's ranges."""
    q, ctx = [], []
    for i in range(case["seqs"]):
        u = (0.37 + 0.6180339887 * i) % 1.0
        v = (0.11 + 0.7548776662 * i) % 1.0
        single = case["kind"] == "window" and i >= case["seqs"] - case["rows"]
        n = 1 if single else case["q_lo"] + int(round(u * (case["q_hi"] - case["q_lo"])))
        q.append(n)
        ctx.append(max(n, case["ctx_lo"] + int(round(v * (case["ctx_hi"] - case["ctx_lo"])))))
    return q, ctx


_BITS = {"f16": 16, "bf16": 16, "fp8": 8, "q4": 4, "q8": 8}


def work(case):
    q, ctx = _lens(case)
    hkv, d = case["hkv"], case["d"]
    if case["kind"] == "commit":
        # an accepted path of a fifth of the tree, read and written, in every layer; the trees' integers
        moved = sum(max(1, n // 5) for n in q) * case["layers"] * hkv * d * 2 * 2
        return {"bytes": 2 * moved + 16 * sum(q), "flops": 0}
    w, sinks = case["window"], case["sinks"]
    token = 2 * hkv * (d * _BITS[case["cache"]] // 8 + (4 * (d // case["group"]) if case["cache"] in ("q4", "q8") else 0))
    keys, pairs = 0, 0
    for n, c in zip(q, ctx):
        if case["kind"] == "tree":
            old = c - n if w <= 0 else min(c - n, w - 1 + sinks)
            keys += old + n
            pairs += n * (old + 1)
        else:
            first = max(0, c - n - w + 1)  # of the first query's window
            keys += c - first + min(sinks, first)
            for p in (c - n, c - 1) if n > 64 else range(c - n, c):
                seen = min(p + 1, w + min(sinks, max(0, p + 1 - w)))
                pairs += seen * (n / 2 if n > 64 else 1)
    t = sum(q)
    return {"bytes": keys * token + 2 * t * case["hq"] * d * 2, "flops": 4 * pairs * case["hq"] * d}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---------------------------------------------------------------- inputs


def _e4m3(codes):
    """Values of FP8 codes: no NaN code, exponent 15 with mantissa 7 is 480."""
    c = codes.to(torch.int32)
    e, m = (c >> 3) & 15, (c & 7).to(torch.float32)
    v = torch.where(e == 0, m * 2.0**-9, torch.ldexp(1 + m / 8, e - 7))
    return torch.where(c >= 128, -v, v)


def _v_shifts(bits):
    """Bit offsets of a value word's tokens: in order at 8 bits; at 4 token k at nibble (k >> 1) | (k & 1) << 2."""
    return [8 * k for k in range(4)] if bits == 8 else [4 * ((k >> 1) | ((k & 1) << 2)) for k in range(8)]


def _pack(codes, shifts):
    """[..., n * len(shifts)] small integers -> [..., n] 32-bit words."""
    c = codes.to(torch.int32).reshape(*codes.shape[:-1], -1, len(shifts))
    return (c << torch.tensor(shifts, dtype=torch.int32, device=c.device)).sum(-1, dtype=torch.int32)


def _affine(x, group, bits):
    """Codes [.., D], scales and biases [.., D / group] (fp16) of the rows x, each group from its least to its largest."""
    g = x.reshape(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / (2**bits - 1)).clamp(min=1e-4).half()
    bias = lo.half()
    code = ((g - bias.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 2**bits - 1)
    return code.reshape(x.shape), scale, bias


def _pages(case, g, nb):
    """The pool's arrays for one layer: random keys and values as the cache's writes leave them."""
    page, hkv, d, kind = case["page"], case["hkv"], case["d"], case["cache"]
    out = {}
    for name, spread in (("k", 1.0), ("v", 0.7)):
        x = torch.empty((nb, page, hkv, d), device=DEV, dtype=torch.float16).normal_(0, spread, generator=g)
        if kind in ("f16", "bf16"):
            out[name] = x.to(torch.float16 if kind == "f16" else torch.bfloat16)
        elif kind == "fp8":
            scale = x.abs().amax((1, 2, 3)).float() / 240
            codes = torch.empty(x.shape, dtype=torch.uint8, device=DEV)
            table = _e4m3(torch.arange(0, 120, device=DEV))  # up to 240, ascending
            mid = (table[1:] + table[:-1]) / 2
            for part in range(0, nb, 4096):  # (the search works in 64-bit indexes)
                y = x[part:part + 4096].float() / scale[part:part + 4096, None, None, None].clamp(min=1e-12)
                at = torch.bucketize(y.abs(), mid)
                codes[part:part + 4096] = (at + (y < 0) * 128).to(torch.uint8)
            out[name], out[name + "_scale"] = codes, scale
        else:
            bits = int(kind[1])
            per = 32 // bits
            tile = min(page, 256 // bits)
            words, scales, biases = [], [], []
            for part in range(0, nb, 1024):
                code, scale, bias = _affine(x[part:part + 1024].float(), case["group"], bits)
                code = code.permute(0, 2, 1, 3)  # [nb, Hkv, page, D]
                if name == "k":
                    words.append(_pack(code, [bits * k for k in range(per)]))
                else:
                    t = code.reshape(code.shape[0], hkv, page // tile, tile, d).transpose(3, 4)
                    words.append(_pack(t, _v_shifts(bits)))
                scales.append(scale.permute(0, 2, 3, 1))  # [nb, Hkv, D / group, page]
                biases.append(bias.permute(0, 2, 3, 1))
            out[name] = torch.cat(words).contiguous()
            out[name + "_scales"] = torch.cat(scales).contiguous()
            out[name + "_biases"] = torch.cat(biases).contiguous()
    return out


def _parents(rs, n):
    """A tree of n drafted tokens in topological order: node 0 the root, others below a random earlier one."""
    return [-1] + [rs.randrange(max(0, (i - 4) // 2), i) if i > 1 else 0 for i in range(1, n)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rs = random.Random(int(seed))
    q, ctx = _lens(case)
    page, s = case["page"], case["seqs"]
    wide = max(-(-c // page) for c in ctx)
    need = [-(-c // page) for c in ctx]
    nb = sum(need) + 3
    order = torch.randperm(nb, device=DEV, generator=g).to(torch.int32)
    tables = torch.full((s, wide), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    st = dict(case=case, q_lens=q, tables=tables, qsl=i32(starts), total=starts[-1], longest=max(ctx), most_q=max(q))
    if case["kind"] != "window":
        parents = [_parents(rs, n) for n in q]
        st["parents"] = i32([p for t in parents for p in t])
    if case["kind"] != "commit":
        st["kv_lens"] = i32(ctx)
        st.update(_pages(case, g, nb))
        dt = torch.bfloat16 if case["cache"] == "bf16" else torch.float16
        st["queries"] = torch.empty((starts[-1], case["hq"], case["d"]), device=DEV, dtype=dt).normal_(
            0, 1.5, generator=g)
        return st
    layers = case["layers"]
    st["kv_before"] = i32([ctx] * layers)
    st["kv_lens"] = st["kv_before"].clone()
    dt = torch.bfloat16 if case["cache"] == "bf16" else torch.float16
    shape = (layers, nb, page, case["hkv"], case["d"])
    st["k"] = torch.empty(shape, device=DEV, dtype=dt).normal_(0, 1, generator=g)
    st["v"] = torch.empty(shape, device=DEV, dtype=dt).normal_(0, 1, generator=g)
    tokens, targets = [], []
    for p in parents:  # most nodes have a child that the target model agrees with
        tok = [rs.randrange(128000) for _ in p]
        tgt = [rs.randrange(128000) for _ in p]
        for i in range(1, len(p)):
            if rs.random() < 0.5:
                tgt[p[i]] = tok[i]
        tokens += tok
        targets += tgt
    st["tokens"] = torch.tensor(tokens, dtype=torch.int64, device=DEV)
    st["targets"] = torch.tensor(targets, dtype=torch.int64, device=DEV)
    return st


# ---------------------------------------------------------------- the plain form


def _plain_cache(st, name):
    """float32 [S, Hkv, L, D]: keys or values of every sequence's tokens, zeros where there is no page."""
    case = st["case"]
    page, hkv, d, kind = case["page"], case["hkv"], case["d"], case["cache"]
    bt = st["tables"].long()
    s, wide = bt.shape
    at = bt.clamp(min=0)
    if kind in ("f16", "bf16"):
        x = st[name][at].float()
    elif kind == "fp8":
        x = _e4m3(st[name][at]) * st[name + "_scale"][at][:, :, None, None, None]
    else:
        bits = int(kind[1])
        per = 32 // bits
        words = st[name][at]
        sh = [bits * k for k in range(per)] if name == "k" else _v_shifts(bits)
        code = (words[..., None] >> torch.tensor(sh, dtype=torch.int32, device=DEV)) & (2**bits - 1)
        code = code.flatten(-2).float()  # keys [S, wide, Hkv, page, D], values [S, wide, Hkv, page / tile, D, tile]
        if name == "v":
            code = code.transpose(-1, -2).reshape(s, wide, hkv, page, d)
        scale, bias = (st[name + e][at].float().transpose(-1, -2).repeat_interleave(case["group"], -1)
                       for e in ("_scales", "_biases"))
        x = (code * scale + bias).transpose(2, 3)
    x = torch.where((bt >= 0)[:, :, None, None, None], x, torch.zeros((), device=DEV))
    return x.reshape(s, wide * page, hkv, d)[:, :st["longest"]].transpose(1, 2).contiguous()


def _ancestors(parents, rows, n):
    """bool [S, n, n]: whether node j is node i or an ancestor of it; `rows` [S, n] places nodes in `parents`, -1: none."""
    s = rows.shape[0]
    par = torch.where(rows >= 0, parents[rows.clamp(min=0)].long(), torch.full((), -1, device=DEV))
    a = torch.eye(n, device=DEV).expand(s, n, n).clone()
    a = a + (par[:, :, None] == torch.arange(n, device=DEV)).float()
    for _ in range(max(1, (n - 1).bit_length())):  # paths twice as long each time
        a = ((a @ a.contiguous()) > 0).float()
    return a > 0


def _rows(st):
    """[S, n] query row of (sequence, token), -1: none."""
    i = torch.arange(st["most_q"], device=DEV)
    lo, hi = st["qsl"][:-1, None].long(), st["qsl"][1:, None].long()
    return torch.where(lo + i < hi, lo + i, torch.full((), -1, device=DEV))


def _plain_attention(st):
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    k, v = _plain_cache(st, "k"), _plain_cache(st, "v")
    rows = _rows(st)
    s, n = rows.shape
    lens = st["kv_lens"].long()[:, None]
    count = (st["qsl"][1:] - st["qsl"][:-1]).long()[:, None]
    before = lens - count  # tokens before the queries'
    i = torch.arange(n, device=DEV)
    key = torch.arange(st["longest"], device=DEV)
    if case["kind"] == "tree":
        anc = _ancestors(st["parents"], rows, n)
        depth = anc.sum(-1) - 1
        node = key[None] - before  # [S, L]
        inside = node.clamp(0, n - 1)[:, None].expand(s, n, -1)
        in_tree = (node >= 0)[:, None]
        seen = torch.where(in_tree, anc.gather(2, inside), torch.ones((), dtype=torch.bool, device=DEV))
        at = torch.where(in_tree, before[:, :, None] + depth.gather(1, node.clamp(0, n - 1))[:, None], key[None, None])
        place = before + depth
    else:
        at = key[None, None]
        place = before + i
        seen = at <= place[:, :, None]
    seen = seen & (key[None, None] < lens[:, :, None])
    if case["window"] > 0:
        seen = seen & ((at > place[:, :, None] - case["window"]) | (at < case["sinks"]))
    x = st["queries"][rows.clamp(min=0)].float()  # [S, n, Hq, D]
    x = x.reshape(s, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(s, hkv, -1, d)
    score = (x @ k.transpose(2, 3).contiguous()) / math.sqrt(d)
    score = score.reshape(s, hkv, n, hq // hkv, -1)
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    out = score.reshape(s, hkv, -1, st["longest"]) @ v
    out = out.reshape(s, hkv, n, hq // hkv, d) / score.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3, 4).reshape(s * n, hq, d)
    back = torch.zeros((st["total"] + 1, hq, d), device=DEV)
    back[torch.where(rows >= 0, rows, torch.full((), st["total"], device=DEV)).reshape(-1)] = out
    return back[:-1].to(st["queries"].dtype)


def _plain_commit(st):
    case = st["case"]
    page, nb, layers = case["page"], st["k"].shape[1], case["layers"]
    rows = _rows(st)
    s, n = rows.shape
    anc = _ancestors(st["parents"], rows, n)
    some = rows >= 0
    at = rows.clamp(min=0)
    par = torch.where(some, st["parents"][at].long(), torch.full((), -1, device=DEV))
    i = torch.arange(n, device=DEV)
    tok, tgt = st["tokens"][at], st["targets"][at]
    agrees = some & (par >= 0) & (tok == tgt.gather(1, par.clamp(min=0)))
    # of several children that agree the first counts
    twin = (par[:, :, None] == par[:, None]) & (i[None, :] < i[:, None]) & agrees[:, None]
    fine = (agrees & ~twin.any(-1)) | (some & (i == 0))
    taken = some & ~(anc & ~fine[:, None]).any(-1)
    count = taken.sum(-1)
    path = torch.full((s, n + 1), -1, dtype=torch.long, device=DEV)
    path.scatter_(1, torch.where(taken, taken.cumsum(-1) - 1, n), i.expand(s, n))
    path = path[:, :n]
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    following = tgt.gather(1, last.clamp(min=0))[:, 0]
    # row j of a tree's place in the cache is afterwards that of its path's node j
    source = torch.where(path >= 0, path, i)
    st["kv_lens"].copy_(st["kv_before"])
    before = st["kv_lens"][0].long() - (st["qsl"][1:] - st["qsl"][:-1]).long()

    def slot(j):
        p = before[:, None] + j
        return st["tables"].long().gather(1, (p // page).clamp(max=st["tables"].shape[1] - 1)) * page + p % page

    src, dst = slot(source)[some], slot(i.expand(s, n))[some]
    for x in (st["k"], st["v"]):
        y = x.reshape(layers, nb * page, -1)
        y[:, dst] = y[:, src]
    st["kv_lens"].copy_((before + count).expand(layers, s))
    return dict(path=path[some].to(torch.int32), accepted=count.to(torch.int32), next=following,
                kv_lens=st["kv_lens"], k=st["k"], v=st["v"])


# ---------------------------------------------------------------- the framework's calls


def _own_cache(st):
    case = st["case"]
    if case["cache"] == "fp8":
        return dict(k_scale=st["k_scale"], v_scale=st["v_scale"])
    if case["cache"] in ("q4", "q8"):
        return dict(k_scales=st["k_scales"], k_biases=st["k_biases"], v_scales=st["v_scales"],
                    v_biases=st["v_biases"], bits=int(case["cache"][1]), group_size=case["group"])
    return {}


def _own_run(st):
    case = st["case"]
    if case["kind"] == "commit":
        from easymlx_amd import PageCache, PageCacheView, tree_accept

        if "pages" not in st:  # the program's cache
            st["pages"] = PageCache([
                PageCacheView(key_cache=st["k"][i], value_cache=st["v"][i], block_tables=st["tables"],
                              kv_lens=st["kv_lens"][i], block_size=case["page"], num_kv_heads=case["hkv"],
                              head_dim=case["d"]) for i in range(case["layers"])])
        st["kv_lens"].copy_(st["kv_before"])
        took = tree_accept(st["tokens"], st["targets"], st["parents"], st["qsl"])
        st["pages"].commit_tree(took.path, took.accepted, st["qsl"])
        return dict(path=took.path, accepted=took.accepted, next=took.next_tokens, kv_lens=st["kv_lens"], k=st["k"],
                    v=st["v"])
    from easymlx_amd import paged_attention, tree_attention

    cache = _own_cache(st)
    window = dict(sliding_window=case["window"], sink_tokens=case["sinks"]) if case["window"] else {}
    if case["kind"] == "tree":
        return tree_attention(st["queries"], st["k"], st["v"], st["tables"], st["kv_lens"], st["qsl"], st["parents"],
                              **window, **cache)
    return paged_attention(st["queries"], st["k"], st["v"], st["tables"], st["kv_lens"], st["qsl"],
                           single_token_decode=st["most_q"] == 1, **window, **cache)


def run(state):
    if own:
        return _own_run(state)
    return _plain_commit(state) if state["case"]["kind"] == "commit" else _plain_attention(state)


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_rows(st, name, i, count):
    """float64 [count, Hkv, D] of sequence i, element by element from the cache's description."""
    case = st["case"]
    page, hkv, d, kind = case["page"], case["hkv"], case["d"], case["cache"]
    t = torch.arange(count, device=DEV)
    b, o = st["tables"][i].long()[t // page], t % page
    if kind in ("f16", "bf16"):
        return st[name][b, o].double()
    if kind == "fp8":
        table = np.zeros(256)
        for c in range(256):
            e, m = (c >> 3) & 15, c & 7
            table[c] = (-1.0 if c & 128 else 1.0) * (m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        value = torch.from_numpy(table).to(DEV)[st[name][b, o].long()]
        return value * st[name + "_scale"].double()[b][:, None, None]
    bits = int(kind[1])
    per, dim, head = 32 // bits, torch.arange(d, device=DEV), torch.arange(hkv, device=DEV)
    bb, oo, hh, dd = b[:, None, None], o[:, None, None], head[None, :, None], dim[None, None]
    if name == "k":
        word = st["k"][bb, hh, oo, dd // per]
        shift = (dd % per) * bits
    else:
        tile = min(page, 256 // bits)
        word = st["v"][bb, hh, oo // tile, dd, (oo % tile) // per]
        k = oo % per
        shift = 8 * k if bits == 8 else 4 * (k // 2 + 4 * (k % 2))
    code = torch.bitwise_and(word.long() >> shift, 2**bits - 1).double()
    grp = dd // case["group"]
    return code * st[name + "_scales"][bb, hh, grp, oo].double() + st[name + "_biases"][bb, hh, grp, oo].double()


def exact(case, seed):
    st = prepare(case, seed)
    q, ctx = _lens(case)
    if case["kind"] == "commit":
        return _exact_commit(st, q, ctx)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros((st["total"], hq, d), dtype=torch.float64, device=DEV)
    parents = st["parents"].tolist() if case["kind"] == "tree" else None
    at = 0
    for i, (n, c) in enumerate(zip(q, ctx)):
        see = np.zeros((n, c), dtype=bool)
        place = np.arange(c)
        if parents is not None:
            for t in range(n):
                p = parents[at + t]
                if p >= 0:
                    see[t] = see[p]
                    place[c - n + t] = place[c - n + p] + 1
                else:
                    see[t, :c - n] = True
                    place[c - n + t] = c - n
                see[t, c - n + t] = True
        else:
            for t in range(n):
                see[t, :c - n + t + 1] = True
        if case["window"] > 0:
            near = place[None] > place[c - n:, None] - case["window"]
            see &= near | (place[None] < case["sinks"])
        see = torch.from_numpy(see).to(DEV)
        k, v = _exact_rows(st, "k", i, c), _exact_rows(st, "v", i, c)
        for h in range(hkv):
            for part in range(0, n, 512):
                m = min(n, part + 512)
                x = st["queries"][at + part:at + m, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
                z = torch.matmul(x.reshape(-1, d), k[:, h].t().contiguous()) / d**0.5
                z = z.reshape(m - part, -1, c).masked_fill(~see[part:m, None], -math.inf)
                w = torch.softmax(z, -1)
                y = torch.matmul(w.reshape(-1, c), v[:, h].contiguous())
                out[at + part:at + m, h * (hq // hkv):(h + 1) * (hq // hkv)] = y.reshape(m - part, -1, d)
        at += n
    return out


def _exact_commit(st, q, ctx):
    case = st["case"]
    page = case["page"]
    tables, parents = st["tables"].tolist(), st["parents"].tolist()
    tokens, targets = st["tokens"].tolist(), st["targets"].tolist()
    path, accepted, following, moves = [], [], [], []
    at = 0
    for i, (n, c) in enumerate(zip(q, ctx)):
        took = [0]
        while True:
            hit = [j for j in range(n) if parents[at + j] == took[-1] and tokens[at + j] == targets[at + took[-1]]]
            if not hit:
                break
            took.append(hit[0])
        path += took + [-1] * (n - len(took))
        accepted.append(len(took))
        following.append(targets[at + took[-1]])
        slot = lambda p: tables[i][p // page] * page + p % page  # noqa: E731
        moves += [(slot(c - n + j), slot(c - n + k)) for k, j in enumerate(took)]
        at += n
    src = torch.tensor([m[0] for m in moves], device=DEV)
    dst = torch.tensor([m[1] for m in moves], device=DEV)
    new = {}
    for name in ("k", "v"):
        x = st[name].flatten(1, 2).clone()
        x[:, dst] = x[:, src]
        new[name] = x.reshape(st[name].shape)
    lens = torch.tensor([c - n + a for n, c, a in zip(q, ctx, accepted)], dtype=torch.int32, device=DEV)
    return dict(path=torch.tensor(path, dtype=torch.int32), accepted=torch.tensor(accepted, dtype=torch.int32),
                next=torch.tensor(following), kv_lens=lens.expand(case["layers"], -1).contiguous(), **new)
