"""Performance cases of the operators around drafted token trees and bounded
caches on paged keys and values.

``listed()`` gives the named cases, ``draw(rng)`` one more of the same ranges.
A case is a dict of plain values; ``kind`` names the operator:

* ``meta``     ``dvattn_tree_metadata``: positions, rotary tables and visible
  lengths of the drafted nodes of every sequence, once per step;
* ``tree``     ``dvattn_tree_paged_sdpa``: attention of the drafted nodes over
  the committed cache and each node's ancestors;
* ``mass``     ``dvattn_paged_key_mass``: the attention weight every cached key
  receives, added to what it has collected;
* ``select``   ``dvattn_kv_select``: the cache rows worth keeping;
* ``compact``  ``dvattn_paged_kv_compact``: kept rows (of an eviction, or of a
  tree's accepted path) moved together.

``run`` computes a case with the operators where ``own`` is true and from
elementary torch operations in 32 bits where it is false; ``exact`` computes it
in 64 bits.  All heads are 128 wide with 16 query heads per KV head.  The
rotated query is part of the operators' definition: float32 products and their
sum, each rounded, and the result rounded to the storage type; an angle is the
float32 product of a position and an inverse frequency.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

E = 128
GQA = 16
SCALE = E ** -0.5
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# The cases.
def listed():
    return [
        # one conversation drafts eight tokens: the smallest call, where latency counts
        dict(name="meta_single", kind="meta", W=1, F=1, S=8, R=128, lo=1000, hi=1000, layout=1),
        # sixteen workers over a shared prompt and each other's segments
        dict(name="meta_workers", kind="meta", W=16, F=17, S=32, R=128, lo=200, hi=4096, layout=2),
        # verification of one conversation's small tree
        dict(name="tree_single_bf16", kind="tree", dtype="bf16", W=1, Hkv=8, F=1, S=8, lo=1000, hi=1000, R=128, bs=16,
             layout=3),
        # a batch of ragged trees, padded to the longest, over a prompt and a segment of its own
        dict(name="tree_batch_fp16", kind="tree", dtype="fp16", W=8, Hkv=4, F=2, S=26, lo=512, hi=4096, R=64, bs=24,
             layout=4),
        # wide trees over long caches: the largest amount of arithmetic
        dict(name="tree_long_bf16", kind="tree", dtype="bf16", W=16, Hkv=8, F=1, S=64, lo=8192, hi=8192, R=128, bs=16,
             layout=5),
        # one conversation's decode step keeps account of its keys
        dict(name="mass_single_bf16", kind="mass", dtype="bf16", W=1, Hkv=8, F=1, S=1, lo=2001, hi=2001, R=128, bs=16,
             layout=6),
        # batched decode, ragged lengths
        dict(name="mass_batch_bf16", kind="mass", dtype="bf16", W=32, Hkv=8, F=1, S=1, lo=1024, hi=8192, R=128, bs=16,
             layout=7),
        # the last tokens of a prompt vote on the whole prompt
        dict(name="mass_window_fp16", kind="mass", dtype="fp16", W=4, Hkv=4, F=2, S=32, lo=8000, hi=8208, R=64, bs=24,
             layout=8),
        # a cache of a thousand tokens cut to half
        dict(name="select_single", kind="select", W=1, Hkv=8, lo=1000, hi=1000, budget=512, first=4, last=64,
             layout=9),
        # long prompts cut to a bounded cache
        dict(name="select_long", kind="select", W=16, Hkv=8, lo=30000, hi=32768, budget=4096, first=4, last=256,
             layout=10),
        # accepted paths of a batch of trees
        dict(name="compact_path_fp16", kind="compact", dtype="fp16", W=32, Hkv=8, lo=64, hi=64, keep=6, shared=True,
             bs=16, layout=11),
        # caches of a batch cut to half, every KV head its own rows
        dict(name="compact_evict_bf16", kind="compact", dtype="bf16", W=16, Hkv=8, lo=8000, hi=8192, keep=4096,
             shared=False, bs=16, layout=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["meta", "tree", "tree", "mass", "mass", "select", "compact"])
        c = dict(kind=kind, W=_log_int(rng, 1, 32), layout=rng.randrange(1 << 30))
        if kind not in ("meta", "select"):
            c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if kind == "meta":
            hi = _log_int(rng, 64, 16384)
            c.update(F=_log_int(rng, 1, 20), S=_log_int(rng, 1, 256), R=rng.choice([32, 64, 128]), hi=hi,
                     lo=max(1, hi // 4))
        elif kind == "tree":
            hi = _log_int(rng, 16, 16384)
            c.update(Hkv=rng.choice([1, 2, 4, 8]), F=rng.choice([1, 1, 2, 3]), S=_log_int(rng, 1, 128), hi=hi,
                     lo=max(1, hi // 4), R=rng.choice([32, 64, 128]), bs=rng.choice([16, 16, 24, 32, 64]))
        elif kind == "mass":
            hi = _log_int(rng, 16, 32768)
            c.update(Hkv=rng.choice([1, 2, 4, 8]), F=rng.choice([1, 1, 2, 3]), S=rng.choice([1, 1, 2, 5, 16, 33]),
                     hi=hi, lo=max(1, hi // 4), R=rng.choice([32, 64, 128]), bs=rng.choice([16, 16, 24, 32, 64]))
            c["lo"] = max(c["lo"], c["S"])
            c["hi"] = max(c["hi"], c["lo"])
        elif kind == "select":
            hi = _log_int(rng, 16, 65536)
            budget = _log_int(rng, 8, max(9, hi // 2))
            c.update(Hkv=rng.choice([1, 2, 4, 8]), hi=hi, lo=max(1, hi // 4), budget=budget,
                     first=rng.randint(0, budget // 4), last=rng.randint(0, budget // 2))
        else:
            hi = _log_int(rng, 8, 16384)
            c.update(Hkv=rng.choice([1, 2, 4, 8]), hi=hi, lo=max(1, hi // 2), keep=_log_int(rng, 1, max(1, hi // 2)),
                     shared=rng.random() < 0.3, bs=rng.choice([16, 16, 24, 32, 64]))
        if _cost(c) <= limit and _scores(c) <= 4e9:
            return c


def _cost(case):
    w = work(case)
    rate = 1e14 if case.get("dtype") == "fp32" else 1e15
    return w["bytes"] / 6e12 + w["flops"] / rate


def _scores(case):
    """Scores that the plain form of an attention case holds at once."""
    if case["kind"] not in ("tree", "mass"):
        return 0
    return case["F"] * case["W"] * case["Hkv"] * GQA * case["S"] * int(_layout(case)["fl"].sum())


# ---------------------------------------------------------------------------
# What a case's numbers fix: lengths, trees and kept rows (the same for every seed).
def _tree(rng, S, n):
    """Parents of a drafted tree of n nodes, breadth first (-1: a child of the
    committed tokens), padded with absent nodes (-2) to S."""
    parents = np.full(S, -2, dtype=np.int64)
    parents[:n] = np.sort(np.minimum(rng.integers(-1, np.maximum(1, np.arange(n) // 2 + 1), size=n), np.arange(n) - 1))
    return parents


def _layout(case):
    rng = np.random.default_rng(case["layout"])
    kind, W = case["kind"], case["W"]
    n = rng.integers(case["lo"], case["hi"], size=W, endpoint=True).astype(np.int64)
    out = dict(n=n)
    if kind in ("meta", "tree"):
        S = case["S"]
        size = rng.integers(max(1, S // 2), S, size=W, endpoint=True)
        size[0] = S
        out["parents"] = np.stack([_tree(rng, S, int(s)) for s in size])
        out["size"] = size
    if kind in ("tree", "mass"):
        F, S = case["F"], case["S"]
        # the committed tokens over the views: a part of them in every view but the
        # last, which is each sequence's own; view lengths are those of the longest
        cuts = np.sort(rng.integers(0, n[:, None], size=(W, F - 1), endpoint=True), axis=1)
        lens = np.diff(np.concatenate([np.zeros((W, 1), np.int64), cuts, n[:, None]], axis=1), axis=1)
        extra = S if kind == "tree" else 0
        fl = lens.max(axis=0)
        fl[-1] += extra
        out.update(lens=lens, fl=fl, off=np.concatenate([[0], np.cumsum(fl)[:-1]]))
    if kind == "meta":
        # view F - 1 - (w mod F) is sequence w's own; the others come before it
        F = case["F"]
        own_view = F - 1 - np.arange(W) % F
        out["order"] = np.stack([[f for f in range(F) if f != v] + [v] for v in own_view])
        out["fl"] = rng.integers(case["lo"], case["hi"], size=F, endpoint=True) + case["S"]
    if kind == "compact":
        heads = 1 if case["shared"] else case["Hkv"]
        keep = np.full((W, heads, case["keep"]), -1, dtype=np.int64)
        for w in range(W):
            k = min(case["keep"], int(n[w]))
            for h in range(heads):
                keep[w, h, :k] = np.sort(rng.choice(int(n[w]), size=k, replace=False))
        out["rows"] = keep
    return out


def _visible(case, lay):
    """Keys each token of a mass case sees, summed over tokens ``[W]``: the S
    tokens are the last ones of the sequence's own view."""
    S = case["S"]
    last = lay["lens"][:, -1:]
    back = S - 1 - np.arange(S)[None, :]
    return (lay["n"][:, None] - last).sum(axis=1) * S + np.maximum(last - back, 0).sum(axis=1)


def work(case):
    """Bytes and operations of one pass: every visible key (and value) of a
    sequence once, queries, outputs and tables once; 2 * E operations per
    product of a query head and a visible key (or value)."""
    kind, W = case["kind"], case["W"]
    lay = _layout(case)
    if kind == "select":
        heads = W * case["Hkv"]
        return dict(bytes=int(lay["n"].sum() * case["Hkv"] * 4 + heads * case["budget"] * 4 + 8 * W),
                    flops=int(lay["n"].sum() * case["Hkv"]))
    S, R = case.get("S"), case.get("R")
    if kind == "meta":
        nodes = case["F"] * W * S
        return dict(bytes=int(nodes * (4 + 8 * R) + 4 * W * (case["F"] + S + 2)), flops=int(nodes * R))
    es, Hkv = ESIZE[case["dtype"]], case["Hkv"]
    row = Hkv * E * es
    if kind == "compact":
        moved = int((lay["rows"] > np.arange(case["keep"])).sum()) * (Hkv if case["shared"] else 1)
        rows = lay["rows"].size * 4
        mass = 0 if case["shared"] else int(lay["n"].sum()) * Hkv * 4 + moved * 4
        return dict(bytes=int(moved * 4 * E * es + rows + mass), flops=moved)
    head = GQA * Hkv * E
    tables = W * S * 4 + int(((lay["n"] + case["bs"] - 1) // case["bs"]).sum()) * 4
    rope = case["F"] * W * S * (8 * R + 4)
    if kind == "tree":
        depth = np.stack([_closure(p).sum(axis=1) for p in lay["parents"]])
        seen = int((lay["n"] * lay["size"]).sum() + depth.sum())
        return dict(bytes=int((lay["n"].sum() + lay["size"].sum()) * 2 * row + 2 * W * S * head * es + rope + tables),
                    flops=int(seen * GQA * Hkv * 4 * E))
    return dict(bytes=int(lay["n"].sum() * (row + 8 * Hkv) + W * S * head * es + rope + tables),
                flops=int(_visible(case, lay).sum() * GQA * Hkv * 2 * E))


def _closure(parents):
    """``[S, S]``: node j is an ancestor of node s, or s itself (one sequence)."""
    S = len(parents)
    see = np.zeros((S, S), dtype=bool)
    for s in range(S):
        if parents[s] >= 0:
            see[s] = see[parents[s]]
        see[s, s] = parents[s] >= -1
    return see


# ---------------------------------------------------------------------------
# Inputs.
def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _rand(gen, shape, dtype, scale=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if scale != 1.0:
        t.mul_(scale)
    return t.to(dtype)


def _inv_freq(R):
    return torch.from_numpy((1e4 ** (-np.arange(0, R, 2, dtype=np.float64) / R)).astype(np.float32)).cuda()


def _cache(case, gen, rng, rows, dt):
    """Block tables of W sequences of ``rows`` rows over scattered pages, and the caches."""
    W, Hkv, bs = case["W"], case["Hkv"], case["bs"]
    per = max(1, (rows + bs - 1) // bs)
    bt = rng.permutation(W * per).reshape(W, per)
    return dict(block_tables=_i32(bt), k_cache=_rand(gen, (W * per, bs, Hkv, E), dt),
                v_cache=_rand(gen, (W * per, bs, Hkv, E), dt))


def _cos_sin(positions, R):
    ang = torch.from_numpy(positions.astype(np.float32)).cuda()[..., None] * _inv_freq(R)
    ang = torch.cat([ang, ang], dim=-1)
    return torch.cos(ang), torch.sin(ang)


def _heavy_tailed(gen, shape):
    """Accumulated attention weights: a few heavy keys, many light ones, some that
    were never attended."""
    m = torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda")) * 1e-2
    return m * (torch.rand(shape, generator=gen, device="cuda") > 0.1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, W = case["kind"], case["W"]
    lay = _layout(case)
    n = lay["n"]
    if kind == "select":
        return dict(kind=kind, mass=_heavy_tailed(gen, (W, case["Hkv"], case["hi"])), first_rows=_i32(np.zeros(W)),
                    lengths=_i32(n), budget=case["budget"], keep_first=case["first"], keep_last=case["last"])
    if kind == "meta":
        return dict(kind=kind, lengths=_i32(lay["fl"] + rng.integers(0, 1000, size=len(lay["fl"]))),
                    order=_i32(lay["order"]), parents=_i32(lay["parents"]), inv_freq=_inv_freq(case["R"]))
    dt = DTYPES[case["dtype"]]
    if kind == "compact":
        st = dict(kind=kind, rows=_i32(lay["rows"]), **_cache(case, gen, rng, case["hi"] + 1, dt))
        st.update(first_rows=_i32(rng.integers(0, 2, size=W)), lengths=_i32(n), mass=None)
        if not case["shared"]:
            st["mass"] = _heavy_tailed(gen, (W, case["Hkv"], case["hi"] + 1))
        return st
    F, S, R = case["F"], case["S"], case["R"]
    lens, fl = lay["lens"], lay["fl"]
    st = dict(kind=kind, lengths=_i32(fl), queries=_rand(gen, (W, GQA * case["Hkv"], S, E), dt, 2.0),
              **_cache(case, gen, rng, int(fl.sum()), dt))
    # rotary positions: a sequence's views one after the other
    after = np.cumsum(lens[:, ::-1], axis=1)[:, ::-1].T  # [F, W]: committed tokens from view f on
    if kind == "tree":
        depth = np.stack([np.maximum(_closure(p).sum(axis=1) - 1, 0) for p in lay["parents"]])
        loc = np.where(lay["parents"][None] >= -1, (lens.T - 1)[:, :, None], -1)  # an absent node sees nothing
        pos = after[:, :, None] + depth[None]
        st.update(parents=_i32(lay["parents"]), tree_views=_i32(np.full(W, F - 1)),
                  tree_rows=_i32(lay["off"][-1] + lens[:, -1]))
    else:
        back = S - 1 - np.arange(S)
        loc = np.broadcast_to((lens.T - 1)[:, :, None], (F, W, S)).copy()
        loc[-1] -= back[None, :]
        pos = after[:, :, None] - 1 - back
        C = int(fl.sum())
        st.update(mass=_heavy_tailed(gen, (W, case["Hkv"], C)), decay=0.99,
                  out=torch.empty((W, case["Hkv"], C), device="cuda"))
    cos, sin = _cos_sin(pos, R)
    st.update(locations=_i32(loc), cos=cos, sin=sin)
    return st


# ---------------------------------------------------------------------------
# The operators, and their plain form.
def run(state):
    s = state
    kind = s["kind"]
    if own:
        import dvattention_amd as dv

        if kind == "meta":
            return dv.dvattn_tree_metadata(s["lengths"], s["order"], s["parents"], s["inv_freq"])
        if kind == "tree":
            return dv.dvattn_tree_paged_sdpa(s["queries"], s["locations"], s["cos"], s["sin"], s["lengths"],
                                             s["k_cache"], s["v_cache"], s["block_tables"], s["parents"],
                                             s["tree_views"], s["tree_rows"], SCALE)
        if kind == "mass":
            return dv.dvattn_paged_key_mass(s["mass"], s["queries"], s["locations"], s["cos"], s["sin"], s["lengths"],
                                            s["k_cache"], s["block_tables"], SCALE, decay=s["decay"], out=s["out"])
        if kind == "select":
            return dv.dvattn_kv_select(s["mass"], s["first_rows"], s["lengths"], s["budget"], s["keep_first"],
                                       s["keep_last"])
        dv.dvattn_paged_kv_compact(s["rows"], s["first_rows"], s["k_cache"], s["v_cache"], s["block_tables"],
                                   mass=s["mass"], lengths=s["lengths"])
        return [s["k_cache"], s["v_cache"]] + ([] if s["mass"] is None else [s["mass"]])
    return {"meta": _plain_meta, "tree": _plain_tree, "mass": _plain_mass, "select": _plain_select,
            "compact": _plain_compact}[kind](s)


def _see(parents):
    """``[W, S, S]``: node j is an ancestor of node s, or s itself.  The path to
    the root is followed by repeated squaring of the step to the parent."""
    W, S = parents.shape
    p = parents.long()
    index = torch.arange(S, device=p.device)
    step = (p[:, :, None] == index) | torch.eye(S, dtype=torch.bool, device=p.device)
    see = step.float()
    for _ in range(max(1, S - 1).bit_length()):
        see = (see @ see > 0).float()
    # a node is absent if the path to the root meets no committed token
    good = ((p >= -1) & (p < index)).float()
    bad_above = see @ (1.0 - good)[:, :, None] > 0
    return (see > 0) & ~bad_above


def _plain_meta(s):
    fl, order, S = s["lengths"].long(), s["order"].long(), s["parents"].shape[1]
    W, F = order.shape
    see = _see(s["parents"])
    there = see.any(-1)
    depth = see.sum(-1) - 1
    own_view = order[:, -1]
    drafted = (own_view[:, None] == torch.arange(F, device=fl.device)).any(0)
    committed = torch.where(drafted, fl - S, fl).clamp(min=0)
    from_here = committed[order].flip(1).cumsum(1).flip(1)  # [W, F] by place in the order
    base = torch.zeros_like(from_here).scatter(1, order, from_here).T  # [F, W]
    position = base[:, :, None] + depth[None]
    there = there[None].expand(F, W, S)
    locations = torch.where(there, (committed - 1)[:, None, None], -1).to(torch.int32)
    angle = position.float()[..., None] * s["inv_freq"]
    angle = torch.cat([angle, angle], dim=-1).double()
    cos = torch.where(there[..., None], torch.cos(angle), 1.0).float()
    sin = torch.where(there[..., None], torch.sin(angle), 0.0).float()
    start = fl.cumsum(0) - fl
    tree_rows = start[own_view] + committed[own_view]
    return locations, cos, sin, own_view.to(torch.int32), tree_rows.to(torch.int32)


def _rotated(q, cos, sin):
    """Queries ``[W, Hq, S, E]`` rotated for every view, rounded to their type,
    in float32: ``[F, W, Hq, S, E]``."""
    h = cos.shape[-1] // 2
    x = q.float()[None]
    c, n = cos[:, :, None, :, :h], sin[:, :, None, :, :h]
    a, b = x[..., :h], x[..., h:2 * h]
    first, second = a * c - b * n, b * c + a * n
    rest = x[..., 2 * h:].expand(*first.shape[:-1], -1)
    return torch.cat([first, second, rest], dim=-1).to(q.dtype).float()


def _stream(s, cache):
    """The first sum(lengths) rows of every sequence, ``[W, Hkv, n, E]`` float32,
    with each row's view ``[n]`` and its place in it ``[n]``."""
    fl = s["lengths"].long()
    bs = cache.shape[1]
    rows = torch.arange(s["block_tables"].shape[1] * bs, device=cache.device)
    end = fl.cumsum(0)
    view = (rows[:, None] >= end).sum(1)
    last = torch.clamp(view, max=fl.shape[0] - 1)
    place = torch.where(view < fl.shape[0], rows - (end - fl)[last], 1 << 30)
    page = s["block_tables"].long()[:, rows // bs]
    return cache[page, rows % bs].permute(0, 2, 1, 3).float(), last, place


def _weights(s, keys, view, seen):
    """Softmax weights ``[W, Hkv, 16, S, n]`` (float32) of the keys that are seen
    ``[W, S, n]``; zeros where a token sees none."""
    q = _rotated(s["queries"], s["cos"], s["sin"])
    F, W, Hq, S, _ = q.shape
    q = q.reshape(F, W, Hq // GQA, GQA * S, E)
    scores = (q @ keys.transpose(-1, -2)[None])  # [F, W, Hkv, 16*S, n]
    scores = (scores[0] if F == 1 else
              torch.gather(scores, 0, view.expand(1, *scores.shape[1:]))[0]).reshape(W, Hq // GQA, GQA, S, -1)
    scores = (scores * SCALE).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _committed(s, view, place):
    loc = s["locations"].long()[view]  # [n, W, S]
    return (place[:, None, None] <= loc).permute(1, 2, 0)


def _plain_tree(s):
    keys, view, place = _stream(s, s["k_cache"])
    values, _, _ = _stream(s, s["v_cache"])
    seen = _committed(s, view, place)
    W, S = s["parents"].shape
    n = view.shape[0]
    node = torch.arange(n, device=view.device)[None] - s["tree_rows"].long()[:, None]  # [W, n]
    inside = (node >= 0) & (node < S) & (view[None] == s["tree_views"].long()[:, None]) & (place < 1 << 30)[None]
    up = torch.gather(_see(s["parents"]), 2, node.clamp(0, S - 1)[:, None].expand(W, S, n))
    p = _weights(s, keys, view, seen | (up & inside[:, None]))
    W, Hkv, _, S, n = p.shape
    out = (p.reshape(W, Hkv, GQA * S, n) @ values).reshape(W, Hkv * GQA, S, E)
    return out.to(s["queries"].dtype)


def _plain_mass(s):
    keys, view, place = _stream(s, s["k_cache"])
    p = _weights(s, keys, view, _committed(s, view, place)).sum((2, 3))
    out = s["mass"] * s["decay"]
    C = min(out.shape[-1], p.shape[-1])
    out[..., :C] += p[..., :C]
    return out


def _plain_select(s):
    mass, budget = s["mass"], s["budget"]
    W, Hkv, C = mass.shape
    index = torch.arange(C, device=mass.device)
    at = s["first_rows"].long()[:, None] + index  # [W, C]
    n = s["lengths"].long()[:, None].clamp(min=0)
    m = torch.gather(mass, 2, at.clamp(max=C - 1)[:, None].expand(W, Hkv, C))
    inside = ((index < n) & (at < C))[:, None].expand(W, Hkv, C)
    held = ((index < s["keep_first"]) | (index >= n - s["keep_last"]))[:, None] & inside
    rank = torch.where(held, 3, torch.where(inside, torch.where(m.isnan(), 1, 2), 0))
    by_mass = torch.sort(m.nan_to_num(0.0, math.inf, -math.inf), dim=-1, descending=True, stable=True).indices
    by_rank = torch.sort(torch.gather(rank, 2, by_mass), dim=-1, descending=True, stable=True)
    rows = torch.gather(by_mass, 2, by_rank.indices)[..., :budget]
    rows = torch.where(by_rank.values[..., :budget] > 0, rows, C).sort(dim=-1).values
    rows = torch.where(rows < C, rows, -1)
    return torch.nn.functional.pad(rows, (0, budget - rows.shape[-1]), value=-1).to(torch.int32)


def _plain_compact(s):
    bt, bs = s["block_tables"].long(), s["k_cache"].shape[1]
    P, _, Hkv, _ = s["k_cache"].shape
    W, _, N = s["rows"].shape
    i = torch.arange(N, device=bt.device)
    first = s["first_rows"].long()[:, None, None]
    rows = s["rows"].long().expand(W, Hkv, N)
    moved = (rows >= i) & (rows < s["lengths"].long()[:, None, None])
    src, dst = first + torch.where(moved, rows, i), (first + i).expand(W, Hkv, N)
    w, h = torch.arange(W, device=bt.device)[:, None, None], torch.arange(Hkv, device=bt.device)[:, None]
    sp, dp = bt[w, src // bs], bt[w, dst // bs]
    s["k_cache"][dp, dst % bs, h] = s["k_cache"][sp, src % bs, h]
    s["v_cache"][dp, dst % bs, h] = s["v_cache"][sp, src % bs, h]
    if s["mass"] is None:
        return [s["k_cache"], s["v_cache"]]
    mass = s["mass"]
    C = mass.shape[-1]
    kept = torch.where(moved, torch.gather(mass, 2, src), 0.0)
    place = torch.arange(C, device=bt.device) - first[:, 0]  # [W, C]
    gone = (place >= 0) & (place < s["lengths"].long()[:, None])
    mass.masked_fill_(gone[:, None], 0.0)
    old = torch.gather(mass, 2, dst)
    mass.scatter_(2, dst, torch.where((i < s["lengths"].long()[:, None, None]).expand(W, Hkv, N), kept, old))
    return [s["k_cache"], s["v_cache"], mass]


# ---------------------------------------------------------------------------
# The same in 64 bits, one sequence and KV head after the other.
def _turn(x, cos, sin):
    """Rotated queries ``[T, 16, E]`` of tables ``[T, R]``, as the operators define them."""
    h = cos.shape[-1] // 2
    x32 = x.to(torch.float32)
    lo, hi = x32[..., :h], x32[..., h:2 * h]
    c, n = cos[:, None, :h], sin[:, None, :h]
    y = x32.clone()
    y[..., :h] = torch.sub(torch.mul(lo, c), torch.mul(hi, n))
    y[..., h:2 * h] = torch.add(torch.mul(hi, c), torch.mul(lo, n))
    return y.to(x.dtype).to(torch.float64)


def _exact_attention(case, st, lay, weights_only):
    f64 = torch.float64
    W, Hkv, F, S, bs = case["W"], case["Hkv"], case["F"], case["S"], case["bs"]
    fl, off, lens = lay["fl"], lay["off"], lay["lens"]
    bt = st["block_tables"].cpu().numpy().astype(np.int64)
    C = int(fl.sum())
    if weights_only:
        result = st["mass"].to(f64) * st["decay"]
    else:
        result = torch.zeros((W, GQA * Hkv, S, E), dtype=f64, device="cuda")
    for w in range(W):
        # every row that some token sees: (view, stream row, seen by token s)
        rows, views, seen = [], [], []
        for f in range(F):
            k = int(lens[w, f])
            rows.append(off[f] + np.arange(k))
            views.append(np.full(k, f))
            if weights_only and f == F - 1:
                seen.append(np.arange(k)[None, :] <= (k - 1 - (S - 1 - np.arange(S)))[:, None])
            elif weights_only:
                seen.append(np.ones((S, k), dtype=bool))
            else:
                seen.append(np.repeat((lay["parents"][w] >= -1)[:, None], k, axis=1))
        if not weights_only:
            rows.append(off[F - 1] + lens[w, F - 1] + np.arange(S))
            views.append(np.full(S, F - 1))
            seen.append(_closure(lay["parents"][w]))
        rows, views = np.concatenate(rows), np.concatenate(views)
        mask = torch.from_numpy(np.concatenate(seen, axis=1)).cuda()
        at = torch.from_numpy(bt[w, rows // bs] * bs + rows % bs).cuda()
        rows = torch.from_numpy(rows).cuda()
        for j in range(Hkv):
            q = st["queries"][w, GQA * j:GQA * (j + 1)].transpose(0, 1)  # [S, 16, E]
            k = st["k_cache"].flatten(0, 1)[at, j].to(f64)
            scores = torch.empty((S, GQA, len(rows)), dtype=f64, device="cuda")
            for f in range(F):
                mine = torch.from_numpy(np.flatnonzero(views == f)).cuda()
                turned = _turn(q, st["cos"][f, w], st["sin"][f, w])
                scores[:, :, mine] = (turned.reshape(-1, E) @ k[mine].T).reshape(S, GQA, -1) * SCALE
            scores.masked_fill_(~mask[:, None], -math.inf)
            p = torch.nan_to_num(torch.softmax(scores, dim=-1))
            if weights_only:
                result[w, j].index_add_(0, rows, p.sum((0, 1)))
            else:
                v = st["v_cache"].flatten(0, 1)[at, j].to(f64)
                result[w, GQA * j:GQA * (j + 1)] = (p.reshape(-1, len(rows)) @ v).reshape(S, GQA, E).transpose(0, 1)
    assert C <= bt.shape[1] * bs
    return result


def exact(case, seed):
    st = prepare(case, seed)
    kind, W = case["kind"], case["W"]
    lay = _layout(case)
    if kind in ("tree", "mass"):
        return _exact_attention(case, st, lay, kind == "mass")
    if kind == "meta":
        F, S, R = case["F"], case["S"], case["R"]
        fl, inv = st["lengths"].cpu().numpy().astype(np.int64), st["inv_freq"].cpu().numpy()
        order = lay["order"]
        committed = fl.copy()
        for v in set(order[:, -1].tolist()):
            committed[v] = max(fl[v] - S, 0)
        loc = np.empty((F, W, S), dtype=np.int64)
        cos, sin = np.empty((F, W, S, R)), np.empty((F, W, S, R))
        for w in range(W):
            see = _closure(lay["parents"][w])
            there = see.any(axis=1)
            total = 0
            for f in reversed(order[w].tolist()):
                total += committed[f]
                angle = ((total + see.sum(axis=1) - 1).astype(np.float32)[:, None] * inv).astype(np.float64)
                angle = np.concatenate([angle, angle], axis=1)
                loc[f, w] = np.where(there, committed[f] - 1, -1)
                cos[f, w] = np.where(there[:, None], np.cos(angle), 1.0)
                sin[f, w] = np.where(there[:, None], np.sin(angle), 0.0)
        start = np.cumsum(fl) - fl
        last = order[:, -1]
        return (torch.from_numpy(loc).to(torch.int32), torch.from_numpy(cos), torch.from_numpy(sin),
                torch.from_numpy(last).to(torch.int32), torch.from_numpy(start[last] + committed[last]).to(torch.int32))
    if kind == "select":
        m = st["mass"].cpu().numpy()
        out = np.full((W, case["Hkv"], case["budget"]), -1, dtype=np.int32)
        for w in range(W):
            n = int(lay["n"][w])
            a, b = case["first"], max(case["first"], n - case["last"])
            for h in range(case["Hkv"]):
                if n <= case["budget"]:
                    out[w, h, :n] = np.arange(n)
                    continue
                free = case["budget"] - a - (n - b)
                best = a + np.argsort(-m[w, h, a:b].astype(np.float64), kind="stable")[:free]
                out[w, h] = np.sort(np.concatenate([np.arange(a), best, np.arange(b, n)]))
        return torch.from_numpy(out)
    f64 = torch.float64
    k, v = st["k_cache"].to(f64), st["v_cache"].to(f64)
    mass = None if st["mass"] is None else st["mass"].to(f64)
    bt, first, bs = st["block_tables"].cpu().numpy(), st["first_rows"].cpu().numpy(), case["bs"]
    for w in range(W):
        for h in range(case["Hkv"]):
            rows = lay["rows"][w, 0 if case["shared"] else h]
            to = np.flatnonzero(rows >= 0)
            src, dst = first[w] + rows[to], first[w] + to
            sp, sr = torch.from_numpy(bt[w, src // bs]).cuda().long(), torch.from_numpy(src % bs).cuda()
            dp, dr = torch.from_numpy(bt[w, dst // bs]).cuda().long(), torch.from_numpy(dst % bs).cuda()
            k[dp, dr, h], v[dp, dr, h] = k[sp, sr, h].clone(), v[sp, sr, h].clone()
            if mass is not None:
                line = mass[w, h].clone()
                mass[w, h, first[w]:first[w] + int(lay["n"][w])] = 0.0
                mass[w, h, torch.from_numpy(dst).cuda()] = line[torch.from_numpy(src).cuda()]
    return [k, v] + ([] if mass is None else [mass])
