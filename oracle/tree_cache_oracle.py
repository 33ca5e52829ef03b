"""64-bit CPU restatements of the tree and bounded-cache operators
(dvattn_tree_metadata, dvattn_tree_paged_sdpa, dvattn_paged_key_mass,
dvattn_kv_select, dvattn_paged_kv_compact), written key by key from their
definitions.  Test infrastructure only.

The rotated query is part of the definition -- float32 products and their sum,
each rounded, the result rounded to the storage type -- as is the float32
product that makes an angle; everything after that is float64.
"""
from __future__ import annotations

import math

import torch

GQA = 16
F64 = torch.float64


def path(parents, s):
    """Node s and its ancestors, or None for an absent node."""
    nodes, j = [], s
    while True:
        nodes.append(j)
        up = int(parents[j])
        if up == -1:
            return nodes
        if up < -1 or up >= j:
            return None
        j = up


def rotate(q, cos, sin):
    """q [n, E] in its type, cos/sin [R] float32 -> [n, E] float64 (rounded to q's type)."""
    h = cos.shape[-1] // 2
    x = q.float()
    a, b = x[:, :h], x[:, h:2 * h]
    c, s = cos[:h], sin[:h]
    y = x.clone()
    y[:, :h] = (a * c) - (b * s)
    y[:, h:2 * h] = (b * c) + (a * s)
    return y.to(q.dtype).to(F64)


def cache_row(block_tables, w, pos, num_blocks, bs):
    """(page, row) of a stream row, or None."""
    if pos < 0 or pos // bs >= block_tables.shape[1]:
        return None
    page = int(block_tables[w, pos // bs])
    return (page, pos % bs) if 0 <= page < num_blocks else None


def visible(w, s, locations, fl, bt, num_blocks, bs, tree=None):
    """[(view, stream row, page, row)] of the keys token (w, s) sees."""
    keys, off = [], 0
    for f, n in enumerate(fl):
        top = min(int(locations[f, w, s]) + 1, n)
        rows = [off + l for l in range(max(top, 0))]
        if tree is not None:
            nodes, tv, first = tree
            if f == tv:
                extra = [first + j for j in nodes]
                rows += [p for p in sorted(extra) if off <= p < off + n and p - off >= max(top, 0)]
        for p in rows:
            at = cache_row(bt, w, p, num_blocks, bs)
            if at is not None:
                keys.append((f, p) + at)
        off += n
    return keys


def attention_rows(scale, locations, queries, cosines, sines, fragment_lengths, k_cache, block_tables, tree_of=None):
    """Yields (w, hkv, s, keys, p [16, n], spread) for every token and KV head: softmax
    weights of the keys it sees, and the largest sum of |q_e k_e| * |scale|, which the
    error of a float32 score scales with.  Keys empty: p is [16, 0]."""
    W, Hq, S, _ = queries.shape
    P, bs, Hkv, _ = k_cache.shape
    fl = [int(x) for x in fragment_lengths]
    for w in range(W):
        for s in range(S):
            tree = tree_of(w, s) if tree_of else None
            keys = [] if tree == "absent" else visible(w, s, locations, fl, block_tables, P, bs, tree)
            for h in range(Hkv):
                q = queries[w, GQA * h:GQA * (h + 1), s]
                if not keys:
                    yield w, h, s, keys, torch.zeros(GQA, 0, dtype=F64), 0.0
                    continue
                k = k_cache[[x[2] for x in keys], [x[3] for x in keys], h].to(F64)
                views = torch.tensor([x[0] for x in keys])
                x = torch.empty(GQA, len(keys), dtype=F64)
                spread = 0.0
                for f in set(views.tolist()):
                    mine = views == f
                    rq = rotate(q, cosines[f, w, s], sines[f, w, s])
                    x[:, mine] = rq @ k[mine].T * scale
                    spread = max(spread, float((rq.abs() @ k[mine].abs().T).nan_to_num(0.0).max()) * abs(scale))
                yield w, h, s, keys, torch.softmax(x, dim=-1), spread


def tree_sdpa(scale, locations, queries, cosines, sines, fragment_lengths, k_cache, v_cache, block_tables, parents,
              tree_views, tree_rows):
    """(out, sum of weight * |v|, spread), float64 [W,Hq,S,Ev] / [W,Hq,S,1]."""
    W, Hq, S, _ = queries.shape
    out = torch.zeros(W, Hq, S, v_cache.shape[3], dtype=F64)
    size = torch.zeros_like(out)
    spread = torch.zeros(W, Hq, S, 1, dtype=F64)

    def tree_of(w, s):
        nodes = path(parents[w], s)
        return "absent" if nodes is None else (nodes, int(tree_views[w]), int(tree_rows[w]))

    for w, h, s, keys, p, sp in attention_rows(scale, locations, queries, cosines, sines, fragment_lengths, k_cache,
                                               block_tables, tree_of):
        if keys:
            v = v_cache[[x[2] for x in keys], [x[3] for x in keys], h].to(F64)
            out[w, GQA * h:GQA * (h + 1), s] = p @ v
            size[w, GQA * h:GQA * (h + 1), s] = p @ v.abs()
            spread[w, GQA * h:GQA * (h + 1), s] = sp
    return out, size, spread


def key_mass(mass, decay, scale, locations, queries, cosines, sines, fragment_lengths, k_cache, block_tables):
    """(out, largest spread), float64 [W,Hkv,C]."""
    out = mass.to(F64) * decay if decay != 0 else torch.zeros(mass.shape, dtype=F64)
    worst = 0.0
    for w, h, s, keys, p, sp in attention_rows(scale, locations, queries, cosines, sines,
                                               [max(int(x), 0) for x in fragment_lengths], k_cache, block_tables):
        worst = max(worst, sp)
        for i, key in enumerate(keys):
            if key[1] < out.shape[2]:
                out[w, h, key[1]] += p[:, i].sum()
    return out, worst


def select(mass, first_rows, lengths, budget, keep_first, keep_last):
    W, Hkv, C = mass.shape
    rows = torch.full((W, Hkv, budget), -1, dtype=torch.int32)
    for w in range(W):
        first = int(first_rows[w])
        n = max(0, min(int(lengths[w]), C - first)) if first >= 0 else 0
        for h in range(Hkv):
            if n <= budget:
                rows[w, h, :n] = torch.arange(n, dtype=torch.int32)
                continue
            m = mass[w, h, first:first + n].double().tolist()
            middle = range(keep_first, n - keep_last)
            heavy = sorted(middle, key=lambda i: (math.isnan(m[i]), 0.0 if math.isnan(m[i]) else -m[i], i))
            kept = sorted(list(range(keep_first)) + heavy[:budget - keep_first - keep_last] +
                          list(range(n - keep_last, n)))
            rows[w, h] = torch.tensor(kept, dtype=torch.int32)
    return rows


def compact(k_cache, v_cache, block_tables, rows, first_rows, lengths=None, mass=None):
    """New (k, v, mass); every source is read before any row is written."""
    P, bs, Hkv, _ = k_cache.shape
    W, heads, N = rows.shape
    k, v, m = k_cache.clone(), v_cache.clone(), None if mass is None else mass.clone()
    for w in range(W):
        first = int(first_rows[w])
        if first < 0:
            continue
        limit = 1 << 31 if lengths is None else int(lengths[w])
        for h in range(Hkv):
            r = rows[w, h if heads > 1 else 0].tolist()
            for i in range(N):
                if i <= r[i] < limit:
                    src, dst = (cache_row(block_tables, w, first + x, P, bs) for x in (r[i], i))
                    if src is not None and dst is not None:
                        k[dst[0], dst[1], h] = k_cache[src[0], src[1], h]
                        v[dst[0], dst[1], h] = v_cache[src[0], src[1], h]
            if m is not None:
                end = min(limit, m.shape[2] - first)
                for i in range(max(end, 0)):
                    ok = i < N and i <= r[i] < end
                    m[w, h, first + i] = mass[w, h, first + r[i]] if ok else 0.0
    return k, v, m


def metadata(fragment_lengths, order, parents, inv_freq, scaling=1.0, dropped=None, committed=None):
    """(locations, cos, sin, tree_views, tree_rows); cos/sin float64 of the float32 angle."""
    F, (W, S), R = len(fragment_lengths), parents.shape, 2 * inv_freq.numel()
    fl = [int(x) for x in fragment_lengths]
    drafted = {int(order[w, F - 1]) for w in range(W)}
    shared = [max(fl[g] - (S if g in drafted else 0), 0) for g in range(F)]
    loc = torch.full((F, W, S), -1, dtype=torch.int32)
    cos, sin = torch.ones(F, W, S, R, dtype=F64), torch.zeros(F, W, S, R, dtype=F64)
    views, rows = torch.empty(W, dtype=torch.int32), torch.empty(W, dtype=torch.int32)
    for w in range(W):
        c = shared if committed is None else [max(int(x), 0) for x in committed[w]]
        o = [int(x) for x in order[w]]
        own = o[-1]
        ok = 0 <= own < F
        views[w] = own if ok else -1
        rows[w] = sum(fl[:own]) + c[own] if ok else 0
        for f in range(F):
            if f not in o:
                continue
            base = sum(c[g] + (0 if dropped is None else int(dropped[w, g])) for g in o[o.index(f):] if 0 <= g < F)
            for s in range(S):
                nodes = path(parents[w], s)
                if nodes is None:
                    continue
                loc[f, w, s] = c[f] - 1
                ang = (torch.tensor(base + len(nodes) - 1, dtype=torch.float32) * inv_freq).to(F64)
                ang = torch.cat([ang, ang])
                cos[f, w, s], sin[f, w, s] = torch.cos(ang) * scaling, torch.sin(ang) * scaling
    return loc, cos, sin, views, rows
