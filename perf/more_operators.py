"""Performance cases of the operators around paged keys and values held in 8 bits.

``listed()`` gives the named cases, ``draw(rng)`` one more of the same ranges.
A case is a dict of plain values; ``kind`` names the operator:

* ``tables``  ``dvattn_block_tables``: block tables, positions and slots of a
  step's tokens from the sequences' lengths and a stack of free pages;
* ``append``  ``dvattn_paged_kv_append_q8``: new keys (rotated) and values
  rounded to 8 bits in their slots, one scale per page and KV head;
* ``paged``   ``dvattn_paged_sdpa_q8``: S tokens per sequence over an 8-bit cache;
* ``varlen``  ``dvattn_varlen_paged_sdpa_q8``: the same for packed tokens.

``run`` computes a case with the operators where ``own`` is true and from
elementary torch operations in 32 bits where it is false; ``exact`` computes it
in 64 bits.  All heads are 128 wide with 16 query heads per KV head.

What the operators are defined by: a cached element is an E4M3 byte times
2^(b - 127) of its page's and KV head's exponent byte b.  An append takes the
smallest exponent, at least -126, under which the largest finite magnitude
written to the page is at most 448; it never lowers the exponent that the page
has, unless row 0 of the page is written (what the page held is gone then).
Rows held under a smaller exponent are rounded again.  Rotated keys and queries
are float32 products and their sum, each rounded, and the result rounded to the
storage type.
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
        # a decode step of a batch: every sequence one token, a few of them a page
        dict(name="tables_decode", kind="tables", W=64, lo=100, hi=8000, bs=16, chunks=0, chunk=1, done=0, layout=1),
        # a busy server's step: decodes, prompts in chunks, sequences that ended
        dict(name="tables_admit", kind="tables", W=512, lo=0, hi=32000, bs=16, chunks=32, chunk=512, done=24, layout=2),
        # the decode step's keys and values: one row in each sequence's last page
        dict(name="append_decode_bf16", kind="append", dtype="bf16", W=32, Hkv=8, lo=1024, hi=8192, chunks=0, chunk=1,
             R=128, bs=16, layout=3),
        # prompts of 2047 tokens
        dict(name="append_prompt_bf16", kind="append", dtype="bf16", W=4, Hkv=8, lo=2047, hi=2050, chunks=4,
             chunk=2047, R=128, bs=16, layout=4),
        # decodes and prompt chunks that start inside a page, pages of 24 rows
        dict(name="append_mixed_fp16", kind="append", dtype="fp16", W=50, Hkv=4, lo=256, hi=8192, chunks=2, chunk=250,
             R=64, bs=24, layout=5),
        # interactive decode of one conversation: the smallest attention call
        dict(name="paged_single_bf16", kind="paged", dtype="bf16", W=1, Hkv=8, S=1, lo=3001, hi=3001, R=128, bs=16,
             layout=6),
        # batched decode, ragged lengths
        dict(name="paged_batch_bf16", kind="paged", dtype="bf16", W=32, Hkv=8, S=1, lo=1024, hi=8192, R=128, bs=16,
             layout=7),
        # long-context decode
        dict(name="paged_long_fp16", kind="paged", dtype="fp16", W=4, Hkv=8, S=1, lo=131072, hi=131072, R=128, bs=64,
             layout=8),
        # verification of four speculated tokens, float32 queries, a page size that is no power of two
        dict(name="paged_verify_fp32", kind="paged", dtype="fp32", W=24, Hkv=4, S=4, lo=512, hi=4096, R=64, bs=24,
             layout=9),
        # prompt prefill in chunks of 2048 tokens, the largest amount of arithmetic
        dict(name="paged_prefill_bf16", kind="paged", dtype="bf16", W=2, Hkv=8, S=2048, lo=3800, hi=4400, R=128,
             bs=16, layout=10),
        # packed decode, every sequence's cache made of one to three views
        dict(name="varlen_views_fp16", kind="varlen", dtype="fp16", W=48, Hkv=4, F=3, lo=64, hi=16384, chunks=0,
             chunk=1, R=64, bs=16, layout=11),
        # continuous batching: decodes and two prompt chunks in one call
        dict(name="varlen_mixed_bf16", kind="varlen", dtype="bf16", W=50, Hkv=4, F=1, lo=256, hi=8192, chunks=2,
             chunk=250, R=128, bs=16, layout=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["tables", "append", "append", "paged", "paged", "paged", "varlen", "varlen"])
        c = dict(kind=kind, layout=rng.randrange(1 << 30), bs=rng.choice([16, 16, 24, 32, 64]))
        if kind != "tables":
            c.update(dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), Hkv=rng.choice([1, 2, 4, 8]),
                     R=rng.choice([32, 64, 128]))
        if kind == "tables":
            W, hi = _log_int(rng, 1, 1024), _log_int(rng, 16, 65536)
            c.update(W=W, lo=hi // 8, hi=hi, chunks=rng.randint(0, W // 4), chunk=_log_int(rng, 1, 512),
                     done=rng.randint(0, W // 8))
        elif kind == "paged":
            S = rng.choice([1, 1, 2, 4, 8, 16, 33, _log_int(rng, 64, 2048)])
            hi = S + _log_int(rng, 64, 131072 if S == 1 else 16384)
            c.update(W=_log_int(rng, 1, 64), S=S, lo=max(S, hi // 8), hi=hi)
        else:
            W, hi = _log_int(rng, 1, 64), _log_int(rng, 64, 16384)
            c.update(W=W, lo=max(1, hi // 8), hi=hi, chunks=rng.randint(0, min(W, 4)), chunk=_log_int(rng, 1, 1024))
            if kind == "varlen":
                c.update(F=rng.choice([1, 1, 2, 3, 4]))
        if _cost(c) <= limit and _scores(c) <= 7e9:
            return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / (3e14 if case.get("dtype") == "fp32" else 1e15)


def _scores(case):
    """Scores that the plain form of an attention case holds at once."""
    if case["kind"] not in ("paged", "varlen"):
        return 0
    lay = _layout(case)
    return len(lay["fl"]) * case["W"] * case["Hkv"] * GQA * int(lay["new"].max()) * int(lay["fl"].sum())


# ---------------------------------------------------------------------------
# What a case's numbers fix: lengths, new tokens and views (the same for every seed).
def _layout(case):
    """``n`` tokens of each sequence with this step's, ``new`` of them this step's;
    attention: views of ``lens [W, F]`` rows and their common lengths ``fl``."""
    rng = np.random.default_rng(case["layout"])
    kind, W = case["kind"], case["W"]
    if kind == "tables":
        n = rng.integers(case["lo"], case["hi"], size=W, endpoint=True).astype(np.int64)
        new = np.ones(W, dtype=np.int64)
        who = rng.permutation(W)
        new[who[:case["chunks"]]] = rng.integers(1, case["chunk"], size=case["chunks"], endpoint=True)
        new[who[case["chunks"]:case["chunks"] + case["done"]]] = -1
        return dict(n=n, new=new)
    if kind == "varlen" or (kind == "append" and case["lo"] < case["hi"] // 2):
        n = np.exp(rng.uniform(math.log(case["lo"]), math.log(case["hi"]), size=W))
        n = np.clip(np.round(n), case["lo"], case["hi"]).astype(np.int64)
    else:
        n = rng.integers(case["lo"], case["hi"], size=W, endpoint=True).astype(np.int64)
    if kind == "paged":
        return dict(n=n, new=np.full(W, case["S"], dtype=np.int64), lens=n[:, None], fl=np.array([n.max()]))
    new = np.ones(W, dtype=np.int64)
    who = rng.choice(W, size=case["chunks"], replace=False)
    new[who] = np.maximum(1, np.minimum(n[who], case["chunk"] - rng.integers(0, 8, size=len(who))))
    if kind == "append":
        return dict(n=n, new=new)
    F = case["F"]
    lens = np.zeros((W, F), dtype=np.int64)
    views = rng.integers(1, F, size=W, endpoint=True)
    for w in range(W):
        # the last view that a sequence has holds this step's tokens
        cuts = np.sort(rng.integers(0, n[w] - new[w], size=views[w] - 1, endpoint=True))
        lens[w, :views[w]] = np.diff(np.concatenate([[0], cuts, [n[w]]]))
    return dict(n=n, new=new, lens=lens, fl=lens.max(axis=0), views=views)


def work(case):
    """Bytes and operations of one pass: every visible row of a sequence once, in
    8 bits, queries, outputs, scales and tables once; 4 * E operations per query
    head and visible key."""
    kind, W, bs = case["kind"], case["W"], case["bs"]
    lay = _layout(case)
    n, new = lay["n"], np.maximum(lay["new"], 0)
    T = int(new.sum())
    pages = (n + bs - 1) // bs
    if kind == "tables":
        gone = int(pages[lay["new"] < 0].sum())
        got = int(((n + new + bs - 1) // bs - pages).sum())
        return dict(bytes=int(T * 12 + W * 28 + 8 * (gone + got)), flops=int(T + W))
    es, Hkv, R = ESIZE[case["dtype"]], case["Hkv"], case["R"]
    row = Hkv * 2 * E
    if kind == "append":
        # of the pages that are written the exponents are read and written
        touched = int(((n - 1) // bs - (n - new) // bs + 1).sum())
        return dict(bytes=int(T * row * (es + 1) + T * (2 * R * es + 8) + touched * 4 * Hkv),
                    flops=int(T * Hkv * (3 * R + 4 * E)))
    F = lay["lens"].shape[1]
    seen = new * n - new * (new - 1) // 2
    head = GQA * Hkv * E
    rope = F * T * ((R if kind == "paged" else R // 2) * 8 + 4)
    return dict(bytes=int(n.sum() * row + pages.sum() * (2 * Hkv + 4) + 2 * T * head * es + rope),
                flops=int(seen.sum() * GQA * Hkv * 4 * E))


# ---------------------------------------------------------------------------
# Inputs.
def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _rand(gen, shape, dtype, scale=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if scale != 1.0:
        t.mul_(scale)
    return t.to(dtype)


def _cos_sin(positions, R):
    """float32 ``[..., R]`` tables of integer positions, both halves alike."""
    ang = np.asarray(positions, dtype=np.float64)[..., None] * 1e4 ** (-np.arange(0, R, 2, dtype=np.float64) / R)
    ang = np.concatenate([ang, ang], axis=-1)
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(ang).astype(np.float32)).cuda())


def _cache(gen, P, bs, Hkv):
    """A pool of P pages as earlier steps left it: bytes of elements whose size
    differs from page to page and head to head, and their exponents."""
    size = torch.exp(0.7 * torch.randn((P, 1, Hkv, 1), generator=gen, device="cuda"))
    x = torch.randn((P, bs, Hkv, E), generator=gen, device="cuda").mul_(size)
    b = _exponent(x.abs().amax((1, 3)))
    return x.mul_(_power(127 - b)[:, None, :, None]).to(torch.float8_e4m3fn), b.to(torch.uint8)


def _pages(rng, counts, logical=None, width=None):
    """Block tables of sequences with ``counts[w]`` pages, scattered over the
    pool; ``logical[w]``: the logical pages that are backed."""
    total = int(sum(counts))
    perm = rng.permutation(total).astype(np.int32)
    bt = np.zeros((len(counts), width or max(1, int(max(counts)))), dtype=np.int32)
    at = 0
    for w, n in enumerate(counts):
        bt[w, logical[w] if logical is not None else np.arange(n)] = perm[at:at + n]
        at += n
    return bt, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, W, bs = case["kind"], case["W"], case["bs"]
    lay = _layout(case)
    n, new = lay["n"], lay["new"]
    if kind == "tables":
        counts = (n + bs - 1) // bs
        width = int(-(-(case["hi"] + case["chunk"]) // bs))
        bt, held = _pages(rng, counts, width=width)
        spare = int(np.maximum(new, 0).sum()) // bs + W
        P = held + spare
        names = rng.permutation(P)  # pages in use and free ones are spread over the pool
        used = np.arange(width)[None, :] < counts[:, None]
        stack = np.zeros(P, dtype=np.int64)
        stack[:spare] = names[held:]
        return dict(kind=kind, lengths=_i32(n), new_tokens=_i32(new), block_tables=_i32(np.where(used, names[bt], -1)),
                    free_pages=_i32(stack), free_count=_i32([spare]), bs=bs, T=int(np.maximum(new, 0).sum()))
    Hkv, R, dt = case["Hkv"], case["R"], DTYPES[case["dtype"]]
    seq = np.repeat(np.arange(W), new)
    T = len(seq)
    cu = np.concatenate([[0], np.cumsum(new)])
    place = np.arange(T) - cu[seq]
    if kind == "append":
        bt, P = _pages(rng, (n + bs - 1) // bs)
        pos = n[seq] - new[seq] + place
        cos, sin = _cos_sin(pos, R)
        k, ks = _cache(gen, P, bs, Hkv)
        v, vs = _cache(gen, P, bs, Hkv)
        # keys and values as the projection of the packed tokens leaves them, side by side
        kv = _rand(gen, (T, 2, Hkv, E), dt) * torch.exp(0.5 * torch.randn((T, 1, 1, 1), generator=gen,
                                                                          device="cuda")).to(dt)
        slots = torch.from_numpy(bt[seq, pos // bs].astype(np.int64) * bs + pos % bs).cuda()
        return dict(kind=kind, keys=kv[:, 0], values=kv[:, 1], slots=slots, cos=cos.to(dt), sin=sin.to(dt), k_cache=k,
                    v_cache=v, k_scales=ks, v_scales=vs)
    lens, fl = lay["lens"], lay["fl"]
    F = len(fl)
    off = np.concatenate([[0], np.cumsum(fl)[:-1]])
    logical = [np.unique(np.concatenate([np.arange(off[f] // bs, (off[f] + lens[w, f] - 1) // bs + 1)
                                         for f in range(F) if lens[w, f]])) for w in range(W)]
    bt, P = _pages(rng, [len(x) for x in logical], logical, int(-(-fl.sum() // bs)))
    k, ks = _cache(gen, P, bs, Hkv)
    v, vs = _cache(gen, P, bs, Hkv)
    st = dict(kind=kind, k_cache=k, v_cache=v, k_scales=ks, v_scales=vs, block_tables=_i32(bt), lengths=_i32(fl))
    if kind == "paged":
        S = case["S"]
        pos = n[:, None] - S + np.arange(S)[None, :]
        cos, sin = _cos_sin(pos[None], R)
        st.update(queries=_rand(gen, (W, GQA * Hkv, S, E), dt, 1.5), locations=_i32(pos[None]), cos=cos, sin=sin)
        return st
    # the last view of a sequence is causal over its own tokens, those before it are whole
    last = lay["views"][seq] - 1
    loc = np.where(np.arange(F)[:, None] <= last[None, :], lens[seq].T - 1, -1)
    loc[last, np.arange(T)] -= new[seq] - 1 - place
    cos, sin = _cos_sin(rng.integers(0, 65536, size=(F, T)) if F > 1 else loc, R)
    st.update(queries=_rand(gen, (T, GQA * Hkv, E), dt, 1.5), locations=_i32(loc), cos=cos[..., :R // 2].contiguous(),
              sin=sin[..., :R // 2].contiguous(), cu_q=_i32(cu), cu_k=_i32(np.concatenate([[0], np.cumsum(n)])),
              most=int(new.max()))
    return st


# ---------------------------------------------------------------------------
# The operators, and their plain form.
def run(state):
    s = state
    kind = s["kind"]
    if own:
        import dvattention_amd as dv

        if kind == "tables":
            return dv.dvattn_block_tables(s["lengths"], s["new_tokens"], s["block_tables"], s["free_pages"],
                                          s["free_count"], s["bs"], s["T"]) + (s["block_tables"], s["free_pages"])
        if kind == "append":
            return dv.dvattn_paged_kv_append_q8(s["keys"], s["values"], s["slots"], s["cos"], s["sin"], s["k_cache"],
                                                s["v_cache"], s["k_scales"], s["v_scales"])
        if kind == "paged":
            return dv.dvattn_paged_sdpa_q8(s["queries"], s["locations"], s["cos"], s["sin"], s["lengths"],
                                           s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"],
                                           s["block_tables"], SCALE)
        return dv.dvattn_varlen_paged_sdpa_q8(s["queries"], s["locations"], s["cos"], s["sin"], s["lengths"],
                                              s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"],
                                              s["block_tables"], s["cu_q"], s["cu_k"], SCALE)
    return {"tables": _plain_tables, "append": _plain_append, "paged": _plain_paged, "varlen": _plain_varlen}[kind](s)


def _plain_tables(s):
    bs, T = s["bs"], s["T"]
    bt, stack = s["block_tables"], s["free_pages"]
    W, width = bt.shape
    P = stack.shape[0]
    before, new = s["lengths"].long().clamp(0, width * bs), s["new_tokens"].long()
    page = torch.arange(width, device=bt.device)
    done = new < 0
    held = (before + bs - 1) // bs
    # the pages of sequences that ended go on the stack, in order
    gone = torch.where(done, held, 0)
    count = s["free_count"].long().clamp(0, P)
    at = count + (gone.cumsum(0) - gone)[:, None] + page
    back = (page < gone[:, None]) & (at < P)
    at, back = at.reshape(-1), back.reshape(-1)
    # (entries that go nowhere are written to a place behind the stack's end)
    wide = torch.cat([stack, stack.new_zeros(1)])
    wide[torch.where(back, at, P)] = bt.reshape(-1)
    stack.copy_(wide[:P])
    have = (count + gone.sum()).clamp(max=P)
    before, held, new = torch.where(done, 0, before), torch.where(done, 0, held), new.clamp(min=0)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    after = before + new
    fits = (after <= width * bs) & (cu[1:] <= T)
    need = torch.where(fits, (after + bs - 1) // bs - held, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= have))
    got = torch.where(granted, need, 0)
    j = page - held[:, None]
    take = (j >= 0) & (j < got[:, None])
    top = (have - 1 - (upto - need)[:, None] - j).clamp(0, P - 1)
    bt.copy_(torch.where(take, stack[top], bt))
    starts = torch.where(granted & ~done, before, -1)
    t = torch.arange(T, device=bt.device)
    w = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    inside = w < W
    w = w.clamp(max=W - 1)
    inside = inside & (starts[w] >= 0)
    pos = torch.where(inside, starts[w] + t - cu[w], 0)
    p = bt[w, pos // bs].long()
    slots = torch.where(inside & (p >= 0) & (p < P), p * bs + pos % bs, -1)
    lengths = torch.where(granted, after, before)
    return (cu.to(torch.int32), starts.to(torch.int32), torch.where(inside, pos, -1).to(torch.int32), slots,
            lengths.to(torch.int32), (have - got.sum()).to(torch.int32).reshape(1), bt, stack)


def _exponent(amax):
    """Biased exponents ``b`` (int32): the smallest, at least 1, with amax <= 448 * 2^(b - 127)."""
    bits = amax.contiguous().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).to(torch.int32)).clamp(min=1)


def _power(e):
    """2^e in float32, exactly (whole e from -126 to 127)."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _values(byte):
    """What E4M3 bytes stand for, in float32."""
    return byte.view(torch.float8_e4m3fn).float()


def _turn_keys(x, cos, sin):
    """Keys ``[T, Hkv, E]`` rotated as PyTorch evaluates it in their type."""
    R = cos.shape[-1]
    a, rest = x[..., :R], x[..., R:]
    half = torch.cat([-a[..., R // 2:], a[..., :R // 2]], dim=-1)
    return torch.cat([a * cos[:, None] + half * sin[:, None], rest], dim=-1)


def _plain_append(s):
    slots, (P, bs, Hkv, _) = s["slots"], s["k_cache"].shape
    page, row = slots // bs, slots % bs
    ids, which = torch.unique(page, return_inverse=True)
    n = ids.shape[0]
    written = torch.zeros((n, bs), dtype=torch.bool, device=slots.device)
    written[which, row] = True
    fresh = written[:, 0]
    out = []
    for x, cache, scales in ((_turn_keys(s["keys"], s["cos"], s["sin"]), s["k_cache"], s["k_scales"]),
                             (s["values"], s["v_cache"], s["v_scales"])):
        x = x.float()
        if s["keys"].dtype == torch.float16:
            x = x.clamp(-61440.0, 61440.0)
        amax = torch.zeros((n, Hkv), device=x.device).scatter_reduce_(
            0, which[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
        old = scales[ids].to(torch.int32)
        b = _exponent(amax)
        b = torch.where(fresh[:, None], b, torch.maximum(b, old))
        # rows that were held: rounded again under the exponent that grew
        shift = torch.where(fresh[:, None], 0, old - b).clamp(min=-126)
        rows = _values(cache.view(torch.uint8)[ids]).mul_(_power(shift)[:, None, :, None]).to(torch.float8_e4m3fn)
        rows = rows.view(torch.uint8)
        rows[which, row] = (x * _power(127 - b)[which][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        cache.view(torch.uint8)[ids] = rows
        scales[ids] = b.to(torch.uint8)
        out += [cache, scales]
    return out[0], out[2], out[1], out[3]


def _rotated(q, cos, sin):
    """Queries ``[W, Hq, S, E]`` rotated for every view, rounded to their type,
    in float32: ``[F, W, Hq, S, E]``; tables of half the width ``[F, W, S, R/2]``."""
    h = cos.shape[-1]
    x = q.float()[None]
    c, n = cos[:, :, None], sin[:, :, None]
    a, b = x[..., :h], x[..., h:2 * h]
    first, second = a * c - b * n, b * c + a * n
    rest = x[..., 2 * h:].expand(*first.shape[:-1], -1)
    return torch.cat([first, second, rest], dim=-1).to(q.dtype).float()


def _stream(s, cache, scales, n):
    """The first n rows of every sequence, ``[W, Hkv, n, E]`` float32."""
    bs = cache.shape[1]
    rows = torch.arange(n, device=cache.device)
    page = s["block_tables"].long()[:, rows // bs]
    x = _values(cache.view(torch.uint8)[page, rows % bs])
    x = x.mul_(_power(scales[page].to(torch.int32) - 127)[..., None])
    return x.permute(0, 2, 1, 3)


def _attend(s, queries, locations, cos, sin):
    """``[W, Hq, S, E]`` queries over the cached rows; locations ``[F, W, S]``."""
    fl = s["lengths"].long()
    W, Hq, S, _ = queries.shape
    width = s["block_tables"].shape[1] * s["k_cache"].shape[1]
    rows = torch.arange(width, device=fl.device)
    end = fl.cumsum(0)
    view = (rows[:, None] >= end).sum(1)
    place = torch.where(view < fl.shape[0], rows - (end - fl)[view.clamp(max=fl.shape[0] - 1)], 1 << 30)
    view = view.clamp(max=fl.shape[0] - 1)
    keys = _stream(s, s["k_cache"], s["k_scales"], width)
    q = _rotated(queries, cos, sin).reshape(-1, W, Hq // GQA, GQA * S, E)
    scores = q @ keys.transpose(-1, -2)[None]  # [F, W, Hkv, 16*S, n]
    scores = scores[0] if q.shape[0] == 1 else torch.gather(scores, 0, view.expand(1, *scores.shape[1:]))[0]
    seen = (place[:, None, None] <= locations.long()[view]).permute(1, 2, 0)  # [W, S, n]
    scores = scores.reshape(W, Hq // GQA, GQA, S, -1).mul_(SCALE).masked_fill_(~seen[:, None, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0)).reshape(W, Hq // GQA, GQA * S, -1)
    values = _stream(s, s["v_cache"], s["v_scales"], width)
    return (p @ values).reshape(W, Hq, S, E).to(queries.dtype)


def _plain_paged(s):
    h = s["cos"].shape[-1] // 2
    return _attend(s, s["queries"], s["locations"], s["cos"][..., :h], s["sin"][..., :h])


def _plain_varlen(s):
    """The packed tokens as rows of a grid [W, most], behind them rows that see nothing."""
    T, Hq, _ = s["queries"].shape
    cu, most = s["cu_q"].long(), s["most"]
    F, W = s["locations"].shape[0], cu.shape[0] - 1
    t = cu[:-1, None] + torch.arange(most, device=cu.device)
    there = t < cu[1:, None]
    at = t.clamp(max=T - 1)
    loc = torch.where(there[None], s["locations"][:, at], -1)
    out = _attend(s, s["queries"][at].transpose(1, 2), loc, s["cos"][:, at], s["sin"][:, at])
    return out.transpose(1, 2)[there]


# ---------------------------------------------------------------------------
# The same in 64 bits, one sequence, page or head after the other.
def _exact_tables(case, st):
    bs, T = st["bs"], st["T"]
    before, new = st["lengths"].tolist(), st["new_tokens"].tolist()
    bt = st["block_tables"].cpu().numpy().astype(np.int64)
    pages = st["free_pages"].tolist()
    count, P = int(st["free_count"]), len(pages)
    stack = pages[:count]
    for w in range(case["W"]):
        if new[w] < 0:
            stack += bt[w, :-(-before[w] // bs)].tolist()
    stack = stack[:P]
    listed_pages = np.array(stack + pages[len(stack):])
    cu, starts, lengths, pos, slots = [0], [], [], np.full(T, -1), np.full(T, -1)
    left, full = len(stack), False
    for w in range(case["W"]):
        k = max(new[w], 0)
        have = 0 if new[w] < 0 else before[w]
        need = -(-(have + k) // bs) - -(-have // bs)
        ok = have + k <= bt.shape[1] * bs and cu[-1] + k <= T
        if ok and need:
            full = full or need > left  # nobody after the first who has to wait gets pages
            ok = not full
            for j in range(need if ok else 0):
                left -= 1
                bt[w, -(-have // bs) + j] = stack[left]
        starts.append(have if ok and new[w] >= 0 else -1)
        for j in range(k if ok else 0):
            pos[cu[-1] + j] = have + j
            slots[cu[-1] + j] = bt[w, (have + j) // bs] * bs + (have + j) % bs
        lengths.append(have + k if ok else have)
        cu.append(cu[-1] + k)
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32)  # noqa: E731
    return (i32(cu), i32(starts), i32(pos), torch.tensor(slots), i32(lengths), i32([left]), i32(bt),
            i32(listed_pages))


def _e4m3(x):
    """float64 numbers of at most 448 rounded to E4M3, ties to even."""
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-300))), -6) - 3)
    return np.rint(x / step) * step


def _exact_append(case, st):
    slots = st["slots"].cpu().numpy()
    bs, R = case["bs"], case["R"]
    dt = st["keys"].dtype
    k = st["keys"].float()
    c, s = st["cos"].float()[:, None], st["sin"].float()[:, None]
    lo, hi = k[..., :R // 2], k[..., R // 2:R]
    # every product and sum rounded to the type
    turn = lambda x, y: (x.to(dt).float() + y.to(dt).float()).to(dt).float()  # noqa: E731
    k = torch.cat([turn(lo * c[..., :R // 2], -hi * s[..., :R // 2]), turn(hi * c[..., R // 2:], lo * s[..., R // 2:]),
                   k[..., R:]], dim=-1)
    out = []
    order = np.argsort(slots, kind="stable")
    page = slots[order] // bs
    begin = np.flatnonzero(np.concatenate([[True], page[1:] != page[:-1]]))
    ids = page[begin]
    group = np.repeat(np.arange(len(ids)), np.diff(np.concatenate([begin, [len(page)]])))
    fresh = slots[order][begin] % bs == 0
    for x, cache, scales in ((k, st["k_cache"], st["k_scales"]), (st["values"], st["v_cache"], st["v_scales"])):
        x = x.double().cpu().numpy()[order]
        b = scales.cpu().numpy().astype(np.int64)
        amax = np.maximum.reduceat(np.abs(x).max(-1), begin, axis=0)
        want = np.maximum(np.ceil(np.log2(np.maximum(amax, 1e-300) / 448.0)), -126).astype(np.int64)
        want = np.where(amax > 448.0 * np.exp2(want), want + 1, want) + 127
        b_old = b[ids]
        b[ids] = np.where(fresh[:, None], want, np.maximum(want, b_old))
        held = cache.double()[torch.from_numpy(ids).cuda()].cpu().numpy()
        shift = np.where(fresh[:, None], 0, b_old - b[ids])
        held = np.where(shift[:, None, :, None] < 0, _e4m3(held * np.exp2(shift)[:, None, :, None]), held)
        held[group, slots[order] % bs] = _e4m3(x * np.exp2(127 - b[ids])[group][..., None])
        full = cache.double()
        full[torch.from_numpy(ids).cuda()] = torch.from_numpy(held).cuda()
        out += [full, torch.from_numpy(b.astype(np.uint8))]
    return out[0], out[2], out[1], out[3]


def _exact_attention(case, st, lay):
    f64 = torch.float64
    W, Hkv, bs = case["W"], case["Hkv"], case["bs"]
    lens, fl, new = lay["lens"], lay["fl"], lay["new"]
    F = len(fl)
    off = np.concatenate([[0], np.cumsum(fl)[:-1]])
    bt = st["block_tables"].cpu().numpy().astype(np.int64)
    packed = case["kind"] == "varlen"
    queries = st["queries"] if packed else st["queries"].transpose(1, 2).reshape(-1, GQA * Hkv, E)
    h = case["R"] // 2
    cos, sin = (st[x].reshape(F, -1, st[x].shape[-1])[..., :h] for x in ("cos", "sin"))
    loc = st["locations"].reshape(F, -1)
    out = torch.zeros(queries.shape, dtype=f64, device="cuda")
    first = np.concatenate([[0], np.cumsum(new)])

    def held(cache, exponents, page, row, j):
        byte = cache.view(torch.uint8)[page, row, j]
        return byte.view(torch.float8_e4m3fn).to(f64) * torch.exp2(exponents[page, j].to(f64) - 127)[:, None]

    for w in range(W):
        a, z = int(first[w]), int(first[w + 1])
        rows = np.concatenate([off[f] + np.arange(lens[w, f]) for f in range(F)])
        page, row = torch.from_numpy(bt[w, rows // bs]).cuda(), torch.from_numpy(rows % bs).cuda()
        hidden = torch.cat([torch.arange(int(lens[w, f]), device="cuda")[None] > loc[f, a:z, None] for f in range(F)], 1)
        for j in range(Hkv):
            k = held(st["k_cache"], st["k_scales"], page, row, j)
            v = held(st["v_cache"], st["v_scales"], page, row, j)
            x = queries[a:z, GQA * j:GQA * (j + 1)].to(torch.float32)
            scores, at = [], 0
            for f in range(F):
                c, n = cos[f, a:z, None], sin[f, a:z, None]
                y = x.clone()
                y[..., :h] = x[..., :h] * c - x[..., h:2 * h] * n
                y[..., h:2 * h] = x[..., h:2 * h] * c + x[..., :h] * n
                y = y.to(queries.dtype).to(f64)
                scores.append((y.reshape(-1, E) @ k[at:at + int(lens[w, f])].T).reshape(z - a, GQA, -1) * SCALE)
                at += int(lens[w, f])
            p = torch.cat(scores, dim=-1).masked_fill_(hidden[:, None], -math.inf)
            p = torch.nan_to_num(torch.softmax(p, dim=-1))
            out[a:z, GQA * j:GQA * (j + 1)] = (p.reshape(-1, len(rows)) @ v).reshape(z - a, GQA, E)
    if packed:
        return out
    return out.reshape(W, case["S"], GQA * Hkv, E).transpose(1, 2).contiguous()


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(case, st)
    if case["kind"] == "append":
        return _exact_append(case, st)
    return _exact_attention(case, st, _layout(case))
