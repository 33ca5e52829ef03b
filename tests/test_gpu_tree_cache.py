"""GPU tests of the operators for drafted token trees and bounded caches
(marked ``gpu``) against their 64-bit restatement in oracle/tree_cache_oracle.py.

Tolerances are bounds, not measurements.  A float32 score is off by at most
(E + 8) roundings of the terms it sums, e = (E + 8) * 2^-24 * sum |q_e k_e| * |scale|,
so a softmax weight by a factor exp(2 e), and sums over n keys by n * 2^-24 more.  An
output element is a weighted sum of v: its error is bounded by the same factor times
sum p |v|, plus the roundings the types bring -- bf16: the weights (2^-8, and the
normaliser sums the rounded ones: twice), a stored partial result (2^-11 of a row's
largest magnitude) and the output (2^-8); fp16: the output (2^-11).  Whole numbers and
moved rows have to be equal.
"""
import math

import pytest
import torch

from oracle import tree_cache_oracle as TO

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 128
SCALE = E ** -0.5


@pytest.fixture(scope="module")
def dv(gpu):
    import dvattention_amd
    return dvattention_amd


def to(dev, d):
    return {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in d.items()}


def random_tree(g, S, absent=0.1):
    parents = torch.full((S,), -1, dtype=torch.int32)
    for s in range(1, S):
        parents[s] = int(torch.randint(-1, s, (1,), generator=g))
        if float(torch.rand((), generator=g)) < absent:
            parents[s] = [-2, s, S + 5][int(torch.randint(0, 3, (1,), generator=g))]
    return parents


def cache_case(g, dtype, W, Hkv, fl, bs, spare=1, bad=False):
    n = sum(max(x, 0) for x in fl)
    maxB = max(1, (n + bs - 1) // bs) + spare
    P = W * maxB + 2
    bt = torch.randperm(P, generator=g)[:W * maxB].to(torch.int32).reshape(W, maxB)
    if bad:  # pages that do not exist, in the middle
        bt[0, maxB // 2] = -3
        bt[-1, 0] = P + 1
    kc = torch.randn(P, bs, Hkv, E, generator=g).to(dtype)
    vc = torch.randn(P, bs, Hkv, E, generator=g).to(dtype)
    return dict(k_cache=kc, v_cache=vc, block_tables=bt, fragment_lengths=torch.tensor(fl, dtype=torch.int32))


def query_case(g, dtype, W, Hkv, F, S, R):
    ang = torch.rand(F, W, S, R, generator=g) * 6.0
    return dict(queries=(torch.randn(W, 16 * Hkv, S, E, generator=g) * 2).to(dtype), cosines=torch.cos(ang),
                sines=torch.sin(ang))


def tree_case(dtype, W, Hkv, S, fl, bs, R, seed, chain=False, bad=False, absent=0.1):
    """Committed lengths differ between sequences; the drafted rows lie in a view of
    each sequence's choice."""
    g = torch.Generator().manual_seed(seed)
    F = len(fl)
    d = cache_case(g, dtype, W, Hkv, fl, bs, bad=bad) | query_case(g, dtype, W, Hkv, F, S, R)
    loc = torch.empty(F, W, S, dtype=torch.int32)
    tv, tr, parents = [], [], []
    for w in range(W):
        own = int(torch.randint(0, F, (1,), generator=g))
        first = max(0, fl[own] - S - w)
        tv.append(own)
        tr.append(sum(fl[:own]) + first)
        for f in range(F):
            loc[f, w] = first - 1 if f == own else int(torch.randint(-1, max(fl[f], 1), (1,), generator=g))
        p = torch.arange(-1, S - 1, dtype=torch.int32) if chain else random_tree(g, S, absent)
        parents.append(p)
    d.update(locations=loc, parents=torch.stack(parents), tree_views=torch.tensor(tv, dtype=torch.int32),
             tree_rows=torch.tensor(tr, dtype=torch.int32))
    return d


def widened(d, rows):
    """The same case under a block table of at least so many rows."""
    W, maxB = d["block_tables"].shape
    wide = torch.full((W, max(maxB, rows // d["k_cache"].shape[1])), -1, dtype=torch.int32)
    wide[:, :maxB] = d["block_tables"]
    return {**d, "block_tables": wide}


def check_tree(dv, gpu, d, dtype, scale=SCALE):
    """Under the given block table, where one launch may take the call, under a wider one,
    which cuts the nodes' key lists into windows, and under a wide one, where pieces of the
    committed keys are merged."""
    want, size, spread = TO.tree_sdpa(scale, **d)
    for case in (widened(d, 80000), widened(d, 2500), d):
        got = compare_tree(dv.dvattn_tree_paged_sdpa(scale=scale, **to(gpu, case)).cpu(), d, dtype, want, size, spread)
    return got, want


def compare_tree(got, d, dtype, want, size, spread):
    n = int(d["fragment_lengths"].clamp(min=0).sum())
    e = 2 * (E + 8) * 2.0 ** -24 * spread + (n + 16) * 2.0 ** -24
    tol = size * torch.expm1(2 * e) + 1e-30
    if dtype == torch.bfloat16:
        tol = tol + 2 * 2.0 ** -8 * size + 2.0 ** -10 * size.amax(-1, keepdim=True) + 2.0 ** -8 * want.abs()
    if dtype == torch.float16:
        tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -24
    assert torch.equal(got.isnan(), want.isnan())
    over = (got.double() - want).abs().nan_to_num(0.0) - tol.nan_to_num(math.inf)
    assert bool((over <= 0).all()), f"largest excess {float(over.max()):.3e}"
    return got


TREES = [
    # W, Hkv, S, view lengths, page size, R
    (1, 1, 1, [6], 16, 128),           # one node
    (2, 2, 2, [40], 16, 64),           # two
    (2, 1, 7, [19, 130], 24, 32),      # two views, pages of 24 keys
    (3, 2, 16, [200], 16, 128),        # one group of nodes, four wave sets not taken
    (2, 1, 17, [90, 33, 70], 8, 20),   # a group of one node behind a full one; R/2 odd
    (1, 2, 33, [300], 32, 0),          # no rotation
    (2, 1, 5, [5], 16, 128),           # nothing committed
    (1, 1, 64, [1100], 16, 128),
    (1, 2, 100, [110], 16, 64),        # a path longer than a wave has lanes; just nodes
    (2, 1, 3, [25, 1, 40, 60], 24, 64),  # four views
    (2, 1, 4, [300, 900], 16, 128),    # windows that meet two views
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TREES)
def test_tree_sdpa(dv, gpu, dtype, shape):
    W, Hkv, S, fl, bs, R = shape
    check_tree(dv, gpu, tree_case(dtype, W, Hkv, S, fl, bs, R, seed=S + len(fl)), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_sdpa_missing_pages(dv, gpu, dtype):
    check_tree(dv, gpu, tree_case(dtype, 2, 2, 12, [60, 50], 8, 64, seed=3, bad=True), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("S", [3, 130])
def test_tree_sdpa_chain_is_causal(dv, gpu, dtype, S):
    """A chain is a causal chunk: dvattn_paged_sdpa with locations that grow by one."""
    d = tree_case(dtype, 2, 1, S, [400], 16, 64, seed=S, chain=True)
    got, _ = check_tree(dv, gpu, d, dtype)
    g = to(gpu, {k: d[k] for k in ("queries", "cosines", "sines", "fragment_lengths", "k_cache", "v_cache",
                                   "block_tables")})
    loc = (d["locations"] + 1 + torch.arange(S, dtype=torch.int32)).to(gpu)
    causal = dv.dvattn_paged_sdpa(locations=loc, scale=SCALE, **g).cpu()
    tol = 4 * torch.finfo(dtype).eps + 2e-5
    assert (got.float() - causal.float()).abs().max() <= tol * max(1.0, float(causal.abs().max()))


def test_tree_of_the_most_nodes(dv, gpu):
    """4096 nodes: a chain of all of them is a causal chunk; its metadata counts depths."""
    S, dt = 4096, torch.float16
    d = to(gpu, tree_case(dt, 1, 1, S, [S + 30], 16, 64, seed=4, chain=True))
    got = dv.dvattn_tree_paged_sdpa(scale=SCALE, **d).float()
    loc = d["locations"] + 1 + torch.arange(S, dtype=torch.int32, device=gpu)
    causal = dv.dvattn_paged_sdpa(locations=loc, scale=SCALE, **{k: d[k] for k in (
        "queries", "cosines", "sines", "fragment_lengths", "k_cache", "v_cache", "block_tables")}).float()
    assert got.isfinite().all()
    tol = 4 * torch.finfo(dt).eps + 2e-5
    assert (got - causal).abs().max() <= tol * max(1.0, float(causal.abs().max()))
    inv = torch.full((2,), 2.0 ** -8, device=gpu)
    loc, cos, sin, views, rows = dv.dvattn_tree_metadata(d["fragment_lengths"], torch.zeros(1, 1, dtype=torch.int32,
                                                         device=gpu), d["parents"], inv)
    angle = (30 + torch.arange(S, device=gpu, dtype=torch.float64)) * 2.0 ** -8
    assert loc.eq(29).all() and views.tolist() == [0] and rows.tolist() == [30]
    assert (cos[0, 0].double() - torch.cos(angle)[:, None]).abs().max() <= 2.0 ** -22
    assert (sin[0, 0].double() - torch.sin(angle)[:, None]).abs().max() <= 2.0 ** -22


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_sdpa_unseen_rows_may_hold_anything(dv, gpu, dtype):
    """NaN and infinity in drafted rows that no node, or only another node, sees:
    siblings of a path, absent nodes' rows, rows behind the tree."""
    d = tree_case(dtype, 2, 1, 9, [80], 16, 128, seed=11, absent=0.0)
    d["parents"][0] = torch.tensor([-1, -1, 0, 0, 1, 2, -2, 6, 4])
    first = int(d["tree_rows"][0])
    for j, x in ((3, math.nan), (6, math.nan), (7, math.inf), (8, -math.inf)):
        page, row = TO.cache_row(d["block_tables"], 0, first + j, d["k_cache"].shape[0], 16)
        d["k_cache"][page, row] = x
        d["v_cache"][page, row] = x
    got, want = check_tree(dv, gpu, d, dtype)
    assert got[0, :, [0, 1, 2, 4, 5]].isfinite().all() and not got[0, :, [6, 7]].any()
    assert want[0, :, 3].isnan().all()  # a node sees its own row


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tree_sdpa_keys_count_once(dv, gpu, dtype):
    """Locations that reach into the drafted rows, drafted rows that leave the view, and
    views that do not exist."""
    d = tree_case(dtype, 3, 1, 10, [64, 40], 16, 64, seed=5)
    own = d["tree_views"].long()
    for w in range(3):
        d["locations"][own[w], w] += torch.arange(10, dtype=torch.int32)  # up to nine drafted rows are committed too
    d["tree_rows"][1] += 4      # the last rows lie past the view
    d["tree_views"][2] = 7      # no such view: the committed keys only
    check_tree(dv, gpu, d, dtype)
    d["tree_rows"][0] -= 60     # before the view (a negative row, or another view's)
    d["tree_views"][2] = -1
    check_tree(dv, gpu, d, dtype)


def test_tree_sdpa_negative_scale_and_empty(dv, gpu):
    d = tree_case(torch.float32, 2, 1, 6, [50], 16, 64, seed=9)
    check_tree(dv, gpu, d, torch.float32, scale=-0.05)
    d["locations"][:] = -1
    d["tree_views"][:] = -1
    got, _ = check_tree(dv, gpu, d, torch.float32)
    assert not got.any()
    e = tree_case(torch.bfloat16, 2, 1, 4, [30], 16, 64, seed=9)
    for name, dim in (("queries", 2), ("cosines", 2), ("sines", 2), ("locations", 2), ("parents", 1)):
        e[name] = e[name].narrow(dim, 0, 0).contiguous()
    assert dv.dvattn_tree_paged_sdpa(scale=SCALE, **to(gpu, e)).shape == (2, 16, 0, E)


@pytest.mark.parametrize("W", [2, 150])
def test_tree_sdpa_without_views(dv, gpu, W):
    """F = 0, with pages and without: zeros, for few nodes and for more than a launch of
    short lists takes."""
    d = tree_case(torch.bfloat16, W, 2, 4, [20], 16, 64, seed=3)
    for name in ("locations", "cosines", "sines", "fragment_lengths"):
        d[name] = d[name][:0].contiguous()
    for pages in (d["block_tables"], d["block_tables"][:, :0].contiguous()):
        out = torch.full((W, 32, 4, E), math.nan, dtype=torch.bfloat16, device=gpu)
        dv.dvattn_tree_paged_sdpa(scale=SCALE, out=out, **to(gpu, {**d, "block_tables": pages}))
        assert not out.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_sdpa_many_short_sequences(dv, gpu, dtype):
    """More nodes than a launch of whole lists takes, few keys each."""
    check_tree(dv, gpu, tree_case(dtype, 90, 2, 7, [9, 14], 16, 64, seed=8), dtype)


# ---------------------------------------------------------------------------
def mass_case(dtype, W, Hkv, S, fl, bs, R, seed, extra=3, bad=False):
    g = torch.Generator().manual_seed(seed)
    F = len(fl)
    d = cache_case(g, dtype, W, Hkv, fl, bs, spare=2, bad=bad) | query_case(g, dtype, W, Hkv, F, S, R)
    del d["v_cache"]
    loc = torch.empty(F, W, S, dtype=torch.int32)
    for f in range(F):
        loc[f] = torch.randint(-1, max(fl[f], 1) + 4, (W, S), generator=g)
    d.update(locations=loc)
    mass = torch.rand(W, Hkv, max(1, sum(max(x, 0) for x in fl) + extra), generator=g)
    return d, mass


def check_mass(dv, gpu, d, mass, decay, in_place=False, scale=SCALE):
    want, spread = TO.key_mass(mass, decay, scale, **d)
    g, m = to(gpu, d), mass.to(gpu)
    out = None if in_place else torch.full_like(m, math.nan)
    got = dv.dvattn_paged_key_mass(m, scale=scale, decay=decay, out=out, **g).cpu()
    if not in_place:
        assert torch.equal(m.cpu(), mass)
    n = int(d["fragment_lengths"].clamp(min=0).sum())
    S = d["queries"].shape[2]
    e = 2 * ((E + 8) * spread + n + 16 * S + 64) * 2.0 ** -24
    tol = (want.abs() + mass * abs(decay)) * (math.expm1(e) + 2.0 ** -22) + 1e-30
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), f"largest excess {float(over.max()):.3e}"
    return got


MASSES = [
    # W, Hkv, S, view lengths, page size, R
    (1, 1, 1, [1], 16, 128),
    (2, 2, 1, [300], 16, 128),
    (3, 1, 1, [70, 5, 190], 24, 64),    # units that meet several views
    (2, 1, 1, [0, 33], 5, 20),
    (2, 2, 2, [130], 16, 0),
    (1, 1, 7, [90, 150], 32, 32),
    (1, 1, 70, [140], 8, 128),          # two launches of tokens
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", MASSES)
def test_key_mass(dv, gpu, dtype, shape):
    W, Hkv, S, fl, bs, R = shape
    d, mass = mass_case(dtype, W, Hkv, S, fl, bs, R, seed=S + len(fl))
    check_mass(dv, gpu, d, mass, 0.75)


def test_key_mass_whole_units(dv, gpu):
    """Tokens that all see whole units of keys, in whole groups (the loop without masks),
    for either sign of the scale."""
    for dtype in DTYPES:
        d, mass = mass_case(dtype, 2, 1, 17, [530], 16, 128, seed=12)
        d["locations"][:] = 529
        check_mass(dv, gpu, d, mass, 1.0)
        check_mass(dv, gpu, d, mass, 1.0, scale=-SCALE)


WINDOWS = [s for s in MASSES if s[2] > 1] + [(3, 2, 8, [50, 0, 300, 9], 16, 64), (1, 2, 9, [517], 24, 128),
                                             (2, 1, 64, [100, 31], 16, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", WINDOWS)
@pytest.mark.parametrize("bad", [False, True])
def test_key_mass_narrow_and_wide_tables(dv, gpu, dtype, shape, bad):
    """The same keys under a block table of their size, where few blocks cover them and the
    waves of a block share the tokens, and under one so wide that a plan cuts them."""
    W, Hkv, S, fl, bs, R = shape
    d, mass = mass_case(dtype, W, Hkv, S, fl, bs, R, seed=S + W, bad=bad)
    d["locations"][-1, 0, 0] = -1
    narrow = check_mass(dv, gpu, d, mass, 0.75)
    d = widened(d, 40000)
    again = check_mass(dv, gpu, d, mass, 0.75)
    assert (narrow - again).abs().max() <= 1e-4 * S
    assert torch.equal(again, check_mass(dv, gpu, d, mass, 0.75, in_place=True))
    d["locations"][:] = 10 ** 6  # every token sees whole views
    check_mass(dv, gpu, d, mass, 1.0, scale=-SCALE)


@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("extra", [-40, 0, 700])
@pytest.mark.parametrize("decay", [0.0, 1.0])
def test_key_mass_capacity_and_decay(dv, gpu, S, extra, decay):
    """Capacities short of the stream and far past it; in place; mass not read for decay 0."""
    d, mass = mass_case(torch.bfloat16, 2, 1, S, [150, 60], 16, 64, seed=2, extra=extra)
    a = check_mass(dv, gpu, d, mass, decay)
    if decay == 0.0:
        nan = torch.full_like(mass, math.nan).to(gpu)
        b = dv.dvattn_paged_key_mass(nan, scale=SCALE, decay=0.0, **to(gpu, d)).cpu()
        c = dv.dvattn_paged_key_mass(None, scale=SCALE, decay=0.0, out=nan, **to(gpu, d)).cpu()
        assert torch.equal(a, b) and torch.equal(a, c)
    else:
        assert torch.equal(a, check_mass(dv, gpu, d, mass, decay, in_place=True))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("S", [1, 5])
def test_key_mass_missing_pages_and_unseen_keys(dv, gpu, dtype, S):
    """Pages that do not exist, tokens that see nothing, NaN in rows no token sees, and
    weights that sum to the number of (token, head) rows with a key."""
    d, mass = mass_case(dtype, 2, 2, S, [70, 50], 8, 64, seed=4, bad=True)
    d["locations"][:, 1, 0] = -1
    d["locations"][1] = d["locations"][1].clamp(max=20)
    for w in range(2):
        for p in range(70 + 21, 120):
            at = TO.cache_row(d["block_tables"], w, p, d["k_cache"].shape[0], 8)
            if at:
                d["k_cache"][at[0], at[1]] = math.nan
    got = check_mass(dv, gpu, d, mass, 0.0)
    assert got.isfinite().all()
    rows = (d["locations"] >= 0).any(0).sum(1) * 16  # (token, head) rows of a KV head
    assert torch.allclose(got.sum(-1), rows[:, None].float().expand(2, 2), rtol=1e-5)


def test_key_mass_nan_stays_in_its_head(dv, gpu):
    """A NaN query makes its own head's weights NaN and leaves keys it does not see alone."""
    for S in (1, 2):
        d, mass = mass_case(torch.float32, 1, 2, S, [60], 16, 0, seed=1)
        d["locations"][:] = 29
        d["queries"][0, 3, 0] = math.nan
        got = dv.dvattn_paged_key_mass(mass.to(gpu), scale=SCALE, **to(gpu, d)).cpu()
        assert got[0, 0, :30].isnan().all() and torch.equal(got[0, 0, 30:], mass[0, 0, 30:])
        assert got[0, 1].isfinite().all()


@pytest.mark.parametrize("S", [1, 2])
def test_key_mass_many_ragged_sequences(dv, gpu, S):
    """More sequences than a wave has lanes, most of them short, and block tables so wide
    that the scores of one token are not kept (more than 1 GiB of them)."""
    g = torch.Generator().manual_seed(S)
    W, fl, bs = 70, [40, 700], 16
    d, mass = mass_case(torch.float16, W, 1, S, fl, bs, 64, seed=S)
    d["locations"][1] = torch.randint(-1, 30, (W, S), generator=g)
    d["locations"][1, ::13] = torch.randint(300, 700, (6, S), generator=g)
    d["locations"][0, 5:9] = -1
    narrow = check_mass(dv, gpu, d, mass, 0.5)
    wide = torch.full((W, 15500), -1, dtype=torch.int32)
    wide[:, :d["block_tables"].shape[1]] = d["block_tables"]
    d["block_tables"] = wide
    assert W * wide.shape[1] * bs * 64 > 1 << 30
    again = check_mass(dv, gpu, d, mass, 0.5)
    assert (narrow - again).abs().max() <= 1e-4


def test_key_mass_windows_of_a_prompt(dv, gpu):
    """Every token of a prompt votes: more tokens than a launch takes, each seeing the
    keys before it, whole parts of the keys seen by later launches only."""
    d, mass = mass_case(torch.bfloat16, 1, 1, 150, [600], 16, 64, seed=6)
    d["locations"][0, 0] = 4 * torch.arange(150, dtype=torch.int32)
    got = check_mass(dv, gpu, d, mass, 0.0)
    assert got[0, 0, 597:].eq(0).all()


def test_key_mass_no_tokens_decays(dv, gpu):
    d, mass = mass_case(torch.bfloat16, 2, 1, 2, [40], 16, 64, seed=8)
    for name, dim in (("queries", 2), ("cosines", 2), ("sines", 2), ("locations", 2)):
        d[name] = d[name].narrow(dim, 0, 0).contiguous()
    got = dv.dvattn_paged_key_mass(mass.to(gpu), scale=SCALE, decay=0.5, **to(gpu, d)).cpu()
    assert torch.equal(got, mass * 0.5)


# ---------------------------------------------------------------------------
def run_select(dv, gpu, mass, first, lengths, budget, kf, kl):
    first, lengths = (torch.tensor(x, dtype=torch.int32) for x in (first, lengths))
    want = TO.select(mass, first, lengths, budget, kf, kl)
    got = dv.dvattn_kv_select(mass.to(gpu), first.to(gpu), lengths.to(gpu), budget, kf, kl).cpu()
    assert torch.equal(got, want)
    return got


@pytest.mark.parametrize("budget,kf,kl", [(1, 0, 0), (37, 4, 9), (40, 40, 0), (40, 3, 37), (500, 10, 100)])
def test_select(dv, gpu, budget, kf, kl):
    g = torch.Generator().manual_seed(budget)
    mass = torch.exp(3 * torch.randn(4, 2, 900, generator=g)) * (torch.rand(4, 2, 900, generator=g) > 0.2)
    run_select(dv, gpu, mass, [0, 100, 5, 899], [900, 333, 38, 1], budget, kf, kl)


def test_select_ranges(dv, gpu):
    """Lengths of zero, below zero and past the capacity; first rows outside it."""
    mass = torch.rand(6, 1, 64, generator=torch.Generator().manual_seed(1))
    run_select(dv, gpu, mass, [0, 0, 10, -1, 64, 70], [0, -5, 1000, 20, 20, 20], 8, 1, 2)


@pytest.mark.parametrize("n", [63, 1025, 5000, 20001])
def test_select_ties_and_specials(dv, gpu, n):
    """Few distinct weights, all equal ones, signed zeros, infinities, negative and NaN."""
    g = torch.Generator().manual_seed(n)
    mass = torch.randint(0, 4, (5, 1, n), generator=g).float()
    mass[1] = 0.0
    mass[1, 0, ::3] = -0.0
    mass[2] = torch.tensor([math.nan, math.inf, -math.inf, -1.0, 0.0, 1e-42, -1e-42, 7.0])[
        torch.randint(0, 8, (n,), generator=g)]
    mass[3] = math.nan
    mass[4] = 1.0 + torch.randint(0, 3, (n,), generator=g) * 2.0 ** -23  # weights that differ in the last bits
    for budget in (1, n // 3, n - 1):
        run_select(dv, gpu, mass, [0] * 5, [n] * 5, budget, min(2, budget // 4), budget // 3)


# ---------------------------------------------------------------------------
def compact_case(dtype, W, Hkv, rows_n, N, bs, seed, heads=None, Ek=E, Ev=E, pool=False):
    g = torch.Generator().manual_seed(seed)
    maxB = (rows_n + bs - 1) // bs
    P = W * maxB + 1
    bt = torch.randperm(P, generator=g)[:W * maxB].to(torch.int32).reshape(W, maxB)
    shape = (P, Hkv, bs) if pool else (P, bs, Hkv)
    kc, vc = (torch.randn(*shape, e, generator=g).to(dtype) for e in (Ek, Ev))
    rows = torch.full((W, heads or Hkv, N), -1, dtype=torch.int32)
    first = torch.randint(0, max(1, rows_n // 4), (W,), generator=g).to(torch.int32)
    lengths = rows_n - first
    for w in range(W):
        for h in range(heads or Hkv):
            k = min(N, int(lengths[w]))
            rows[w, h, :k] = torch.randperm(int(lengths[w]), generator=g)[:k].sort().values.to(torch.int32)
    mass = torch.rand(W, Hkv, rows_n + 5, generator=g)
    return kc, vc, bt, rows, first, lengths.to(torch.int32), mass


def check_compact(dv, gpu, kc, vc, bt, rows, first, lengths, mass, pool=False):
    view = (lambda t: t.permute(0, 2, 1, 3)) if pool else (lambda t: t)
    k_ref, v_ref, m_ref = TO.compact(view(kc), view(vc), bt, rows, first, lengths, mass)
    kg, vg = kc.to(gpu), vc.to(gpu)
    mg = None if mass is None else mass.to(gpu)
    dv.dvattn_paged_kv_compact(rows.to(gpu), first.to(gpu), view(kg), view(vg), bt.to(gpu), mass=mg,
                               lengths=None if lengths is None else lengths.to(gpu))
    assert torch.equal(view(kg).cpu(), k_ref) and torch.equal(view(vg).cpu(), v_ref)
    if mass is not None:
        assert torch.equal(mg.cpu(), m_ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [None, 1])
@pytest.mark.parametrize("pool", [False, True])
def test_compact(dv, gpu, dtype, heads, pool):
    case = compact_case(dtype, 3, 4, 150, 60, 16, seed=1, heads=heads, pool=pool)
    check_compact(dv, gpu, *case, pool=pool)
    check_compact(dv, gpu, *case[:5], None, None, pool=pool)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Ek,Ev", [(100, 36), (7, 130), (128, 0), (0, 64)])
def test_compact_head_dims(dv, gpu, dtype, Ek, Ev):
    """Rows that 16-byte vectors do not fit, and caches without keys or values."""
    check_compact(dv, gpu, *compact_case(dtype, 2, 2, 90, 40, 8, seed=2, Ek=Ek, Ev=Ev))


def test_compact_refuses_overlapping_rows(dv, gpu):
    kc, vc, bt, rows, first, lengths, mass = (t.to(gpu) for t in compact_case(torch.float16, 1, 2, 40, 10, 16, seed=2))
    with pytest.raises(RuntimeError, match="memory"):
        dv.dvattn_paged_kv_compact(rows, first, kc[:, :, :1].expand(-1, -1, 2, -1), vc, bt)


def test_compact_many_rows(dv, gpu):
    """Several batches of rows, where sources of later batches lie among the
    destinations of earlier ones' neighbours."""
    kc, vc, bt, rows, first, lengths, mass = compact_case(torch.float16, 1, 1, 6000, 5500, 16, seed=3)
    check_compact(dv, gpu, kc, vc, bt, rows, first, lengths, mass)


def test_compact_any_entries(dv, gpu):
    """Entries out of order, twice, below their place, past the range, on missing pages."""
    kc, vc, bt, rows, first, lengths, mass = compact_case(torch.bfloat16, 3, 2, 200, 120, 16, seed=4)
    g = torch.Generator().manual_seed(5)
    rows = torch.randint(-3, 210, rows.shape, generator=g).to(torch.int32)
    rows[:, :, 10:20] = 77
    lengths[1] = 90
    bt[0, 9] = -1
    bt[2, 1] = 1 << 20
    first[1] = 3
    check_compact(dv, gpu, kc, vc, bt, rows, first, lengths, mass)
    first[2] = -4
    lengths[0] = -2
    check_compact(dv, gpu, kc, vc, bt, rows, first, lengths, mass)
    check_compact(dv, gpu, kc, vc, bt, rows[:, :, :0].contiguous(), first, lengths, mass)


# ---------------------------------------------------------------------------
def meta_inputs(W, F, S, R, seed, absent=0.15):
    g = torch.Generator().manual_seed(seed)
    fl = torch.randint(S, 3 * S + 400, (F,), generator=g).to(torch.int32)
    order = torch.stack([torch.randperm(F, generator=g) for _ in range(W)]).to(torch.int32)
    parents = torch.stack([random_tree(g, S, absent) for _ in range(W)])
    inv = (1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))).float()
    return fl, order, parents, inv


def check_meta(dv, gpu, fl, order, parents, inv, scaling=1.0):
    want = TO.metadata(fl, order, parents, inv, scaling)
    got = [t.cpu() for t in dv.dvattn_tree_metadata(fl.to(gpu), order.to(gpu), parents.to(gpu), inv.to(gpu), scaling)]
    for i in (0, 3, 4):
        assert torch.equal(got[i], want[i])
    for i in (1, 2):  # cosf and sinf: a few units in the last place of values up to 1
        assert (got[i].double() - want[i]).abs().max().item() <= 4 * 2.0 ** -24 * max(1.0, abs(scaling)) \
            if want[i].numel() else got[i].numel() == 0


@pytest.mark.parametrize("W,F,S,R", [(1, 1, 1, 128), (3, 2, 9, 64), (2, 5, 70, 20), (5, 40, 3, 0), (2, 3, 200, 32)])
def test_tree_metadata(dv, gpu, W, F, S, R):
    check_meta(dv, gpu, *meta_inputs(W, F, S, R, seed=S), scaling=1.25)


def test_tree_metadata_orders(dv, gpu):
    """Views missing from an order, named twice, outside the range; own views shorter
    than the tree; an order whose own view does not exist."""
    fl, order, parents, inv = meta_inputs(4, 4, 12, 32, seed=1)
    fl[2] = 5
    order[0] = torch.tensor([-1, -1, 0, 2])
    order[1] = torch.tensor([1, 3, 1, 2])
    order[2] = torch.tensor([9, 0, 1, 3])
    order[3] = torch.tensor([0, 1, 2, -1])
    check_meta(dv, gpu, fl, order, parents, inv)


def test_tree_metadata_without_nodes_or_views(dv, gpu):
    """The place of the drafted rows is written for S = 0 and F = 0 too."""
    fl, order, parents, inv = meta_inputs(3, 2, 4, 64, seed=3)
    loc, cos, _, views, rows = dv.dvattn_tree_metadata(fl.to(gpu), order.to(gpu), parents[:, :0].contiguous().to(gpu),
                                                       inv.to(gpu))
    own = order[:, -1].long()
    want = [int(fl[:o + 1].sum()) if 0 <= o < 2 else 0 for o in own.tolist()]  # S = 0: behind the view's rows
    assert loc.shape == (2, 3, 0) and cos.shape == (2, 3, 0, 64)
    assert views.tolist() == [o if 0 <= o < 2 else -1 for o in own.tolist()] and rows.tolist() == want
    views, rows = dv.dvattn_tree_metadata(fl[:0].to(gpu), order[:, :0].contiguous().to(gpu), parents.to(gpu),
                                          inv.to(gpu))[3:]
    assert views.tolist() == [-1] * 3 and rows.tolist() == [0] * 3


@pytest.mark.parametrize("round_to", [None, torch.bfloat16, torch.float16])
def test_tree_metadata_chain_is_view_metadata(dv, gpu, round_to):
    """One sequence drafting a chain: the tables of S ordinary new tokens, bit for bit."""
    S, F = 7, 4
    fl, order, _, inv = meta_inputs(1, F, S, 64, seed=3)
    parents = torch.arange(-1, S - 1, dtype=torch.int32)[None]
    a = dv.dvattn_tree_metadata(fl.to(gpu), order.to(gpu), parents.to(gpu), inv.to(gpu), 1.0, round_to)
    b = dv.dvattn_view_metadata(fl.to(gpu), order.to(gpu), S, inv.to(gpu), 1.0, round_to)
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    own = int(order[0, -1])
    assert torch.equal(a[0][own, 0], b[0][own, 0, :1].expand(S) - 1)


# ---------------------------------------------------------------------------
def everything(dv, gpu, dtype):
    """One call of each operator on inputs of its own; returns (run, state to restore)."""
    trees = [to(gpu, widened(tree_case(dtype, 2, 2, 10, [60, 90], 16, 64, seed=21), n)) for n in (0, 2500, 80000)]
    md, mass = mass_case(dtype, 2, 2, 1, [200], 16, 64, seed=22)
    md3, mass3 = mass_case(dtype, 2, 2, 3, [200], 16, 64, seed=23)
    mdw = to(gpu, widened(md3, 40000))
    md, md3, mass, mass3 = to(gpu, md), to(gpu, md3), mass.to(gpu), mass3.to(gpu)
    fl, order, parents, inv = (t.to(gpu) for t in meta_inputs(2, 2, 10, 64, seed=24))
    kc, vc, bt, rows, first, lengths, cm = (t.to(gpu) for t in compact_case(dtype, 2, 2, 150, 60, 16, seed=25))
    k0, v0, cm0, mass_out = kc.clone(), vc.clone(), cm.clone(), torch.empty_like(mass)
    mass3_out, massw_out = torch.empty_like(mass3), torch.empty_like(mass3)

    def run():
        kc.copy_(k0), vc.copy_(v0), cm.copy_(cm0)
        out = [dv.dvattn_tree_paged_sdpa(scale=SCALE, **d) for d in trees]
        out.append(dv.dvattn_paged_key_mass(mass, scale=SCALE, decay=0.5, out=mass_out, **md))
        out.append(dv.dvattn_paged_key_mass(mass3, scale=SCALE, decay=0.5, out=mass3_out, **md3))
        out.append(dv.dvattn_paged_key_mass(mass3, scale=SCALE, decay=0.5, out=massw_out, **mdw))
        out += dv.dvattn_tree_metadata(fl, order, parents, inv)
        out.append(dv.dvattn_kv_select(mass, first, lengths, 40, 2, 5))
        dv.dvattn_paged_kv_compact(rows, first, kc, vc, bt, mass=cm, lengths=lengths)
        return out + [kc, vc, cm]

    return run


@pytest.mark.parametrize("dtype", DTYPES)
def test_capture_and_streams(dv, gpu, dtype):
    """The same bits from eager calls, another stream and replays of a captured graph."""
    run = everything(dv, gpu, dtype)
    eager = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.clone() for t in run()]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        for t in captured:
            t.zero_()
        again = [t.clone() for t in run()]
        torch.cuda.synchronize()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(eager, again, captured))


def test_pages_beyond_4_gib(dv, gpu):
    """The same bits from pages whose bytes lie past 2^32 of a cache."""
    bs, far = 16, (1 << 20) + 100  # pages of 4 KiB
    big = [torch.empty(far + 300, bs, 1, E, dtype=torch.float16, device=gpu) for _ in range(2)]
    table = lambda bt: torch.where(bt >= 0, bt + far, bt)

    def place(d):
        n = d["k_cache"].shape[0]
        out = dict(d, k_cache=big[0], block_tables=table(d["block_tables"]))
        big[0][far:far + n] = d["k_cache"]
        if "v_cache" in d and "parents" in d:
            big[1][far:far + n] = d["v_cache"]
            out["v_cache"] = big[1]
        return out

    tree = tree_case(torch.float16, 2, 1, 6, [60, 90], bs, 64, seed=41)
    for rows in (0, 2500, 80000):
        d = to(gpu, widened(tree, rows))
        assert torch.equal(dv.dvattn_tree_paged_sdpa(scale=SCALE, **d),
                           dv.dvattn_tree_paged_sdpa(scale=SCALE, **place(d)))
    for S, rows in ((1, 0), (3, 0), (3, 40000)):
        md, mass = mass_case(torch.float16, 2, 1, S, [200], bs, 64, seed=42)
        md = to(gpu, widened(md, rows))
        out = [dv.dvattn_paged_key_mass(mass.to(gpu), scale=SCALE, **x) for x in (md, place(md))]
        assert torch.equal(*out)
    kc, vc, bt, rows, first, lengths, _ = (t.to(gpu) for t in compact_case(torch.float16, 2, 1, 150, 60, bs, seed=43,
                                                                           heads=1))
    n = kc.shape[0]
    big[0][far:far + n], big[1][far:far + n] = kc, vc
    dv.dvattn_paged_kv_compact(rows, first, kc, vc, bt, lengths=lengths)
    dv.dvattn_paged_kv_compact(rows, first, big[0], big[1], table(bt), lengths=lengths)
    assert torch.equal(big[0][far:far + n], kc) and torch.equal(big[1][far:far + n], vc)


def test_drafted_and_bounded_decoding(dv, gpu):
    """The operators together: a cache that collects key mass, is cut to a budget per KV
    head, drafts a tree, attends with it, keeps an accepted path and goes on -- against a
    simulation that holds every KV head's kept keys as plain lists."""
    dt = torch.float32
    g = torch.Generator().manual_seed(31)
    W, Hkv, R, bs, n0, budget = 2, 2, 64, 16, 90, 40
    inv = (1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float()
    maxB = 8
    P = W * maxB
    bt = torch.randperm(P, generator=g).to(torch.int32).reshape(W, maxB).to(gpu)
    kc, vc = torch.zeros(P, bs, Hkv, E, device=gpu), torch.zeros(P, bs, Hkv, E, device=gpu)
    zero = torch.zeros(W, dtype=torch.int32, device=gpu)
    keys = [[[] for _ in range(Hkv)] for _ in range(W)]  # (rotated key, value) of each kept row, float64

    def tables(pos):
        ang = torch.as_tensor(pos, dtype=torch.float32)[..., None] * inv
        ang = torch.cat([ang, ang], -1)
        return torch.cos(ang), torch.sin(ang)

    def append(rows, pos, keep):
        """New tokens in rows ``[W,S]`` at rotary positions ``[W,S]``."""
        S = rows.shape[1]
        k, v = torch.randn(W, Hkv, S, E, generator=g), torch.randn(W, Hkv, S, E, generator=g)
        c, s = tables(pos)
        dv.dvattn_paged_kv_append(k.to(gpu), v.to(gpu), rows.to(gpu), c.to(gpu), s.to(gpu), kc, vc, bt)
        new = [[[(dv.apply_rotary_pos_emb(k[w, h, i][None, None], c[w, i][None], s[w, i][None])[0, 0].double(),
                  v[w, h, i].double()) for i in range(S)] for h in range(Hkv)] for w in range(W)]
        if keep:
            for w in range(W):
                for h in range(Hkv):
                    keys[w][h] += new[w][h]
        return new

    def attend(q, pos, w, h, seen):
        c, s = tables(pos)
        rq = TO.rotate(q, c, s)
        k, v = torch.stack([x[0] for x in seen]), torch.stack([x[1] for x in seen])
        p = torch.softmax(rq @ k.T * SCALE, -1)
        return p @ v, p.sum(0)

    # sum |q_e k_e| * scale < 25: a score is off by (E + 8) 2^-24 * 25 = 2.0e-4 at most, a weight by a
    # factor exp(4.1e-4), an output by that times |v| < 5
    tol = 2.1e-3
    append(torch.arange(n0, dtype=torch.int32).repeat(W, 1), torch.arange(n0).repeat(W, 1), True)
    mass = torch.zeros(W, Hkv, maxB * bs, device=gpu)
    sim_mass = [[torch.zeros(n0, dtype=torch.float64) for _ in range(Hkv)] for _ in range(W)]
    length, position = n0, n0
    for step in range(3):  # decode steps that keep account
        append(torch.full((W, 1), length, dtype=torch.int32), torch.full((W, 1), position), True)
        length += 1
        q = torch.randn(W, 16 * Hkv, 1, E, generator=g) * 2
        c, s = tables(torch.full((1, W, 1), position))
        args = (q.to(gpu), torch.full((1, W, 1), length - 1, dtype=torch.int32, device=gpu), c.to(gpu), s.to(gpu),
                torch.tensor([length], dtype=torch.int32, device=gpu), kc)
        out = dv.dvattn_paged_sdpa(*args, vc, bt, SCALE).cpu().double()
        dv.dvattn_paged_key_mass(mass, *args, bt, SCALE)
        for w in range(W):
            for h in range(Hkv):
                o, p = attend(q[w, 16 * h:16 * h + 16, 0], position, w, h, keys[w][h])
                assert (out[w, 16 * h:16 * h + 16, 0] - o).abs().max() <= tol
                sim_mass[w][h] = torch.cat([sim_mass[w][h], torch.zeros(1, dtype=torch.float64)]) + p
        position += 1
    # cut every KV head's cache to the budget
    lengths = torch.full((W,), length, dtype=torch.int32, device=gpu)
    rows = dv.dvattn_kv_select(mass, zero, lengths, budget, 4, 8)
    dv.dvattn_paged_kv_compact(rows, zero, kc, vc, bt, mass=mass, lengths=lengths)
    for w in range(W):
        for h in range(Hkv):
            r = TO.select(sim_mass[w][h].float()[None, None], [0], [length], budget, 4, 8)[0, 0].tolist()
            assert r == rows[w, h].tolist()
            keys[w][h] = [keys[w][h][i] for i in r]
    assert not mass[:, :, budget:].any()
    length = budget
    # a tree of drafted tokens behind the kept rows
    parents = torch.tensor([[-1, -1, 0, 0, 1, 3, -2], [-1, 0, 1, 1, 0, 3, 5]], dtype=torch.int32)
    S = parents.shape[1]
    depth = torch.tensor([[len(TO.path(parents[w], s) or [0]) - 1 for s in range(S)] for w in range(W)])
    fl = torch.tensor([length + S], dtype=torch.int32, device=gpu)
    order = torch.zeros(W, 1, dtype=torch.int32, device=gpu)
    loc, _, _, views, first = dv.dvattn_tree_metadata(fl, order, parents.to(gpu), inv.to(gpu))
    assert first.tolist() == [length] * W
    # rows count what is kept, positions what was seen
    c, s = tables((position + depth)[None])
    new = append((first.cpu()[:, None] + torch.arange(S, dtype=torch.int32)).to(torch.int32), position + depth, False)
    q = torch.randn(W, 16 * Hkv, S, E, generator=g) * 2
    out = dv.dvattn_tree_paged_sdpa(q.to(gpu), loc, c.to(gpu), s.to(gpu), fl, kc, vc, bt, parents.to(gpu), views, first,
                                    SCALE).cpu().double()
    for w in range(W):
        for n in range(S):
            nodes = TO.path(parents[w], n)
            for h in range(Hkv):
                got = out[w, 16 * h:16 * h + 16, n]
                if nodes is None:
                    assert not got.any()
                    continue
                o, _ = attend(q[w, 16 * h:16 * h + 16, n], position + int(depth[w, n]), w, h,
                              keys[w][h] + [new[w][h][j] for j in nodes])
                assert (got - o).abs().max() <= tol
    # the accepted paths stay
    accepted = [[0, 3, 5], [0, 1, 3]]
    dv.dvattn_paged_kv_compact(torch.tensor(accepted, dtype=torch.int32, device=gpu)[:, None], first, kc, vc, bt)
    for w in range(W):
        for h in range(Hkv):
            keys[w][h] += [new[w][h][j] for j in accepted[w]]
    length, position = length + 3, position + 3
    append(torch.full((W, 1), length, dtype=torch.int32), torch.full((W, 1), position), True)
    length += 1
    q = torch.randn(W, 16 * Hkv, 1, E, generator=g) * 2
    c, s = tables(torch.full((1, W, 1), position))
    out = dv.dvattn_paged_sdpa(q.to(gpu), torch.full((1, W, 1), length - 1, dtype=torch.int32, device=gpu), c.to(gpu),
                               s.to(gpu), torch.tensor([length], dtype=torch.int32, device=gpu), kc, vc, bt,
                               SCALE).cpu().double()
    for w in range(W):
        for h in range(Hkv):
            o, _ = attend(q[w, 16 * h:16 * h + 16, 0], position, w, h, keys[w][h])
            assert (out[w, 16 * h:16 * h + 16, 0] - o).abs().max() <= tol
