"""GPU tests of the tree and bounded-cache operators at the sizes that choose the
less common ways through their kernels (marked ``gpu``): one token's key mass with
several units of keys per wave, lists of more rows than a block's registers hold, one
node per sequence through the multi-query kernel, many views, and every key's weight
read off the output.  Oracles and tolerances: test_gpu_tree_cache."""
import math

import pytest
import torch

from test_gpu_tree_cache import (DTYPES, E, SCALE, check_mass, check_tree, compare_tree, dv, mass_case,  # noqa: F401
                                 run_select, to, tree_case, widened)
from oracle import tree_cache_oracle as TO

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Key mass of one token: two and four units of 64 keys (fp32: 32) per wave from 2^20
# and 2^21 (fp32: 2^19 and 2^20) rows of block tables on.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("units", [2, 4])
@pytest.mark.parametrize("fl,bs,bad", [
    ([2050], 16, False),             # whole units and a ragged end
    ([700, 450, 900, 3], 16, True),  # views that meet inside a wave's later units; missing pages
    ([100] * 9 + [0, 61], 24, False),
])
def test_key_mass_several_units(dv, gpu, dtype, units, fl, bs, bad):  # noqa: F811
    d, mass = mass_case(dtype, 2, 2, 1, fl, bs, 64, seed=len(fl), bad=bad)
    d["locations"][0, 0] = 10 ** 6  # one sequence sees a whole view
    narrow = check_mass(dv, gpu, d, mass, 0.75)
    rows = units * (1 << 17) // (2 if dtype == torch.float32 else 1)
    wide = widened(d, -(-rows // bs) * bs)
    again = check_mass(dv, gpu, wide, mass, 0.75)
    assert (narrow - again).abs().max() <= 1e-4
    assert torch.equal(again, check_mass(dv, gpu, wide, mass, 0.75, in_place=True))
    check_mass(dv, gpu, wide, mass, 0.0, scale=-SCALE)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S,rows", [(1, 0), (4, 0), (4, 60000)])
def test_key_mass_many_views(dv, gpu, dtype, S, rows):  # noqa: F811
    """Seventeen short views, empty ones among them, for each way through the kernels."""
    fl = [33, 0, 70, 15, 16, 17, 1, 64, 0, 40, 90, 5, 31, 32, 48, 60, 7]
    d, mass = mass_case(dtype, 2, 1, S, fl, 16, 64, seed=S)
    d["locations"][5:9, 1] = -1
    check_mass(dv, gpu, widened(d, rows), mass, 0.5)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fl", [[1], [90], [30, 0, 50, 7]])
def test_tree_sdpa_one_node(dv, gpu, dtype, fl):  # noqa: F811
    """One node per sequence under a table so wide that the multi-query kernel takes it."""
    d = tree_case(dtype, 3, 2, 1, fl, 16, 64, seed=7, absent=0.0)
    want, size, spread = TO.tree_sdpa(SCALE, **d)
    got = dv.dvattn_tree_paged_sdpa(scale=SCALE, **to(gpu, widened(d, 1 << 20))).cpu()
    compare_tree(got, d, dtype, want, size, spread)
    d["parents"][1] = -2
    out = dv.dvattn_tree_paged_sdpa(scale=SCALE, **to(gpu, widened(d, 1 << 20))).cpu()
    assert not out[1].any() and torch.equal(out[0], got[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [5, 17])
@pytest.mark.parametrize("S", [1, 6, 20])
def test_tree_sdpa_many_views(dv, gpu, dtype, F, S):  # noqa: F811
    """More views than the short-list kernel holds the queries of."""
    fl = [S + 3 + 7 * (f % 4) if f % 5 else 2 * S for f in range(F)]
    check_tree(dv, gpu, tree_case(dtype, 2, 1, S, fl, 16, 64, seed=F + S), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S,fl", [(9, [120]), (20, [60, 40]), (1, [100])])
def test_tree_sdpa_weight_of_every_key(dv, gpu, dtype, S, fl):  # noqa: F811
    """The value of stream row l is the l-th unit vector, so an output's elements are its
    keys' weights: in float32 each is held to its own size, however small, and a key lost
    or counted twice is off by all of it."""
    d = tree_case(dtype, 2, 2, S, fl, 16, 64, seed=S)
    P, bs = d["k_cache"].shape[:2]
    d["v_cache"].zero_()
    for w in range(2):
        for pos in range(sum(fl)):
            page, row = TO.cache_row(d["block_tables"], w, pos, P, bs)
            d["v_cache"][page, row, :, pos] = 1.0
    got, want = check_tree(dv, gpu, d, dtype)
    if dtype == torch.float32:
        assert torch.equal(got != 0, want != 0)
    sums = got.double().sum(-1)
    assert ((sums - (want.sum(-1) > 0).double()).abs() <= 2.0 ** -6).all()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("m", [32767, 32768, 32769, 40001, 70000])
@pytest.mark.parametrize("kind", ["wide", "narrow", "few", "special"])
def test_select_long_lists(dv, gpu, m, kind):  # noqa: F811
    """Up to and past the 32768 competing rows that a block's registers hold: weights of
    many sizes (few share the deciding digit), of one size (more than the short list
    holds do), few distinct ones, and specials."""
    g = torch.Generator().manual_seed(m)
    kf, kl, first = 3, 21, 1000
    n = m + kf + kl
    if kind == "wide":
        mass = torch.exp(3 * torch.randn(2, 1, first + n + 17, generator=g))
    elif kind == "narrow":
        mass = 1.0 + torch.rand(2, 1, first + n + 17, generator=g) * 2.0 ** -5
    elif kind == "few":
        mass = torch.randint(0, 3, (2, 1, first + n + 17), generator=g).float()
    else:
        mass = torch.tensor([math.nan, math.inf, -math.inf, -1.0, 0.0, -0.0, 1e-42, 7.0])[
            torch.randint(0, 8, (2, 1, first + n + 17), generator=g)]
    for budget in (kf + kl + 1, n // 4, n - 1):
        run_select(dv, gpu, mass, [0, first], [n, n], budget, kf, kl)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 5, 17])
@pytest.mark.parametrize("what", ["nan key", "inf key", "nan query", "every key"])
def test_tree_sdpa_nan_reaches_the_output(dv, gpu, dtype, S, what):  # noqa: F811
    """A NaN score among the committed keys makes a node's output NaN, whichever piece of
    the keys it is in and whatever the others hold; heads whose query turns an infinite
    key to -infinity only lose that key."""
    fl = [1500]
    d = tree_case(dtype, 2, 1, S, fl, 16, 64, seed=S, absent=0.0)
    d["parents"][:] = -1  # (the drafted rows alone would hide a lost piece)
    P, bs = d["k_cache"].shape[:2]
    if what == "nan query":
        d["queries"][0, 3] = math.nan
    elif what == "every key":
        for pos in range(1500 - S - 1):
            page, row = TO.cache_row(d["block_tables"], 0, pos, P, bs)
            d["k_cache"][page, row] = math.nan
    else:
        page, row = TO.cache_row(d["block_tables"], 0, 700, P, bs)
        if what == "nan key":
            d["k_cache"][page, row] = math.nan
        else:
            d["k_cache"][page, row, :, 100] = math.inf  # (a dim that is not rotated)
    want, size, spread = TO.tree_sdpa(SCALE, **d)
    spread = spread.nan_to_num(0.0, posinf=0.0).clamp(max=1e6)
    if what == "inf key":  # e as without the key: its weight is 0 where the row is finite
        spread = TO.tree_sdpa(SCALE, **{**d, "k_cache": d["k_cache"].clamp(max=100.0)})[2]
    assert want[0].isnan().any() and not want[1].isnan().any()
    for rows in (0, 2500, 80000, 1 << 20):
        got = dv.dvattn_tree_paged_sdpa(scale=SCALE, **to(gpu, widened(d, rows))).cpu()
        assert torch.equal(got.isnan(), want.isnan()), f"table of {rows} rows"
        compare_tree(got, d, dtype, want, size, spread)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S,rows", [(1, 0), (1, 1 << 18), (3, 0), (3, 60000), (70, 0)])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_key_mass_of_nan_and_infinite_keys(dv, gpu, dtype, S, rows, what):  # noqa: F811
    """A NaN score makes every weight of its (token, head) NaN, an infinite key does so for
    the heads that score it +infinity and weighs nothing for the others; other sequences
    and rows past what is seen keep their own."""
    d, mass = mass_case(dtype, 2, 1, S, [300], 16, 64, seed=S)
    d["locations"][0, 0] = 250
    page, row = TO.cache_row(d["block_tables"], 0, 100, d["k_cache"].shape[0], 16)
    d["k_cache"][page, row, :, 100] = what
    want, _ = TO.key_mass(mass, 0.5, SCALE, **d)
    assert want[0, 0, :251].isnan().all() and want[0, 0, 251:].isfinite().all() and want[1].isfinite().all()
    got = dv.dvattn_paged_key_mass(mass.to(gpu), scale=SCALE, decay=0.5, **to(gpu, widened(d, rows))).cpu()
    assert torch.equal(got.isnan(), want.isnan())
    check_mass(dv, gpu, widened({**d, "locations": d["locations"].clamp(max=99)}, rows), mass, 0.5)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_ctypes_entries(dv, gpu, dtype):  # noqa: F811
    """The C entries through dvattention_amd.capi give the operators' bits, with a workspace
    of the caller's and without."""
    from dvattention_amd import capi
    from test_gpu_tree_cache import compact_case, meta_inputs

    names = ("locations", "queries", "cosines", "sines", "fragment_lengths", "k_cache", "v_cache", "block_tables",
             "parents", "tree_views", "tree_rows")
    for rows in (0, 2500, 80000):
        d = to(gpu, widened(tree_case(dtype, 2, 2, 6, [60, 90], 16, 64, seed=2), rows))
        want = dv.dvattn_tree_paged_sdpa(scale=SCALE, **d)
        for ws in (None, torch.empty(64 << 20, dtype=torch.uint8, device=gpu)):
            out = torch.full_like(want, math.nan)
            assert torch.equal(capi.tree_paged_sdpa(out, SCALE, *(d[n] for n in names), workspace=ws), want)
    for S in (1, 3):
        d, mass = mass_case(dtype, 2, 2, S, [90, 40], 16, 64, seed=2)
        d, mass = to(gpu, d), mass.to(gpu)
        want = dv.dvattn_paged_key_mass(mass, scale=SCALE, decay=0.5, out=torch.empty_like(mass), **d)
        out = capi.paged_key_mass(torch.empty_like(mass), mass, 0.5, SCALE, *(d[n] for n in names[:6]), d["block_tables"])
        assert torch.equal(out, want)
    kc, vc, bt, rows, first, lengths, mass = (t.to(gpu) for t in compact_case(dtype, 2, 2, 150, 60, 16, seed=3))
    want = dv.dvattn_kv_select(mass, first, lengths, 40, 2, 5)
    assert torch.equal(capi.kv_select(torch.empty_like(want), mass, first, lengths, 2, 5), want)
    a, b = [t.clone() for t in (kc, vc, mass)], [t.clone() for t in (kc, vc, mass)]
    dv.dvattn_paged_kv_compact(rows, first, a[0], a[1], bt, mass=a[2], lengths=lengths)
    capi.kv_compact(b[0], b[1], bt, rows, first, lengths=lengths, mass=b[2])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    fl, order, parents, inv = (t.to(gpu) for t in meta_inputs(2, 3, 9, 64, seed=4))
    counts = torch.arange(6, dtype=torch.int32, device=gpu).view(2, 3)
    for kw in ({}, dict(committed=counts * 11, dropped=counts)):
        want = dv.dvattn_tree_metadata(fl, order, parents, inv, 1.5, torch.bfloat16, **kw)
        got = capi.tree_metadata(*(torch.empty_like(t) for t in want), fl, order, parents, inv, 1.5, torch.bfloat16,
                                 **kw)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
