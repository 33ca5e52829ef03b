"""GPU tests of what bytes and exponents of an 8-bit cache stand for (marked ``gpu``):
exponents that are no number, empty pages, the largest and smallest ones, views that begin at
negative positions.  Oracle and tolerances: test_gpu_cache8.py.
"""
import math

import pytest
import torch

from oracle import cache8_oracle as CO
from test_gpu_cache8 import (CACHE, DTYPES, SCALE, append_case, case, check, check_append, compare, dv,  # noqa: F401
                             packed, to)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 4, 7, 20])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_sdpa_exponent_that_is_no_number(dv, gpu, dtype, S, which):  # noqa: F811
    """Causal rows; from the last token on, or the last but one, row 0 of a page whose exponent
    is 255 is seen.  Its bytes are large, small, of both signs and zero; all its elements are
    NaN for the tokens that see it and nothing to the others."""
    n = 129 if S == 1 else 130  # rows 128 ..: page 8
    d = case(dtype, 2, 2, S, [n], 16, 128, seed=S, causal=True)
    page = int(d["block_tables"][1, 8])
    d["k_cache"].view(torch.uint8)[page, 0, 0] = 0
    d["v_cache"].view(torch.uint8)[page, 0, 1, ::2] = 0
    for x in which:
        d[x + "_scales"][page] = 255
    got = check(dv, gpu, d, dtype)
    seen = 1 if S == 1 else 2
    assert got[1, :, S - seen:].isnan().all() and got[0].isfinite().all() and got[1, :, :S - seen].isfinite().all()
    d["locations"][0, 1] += 1 - seen  # the last token alone sees it
    if S > 1:
        got = check(dv, gpu, d, dtype)
        assert got[1, :, S - 1].isnan().all() and got[1, :, :S - 1].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 4, 20])
def test_sdpa_exponent_that_is_no_number_in_a_heads_low_scores(dv, gpu, dtype, S):  # noqa: F811
    """Keys whose bytes would make every score of a head very small are NaN all the same."""
    d = case(dtype, 1, 1, S, [40], 16, 0, seed=S)
    d["locations"][:] = 39
    page = int(d["block_tables"][0, 1])
    d["queries"] = d["queries"].abs()
    d["k_cache"].view(torch.uint8)[page] = 0xb8  # -1
    d["k_scales"][page] = 255
    assert check(dv, gpu, d, dtype).isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 4, 7, 20])
@pytest.mark.parametrize("bs", [16, 24])
def test_sdpa_empty_page_of_any_bytes(dv, gpu, dtype, S, bs):  # noqa: F811
    """Exponent 0: the page's elements count as zeros whatever its bytes are, NaN among them."""
    d = case(dtype, 2, 2, S, [70, 90], bs, 64, seed=S, causal=True)
    d["locations"][0] = 60
    plain = {n: d[n].clone() for n in CACHE}
    for w in range(2):
        for b in (1, 4):
            page = int(d["block_tables"][w, b])
            d["k_scales"][page, w], d["v_scales"][page, 1] = 0, 0
            d["k_cache"].view(torch.uint8)[page, :, w, 3::5] = 0x7f
            d["v_cache"].view(torch.uint8)[page, :, 1, ::3] = 0xff
            plain["k_cache"].view(torch.uint8)[page, :, w], plain["v_cache"].view(torch.uint8)[page, :, 1] = 0, 0
    want = CO.sdpa(SCALE, **{**d, **plain})
    assert want[0].isfinite().all()
    compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, 160, *want)
    v, w, s = packed(d, 2, S, [S, max(1, S // 2)])
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    compare(out, dtype, 160, *(x[w, :, s] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 4, 7, 20])
@pytest.mark.parametrize("bs", [1, 16, 24])
@pytest.mark.parametrize("neg,n", [(5, 40), (32, 200), (70, 64), (37, 150)])
def test_sdpa_view_at_a_negative_position(dv, gpu, dtype, S, bs, neg, n):  # noqa: F811
    """A negative length counts as no keys; the rows of the next view that it puts at negative
    positions are absent, the others are not."""
    d = case(dtype, 2, 2, S, [0, n], bs, 64, seed=S + neg, causal=True)
    d["locations"][0] = 3
    d["fragment_lengths"][0] = -neg
    want = CO.sdpa(SCALE, **d)
    if n <= neg:
        assert not want[0].any()
    compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, n, *want)
    v, w, s = packed(d, 2, S, [S, max(1, S // 2)])
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    compare(out, dtype, n, *(x[w, :, s] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 4, 20])
def test_sdpa_view_far_before_all_positions(dv, gpu, dtype, S):  # noqa: F811
    """Negative lengths that add up to -2^32: the view behind them has no rows, wherever its
    positions lie modulo 2^32."""
    d = case(dtype, 2, 1, S, [40, 0, 0, 40], 16, 64, seed=S)
    d["locations"][0], d["locations"][3] = 30, 39
    d["fragment_lengths"][0] = 40
    d["fragment_lengths"][1:3] = -2 ** 31
    want = CO.sdpa(SCALE, **d)
    alone = CO.sdpa(SCALE, **{**d, "fragment_lengths": torch.tensor([40, 0, 0, 0], dtype=torch.int32)})
    assert torch.equal(want[0], alone[0])
    compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, 40, *want)
    v, w, s = packed(d, 2, S, [S, max(1, S // 2)])
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    compare(out, dtype, 40, *(x[w, :, s] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("old", [0, 1, 5, 250, 253, 254])
@pytest.mark.parametrize("Hkv,T,bs,R", [(1, 1, 16, 0), (2, 1, 16, 32), (5, 9, 16, 0), (2, 40, 48, 64), (1, 9, 16, 20)])
def test_append_under_every_exponent(dv, gpu, dtype, old, Hkv, T, bs, R):  # noqa: F811
    """Rows behind row 0 of a page whose exponent is the largest or the smallest there is, of
    the type's largest and smallest numbers and ordinary ones; what an empty page (0) holds
    counts as zeros."""
    g = torch.Generator().manual_seed(old + T)
    for size in (1.0, 2.0 ** -120 if dtype != torch.float16 else 2.0 ** -13, float(torch.finfo(dtype).max) / 2.0 ** 7):
        d = append_case(g, dtype, dtype, 1, Hkv, T, 3, bs, R)
        for x in ("keys", "values"):
            d[x] = (d[x].double().clamp(-60, 60) * size).to(dtype)
        d["k_scales"][:], d["v_scales"][:] = old, old
        if old == 0:
            for x in ("k_cache", "v_cache"):
                d[x].view(torch.uint8)[1, :, 0, 5] = 0x7f
        check_append(dv, gpu, d, bs + 3 + torch.arange(T)[None])


def test_append_exponents_from_finite_numbers(dv, gpu):  # noqa: F811
    """Infinities and NaN beside ordinary numbers leave the page's exponent to those."""
    g = torch.Generator().manual_seed(2)
    for dtype in DTYPES:
        d = append_case(g, dtype, dtype, 1, 2, 30, 3, 16, 0)
        for t, x in ((2, math.inf), (3, math.nan), (20, -math.inf)):
            d["keys"][0, 0, t, 7], d["values"][0, 1, t, 9] = x, x
        got = check_append(dv, gpu, d, 16 + torch.arange(30)[None])
        assert got[2].view(torch.uint8)[1:].max() < 140
