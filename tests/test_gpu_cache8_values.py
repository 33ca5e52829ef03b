"""GPU tests of what bytes and exponents of an 8-bit cache stand for (marked ``gpu``):
exponents that are no number, empty pages, the largest and smallest ones, views that begin at
negative positions.  Oracle and tolerances: test_gpu_cache8.py.
"""
import pytest
import torch

from oracle import cache8_oracle as CO
from test_gpu_cache8 import (CACHE, DTYPES, SCALE, case, check, compare, dv,  # noqa: F401
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
