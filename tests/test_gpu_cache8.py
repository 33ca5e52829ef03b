"""GPU tests of the operators around 8-bit caches (marked ``gpu``) against their
64-bit restatement in oracle/cache8_oracle.py.

Tables and appended bytes have to be equal.  The attention's tolerances are bounds.  A
float32 score sums E exact products of K and Q (fp32 calls: two of them per element, the
parts of Q, whose last remainder is below 2^-24 of q and 2^-39 of the head's largest; three
are counted), so it is off by at most e =
(m E + 8) * 2^-24 * sum |q_e k_e| * |scale| with m = 3 for fp32 and 1 else, and a softmax
weight by a factor exp(2 e); a sum over n keys adds (m n + 16) * 2^-24.  To that come, times
the sum of weight * |v|: for bf16 the weights' rounding twice (the normaliser sums the
rounded ones), 2^-8 each, and a stored partial result, 2^-10 of the row's largest; for fp16
the weights as two bf16 numbers, 2^-16; for fp32 as three, 2^-24; and the output's own
rounding, 2^-8 (bf16) or 2^-11 (fp16).
"""
import math

import pytest
import torch

from oracle import cache8_oracle as CO
from oracle import tree_cache_oracle as TO

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 128
SCALE = E ** -0.5
CACHE = ("k_cache", "v_cache", "k_scales", "v_scales")


@pytest.fixture(scope="module")
def dv(gpu):
    import dvattention_amd
    return dvattention_amd


def to(dev, d):
    return {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in d.items()}


def pool(g, P, bs, Hkv):
    """Random E4M3 numbers without NaN, exponents that differ from page to page."""
    out = {}
    for n in ("k", "v"):
        x = (torch.randn(P, bs, Hkv, E, generator=g) * 100).clamp(-448, 448)
        out[n + "_cache"] = x.to(torch.float8_e4m3fn)
        out[n + "_scales"] = torch.randint(118, 123, (P, Hkv), generator=g).to(torch.uint8)
    return out


def case(dtype, W, Hkv, S, fl, bs, R, seed, bad=False, causal=False):
    g = torch.Generator().manual_seed(seed)
    F, n = len(fl), sum(fl)
    maxB = max(1, -(-n // bs)) + 1
    P = W * maxB + 2
    bt = torch.randperm(P, generator=g)[:W * maxB].to(torch.int32).reshape(W, maxB)
    if bad:  # pages that do not exist
        bt[0, maxB // 2] = -3
        bt[-1, 0] = P + 1
    loc = torch.empty(F, W, S, dtype=torch.int32)
    for f in range(F):
        loc[f] = torch.randint(-1, max(fl[f], 1) + 3, (W, S), generator=g)
    if causal:
        loc[-1] = fl[-1] - S + torch.arange(S, dtype=torch.int32)
    ang = torch.rand(F, W, S, R, generator=g) * 6.0
    return dict(queries=(torch.randn(W, 16 * Hkv, S, E, generator=g) * 1.5).to(dtype), locations=loc,
                cosines=torch.cos(ang), sines=torch.sin(ang), fragment_lengths=torch.tensor(fl, dtype=torch.int32),
                block_tables=bt, **pool(g, P, bs, Hkv))


def compare(got, dtype, n, want, size, spread):
    m = 3 if dtype == torch.float32 else 1
    e = (m * E + 8) * 2.0 ** -24 * spread + (m * n + 16) * 2.0 ** -24
    tol = size * torch.expm1(2 * e) + 1e-30
    if dtype == torch.bfloat16:
        tol = tol + 2 * 2.0 ** -8 * size + 2.0 ** -10 * size.amax(-1, keepdim=True) + 2.0 ** -8 * want.abs()
    elif dtype == torch.float16:
        tol = tol + 2.0 ** -16 * size + 2.0 ** -11 * want.abs() + 2.0 ** -24
    else:
        tol = tol + 2.0 ** -24 * size
    got = got.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    over = (got.double() - want).abs().nan_to_num(0.0) - tol.nan_to_num(math.inf)
    assert bool((over <= 0).all()), f"largest excess {float(over.max()):.3e}"


def packed(d, W, S, lens):
    """The [W,S] case with lens[w] tokens of each sequence, packed; and what it keeps."""
    at = [(w, s) for w in range(W) for s in range(lens[w])]
    w, s = torch.tensor([x[0] for x in at]), torch.tensor([x[1] for x in at])
    h = d["cosines"].shape[-1] // 2
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    v = dict(queries=d["queries"][w, :, s].contiguous(), locations=d["locations"][:, w, s].contiguous(),
             cosines=d["cosines"][:, w, s, :h].contiguous(), sines=d["sines"][:, w, s, :h].contiguous(),
             cu_seqlens_q=cu, **{k: d[k] for k in CACHE + ("fragment_lengths", "block_tables")})
    return v, w, s


def check(dv, gpu, d, dtype, scale=SCALE):
    """Both forms of the call: the token grid and the packed tokens."""
    want = CO.sdpa(scale, **d)
    n = int(d["fragment_lengths"].clamp(min=0).sum())
    got = dv.dvattn_paged_sdpa_q8(scale=scale, **to(gpu, d))
    compare(got, dtype, n, *want)
    W, _, S, _ = d["queries"].shape
    lens = [S if w % 2 == 0 else max(1, S // 2) for w in range(W)]
    v, w, s = packed(d, W, S, lens)
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=scale, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    compare(out, dtype, n, *(x[w, :, s] for x in want))
    return got


SHAPES = [
    # W, Hkv, S, view lengths, page size, R
    (1, 1, 1, [1], 16, 128),             # one key
    (1, 1, 1, [3001], 16, 128),          # one conversation
    (3, 2, 1, [200], 16, 64),
    (2, 4, 1, [700], 64, 128),           # four waves of a workgroup
    (2, 3, 1, [97], 5, 32),              # a page that ends inside every stage
    (2, 1, 1, [130], 1, 128),            # pages of one row
    (2, 8, 2, [333], 24, 20),            # R/2 no multiple of eight
    (2, 1, 3, [64, 0, 90], 16, 128),     # three views, one of them empty
    (1, 2, 5, [31, 33, 7, 70, 1], 16, 64),
    (1, 1, 1, [40] * 70, 16, 64),        # more views than a wave has lanes
    (2, 2, 16, [150], 16, 0),            # no rotation
    (2, 1, 17, [90, 60], 32, 128),       # a group of one token behind a full one
    (1, 2, 40, [300], 24, 64),
    (90, 1, 1, [50], 16, 64),            # more rows than lanes
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_sdpa(dv, gpu, dtype, shape):
    W, Hkv, S, fl, bs, R = shape
    check(dv, gpu, case(dtype, W, Hkv, S, fl, bs, R, seed=S + len(fl)), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [2, 4, 8, 33])
def test_sdpa_causal(dv, gpu, dtype, S):
    check(dv, gpu, case(dtype, 2, 2, S, [30, 420], 16, 128, seed=S, causal=True), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 6, 20])
def test_sdpa_missing_pages(dv, gpu, dtype, S):
    check(dv, gpu, case(dtype, 3, 2, S, [120, 70], 8, 64, seed=3, bad=True), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_rows_without_keys_and_negative_scale(dv, gpu, dtype):
    d = case(dtype, 2, 2, 4, [50, 30], 16, 64, seed=9)
    d["locations"][:, 0] = -1
    got = check(dv, gpu, d, dtype)
    assert not got[0].any()
    check(dv, gpu, d, dtype, scale=-0.05)
    check(dv, gpu, d, dtype, scale=0.0)
    d["fragment_lengths"][0] = -5  # counts as none; the view behind it starts five rows earlier
    d["locations"][1] = torch.randint(5, 25, (2, 4), dtype=torch.int32)
    d["locations"][0] = 3
    dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_empty_calls(dv, gpu, dtype):
    d = case(dtype, 2, 1, 3, [20], 16, 64, seed=1)
    for name in ("locations", "cosines", "sines", "fragment_lengths"):
        d[name] = d[name][:0].contiguous()
    for bt in (d["block_tables"], d["block_tables"][:, :0].contiguous()):
        out = torch.full((2, 16, 3, E), math.nan, dtype=dtype, device=gpu)
        dv.dvattn_paged_sdpa_q8(scale=SCALE, out=out, **to(gpu, {**d, "block_tables": bt}))
        assert not out.any()
    d = case(dtype, 2, 1, 3, [20], 16, 64, seed=1)
    for name, dim in (("queries", 2), ("locations", 2), ("cosines", 2), ("sines", 2)):
        d[name] = d[name].narrow(dim, 0, 0).contiguous()
    assert dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)).shape == (2, 16, 0, E)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 3, 20])
def test_sdpa_unseen_rows_may_hold_anything(dv, gpu, dtype, S):
    """NaN bytes and exponents of 255 in rows that no token of a sequence sees, in pages
    and behind the last page; NaN in a row that only the later tokens see."""
    d = case(dtype, 2, 2, S, [64, 70], 16, 128, seed=5, causal=True)
    d["locations"][0] = 40
    d["locations"][1] -= 4  # the last four rows of the second view
    kc, vc = d["k_cache"].view(torch.uint8), d["v_cache"].view(torch.uint8)
    bt, P = d["block_tables"], kc.shape[0]
    for w in range(2):
        for row in list(range(41, 64)) + list(range(130, 134)):
            page, r = TO.cache_row(bt, w, row, P, 16)
            kc[page, r], vc[page, r] = 0x7f, 0xff
        page = int(bt[w, 3])  # rows 48 .. 63: unseen as a whole
        d["k_scales"][page], d["v_scales"][page] = 255, 255
    got = check(dv, gpu, d, dtype)
    assert got.isfinite().all()
    # the row of the last token: NaN for it, and for it alone
    page, r = TO.cache_row(bt, 0, 129, P, 16)
    vc[page, r] = 0x7f
    got = check(dv, gpu, d, dtype)
    assert got[0, :, S - 1].isnan().all() and got[1].isfinite().all() and got[0, :, :S - 1].isfinite().all()
    kc[page, r, 1] = 0x7f  # and a NaN key
    got = check(dv, gpu, d, dtype)
    assert got[0, :, :S - 1].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_exponents_of_all_sizes(dv, gpu, dtype):
    """Pages of very different size beside each other: an empty one (0), tiny and large."""
    d = case(dtype, 2, 2, 3, [200], 16, 64, seed=7, causal=True)
    g = torch.Generator().manual_seed(2)
    d["k_scales"] = torch.randint(100, 123, d["k_scales"].shape, generator=g).to(torch.uint8)
    d["v_scales"] = torch.randint(90, 132, d["v_scales"].shape, generator=g).to(torch.uint8)
    for p in d["block_tables"][:, 2].tolist():
        d["k_scales"][p], d["v_scales"][p] = 0, 0
    check(dv, gpu, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_sharp_softmax(dv, gpu, dtype):
    """Scores that rise key by key by more than the running maximum's slack."""
    d = case(dtype, 1, 1, 2, [300], 16, 0, seed=7, causal=True)
    x = torch.linspace(-300, 300, 320).reshape(-1, 16)
    d["k_cache"] = d["k_cache"].clone()
    flat = d["k_cache"].view(torch.uint8)
    for b, page in enumerate(d["block_tables"][0].tolist()[:20]):
        flat[page, :, 0] = (x[b][:, None].expand(16, E)).to(torch.float8_e4m3fn).view(torch.uint8)
    d["k_scales"][:] = 122
    d["queries"] = d["queries"].abs()
    check(dv, gpu, d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S", [1, 4])
def test_sdpa_far_into_a_large_cache(dv, gpu, dtype, S):
    """Rows behind 2^32 bytes of a cache: the same as those rows alone."""
    d = to(gpu, case(dtype, 2, 8, S, [500], 16, 128, seed=4, causal=True))
    want = dv.dvattn_paged_sdpa_q8(scale=SCALE, **d)
    P = (1 << 32) // (16 * 8 * E) + 300
    n = d["k_cache"].shape[0]
    for name in CACHE:
        shape = (P,) + tuple(d[name].shape[1:])
        big = torch.zeros(shape, dtype=torch.uint8, device=gpu)
        big[P - n:] = d[name].view(torch.uint8)
        d[name] = big
    d["block_tables"] = d["block_tables"] + (P - n)
    assert torch.equal(dv.dvattn_paged_sdpa_q8(scale=SCALE, **d), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_agrees_with_the_wide_cache(dv, gpu, dtype):
    """A cache whose elements the 16-bit types hold exactly: the operators without _q8."""
    d = case(dtype, 5, 2, 1, [900], 16, 128, seed=8)
    wide = dict(d)
    for n in ("k", "v"):
        wide[n + "_cache"] = CO.dequantised(d[n + "_cache"], d[n + "_scales"]).to(dtype)
        del wide[n + "_scales"]
    a = dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)).float()
    b = dv.dvattn_paged_sdpa(scale=SCALE, **to(gpu, wide)).float()
    tol = {torch.float32: 2e-5, torch.float16: 2e-3, torch.bfloat16: 2e-2}[dtype]
    assert (a - b).abs().max() <= tol * b.abs().max()


def test_varlen_tokens_behind_the_last_sequence(dv, gpu):
    """Padding tokens see nothing and come out as zeros; a table of many empty sequences."""
    d = case(torch.bfloat16, 2, 1, 3, [80], 16, 64, seed=1, causal=True)
    v, w, s = packed(d, 2, 3, [3, 2])
    pad = 7
    v["queries"] = torch.cat([v["queries"], torch.full((pad, 16, E), math.nan, dtype=torch.bfloat16)])
    v["locations"] = torch.cat([v["locations"], torch.full((1, pad), -1, dtype=torch.int32)], 1)
    v["cosines"] = torch.cat([v["cosines"], torch.full((1, pad, 32), math.nan)], 1)
    v["sines"] = torch.cat([v["sines"], torch.full((1, pad, 32), math.nan)], 1)
    want = [x[w, :, s] for x in CO.sdpa(SCALE, **d)]
    for empty in (0, 100):  # empty sequences between the two
        cu = [0, 3] + [3] * empty + [5]
        x = dict(v, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32),
                 block_tables=torch.cat([d["block_tables"][:1], torch.full((empty, d["block_tables"].shape[1]), -1,
                                                                           dtype=torch.int32), d["block_tables"][1:]]))
        vd = to(gpu, x)
        out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
        compare(out[:5], torch.bfloat16, 80, *want)
        assert not out[5:].any()


def test_sdpa_refusals(dv, gpu):
    d = to(gpu, case(torch.bfloat16, 2, 1, 2, [40], 16, 64, seed=1))
    ok = dv.dvattn_paged_sdpa_q8(scale=SCALE, **d)
    assert torch.equal(ok, dv.dvattn_paged_sdpa_q8(scale=SCALE, **{**d, "k_cache": d["k_cache"].view(torch.uint8),
                                                  "k_scales": d["k_scales"].view(torch.float8_e8m0fnu)}))
    bad = [dict(k_cache=d["k_cache"].float()), dict(v_cache=d["v_cache"].view(torch.float8_e5m2)),
           dict(k_scales=d["k_scales"].float()), dict(k_scales=d["k_scales"][:-1].contiguous()),
           dict(v_scales=d["v_scales"].t()), dict(v_cache=d["v_cache"][:, :8].contiguous()),
           dict(queries=d["queries"][:, :8].contiguous()), dict(locations=d["locations"].long()),
           dict(cosines=d["cosines"].double()), dict(block_tables=d["block_tables"][:1].contiguous()),
           dict(k_cache=d["k_cache"].cpu()), dict(k_cache=d["k_cache"][:, :, :, :64].contiguous())]
    for x in bad:
        with pytest.raises(RuntimeError):
            dv.dvattn_paged_sdpa_q8(scale=SCALE, **{**d, **x})


# ---------------------------------------------------------------------------
# Appends.
def append_case(g, dtype, rope, W, Hkv, S, P, bs, R, size=1.0):
    x = {n: (torch.randn(W, S, Hkv, E, generator=g) * size * torch.exp(torch.randn(W, S, 1, 1, generator=g))).to(dtype)
         for n in ("keys", "values")}
    ang = torch.rand(W, S, R, generator=g) * 6.0
    return dict(keys=x["keys"].transpose(1, 2), values=x["values"].transpose(1, 2), cos=torch.cos(ang).to(rope),
                sin=torch.sin(ang).to(rope), **pool(g, P, bs, Hkv))


def check_append(dv, gpu, d, slots):
    want = CO.append(*(d[n] for n in CACHE), slots, d["keys"], d["values"], d["cos"], d["sin"])
    x = to(gpu, d)
    got = dv.dvattn_paged_kv_append_q8(x["keys"], x["values"], slots.to(gpu), x["cos"], x["sin"],
                                       *(x[n] for n in CACHE))
    for a, b, name in zip(got, want, CACHE):
        a = a.view(torch.uint8).cpu()
        if "cache" in name:  # NaN has two bytes
            a, b = torch.where((a & 0x7f) == 0x7f, 0x7f, a), torch.where((b & 0x7f) == 0x7f, 0x7f, b)
        assert torch.equal(a, b), f"{name}: {int((a != b).sum())} of {a.numel()}"
    return got


@pytest.mark.parametrize("dtype,rope", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                        (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                        (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("W,Hkv,S,bs,R", [(1, 1, 1, 16, 128), (3, 8, 1, 16, 64), (2, 2, 37, 16, 128),
                                          (2, 3, 50, 24, 20), (1, 1, 150, 64, 0), (2, 2, 9, 1, 32),
                                          (1, 2, 600, 16, 128), (1, 12, 700, 5, 64)])
def test_append(dv, gpu, dtype, rope, W, Hkv, S, bs, R):
    """Consecutive tokens from a place inside a page on, one page after the other."""
    g = torch.Generator().manual_seed(S + bs)
    per = -(-S // bs) + 2
    d = append_case(g, dtype, rope, W, Hkv, S, W * per + 3, bs, R)
    bt = torch.randperm(W * per + 3, generator=g)[:W * per].reshape(W, per)
    start = torch.randint(0, bs + 1, (W, 1), generator=g)
    pos = start + torch.arange(S)
    check_append(dv, gpu, d, torch.gather(bt, 1, pos // bs) * bs + pos % bs)


@pytest.mark.parametrize("S", [40, 700])
def test_append_slots_of_any_order(dv, gpu, S):
    """Slots scattered over few pages, many of them named twice or more, some of them out of the
    cache: the last token of a slot is held."""
    g = torch.Generator().manual_seed(S)
    d = append_case(g, torch.bfloat16, torch.bfloat16, 1, 2, S, 6, 16, 64)
    for hi in (96, 300):
        slots = torch.randint(-20, hi, (1, S), generator=g)
        check_append(dv, gpu, d, slots)
    check_append(dv, gpu, d, torch.full((1, S), 37))
    check_append(dv, gpu, d, torch.arange(S)[None].flip(1) % 96)  # backwards
    far = torch.full((1, S), 96)
    far[0, ::2], far[0, 1] = -(1 << 62), (1 << 62)
    got = check_append(dv, gpu, d, far)  # nothing written
    assert torch.equal(got[0].cpu().view(torch.uint8), d["k_cache"].view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_grows_and_starts_anew(dv, gpu, dtype):
    """Token after token of rising and falling size into one page, an element at a time
    outgrowing what the page holds; then its row 0 again."""
    g = torch.Generator().manual_seed(1)
    d = append_case(g, dtype, dtype, 1, 1, 20, 3, 16, 0)
    d["k_scales"][:], d["v_scales"][:] = 0, 0
    d["k_cache"].view(torch.uint8).zero_()
    for i in range(17):
        row = i % 16
        size = 2.0 ** (5 * ((i * 7) % 5) - 12)
        x = {n: (d[n][:, :, i:i + 1] * size).to(dtype) for n in ("keys", "values")}
        got = check_append(dv, gpu, {**d, **x, "cos": d["cos"][:, i:i + 1], "sin": d["sin"][:, i:i + 1]},
                           torch.tensor([[16 + row]]))
        d.update({n: t.cpu() for n, t in zip(CACHE, got)})
    assert int(d["k_scales"][0, 0]) == 0 and int(d["k_scales"][2, 0]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_special_numbers(dv, gpu, dtype):
    """NaN, infinities, the largest and smallest numbers of the type, zeros; a page whose
    exponent is no number."""
    g = torch.Generator().manual_seed(3)
    d = append_case(g, dtype, dtype, 1, 1, 64, 4, 16, 32)
    v = d["values"]
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    v[0, 0, 3, 5], v[0, 0, 3, 9], v[0, 0, 17, 1] = math.nan, math.inf, -math.inf
    v[0, 0, 32:48] *= 0
    v[0, 0, 40, 2], v[0, 0, 41, 3] = small, -small
    v[0, 0, 50, 7], v[0, 0, 51, 8] = big, -big
    d["keys"][0, 0, 5, 40] = math.inf
    d["keys"][0, 0, 20, 1] = math.nan
    slots = (1 + torch.arange(64))[None] % 64
    d["k_scales"][1], d["v_scales"][0] = 255, 254
    check_append(dv, gpu, d, slots)
    check_append(dv, gpu, d, slots[:, :].roll(1, 1))


def test_append_layouts(dv, gpu):
    """Packed tokens, strided heads, off 16-byte alignment, one rotation for all, and tables
    that broadcast."""
    g = torch.Generator().manual_seed(6)
    T, Hkv, bs, R = 45, 2, 16, 64
    d = append_case(g, torch.bfloat16, torch.bfloat16, 1, Hkv, T, 8, bs, R)
    wide = torch.randn(T, Hkv, 2 * E + 1, generator=g).to(torch.bfloat16)
    k, v = wide[..., 1:E + 1], wide[..., E + 1:]
    slots = 3 + torch.arange(T)
    want = CO.append(*(d[n] for n in CACHE), slots[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None], d["cos"],
                     d["sin"])
    x = to(gpu, d)
    w = wide.to(gpu)
    dv.dvattn_paged_kv_append_q8(w[..., 1:E + 1], w[..., E + 1:], slots.to(gpu), x["cos"][0], x["sin"][0],
                                 *(x[n] for n in CACHE))
    for n, b in zip(CACHE, want):
        assert torch.equal(x[n].view(torch.uint8).cpu(), b)
    one = {**d, "cos": d["cos"][:, :1].expand(1, T, R), "sin": d["sin"][:, :1].expand(1, T, R)}
    want = CO.append(*(d[n] for n in CACHE), slots[None], d["keys"], d["values"], one["cos"], one["sin"])
    x = to(gpu, d)
    dv.dvattn_paged_kv_append_q8(x["keys"], x["values"], slots[None].to(gpu), x["cos"][0, 0], x["sin"][0, 0],
                                 *(x[n] for n in CACHE))
    for n, b in zip(CACHE, want):
        assert torch.equal(x[n].view(torch.uint8).cpu(), b)


def test_append_refusals(dv, gpu):
    g = torch.Generator().manual_seed(6)
    d = to(gpu, append_case(g, torch.bfloat16, torch.bfloat16, 1, 2, 5, 4, 16, 64))
    slots = torch.arange(5, device=gpu)[None]

    def call(**kw):
        x = {**d, "slots": slots, **kw}
        dv.dvattn_paged_kv_append_q8(x["keys"], x["values"], x["slots"], x["cos"], x["sin"], *(x[n] for n in CACHE))

    call()
    bad = [dict(slots=slots.int()), dict(slots=slots[:, :3].contiguous()), dict(values=d["values"].float()),
           dict(values=d["values"][:, :1]), dict(cos=d["cos"].half()), dict(sin=d["sin"][..., :32]),
           dict(keys=d["keys"][..., ::2], values=d["values"][..., ::2]), dict(k_cache=d["k_cache"].view(torch.int8)),
           dict(k_cache=d["v_cache"]), dict(k_scales=d["v_scales"]), dict(keys=d["keys"].cpu()),
           dict(k_scales=d["k_scales"][:, :1].contiguous()), dict(k_cache=d["k_cache"][:, :, :1].contiguous())]
    for x in bad:
        with pytest.raises(RuntimeError):
            call(**x)


# ---------------------------------------------------------------------------
# Tables.
def table_case(g, W, width, bs, T, spare, done=0.1, most=40):
    counts = torch.randint(0, width * bs + 1, (W,), generator=g)
    new = torch.randint(0, most + 1, (W,), generator=g)
    new[torch.rand(W, generator=g) < 0.3] = 1
    new[torch.rand(W, generator=g) < done] = -1
    held = -(-counts // bs)
    total = int(held.sum())
    P = total + spare + 3
    names = torch.randperm(P, generator=g)
    bt = torch.full((W, width), -1, dtype=torch.int32)
    at = 0
    for w in range(W):
        bt[w, :held[w]] = names[at:at + held[w]].int()
        at += int(held[w])
    stack = torch.full((P,), -7, dtype=torch.int32)
    stack[:spare] = names[at:at + spare].int()
    return dict(lengths=counts.int(), new_tokens=new.int(), block_tables=bt, free_pages=stack,
                free_count=torch.tensor([spare], dtype=torch.int32), block_size=bs, max_tokens=T)


def check_tables(dv, gpu, d, in_place=False):
    want = CO.tables(d["lengths"], d["new_tokens"], d["block_tables"], d["free_pages"], d["free_count"],
                     d["block_size"], d["max_tokens"])
    x = to(gpu, d)
    got = dv.dvattn_block_tables(in_place=in_place, **x)
    for a, b, name in zip(got, want, ("cu", "starts", "positions", "slots", "lengths", "count")):
        assert a.cpu().tolist() == (b if isinstance(b, list) else [b]), name
    assert torch.equal(x["block_tables"].cpu().long(), torch.from_numpy(want[6]))
    assert x["free_pages"].cpu().tolist() == want[7]
    assert (got[4] is x["lengths"]) == in_place and (got[5] is x["free_count"]) == in_place
    if not in_place:  # the same again: nothing that the call reads has changed
        assert torch.equal(x["lengths"].cpu(), d["lengths"])
        again = dv.dvattn_block_tables(**x)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("W,width,bs,T,spare", [
    (1, 4, 16, 50, 4), (5, 6, 16, 200, 30), (64, 8, 16, 3000, 200), (200, 20, 24, 9000, 900),
    (64, 8, 16, 500, 200),     # packed tokens run out
    (100, 10, 4, 5000, 60),    # pages run out
    (37, 3, 1, 100, 5), (1500, 3, 16, 40000, 4000), (8192, 1, 16, 70000, 9000),
])
def test_tables(dv, gpu, W, width, bs, T, spare, in_place):
    check_tables(dv, gpu, table_case(torch.Generator().manual_seed(W), W, width, bs, T, spare), in_place)


def test_tables_edges(dv, gpu):
    g = torch.Generator().manual_seed(3)
    d = table_case(g, 30, 5, 16, 400, 40)
    for kw in (dict(free_count=torch.tensor([0], dtype=torch.int32)),
               dict(free_count=torch.tensor([-4], dtype=torch.int32)),
               dict(free_count=torch.tensor([1 << 30], dtype=torch.int32)),
               dict(new_tokens=torch.full((30,), -1, dtype=torch.int32)),   # all end
               dict(new_tokens=torch.zeros(30, dtype=torch.int32)),
               dict(new_tokens=torch.full((30,), 2 ** 31 - 1, dtype=torch.int32)),
               dict(lengths=torch.full((30,), -3, dtype=torch.int32)),
               dict(lengths=torch.full((30,), 2 ** 31 - 1, dtype=torch.int32)),
               dict(max_tokens=0), dict(max_tokens=1), dict(max_tokens=5000)):
        check_tables(dv, gpu, {**d, **kw})
    none = dict(lengths=torch.empty(0, dtype=torch.int32), new_tokens=torch.empty(0, dtype=torch.int32),
                block_tables=torch.empty(0, 4, dtype=torch.int32), free_pages=d["free_pages"],
                free_count=d["free_count"], block_size=16, max_tokens=3)
    check_tables(dv, gpu, none)
    check_tables(dv, gpu, {**none, "max_tokens": 5000})


def test_tables_refusals(dv, gpu):
    d = to(gpu, table_case(torch.Generator().manual_seed(1), 4, 5, 16, 100, 40))
    shared = torch.zeros(200, dtype=torch.int32, device=gpu)
    for kw in (dict(lengths=d["lengths"].long()), dict(new_tokens=d["new_tokens"][:3].contiguous()),
               dict(block_tables=d["block_tables"][:2].contiguous()), dict(free_count=d["free_count"].expand(2)),
               dict(block_size=0), dict(max_tokens=-1), dict(free_pages=d["free_pages"].cpu()),
               dict(block_tables=shared[:20].view(4, 5), free_pages=shared[10:90])):
        with pytest.raises(RuntimeError):
            dv.dvattn_block_tables(**{**d, **kw})


# ---------------------------------------------------------------------------
# Together: a server's steps.
def serve(dv, gpu, steps, dtype, Hkv=2, bs=16, R=64, seed=0):
    """Steps of six sequences (prompts, decodes, one that ends and starts anew) through
    tables, append and attention; the outputs and the last state."""
    g = torch.Generator().manual_seed(seed)
    W, width, P, T = 6, 12, 60, 90
    st = dict(lengths=torch.zeros(W, dtype=torch.int32, device=gpu), free_count=torch.tensor([P], dtype=torch.int32,
              device=gpu), block_tables=torch.full((W, width), -1, dtype=torch.int32, device=gpu),
              free_pages=torch.randperm(P, generator=g).int().to(gpu))
    cache = [torch.zeros(P, bs, Hkv, E, dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)] + \
            [torch.zeros(P, Hkv, dtype=torch.float8_e8m0fnu if i else torch.uint8, device=gpu) for i in range(2)]
    cache[3].view(torch.uint8).zero_()
    fl = torch.tensor([width * bs], dtype=torch.int32, device=gpu)
    history = []
    for step in range(steps):
        new = torch.tensor([1, 1, 17, 1, 0, 3] if step else [40, 9, 1, 16, 5, 0], dtype=torch.int32)
        if step % 4 == 3:
            new[step // 4 % W] = -1
        cu, starts, pos, slots, st["lengths"], st["free_count"] = dv.dvattn_block_tables(
            st["lengths"], new.to(gpu), st["block_tables"], st["free_pages"], st["free_count"], bs, T)
        kv = torch.randn(T, 2 * Hkv, E, generator=g).to(dtype).to(gpu)
        q = torch.randn(T, 16 * Hkv, E, generator=g).to(dtype).to(gpu)
        ang = pos[:, None].float() * (1e4 ** (-torch.arange(R // 2, device=gpu) / (R // 2)))
        cos, sin = torch.cos(ang), torch.sin(ang)
        dv.dvattn_paged_kv_append_q8(kv[:, :Hkv], kv[:, Hkv:], slots, torch.cat([cos, cos], -1),
                                     torch.cat([sin, sin], -1), *cache)
        out = dv.dvattn_varlen_paged_sdpa_q8(q, pos[None], cos[None], sin[None], fl, *cache, st["block_tables"], cu,
                                             cu, SCALE)
        history.append(dict(new=new, pos=pos, slots=slots, cu=cu, out=out, q=q, kv=kv, cos=cos, sin=sin,
                            bt=st["block_tables"].clone(), cache=[c.clone() for c in cache]))
    return history, st, cache, fl


@pytest.mark.parametrize("dtype", DTYPES)
def test_serving_steps(dv, gpu, dtype):
    """Each step against the oracle on the caches it read, and the caches against the tokens
    that went in: within E4M3's rounding (twice where a page's scale grew)."""
    history, st, cache, fl = serve(dv, gpu, 7, dtype)
    seen = {}
    for step, h in enumerate(history):
        n = int(h["cu"][-1])
        if step in (0, 3, 6):
            c = [x.cpu() for x in h["cache"]]
            want = CO.varlen_sdpa(SCALE, h["pos"][None, :n].cpu(), h["q"][:n].cpu(), h["cos"][None, :n].cpu(),
                                  h["sin"][None, :n].cpu(), fl.cpu(), *c, h["bt"].cpu(), h["cu"].cpu())
            compare(h["out"][:n], dtype, 192, *want)
        assert not h["out"][n:].any() and (h["slots"][n:] == -1).all()
        for t in range(n):
            if int(h["slots"][t]) >= 0:
                seen[int(h["slots"][t])] = h["kv"][t, 2:].double().cpu()
    v = CO.dequantised(cache[1].cpu(), cache[3].cpu()).flatten(0, 1)
    live = {int(p) * 16 + r for w in range(6) for i in range(int(st["lengths"][w])) for p, r in
            [(st["block_tables"][w, i // 16], i % 16)]}
    assert live <= set(seen)
    unit = torch.exp2(cache[3].view(torch.uint8).cpu().double() - 127)
    for s in live:
        # half a step of E4M3 each time it was rounded: relative 2^-4, at least 2^-10 of the unit
        assert ((v[s] - seen[s]).abs() <= 2 * (2.0 ** -4 * seen[s].abs() + 2.0 ** -10 * unit[s // 16][:, None])).all()


def test_serving_is_deterministic_on_another_stream(dv, gpu):
    a, _, _, _ = serve(dv, gpu, 4, torch.bfloat16)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        b, _, _, _ = serve(dv, gpu, 4, torch.bfloat16)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x["out"], y["out"]) and all(torch.equal(i.view(torch.uint8), j.view(torch.uint8))
                                                       for i, j in zip(x["cache"], y["cache"]))


def test_serving_step_in_a_graph(dv, gpu):
    """A decode step captured with its state in place and replayed, eager work and
    synchronizations in between: every replay is the eager step."""
    W, Hkv, bs, R, width, P = 4, 2, 16, 64, 6, 30
    g = torch.Generator().manual_seed(0)
    inputs = [(torch.randn(W, 2 * Hkv, E, generator=g).bfloat16().to(gpu),
               torch.randn(W, 16 * Hkv, E, generator=g).bfloat16().to(gpu)) for _ in range(40)]
    pages = torch.randperm(P, generator=g).int().to(gpu)

    def fresh():
        return dict(lengths=torch.tensor([0, 15, 3, 30], dtype=torch.int32, device=gpu),
                    count=torch.tensor([P - 5], dtype=torch.int32, device=gpu),
                    bt=torch.tensor([[-1] * 6, [pages[-1]] + [-1] * 5, [pages[-2]] + [-1] * 5,
                                     [pages[-3], pages[-4]] + [-1] * 4], dtype=torch.int32, device=gpu),
                    stack=pages.clone(), kc=torch.zeros(P, bs, Hkv, E, dtype=torch.uint8, device=gpu),
                    vc=torch.zeros(P, bs, Hkv, E, dtype=torch.uint8, device=gpu),
                    ks=torch.zeros(P, Hkv, dtype=torch.uint8, device=gpu),
                    vs=torch.zeros(P, Hkv, dtype=torch.uint8, device=gpu), kv=inputs[0][0].clone(),
                    q=inputs[0][1].clone())

    new = torch.ones(W, dtype=torch.int32, device=gpu)
    fl = torch.tensor([width * bs], dtype=torch.int32, device=gpu)
    freq = 1e4 ** (-torch.arange(R // 2, device=gpu) / (R // 2))

    def step(s):
        cu, _, pos, slots, _, _ = dv.dvattn_block_tables(s["lengths"], new, s["bt"], s["stack"], s["count"], bs, W,
                                                         in_place=True)
        ang = pos[:, None].float() * freq
        cos, sin = torch.cos(ang), torch.sin(ang)
        dv.dvattn_paged_kv_append_q8(s["kv"][:, :Hkv], s["kv"][:, Hkv:], slots, torch.cat([cos, cos], -1),
                                     torch.cat([sin, sin], -1), s["kc"], s["vc"], s["ks"], s["vs"])
        return dv.dvattn_varlen_paged_sdpa_q8(s["q"], pos[None], cos[None], sin[None], fl, s["kc"], s["vc"], s["ks"],
                                              s["vs"], s["bt"], cu, cu, SCALE)

    eager, warm, s = fresh(), fresh(), fresh()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(s)
    for i in range(40):
        for x in (eager, s):
            x["kv"].copy_(inputs[i][0])
            x["q"].copy_(inputs[i][1])
        want = step(eager)
        graph.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for name in ("lengths", "count", "bt", "kc", "vc", "ks", "vs"):
            assert torch.equal(s[name], eager[name]), (i, name)
    assert s["lengths"].tolist() == [40, 55, 43, 70]


def test_capi_matches_and_keeps_to_its_workspace(gpu):
    """The C entries through ctypes, with a workspace of just the queried size between
    guards that stay untouched."""
    import ctypes

    from dvattention_amd import capi
    for S in (1, 5, 40):
        d = to(gpu, case(torch.bfloat16, 3, 4, S, [2000], 16, 128, seed=S, causal=True))
        s = capi.paged_shape(d["queries"], d["locations"], d["cosines"], d["k_cache"], d["v_cache"],
                             d["block_tables"])
        need = capi.lib().dvattn_paged_sdpa_q8_workspace_size(2, ctypes.byref(s), 0)
        buf = torch.full((need + 512,), 0xa5, dtype=torch.uint8, device=gpu)
        out = torch.empty_like(d["queries"])
        ws = buf[256:256 + need]
        assert ws.numel() == need
        capi.paged_sdpa_q8(out, SCALE, workspace=ws, **d)
        assert buf[:256].eq(0xa5).all() and buf[256 + need:].eq(0xa5).all()
        import dvattention_amd as dv
        assert torch.equal(out, dv.dvattn_paged_sdpa_q8(scale=SCALE, **d))
