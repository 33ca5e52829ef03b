"""Scores far above 2^31, finite as floats (marked ``gpu``): each row of attention is the row
of V under its largest visible score, exactly, and a key's mass the number of queries whose
largest it is.

Every key is one number c repeated, no two alike, and every query one number, positive or
negative, so that a score is c times a number of the query, exactly up to one rounding of the
scaled score; two scores differ by a sixteenth at least.  The keys are E4M3 numbers, held in
all types.
"""
import pytest
import torch

from test_gpu_parity import dv  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E, Hkv, N, BS = 128, 2, 200, 16


def numbers():
    """200 E4M3 numbers, no two alike, in an order that goes up and down."""
    x = torch.arange(1, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    x = torch.cat([x[-N // 2:], -x[-N // 2:]])
    return x[torch.randperm(N, generator=torch.Generator().manual_seed(5))]


def make(dtype, W, S, up, seed):
    """Queries of 2^up and scores of up to 2^(up + 16), one view whose rows rise causally."""
    g = torch.Generator().manual_seed(seed)
    c = numbers()
    maxB = -(-N // BS)
    P = W * maxB + 2
    bt = torch.randperm(P, generator=g)[:W * maxB].to(torch.int32).reshape(W, maxB)
    k = torch.zeros(P, BS, Hkv, E)
    v = (torch.randn(P, BS, Hkv, E, generator=g) * 8).to(torch.float8_e4m3fn).float()
    at = torch.arange(N)
    for w in range(W):
        k[bt[w].long()[at // BS], at % BS] = c[:, None, None].expand(N, Hkv, E)
    sign = torch.randint(0, 2, (W, 16 * Hkv, S, 1), generator=g) * 2 - 1
    q = (sign * 2.0 ** up).float().expand(W, 16 * Hkv, S, E)
    loc = torch.randint(0, N, (W, 1), generator=g) + torch.arange(S)
    loc[0] = N - S + torch.arange(S)
    loc = loc.clamp(max=N - 1).to(torch.int32)[None]
    best = torch.empty(W, 16 * Hkv, S, dtype=torch.long)  # row of the largest score
    for w in range(W):
        for s in range(S):
            seen = c[:int(loc[0, w, s]) + 1]
            best[w, :, s] = torch.where(sign[w, :, s, 0] > 0, seen.argmax(), seen.argmin())
    want = torch.empty(W, 16 * Hkv, S, E)
    for w in range(W):
        for h in range(16 * Hkv):
            want[w, h] = v[bt[w].long()[best[w, h] // BS], best[w, h] % BS, h // 16]
    d = dict(queries=q.to(dtype).contiguous(), locations=loc.contiguous(), cosines=torch.zeros(1, W, S, 0),
             sines=torch.zeros(1, W, S, 0), fragment_lengths=torch.tensor([N], dtype=torch.int32),
             k_cache=k.to(dtype), v_cache=v.to(dtype), block_tables=bt)
    return d, want.to(dtype), best


def to(dev, d):
    return {n: t.to(dev) for n, t in d.items()}


def packed(d, want):
    W, S = d["locations"].shape[1:]
    out = {**d, "queries": d["queries"].transpose(1, 2).flatten(0, 1).contiguous(),
           "locations": d["locations"].flatten(1, 2).contiguous(), "cosines": d["cosines"].flatten(1, 2),
           "sines": d["sines"].flatten(1, 2)}
    cu = torch.arange(0, W * S + 1, S, dtype=torch.int32, device=d["locations"].device)
    return dict(out, cu_seqlens_q=cu, cu_seqlens_k=cu), want.transpose(1, 2).flatten(0, 1)


# (fp16: 2^15 is the largest power of two, the rest is the scale's)
CASES = [(t, up, scale) for t in DTYPES for up, scale in ((15, 2.0 ** 5), (15, -(2.0 ** 30)), (15, 2.0 ** 85))]
CASES += [(t, up, 1.0) for t in DTYPES[::2] for up in (30, 60, 100)]


@pytest.mark.parametrize("dtype,up,scale", CASES)
@pytest.mark.parametrize("S", [1, 2, 4, 9, 20, 33])
def test_attention(dv, gpu, dtype, up, scale, S):  # noqa: F811
    d, want, _ = make(dtype, 3, S, up, seed=S)
    if scale < 0:
        d["queries"] = -d["queries"]
    x = to(gpu, d)
    assert torch.equal(dv.dvattn_paged_sdpa(scale=scale, **x).cpu(), want)
    p, flat = packed(x, want)
    assert torch.equal(dv.dvattn_varlen_paged_sdpa(scale=scale, **p).cpu(), flat)
    at = torch.arange(N)
    views = [torch.stack([d[n][d["block_tables"][w].long()[at // BS], at % BS].transpose(0, 1) for w in range(3)])
             for n in ("k_cache", "v_cache")]
    got = dv.dvattn_sdpa(x["queries"][None], x["locations"], [views[0].to(gpu)], [views[1].to(gpu)], scale,
                         x["fragment_lengths"])
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype,up,scale", CASES)
@pytest.mark.parametrize("S", [1, 2, 4, 9, 20, 33])
@pytest.mark.parametrize("b", [127, 134])
def test_attention_over_8_bits(dv, gpu, dtype, up, scale, S, b):  # noqa: F811
    d, want, _ = make(dtype, 3, S, up, seed=S)
    if scale < 0:
        d["queries"] = -d["queries"]
    for n in ("k", "v"):
        d[n + "_cache"] = d[n + "_cache"].float().to(torch.float8_e4m3fn)
        d[n + "_scales"] = torch.full((d["k_cache"].shape[0], Hkv), b if n == "k" else 127, dtype=torch.uint8)
    x = to(gpu, d)
    assert torch.equal(dv.dvattn_paged_sdpa_q8(scale=scale, **x).cpu(), want)
    p, flat = packed(x, want)
    assert torch.equal(dv.dvattn_varlen_paged_sdpa_q8(scale=scale, **p).cpu(), flat)


@pytest.mark.parametrize("up,b", [(-30, 237), (-60, 244), (-100, 240), (-2, 230), (40, 190), (100, 100), (110, 60)])
@pytest.mark.parametrize("S", [1, 3, 20])
def test_float32_queries_and_keys_of_other_sizes(dv, gpu, up, b, S):  # noqa: F811
    """Queries of 2^up against keys under the exponent b: no score leaves the floats, whatever
    the sizes of the two are."""
    d, want, _ = make(torch.float32, 3, S, up, seed=S)
    for n in ("k", "v"):
        d[n + "_cache"] = d[n + "_cache"].to(torch.float8_e4m3fn)
        d[n + "_scales"] = torch.full((d["k_cache"].shape[0], Hkv), b if n == "k" else 127, dtype=torch.uint8)
    x = to(gpu, d)
    scale = 2.0 ** (147 - up - b)  # the largest scores around 2^36
    assert torch.equal(dv.dvattn_paged_sdpa_q8(scale=scale, **x).cpu(), want)
    p, flat = packed(x, want)
    assert torch.equal(dv.dvattn_varlen_paged_sdpa_q8(scale=scale, **p).cpu(), flat)
