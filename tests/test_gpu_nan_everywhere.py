"""NaN keys and values in many places of a long row, so that every piece of a split row, or
all pieces of one round of its merge, holds one (marked ``gpu``): the output is NaN, and
rows that see none of them are as they were.
"""
import math

import pytest
import torch

from test_gpu_parity import dv  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E, Hkv, BS, SCALE = 128, 4, 16, 128 ** -0.5


def make(gpu, dtype, S, n, q8):
    """Two sequences of n rows, whose tokens are the last S of them."""
    g = torch.Generator(device=gpu).manual_seed(S + n)
    maxB = -(-n // BS)
    loc = (n - S + torch.arange(S, dtype=torch.int32, device=gpu)).expand(1, 2, S).contiguous()
    d = dict(queries=torch.randn(2, 16 * Hkv, S, E, generator=g, device=gpu).to(dtype), locations=loc,
             cosines=torch.zeros(1, 2, S, 0, device=gpu), sines=torch.zeros(1, 2, S, 0, device=gpu),
             fragment_lengths=torch.tensor([n], dtype=torch.int32, device=gpu),
             block_tables=torch.randperm(2 * maxB, generator=g, device=gpu).to(torch.int32).reshape(2, maxB))
    for x in "kv":
        rows = torch.randn(2 * maxB, BS, Hkv, E, generator=g, device=gpu)
        d[x + "_cache"] = rows.to(torch.float8_e4m3fn if q8 else dtype)
        if q8:
            d[x + "_scales"] = torch.full((2 * maxB, Hkv), 127, dtype=torch.uint8, device=gpu)
    return d


def packed(d):
    W, S = d["locations"].shape[1:]
    out = {**d, "queries": d["queries"].transpose(1, 2).flatten(0, 1).contiguous(),
           "locations": d["locations"].flatten(1, 2).contiguous(), "cosines": d["cosines"].flatten(1, 2),
           "sines": d["sines"].flatten(1, 2)}
    cu = torch.arange(0, W * S + 1, S, dtype=torch.int32, device=d["locations"].device)
    return dict(out, cu_seqlens_q=cu, cu_seqlens_k=cu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("S", [1, 2, 4, 9, 20])
@pytest.mark.parametrize("n", [700, 9000])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("part", [1.0, 0.6, 0.1])
def test_nan_in_every_piece(dv, gpu, dtype, q8, S, n, where, part):  # noqa: F811
    """Every fifth row of sequence 1, for KV head 2, up to `part` of its length."""
    one, many = (dv.dvattn_paged_sdpa_q8, dv.dvattn_varlen_paged_sdpa_q8) if q8 else (
        dv.dvattn_paged_sdpa, dv.dvattn_varlen_paged_sdpa)
    d = make(gpu, dtype, S, n, q8)
    before = one(scale=SCALE, **d)
    at = torch.arange(0, int(part * n), 5, device=gpu)
    page = d["block_tables"][1].long()[at // BS]
    cache = d[where + "_cache"]
    if q8:
        cache.view(torch.uint8)[page, at % BS, 2] = 0x7f
    else:
        cache[page, at % BS, 2] = math.nan
    for out in (one(scale=SCALE, **d),
                many(scale=SCALE, **packed(d)).unflatten(0, (2, S)).transpose(1, 2)):
        assert out[1, 32:48].isnan().all()
        rest = torch.ones(2, 16 * Hkv, dtype=torch.bool, device=gpu)
        rest[1, 32:48] = False
        assert out[rest].isfinite().all()
    assert torch.equal(one(scale=SCALE, **d)[rest], before[rest])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 3, 9, 20])
@pytest.mark.parametrize("lens", [[16], [60], [40, 700], [3000]])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("step", [1, 5])
def test_nan_in_contiguous_views(dv, gpu, dtype, S, lens, where, step):  # noqa: F811
    """Every row, or every fifth, of every view of KV head 2 of sequence 1."""
    g = torch.Generator(device=gpu).manual_seed(S)
    F = len(lens)
    q = torch.randn(F, 2, 16 * Hkv, S, E, generator=g, device=gpu).to(dtype)
    views = {x: [torch.randn(2, Hkv, n, E, generator=g, device=gpu).to(dtype) for n in lens] for x in "kv"}
    loc = torch.stack([torch.full((2, S), n - 1, dtype=torch.int32, device=gpu) for n in lens])
    fl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    before = dv.dvattn_sdpa(q, loc, views["k"], views["v"], SCALE, fl)
    for x in views[where]:
        x[1, 2, ::step] = math.nan
    out = dv.dvattn_sdpa(q, loc, views["k"], views["v"], SCALE, fl)
    assert out[1, 32:48].isnan().all()
    rest = torch.ones(2, 16 * Hkv, dtype=torch.bool, device=gpu)
    rest[1, 32:48] = False
    assert torch.equal(out[rest], before[rest])
