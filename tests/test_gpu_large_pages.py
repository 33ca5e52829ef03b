"""Attention over pages of more than 2^20 rows (marked ``gpu``): a view that begins near the
end of one page and goes on in the next, against the oracles on the same rows in pages of 16.
Tolerances: test_gpu_parity.close and test_gpu_cache8.compare.
"""
import pytest
import torch

import test_gpu_cache8 as C8
from oracle import cache8_oracle as CO
from oracle import dvattn_oracle as O
from test_gpu_parity import close, dv, rand_paged, run_paged, to  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
N, BEFORE = 300, 150


def in_large_pages(gpu, d, bs, names):
    """The one-view case d as the second of two views, BEFORE of its rows at the end of page 2
    and the others at the start of page 0; of the first view nothing is seen."""
    W, S = d["locations"].shape[1:]
    pages, small = torch.tensor([[2, 0]], dtype=torch.int32), d["block_tables"][0].long()
    at = torch.arange(N)
    pos = bs - BEFORE + at
    row = pages[0].long()[pos // bs] * bs + pos % bs
    out = dict(queries=d["queries"], block_tables=pages, locations=torch.cat([torch.full((1, W, S), -1, dtype=torch.int32),
                                                                              d["locations"]]),
               cosines=d["cosines"].expand(2, -1, -1, -1).contiguous(),
               sines=d["sines"].expand(2, -1, -1, -1).contiguous(),
               fragment_lengths=torch.tensor([bs - BEFORE, N], dtype=torch.int32))
    for n in names:
        big = torch.zeros((3 * bs,) + tuple(d[n].shape[2:]), dtype=d[n].dtype, device=gpu)
        big.view(torch.uint8)[row.to(gpu)] = d[n].flatten(0, 1).view(torch.uint8)[(small[at // 16] * 16 + at % 16)].to(gpu)
        out[n] = big.reshape((3, bs) + tuple(d[n].shape[2:]))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 4, 20, 33])
@pytest.mark.parametrize("bs", [1 << 21, 1100003])
def test_paged(dv, gpu, dtype, S, bs):  # noqa: F811
    loc = (N - S + torch.arange(S, dtype=torch.int32)).reshape(1, 1, S)
    d = rand_paged(1, 1, S, 1, 16, [N], 64, dtype, seed=S, loc=loc)
    big = in_large_pages(gpu, d, bs, ("k_cache", "v_cache"))
    close(run_paged(dv, big, 0.1, gpu), O.paged_sdpa(0.1, **d), dtype, f"S={S}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 4, 20, 33])
@pytest.mark.parametrize("bs", [1 << 21, 1100003])
def test_cache8(dv, gpu, dtype, S, bs):  # noqa: F811
    d = C8.case(dtype, 1, 1, S, [N], 16, 64, seed=S, causal=True)
    d["k_scales"][:], d["v_scales"][:] = 120, 121
    big = in_large_pages(gpu, d, bs, ("k_cache", "v_cache"))
    big.update(k_scales=d["k_scales"][:3], v_scales=d["v_scales"][:3])
    want = CO.sdpa(C8.SCALE, **d)
    C8.compare(dv.dvattn_paged_sdpa_q8(scale=C8.SCALE, **to(big, gpu)), dtype, N, *want)
