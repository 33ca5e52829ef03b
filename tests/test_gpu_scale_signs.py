"""Attention under a negative scale and a scale of zero (marked ``gpu``), over the numbers
of tokens at which the operators change kernels, with causal rows, rows without keys, views
that end inside a stage and pages that do not exist: a key that a token does not see has no
weight, whatever the scale's sign; under a scale of zero all keys seen weigh the same.
Tolerances: test_gpu_parity.close, test_gpu_cache8.compare and test_gpu_tree_cache.compare_tree.
"""
import numpy as np
import pytest
import torch

import test_gpu_cache8 as C8
import test_gpu_tree_cache as TC
from oracle import dvattn_oracle as O
from test_gpu_parity import close, dv, rand_paged, rand_varlen, run_paged, run_varlen  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SCALES = [-0.05, 0.0]


def locations(F, W, S, lens, seed):
    """Causal rows in the last view, rows of any length in the others, one sequence without keys."""
    rng = np.random.default_rng(seed)
    loc = rng.integers(-1, max(lens) + 3, size=(F, W, S))
    loc[-1] = lens[-1] - S + np.arange(S)
    loc[:, 0] = -1
    return loc


def folded(scale, queries):
    """(scale, queries) of a positive scale with the same scores, exactly: the oracle hides
    keys before it scales."""
    return (-scale, -queries) if scale < 0 else (1.0, queries * 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("S", [1, 2, 4, 8, 9, 20, 33])
@pytest.mark.parametrize("bs", [16, 24])
def test_paged(dv, gpu, dtype, scale, S, bs):  # noqa: F811
    lens = [61, 300]
    d = rand_paged(2, 3, S, 2, bs, lens, 64, dtype, seed=S + bs, loc=locations(2, 3, S, lens, S))
    out = run_paged(dv, d, scale, gpu)
    scale, d["queries"] = folded(scale, d["queries"])
    close(out, O.paged_sdpa(scale, **d), dtype, f"S={S}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 4, 20, 33, 0, 2], [3, 5]])
def test_varlen(dv, gpu, dtype, scale, counts):  # noqa: F811
    W, T = len(counts), sum(counts)
    d = rand_varlen(2, W, T, np.concatenate([[0], np.cumsum(counts)]), 2, 16, [90, 401], 64, dtype, seed=T)
    out = run_varlen(dv, d, scale, gpu)
    scale, d["queries"] = folded(scale, d["queries"])
    close(out, O.varlen_paged_sdpa(scale, **d), dtype, f"{counts}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("S,lens", [(1, [40, 7]), (2, [300, 45]), (9, [300, 45]), (20, [70, 1, 133])])
def test_contiguous(dv, gpu, dtype, scale, S, lens):  # noqa: F811
    F, W, Hkv = len(lens), 3, 2
    g = torch.Generator().manual_seed(S)
    q = torch.randn(F, W, 16 * Hkv, S, 128, generator=g).to(dtype)
    ks = [torch.randn(W, Hkv, L, 128, generator=g).to(dtype) for L in lens]
    vs = [torch.randn(W, Hkv, L, 128, generator=g).to(dtype) for L in lens]
    loc = torch.from_numpy(locations(F, W, S, lens, S).astype(np.int32))
    fl = torch.tensor(lens, dtype=torch.int32)
    out = dv.dvattn_sdpa(q.to(gpu), loc.to(gpu), [k.to(gpu) for k in ks], [v.to(gpu) for v in vs], scale, fl.to(gpu))
    scale, q = folded(scale, q)
    close(out, O.contig_sdpa(scale, loc, q, fl, ks, vs), dtype, f"S={S}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("S", [1, 2, 4, 7, 9, 20, 33])
def test_cache8(dv, gpu, dtype, scale, S):  # noqa: F811
    """The token grid and the packed tokens (C8.check) over an 8-bit cache."""
    C8.check(dv, gpu, C8.case(dtype, 2, 2, S, [30, 420], 16, 128, seed=S, causal=True), dtype, scale=scale)
    d = C8.case(dtype, 3, 2, S, [120, 70], 24, 64, seed=3, bad=True)
    d["locations"][:, 1] = -1
    C8.check(dv, gpu, d, dtype, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("S", [1, 5, 17, 40])
def test_tree(dv, gpu, dtype, scale, S):  # noqa: F811
    TC.check_tree(dv, gpu, TC.tree_case(dtype, 2, 2, S, [33, 210], 16, 64, seed=S, bad=True), dtype, scale=scale)
