"""GPU tests of the paths that the operators around 8-bit caches choose by size (marked
``gpu``): runs shared by waves, scans of many slots, workgroups of eight KV heads, pairs of
tokens, calls of more rows than a launch takes, captured calls and calls on two streams.
Tolerances as in test_gpu_cache8.py.
"""
import pytest
import torch

from test_gpu_cache8 import (CACHE, DTYPES, SCALE, append_case, case, check, check_append, compare, dv,  # noqa: F401
                             packed, to)
from oracle import cache8_oracle as CO

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Appends.
@pytest.mark.parametrize("dtype,rope", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                        (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("Hkv,T,bs,R", [(1, 100, 32, 128), (3, 150, 64, 64), (2, 300, 130, 128), (8, 90, 256, 32),
                                        (5, 700, 300, 0), (1, 17, 24, 16)])
@pytest.mark.parametrize("size", [0.01, 30.0])
def test_append_long_pages(dv, gpu, dtype, rope, Hkv, T, bs, R, size):
    """Runs of more than 16 rows, from inside a page on and into the middle of another, over
    pages whose exponents they raise (30) or do not (0.01)."""
    g = torch.Generator().manual_seed(T + bs)
    P = -(-T // bs) + 3
    d = append_case(g, dtype, rope, 1, Hkv, T, P, bs, R, size=size)
    perm = torch.randperm(P, generator=g)
    pos = bs // 3 + torch.arange(T)
    check_append(dv, gpu, d, (perm[pos // bs] * bs + pos % bs)[None])


@pytest.mark.parametrize("T", [1500, 5000, 9000, 18000])
def test_append_many_tokens(dv, gpu, T):
    """Tiles of several tokens, slots compared in several steps: a prompt whose page in the
    middle also gets the last token and the first, and whose other page is written twice."""
    g = torch.Generator().manual_seed(T)
    P = T // 16 + 3
    d = append_case(g, torch.bfloat16, torch.bfloat16, 1, 1, T, P, 16, 32)
    pos = 5 + torch.arange(T)
    perm = torch.randperm(P, generator=g)
    slots = perm[pos // 16] * 16 + pos % 16
    slots[-1] = slots[T // 2] // 16 * 16 + 3
    slots[0] = slots[T // 2] // 16 * 16 + 2
    slots[T // 3:T // 3 + 40] = slots[T // 3 + 40:T // 3 + 80].clone()
    check_append(dv, gpu, d, slots[None])


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_single_tokens(dv, gpu, dtype):
    """One token of each sequence, its row of the page anywhere: four KV heads to a wave, the
    last of them fewer; heads of one page whose exponents rise and do not."""
    g = torch.Generator().manual_seed(8)
    for Hkv in (1, 3, 4, 6, 9):
        W, bs = 50, 16
        d = append_case(g, dtype, dtype, W, Hkv, 1, W + 2, bs, 64)
        scale = torch.tensor([0.01, 1.0, 40.0]).repeat(Hkv)[:Hkv, None, None]
        d["keys"], d["values"] = (d["keys"] * scale).to(dtype), (d["values"] * scale.flip(0)).to(dtype)
        row = torch.randint(0, bs, (W,), generator=g)
        row[:5], row[5:9] = 0, 15
        check_append(dv, gpu, d, (torch.randperm(W + 2, generator=g)[:W] * bs + row)[:, None])


@pytest.mark.parametrize("bs,P", [(48, 20), (1500, 3)])
def test_append_slots_of_any_order_in_long_pages(dv, gpu, bs, P):
    """Several runs and single tokens in each page, rows named twice, rows behind the 1024th."""
    g = torch.Generator().manual_seed(bs)
    T = 1300
    d = append_case(g, torch.bfloat16, torch.bfloat16, 1, 3, T, P, bs, 64, size=20.0)
    check_append(dv, gpu, d, torch.randint(-5, P * bs, (1, T), generator=g))
    slots = torch.cat([torch.arange(100) + int(x) for x in torch.randint(0, P * bs - 100, (13,), generator=g)])
    check_append(dv, gpu, d, slots[None])


def test_append_runs_across_sequences(dv, gpu):
    """The last slots of a sequence and the first of the next are consecutive, in one page."""
    g = torch.Generator().manual_seed(5)
    W, S = 6, 10
    for Hkv in (1, 2):
        d = append_case(g, torch.float16, torch.float16, W, Hkv, S, 6, 16, 64)
        check_append(dv, gpu, d, 4 + torch.arange(W * S).reshape(W, S))


def test_append_refuses_overlapping_caches(dv, gpu):
    """Caches or scales that share a part of their memory."""
    d = to(gpu, append_case(torch.Generator().manual_seed(1), torch.bfloat16, torch.bfloat16, 1, 2, 5, 4, 16, 64))
    slots = torch.arange(5, device=gpu)[None]
    rows, bytes_ = torch.zeros(5, 16, 2, 128, dtype=torch.uint8, device=gpu), torch.zeros(5, 2, dtype=torch.uint8,
                                                                                        device=gpu)
    for bad in (dict(k_cache=rows[:4], v_cache=rows[1:]), dict(k_scales=bytes_[:4], v_scales=bytes_[1:])):
        x = {**d, **bad}
        with pytest.raises(RuntimeError):
            dv.dvattn_paged_kv_append_q8(x["keys"], x["values"], slots, x["cos"], x["sin"], *(x[n] for n in CACHE))


# ---------------------------------------------------------------------------
# Attention.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [1, 2])
def test_sdpa_eight_heads_a_workgroup(dv, gpu, dtype, F):
    fl = [4200] if F == 1 else [2300, 1900]
    d = case(dtype, 16, 8, 1, fl, 16, 128, seed=2)
    d["locations"][:] = torch.randint(-1, 700, d["locations"].shape, generator=torch.Generator().manual_seed(1))
    d["locations"][0, 3], d["locations"][0, 7] = 2299, 2222
    check(dv, gpu, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S,bs", [(5, 16), (7, 24), (8, 1), (9, 64)])
def test_sdpa_few_tokens(dv, gpu, dtype, S, bs):
    """Pairs of tokens, and where calls go over to the multi-query kernel."""
    check(dv, gpu, case(dtype, 3, 2, S, [140, 75], bs, 64, seed=S), dtype)
    check(dv, gpu, case(dtype, 2, 3, S, [200], bs, 128, seed=S, causal=True), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W,S", [(2500, 1), (700, 4), (2100, 12)])
def test_sdpa_more_rows_than_a_launch(dv, gpu, dtype, W, S):
    """Seven sequences, each many times."""
    few = case(dtype, 7, 1, S, [20], 16, 32, seed=3)
    want = CO.sdpa(SCALE, **few)
    i = torch.arange(W) % 7
    d = {**few, "queries": few["queries"][i], "block_tables": few["block_tables"][i],
         **{n: few[n][:, i].contiguous() for n in ("locations", "cosines", "sines")}}
    compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, 20, *(x[i] for x in want))
    v, w, s = packed(d, W, S, [S - k % 2 if S > 1 else 1 for k in range(W)])
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    compare(out, dtype, 20, *(x[w % 7, :, s] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_varlen_of_all_lengths(dv, gpu, dtype):
    """Sequences of 0 to 33 tokens in one call, three views of different lengths."""
    lens = [0, 1, 2, 3, 4, 5, 16, 17, 18, 20, 33, 1, 0, 2]
    S, W = max(lens), len(lens)
    d = case(dtype, W, 2, S, [64, 37, 90], 16, 64, seed=4)
    v, w, s = packed(d, W, S, lens)
    vd = to(gpu, v)
    out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
    want = [x[w, :, s] for x in CO.sdpa(SCALE, **d)]
    compare(out, dtype, 191, *want)


@pytest.mark.parametrize("S", [2, 20])
def test_sdpa_of_tokens_far_into_a_large_cache(dv, gpu, S):
    """Rows behind 2^32 bytes of a cache: the same as those rows alone."""
    d = to(gpu, case(torch.bfloat16, 2, 8, S, [500], 16, 128, seed=4, causal=True))
    want = dv.dvattn_paged_sdpa_q8(scale=SCALE, **d)
    P = (1 << 32) // (16 * 8 * 128) + 300
    n = d["k_cache"].shape[0]
    for name in CACHE:
        big = torch.zeros((P,) + tuple(d[name].shape[1:]), dtype=torch.uint8, device=gpu)
        big[P - n:] = d[name].view(torch.uint8)
        d[name] = big
    d["block_tables"] = d["block_tables"] + (P - n)
    assert torch.equal(dv.dvattn_paged_sdpa_q8(scale=SCALE, **d), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sdpa_small_queries_beside_large(dv, gpu, dtype):
    """A query head whose elements differ by many powers of two, one of zeros, one tiny."""
    d = case(dtype, 1, 1, 3, [90], 16, 32, seed=6)
    q = d["queries"].float()
    q[0, 0] *= 2.0 ** torch.arange(0, -16, -0.125)[:128]
    q[0, 1], q[0, 2] = 0.0, q[0, 2] * 2.0 ** -13
    d["queries"] = q.to(dtype)
    check(dv, gpu, d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S", [1, 2, 6, 20])
def test_sdpa_captured_and_on_two_streams(dv, gpu, dtype, S):
    """Both forms captured into one graph, replayed over changing caches between eager calls;
    the same call on two streams at a time."""
    d = case(dtype, 3, 2, S, [300], 16, 64, seed=1)
    v, _, _ = packed(d, 3, S, [S, max(1, S // 2), 1])
    d, v = to(gpu, d), to(gpu, v)
    v.update({n: d[n] for n in CACHE})

    def both():
        return (dv.dvattn_paged_sdpa_q8(scale=SCALE, **d),
                dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=v["cu_seqlens_q"], **v))

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(6):
        d["k_scales"].copy_(torch.full_like(d["k_scales"], 116 + i))
        d["v_cache"].view(torch.uint8).copy_(d["v_cache"].view(torch.uint8).roll(1, 0))
        want = both()
        graph.replay()
        if i % 2 == 0:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
    torch.cuda.synchronize()
    got = []
    for st in (side, torch.cuda.Stream(gpu)):
        with torch.cuda.stream(st):
            got += [both() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 20])
@pytest.mark.parametrize("bs", [1, 16, 24])
def test_sdpa_views_behind_all_positions(dv, gpu, dtype, S, bs):
    """A view that starts behind what a position can count has no rows; nor have the first rows
    of one behind a negative length."""
    d = case(dtype, 2, 1, S, [60, 5, 40], bs, 32, seed=S)
    d["locations"][0], d["locations"][1], d["locations"][2] = 59, -1, 39
    alone = {**d, "fragment_lengths": torch.tensor([60, 0, 0], dtype=torch.int32)}
    want = CO.sdpa(SCALE, **alone)
    for lens in ([60, 2147483647, 40], [60, 2147483647 - 61, 40]):
        d["fragment_lengths"] = torch.tensor(lens, dtype=torch.int32)
        compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, 60, *want)
        v, w, s = packed(d, 2, S, [S, S])
        vd = to(gpu, v)
        out = dv.dvattn_varlen_paged_sdpa_q8(scale=SCALE, cu_seqlens_k=vd["cu_seqlens_q"], **vd)
        compare(out, dtype, 60, *(x[w, :, s] for x in want))
    # two such views: positions behind 2^32
    d["fragment_lengths"] = torch.tensor([60, 2147483647, 2147483647, 40], dtype=torch.int32)
    loc = d["locations"]
    d.update({n: torch.cat([d[n], d[n][:1]]) for n in ("cosines", "sines")},
             locations=torch.stack([loc[0], loc[1], loc[1], loc[2]]))
    compare(dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, d)), dtype, 60, *want)
    few = case(dtype, 2, 1, S, [-7, 40], bs, 32, seed=S)
    few["locations"][0], few["locations"][1] = -1, 30
    dv.dvattn_paged_sdpa_q8(scale=SCALE, **to(gpu, few))
    torch.cuda.synchronize()
