"""Host-side tests of the entry points around 8-bit caches (CPU only): the C ABI
refuses bad calls before it touches a pointer, the torch operators have no CPU
kernels, and the oracle of the format agrees with torch's E4M3."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import cache8_oracle as CO

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
P = 0x1000  # never dereferenced: every call below is refused, or empty


@pytest.fixture(scope="module")
def lib():
    from dvattention_amd import capi
    return capi.lib()


def shape(**kw):
    from dvattention_amd import capi
    base = dict(F=1, W=2, Hq=16, Hkv=1, E=128, Ev=128, S=4, block_size=16, max_blocks_per_seq=4, total_q_tokens=8,
                num_blocks=8, rotary_dim=64)
    base.update(kw)
    return capi.Shape(**base)


def paged(lib, s, ws_bytes=1 << 40, dtype=2, **ptr):
    a = dict(out=P, loc=P, q=P, cos=P, sin=P, fl=P, kc=P, vc=P, ks=P, vs=P, bt=P, ws=P)
    a.update({k: v for k, v in ptr.items() if k in a})
    return lib.dvattn_paged_sdpa_q8(dtype, a["out"], 0.1, a["loc"], a["q"], a["cos"], a["sin"], a["fl"], a["kc"],
                                    a["vc"], a["ks"], a["vs"], a["bt"], ctypes.byref(s), a["ws"], ws_bytes, None)


def varlen(lib, s, ws_bytes=1 << 40, dtype=2, **ptr):
    a = dict(out=P, loc=P, q=P, cos=P, sin=P, fl=P, kc=P, vc=P, ks=P, vs=P, bt=P, cu=P, ws=P)
    a.update({k: v for k, v in ptr.items() if k in a})
    return lib.dvattn_varlen_paged_sdpa_q8(dtype, a["out"], 0.1, a["loc"], a["q"], a["cos"], a["sin"], a["fl"],
                                           a["kc"], a["vc"], a["ks"], a["vs"], a["bt"], a["cu"], ctypes.byref(s),
                                           a["ws"], ws_bytes, None)


def append(lib, s, dtype=2, rope=2, **ptr):
    from dvattention_amd import capi
    a = dict(kc=P, vc=2 * P, ks=P, vs=2 * P, slots=P, k=P, v=P, cos=P, sin=P)
    a.update({k: v for k, v in ptr.items() if k in a})
    lay = capi.KvLayout()
    return lib.dvattn_paged_kv_append_q8(dtype, rope, a["kc"], a["vc"], a["ks"], a["vs"], a["slots"], a["k"], a["v"],
                                         a["cos"], a["sin"], ctypes.byref(s), ctypes.byref(lay), None)


def tables(lib, s, T=8, **ptr):
    a = dict(cu=P, starts=P, pos=P, slots=P, nl=P, nc=P, bt=P, fp=P, ln=P, nt=P, fc=P)
    a.update({k: v for k, v in ptr.items() if k in a})
    return lib.dvattn_block_tables(a["cu"], a["starts"], a["pos"], a["slots"], a["nl"], a["nc"], a["bt"], a["fp"],
                                   a["ln"], a["nt"], a["fc"], T, ctypes.byref(s), None)


def error(lib):
    return lib.dvattn_last_error().decode()


@pytest.mark.parametrize("call", [paged, varlen])
@pytest.mark.parametrize("kw,status,needle", [
    (dict(Hq=32), UNSUPPORTED, "GQA 16"),
    (dict(Hkv=-1), INVALID, "Hkv"),
    (dict(E=64), UNSUPPORTED, "E == Ev == 128"),
    (dict(Ev=64), UNSUPPORTED, "E == Ev == 128"),
    (dict(rotary_dim=63), UNSUPPORTED, "rotary_dim"),
    (dict(rotary_dim=130), UNSUPPORTED, "rotary_dim"),
    (dict(block_size=0), INVALID, "block_size"),
    (dict(S=-1, total_q_tokens=-1), INVALID, "negative"),
    (dict(F=-1), INVALID, "negative"),
    (dict(max_blocks_per_seq=-1), INVALID, "max_blocks_per_seq"),
    (dict(num_blocks=1 << 28), UNSUPPORTED, "2^32 rows"),
])
def test_attention_shapes_refused(lib, call, kw, status, needle):
    assert call(lib, shape(**kw)) == status
    assert needle in error(lib)


@pytest.mark.parametrize("call", [paged, varlen])
@pytest.mark.parametrize("name", ["out", "q", "loc", "fl", "cos", "sin", "kc", "vc", "ks", "vs", "bt", "cu"])
def test_attention_null_pointers_refused(lib, call, name):
    if name == "cu" and call is paged:
        return
    assert call(lib, shape(), **{name: None}) == INVALID
    assert "null" in error(lib)


@pytest.mark.parametrize("call", [paged, varlen])
@pytest.mark.parametrize("name,off,word", [("out", 8, "out"), ("q", 2, "queries"), ("kc", 4, "k_cache"),
                                           ("vc", 8, "v_cache"), ("loc", 2, "locations"), ("cos", 1, "cosines"),
                                           ("bt", 2, "block_tables"), ("ws", 8, "workspace")])
def test_attention_misaligned_pointers_refused(lib, call, name, off, word):
    assert call(lib, shape(), **{name: P + off}) == INVALID
    assert word in error(lib) and "aligned" in error(lib)


@pytest.mark.parametrize("call,size", [(paged, "dvattn_paged_sdpa_q8_workspace_size"),
                                       (varlen, "dvattn_varlen_paged_sdpa_q8_workspace_size")])
def test_attention_workspace(lib, call, size):
    for dtype in (0, 1, 2):
        for kw in (dict(S=1, total_q_tokens=2), dict(), dict(S=100, total_q_tokens=300, W=3, Hkv=8, Hq=128)):
            need = getattr(lib, size)(dtype, ctypes.byref(shape(**kw)), 0)
            assert need > 0
            assert call(lib, shape(**kw), ws_bytes=need - 1, dtype=dtype) == WORKSPACE
            assert call(lib, shape(**kw), ws=None, dtype=dtype) == WORKSPACE
    assert getattr(lib, size)(7, ctypes.byref(shape()), 0) == 0
    assert call(lib, shape(), dtype=3) == UNSUPPORTED
    for kw in (dict(S=0, total_q_tokens=0), dict(Hkv=0)):
        assert call(lib, shape(**kw), ws_bytes=0, ws=None, out=None, q=None) == 0


def test_varlen_without_sequences_refused(lib):
    assert varlen(lib, shape(W=0)) == INVALID


@pytest.mark.parametrize("kw,status,needle", [
    (dict(E=64), UNSUPPORTED, "E == Ev == 128"), (dict(Ev=256), UNSUPPORTED, "E == Ev == 128"),
    (dict(rotary_dim=7), UNSUPPORTED, "rotary_dim"), (dict(block_size=-2), INVALID, "block_size"),
    (dict(W=-1), INVALID, "negative"), (dict(num_blocks=-1), INVALID, "num_blocks"),
    (dict(num_blocks=1 << 28), UNSUPPORTED, "2^32 rows"), (dict(W=1 << 15, S=1 << 15), UNSUPPORTED, "tokens"),
])
def test_append_shapes_refused(lib, kw, status, needle):
    assert append(lib, shape(**kw)) == status
    assert needle in error(lib)


def test_append_pointers_and_types_refused(lib):
    for name in ("kc", "vc", "ks", "vs", "slots", "k", "v", "cos", "sin"):
        assert append(lib, shape(), **{name: None}) == INVALID
    for name, off in (("kc", 8), ("vc", 4), ("slots", 4), ("k", 1), ("cos", 1)):
        assert append(lib, shape(), **{name: 4 * P + off}) == INVALID
        assert "aligned" in error(lib)
    assert append(lib, shape(), vc=P) == INVALID and "both" in error(lib)
    assert append(lib, shape(), vs=P) == INVALID and "both" in error(lib)
    assert append(lib, shape(), dtype=2, rope=1) == UNSUPPORTED
    assert append(lib, shape(), dtype=9) == UNSUPPORTED
    for kw in (dict(W=0), dict(S=0), dict(Hkv=0)):
        assert append(lib, shape(**kw), k=None, v=None, slots=None) == 0


def test_tables_refused(lib):
    for name in ("cu", "starts", "pos", "slots", "nl", "nc", "bt", "fp", "ln", "nt", "fc"):
        assert tables(lib, shape(), **{name: None}) == INVALID
        assert tables(lib, shape(), **{name: P + (4 if name == "slots" else 2)}) == INVALID
        assert "aligned" in error(lib)
    assert tables(lib, shape(), T=-1) == INVALID
    assert tables(lib, shape(W=-1)) == INVALID
    assert tables(lib, shape(W=8193)) == UNSUPPORTED
    assert tables(lib, shape(block_size=0)) == INVALID
    assert tables(lib, shape(num_blocks=-1)) == INVALID


def test_operators_have_no_cpu_kernels():
    import dvattention_amd as dv
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q = torch.zeros(1, 16, 1, 128)
    kc, sc = torch.zeros(2, 16, 1, 128, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)
    cs = torch.zeros(1, 1, 1, 64)
    with pytest.raises(NotImplementedError):
        dv.dvattn_paged_sdpa_q8(q, i32(1, 1, 1), cs, cs, i32(1), kc, kc, sc, sc, i32(1, 2), 0.1)
    with pytest.raises(NotImplementedError):
        dv.dvattn_varlen_paged_sdpa_q8(q[:, :, 0], i32(1, 1), cs[0, :, :, :32], cs[0, :, :, :32], i32(1), kc, kc, sc,
                                       sc, i32(1, 2), i32(2), i32(2), 0.1)
    with pytest.raises(NotImplementedError):
        dv.dvattn_paged_kv_append_q8(torch.zeros(1, 1, 128), torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.long),
                                     torch.zeros(64), torch.zeros(64), kc, kc.clone(), sc, sc.clone())
    with pytest.raises(NotImplementedError):
        dv.dvattn_block_tables(i32(1), i32(1), i32(1, 2), i32(2), i32(1), 16, 1)


def test_reference_module_offers_them():
    import dvattention_amd as dv
    import dvattn.attention as ref
    for name in ("dvattn_block_tables", "dvattn_paged_kv_append_q8", "dvattn_paged_sdpa_q8",
                 "dvattn_varlen_paged_sdpa_q8"):
        assert getattr(ref, name) is getattr(dv, name) and name in ref.__all__ and name in dv.__all__


def test_oracle_rounding_is_e4m3():
    """The oracle's rounding against torch's type: every byte is a fixed point, and what
    lies between two neighbours goes where torch's conversion sends it."""
    b = torch.arange(256, dtype=torch.uint8)
    v = b.view(torch.float8_e4m3fn).double().numpy()
    fine = ~np.isnan(v)
    assert np.array_equal(CO.e4m3(v[fine]), v[fine])
    x = np.concatenate([np.linspace(-448, 448, 9973), np.linspace(-0.03, 0.03, 4001),
                        (np.sort(v[fine])[1:] + np.sort(v[fine])[:-1]) / 2])
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(CO.e4m3(x.astype(np.float32).astype(np.float64)), want)


@pytest.mark.parametrize("amax,b", [(0.0, 1), (1e-45, 1), (448.0, 127), (448.0001, 128), (449.0, 128), (1.75, 119),
                                    (1.7500001, 120), (61440.0, 135), (3.3e38, 247), (2.0 ** -126, 1)])
def test_oracle_exponents(amax, b):
    assert CO.exponent(float(np.float32(amax))) == b


def test_oracle_tables_by_hand():
    """Pages of 4 rows: one sequence goes on in its page, one needs a page, one ends and
    gives two back, one is refused as its row is full."""
    cu, starts, pos, slots, lengths, count, bt, stack = CO.tables(
        [5, 4, 7, 8], [2, 1, -1, 1], [[3, 1], [0, -1], [5, 2], [6, 7]], [4, 9, 9, 9, 9, 9, 9, 9], 1, 4, 6)
    assert cu == [0, 2, 3, 3, 4] and starts == [5, 4, -1, -1] and lengths == [7, 5, 0, 8]
    assert pos == [5, 6, 4, -1, -1, -1] and count == 2 and stack[:3] == [4, 5, 2]
    assert slots == [5, 6, 8, -1, -1, -1] and bt.tolist() == [[3, 1], [0, 2], [5, 2], [6, 7]]
