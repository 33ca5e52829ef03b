"""Host-side tests of the tree and bounded-cache entry points (CPU only): the C ABI
refuses bad calls before it touches a pointer, the torch operators have no CPU
kernels, and the Python wrappers check what they allocate."""
import ctypes

import pytest
import torch

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from dvattention_amd import capi
    return capi.lib()


def shape(**kw):
    from dvattention_amd import capi
    base = dict(F=1, W=2, Hq=16, Hkv=1, E=128, Ev=128, S=4, block_size=16, max_blocks_per_seq=4, total_q_tokens=0,
                num_blocks=8, rotary_dim=64)
    base.update(kw)
    return capi.Shape(**base)


P = 0x1000  # never dereferenced: every call below is refused, or empty


def error(lib):
    return lib.dvattn_last_error().decode()


def tree(lib, s, ws_bytes=1 << 40, dtype=2, at=(), **ptr):
    a = dict(out=P, loc=P, q=P, cos=P, sin=P, fl=P, kc=P, vc=P, bt=P, parents=P, views=P, rows=P, ws=P)
    a.update(ptr)
    return lib.dvattn_tree_paged_sdpa(dtype, a["out"], 0.1, a["loc"], a["q"], a["cos"], a["sin"], a["fl"], a["kc"],
                                      a["vc"], a["bt"], a["parents"], a["views"], a["rows"], ctypes.byref(s),
                                      a["ws"], ws_bytes, None)


def mass(lib, s, ws_bytes=1 << 40, dtype=2, capacity=64, decay=1.0, **ptr):
    a = dict(out=P, mass=P, loc=P, q=P, cos=P, sin=P, fl=P, kc=P, bt=P, ws=P)
    a.update(ptr)
    return lib.dvattn_paged_key_mass(dtype, a["out"], a["mass"], decay, capacity, 0.1, a["loc"], a["q"], a["cos"],
                                     a["sin"], a["fl"], a["kc"], a["bt"], ctypes.byref(s), a["ws"], ws_bytes, None)


@pytest.mark.parametrize("call", [tree, mass])
@pytest.mark.parametrize("kw,status,needle", [
    (dict(Hq=32), UNSUPPORTED, "GQA 16"),
    (dict(E=64), UNSUPPORTED, "E == Ev == 128"),
    (dict(rotary_dim=63), UNSUPPORTED, "rotary_dim"),
    (dict(rotary_dim=130), UNSUPPORTED, "rotary_dim"),
    (dict(block_size=0), INVALID, "block_size"),
    (dict(S=-1), INVALID, "negative"),
    (dict(max_blocks_per_seq=-1), INVALID, "max_blocks_per_seq"),
    (dict(num_blocks=1 << 28), UNSUPPORTED, "2^32 rows"),
])
def test_attention_shapes_refused(lib, call, kw, status, needle):
    assert call(lib, shape(**kw)) == status
    assert needle in error(lib)


@pytest.mark.parametrize("call,names", [
    (tree, ("out", "loc", "q", "cos", "sin", "fl", "kc", "vc", "bt", "parents", "views", "rows", "ws")),
    (mass, ("out", "mass", "loc", "q", "cos", "sin", "fl", "kc", "bt", "ws")),
])
def test_null_and_misaligned_pointers_refused(lib, call, names):
    s = shape(max_blocks_per_seq=400)  # (short sequences' trees need no workspace)
    for name in names:
        assert call(lib, s, **{name: None}) in (INVALID, WORKSPACE), name
        assert call(lib, s, **{name: P + 2}) == INVALID, name
        assert "aligned" in error(lib), name


def test_workspace_refused(lib):
    for call, size in ((tree, lib.dvattn_tree_paged_sdpa_workspace_size),
                       (mass, lib.dvattn_paged_key_mass_workspace_size)):
        for S in (1, 4):
            s = shape(S=S, max_blocks_per_seq=400)
            need = size(2, ctypes.byref(s), 64 if call is mass else 0)
            assert need > 0
            assert call(lib, s, ws_bytes=need - 1) == WORKSPACE
            assert "workspace" in error(lib)
        assert call(lib, shape(), dtype=7) == UNSUPPORTED


def test_limits_refused(lib):
    assert tree(lib, shape(S=4097)) == UNSUPPORTED and "drafted nodes" in error(lib)
    assert mass(lib, shape(), capacity=-1) == INVALID
    assert mass(lib, shape(W=1 << 20, S=1), capacity=1 << 20) == UNSUPPORTED and "blocks" in error(lib)
    assert mass(lib, shape(W=1 << 20, S=1 << 12)) == UNSUPPORTED
    assert mass(lib, shape(max_blocks_per_seq=1 << 30)) == UNSUPPORTED and "2^32" in error(lib)


def test_workspace_is_bounded(lib):
    """Scores of one token are kept up to 1 GiB; tokens go through in bounded launches."""
    size = lib.dvattn_paged_key_mass_workspace_size
    wide = shape(S=1, W=64, Hkv=8, Hq=128, max_blocks_per_seq=8192, num_blocks=1 << 16)
    assert size(2, ctypes.byref(wide), 0) < 2 << 30
    a, b = (shape(S=s, W=1, max_blocks_per_seq=4096) for s in (64, 64 * 32))
    queries = 16 * 128 * 2
    assert size(2, ctypes.byref(b), 0) - size(2, ctypes.byref(a), 0) == (b.S - a.S) * queries


def test_tree_workspace(lib):
    """None where one launch goes through a node's whole key list; windows of the lists, then
    the pieces of the committed keys, beyond."""
    size = lib.dvattn_tree_paged_sdpa_workspace_size
    need = lambda dtype, **kw: size(dtype, ctypes.byref(shape(**kw)), 0)
    assert need(2) == 0 and need(0, S=100, max_blocks_per_seq=20) == 0
    slot = (16 * 128 + 32) * 4
    for kw in (dict(max_blocks_per_seq=100), dict(max_blocks_per_seq=300, S=9), dict(max_blocks_per_seq=500, W=1, S=1)):
        n = need(2, **kw)
        s = shape(**kw)
        nodes = s.W * s.S * s.Hkv
        assert n > 0 and n % (nodes * slot) == 0
        windows = n // (nodes * slot)
        assert windows * 640 >= s.max_blocks_per_seq * 16 and windows <= s.max_blocks_per_seq * 16 / 128 + 1
    pieces = need(2, S=64, max_blocks_per_seq=10 ** 6)
    assert pieces > 0 and pieces == need(2, S=64, max_blocks_per_seq=2 ** 20) == need(2, F=60, S=64)
    assert need(2, F=0, W=100, Hkv=8, Hq=128, max_blocks_per_seq=0) == 0  # nothing to see, many nodes
    assert need(2, W=-1) == need(2, max_blocks_per_seq=-1) == 0
    assert need(2, W=2 ** 31 - 1, Hkv=2 ** 31 - 1, S=300) >= 0


def test_empty_calls_succeed(lib):
    for kw in (dict(W=0), dict(Hkv=0, Hq=0)):
        assert tree(lib, shape(**kw)) == 0 and mass(lib, shape(**kw)) == 0
    assert tree(lib, shape(S=0)) == 0 and mass(lib, shape(), capacity=0) == 0
    assert select(lib, W=0) == 0 and select(lib, budget=0, kf=0, kl=0) == 0
    assert compact(lib, shape(W=0)) == 0 and compact(lib, shape(), N=0) == 0
    assert meta(lib, W=0) == 0


def select(lib, capacity=100, W=2, Hkv=1, budget=8, kf=1, kl=2, rows=P, m=P, first=P, lengths=P):
    return lib.dvattn_kv_select(rows, m, first, lengths, capacity, W, Hkv, budget, kf, kl, None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(kf=5, kl=4), INVALID, "budget"),
    (dict(kf=2**31 - 1, kl=2**31 - 1), INVALID, "budget"),
    (dict(kf=-1), INVALID, "negative"),
    (dict(budget=-1, kf=0, kl=0), INVALID, "negative"),
    (dict(capacity=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (dict(W=1 << 20, Hkv=1 << 12), UNSUPPORTED, "2^22"),
    (dict(rows=None), INVALID, "null"),
    (dict(m=None), INVALID, "null"),
    (dict(first=None), INVALID, "null"),
    (dict(lengths=None), INVALID, "null"),
    (dict(m=P + 2), INVALID, "aligned"),
])
def test_select_refused(lib, kw, status, needle):
    assert select(lib, **kw) == status
    assert needle in error(lib)


def compact(lib, s, row_heads=1, N=4, dtype=2, capacity=64, layout=True, **ptr):
    from dvattention_amd import capi
    a = dict(kc=P, vc=P, bt=P, rows=P, first=P, lengths=P, mass=P)
    a.update(ptr)
    if N == 0:
        a["mass"] = None
    lay = capi.KvLayout()
    return lib.dvattn_paged_kv_compact(dtype, a["kc"], a["vc"], a["bt"], a["rows"], row_heads, N, a["first"],
                                       a["lengths"], a["mass"], capacity, ctypes.byref(s),
                                       ctypes.byref(lay) if layout else None, None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(row_heads=2), INVALID, "heads"),
    (dict(N=-1), INVALID, "negative"),
    (dict(capacity=-1), INVALID, "negative"),
    (dict(lengths=None), INVALID, "lengths"),
    (dict(rows=None), INVALID, "null"),
    (dict(first=None), INVALID, "null"),
    (dict(bt=None), INVALID, "null"),
    (dict(kc=None), INVALID, "null"),
    (dict(vc=None), INVALID, "null"),
    (dict(kc=P + 1), INVALID, "aligned"),
    (dict(rows=P + 2), INVALID, "aligned"),
    (dict(dtype=9), UNSUPPORTED, "dtype"),
    (dict(layout=False), INVALID, "layout"),
    (dict(capacity=(1 << 30) + 1), UNSUPPORTED, "2^30"),
])
def test_compact_refused(lib, kw, status, needle):
    assert compact(lib, shape(), **kw) == status
    assert needle in error(lib)


@pytest.mark.parametrize("kw,needle", [
    (dict(block_size=0), "block_size"), (dict(num_blocks=-1), "num_blocks"), (dict(E=9000), "8192"),
    (dict(W=1 << 15), "2^15"), (dict(Ev=-1), "negative"),
])
def test_compact_shapes_refused(lib, kw, needle):
    assert compact(lib, shape(**kw)) in (INVALID, UNSUPPORTED)
    assert needle in error(lib)


def meta(lib, F=1, W=2, S=4, R=64, round_dtype=-1, **ptr):
    names = ("loc", "cos", "sin", "views", "rows", "fl", "order", "parents", "inv")
    a = {n: ptr.get(n, P) for n in names}
    return lib.dvattn_tree_metadata(*(a[n] for n in names), 1.0, round_dtype, F, W, S, R, None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(W=-1), INVALID, "negative"),
    (dict(R=7), UNSUPPORTED, "rotary_dim"),
    (dict(R=-2), UNSUPPORTED, "rotary_dim"),
    (dict(round_dtype=5), UNSUPPORTED, "round_dtype"),
    (dict(S=4097), UNSUPPORTED, "drafted nodes"),
    (dict(F=4097), UNSUPPORTED, "views"),
    (dict(F=4096, W=1 << 10, S=4096), UNSUPPORTED, "one launch"),
    (dict(loc=None), INVALID, "null"),
    (dict(parents=None), INVALID, "null"),
    (dict(views=None), INVALID, "null"),
    (dict(views=None, S=0), INVALID, "null"),
    (dict(rows=None, F=0), INVALID, "null"),
    (dict(order=None, S=0), INVALID, "null"),
    (dict(F=0, W=1 << 24), UNSUPPORTED, "one launch"),
    (dict(inv=None), INVALID, "null"),
    (dict(cos=P + 2), INVALID, "aligned"),
])
def test_metadata_refused(lib, kw, status, needle):
    assert meta(lib, **kw) == status
    assert needle in error(lib)


def test_wrappers_and_operators_refuse_host_tensors():
    import dvattention_amd as dv
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="mass or out"):
        dv.dvattn_paged_key_mass(None, None, None, None, None, None, None, None, 1.0, decay=0.0)
    with pytest.raises(ValueError, match="budget"):
        dv.dvattn_kv_select(torch.zeros(1, 1, 4), i, i, 3, rows=torch.zeros(1, 1, 2, dtype=torch.int32))
    with pytest.raises(NotImplementedError):
        dv.dvattn_kv_select(torch.zeros(1, 1, 4), i, i, 2)
    with pytest.raises(NotImplementedError):
        dv.dvattn_paged_kv_compact(i.view(1, 1, 1), i, torch.zeros(1, 4, 1, 8), torch.zeros(1, 4, 1, 8), i.view(1, 1))
