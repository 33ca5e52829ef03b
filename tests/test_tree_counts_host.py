"""Host-side refusals of the tree metadata's optional counts (CPU only)."""
import pytest
import torch

INVALID, UNSUPPORTED = 1, 2
P = 0x1000  # never dereferenced: every call below is refused, or empty


@pytest.fixture(scope="module")
def lib():
    from dvattention_amd import capi
    return capi.lib()


def meta(lib, F=1, W=2, S=4, R=64, **ptr):
    names = ("loc", "cos", "sin", "views", "rows", "fl", "order", "parents", "committed", "dropped", "inv")
    a = {n: ptr.get(n, P) for n in names}
    return lib.dvattn_tree_metadata_counts(*(a[n] for n in names), 1.0, -1, F, W, S, R, None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(dropped=P + 2), INVALID, "dropped"),
    (dict(committed=P + 1), INVALID, "committed"),
    (dict(dropped=None, loc=None), INVALID, "null"),
    (dict(W=-1), INVALID, "negative"),
    (dict(S=4097), UNSUPPORTED, "drafted nodes"),
])
def test_counts_refused(lib, kw, status, needle):
    assert meta(lib, **kw) == status
    assert needle in lib.dvattn_last_error().decode()


def test_empty_calls_succeed(lib):
    assert meta(lib, W=0) == 0 and meta(lib, W=0, dropped=None, committed=None) == 0


def test_schema_keeps_the_earlier_calls():
    import dvattention_amd  # noqa: F401
    schema = str(torch.ops.libdvatt.dvattn_tree_metadata.default._schema)
    assert "ScalarType? round_to=None, Tensor? dropped=None, Tensor? committed=None" in schema


def test_compaction_refuses_one_array_as_both_caches(lib):
    """Keys and values are moved separately: rows of an array that is both would be moved twice."""
    import ctypes

    from dvattention_amd import capi
    s = capi.Shape(F=0, W=2, Hq=0, Hkv=1, E=128, Ev=128, S=0, block_size=16, max_blocks_per_seq=4, total_q_tokens=0,
                   num_blocks=8, rotary_dim=0)
    lay = capi.KvLayout()
    p = ctypes.c_void_p(P)
    assert lib.dvattn_paged_kv_compact(2, p, p, p, p, 1, 4, p, None, None, 0, ctypes.byref(s), ctypes.byref(lay),
                                       None) == INVALID
    assert "same array" in lib.dvattn_last_error().decode()


@pytest.mark.parametrize("kw,capacity", [
    (dict(W=256, Hkv=1, Hq=16, S=4), 1 << 62),                   # W * Hkv * rows past 2^63
    (dict(W=256, Hkv=1, Hq=16, S=1), (1 << 63) - 1),
    (dict(W=1 << 20, S=1 << 22, F=1 << 21), 64),                  # W * S * F past 2^62
    (dict(W=1 << 22, S=2, F=0, max_blocks_per_seq=0), 64),        # one block of the plan too many
    (dict(W=(1 << 22) - 1, S=2, F=1, max_blocks_per_seq=0), 64),
])
def test_key_mass_beyond_a_launch_refused(lib, kw, capacity):
    """Sizes whose products leave 63 bits, and calls one launch cannot hold."""
    import ctypes

    from dvattention_amd import capi
    base = dict(F=1, W=2, Hq=16, Hkv=1, E=128, Ev=128, S=4, block_size=16, max_blocks_per_seq=4, total_q_tokens=0,
                num_blocks=8, rotary_dim=64)
    s = capi.Shape(**{**base, **kw})
    p = ctypes.c_void_p(P)
    for dtype in (0, 2):
        got = lib.dvattn_paged_key_mass(dtype, p, p, 1.0, capacity, 0.1, p, p, p, p, p, p, p, ctypes.byref(s), p,
                                        (1 << 64) - 1, None)
        assert got == UNSUPPORTED and "too many blocks" in lib.dvattn_last_error().decode()
