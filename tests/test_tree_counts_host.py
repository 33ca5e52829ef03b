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
