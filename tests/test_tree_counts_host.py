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
