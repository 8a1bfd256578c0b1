"""The requests of a speculative step know what their index buffers hold."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from test_step_host import accept, norm, norm_backward, plan, tree

FIELDS = {
    plan: dict(int32="blockLists listIndex lengths newTokens parents tables totalLengths rowStarts positions masks", int64="slots"),
    accept: dict(int32="rowStarts parents draftTokens targetTokens lengths blockTables acceptedCounts acceptedRows nextTokens newLengths",
                 int64="slots"),
    norm: dict(int32="positions", int64="slots", float32="invFreq"),
    norm_backward: dict(int32="positions", int64="slots", float32="invFreq dQWeight dKWeight"),
    tree: dict(int32="blockTables cacheLengths rowStarts masks positions", float16="kScaleBuffer vScaleBuffer"),
}
CASES = [(make, kind, name) for make, kinds in FIELDS.items() for kind, names in kinds.items() for name in names.split()]


@pytest.mark.parametrize("make,kind,name", CASES, ids=[f"{m.__name__}-{n}" for m, _, n in CASES])
def test_other_types_are_refused(make, kind, name):
    """An int64 tensor where int32 is read would pass every check of its size."""
    torch = pytest.importorskip("torch")
    request = make()
    for other in {"int32", "int64", "float32", "float64", "float16", "bool"} - {kind}:
        for value in (np.zeros(4096, other), torch.zeros(4096, dtype=getattr(torch, other))):
            with pytest.raises(TypeError, match=f"{name}.*{kind}"):
                setattr(request, name, value)
            with pytest.raises(TypeError, match=f"{name}.*{kind}"):
                make(**{name: value})
    for value in (np.zeros(4096, kind), torch.zeros(4096, dtype=getattr(torch, kind)), None):
        setattr(request, name, value)
        assert getattr(request, name) is value
    if kind.startswith("int"):
        setattr(request, name, np.zeros(4096, "u" + kind))


def test_buffers_without_a_type_are_taken():
    request = tree()
    from pagedattentionmetal_b200._cabi import PamBuffer
    request.cacheLengths = PamBuffer(4096, 64)
    assert request._c.cache_lengths.bytes == 64
    request.q = np.zeros(64, np.uint16)                 # (rows: the layer says what they hold)
    assert isinstance(request, pam.PagedTreeAttentionRequest)


def views():
    torch = pytest.importorskip("torch")
    wide = np.zeros((6, 512), np.float16)
    return wide, torch.from_numpy(wide)


def test_views_of_rows_reach_from_their_first_to_their_last_element():
    for wide in views():
        address = wide.ctypes.data if isinstance(wide, np.ndarray) else wide.data_ptr()
        for view in (wide[:, 128:256], wide[:, 128:256].reshape(6, 2, 64)):
            request = tree(v=view, vStride=512)
            assert request._c.v.ptr == address + 256 and request._c.v.bytes == (5 * 512 + 128) * 2


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_rows_that_are_not_in_one_piece_are_refused(name):
    for wide in views():
        for view in (wide[:, ::2], wide.T, wide.reshape(6, 8, 64)[:, ::2], wide.reshape(6, 8, 64)[:, :, :32]):
            with pytest.raises(ValueError, match=name):
                tree(**{name: view})
    with pytest.raises(ValueError, match=name):
        tree(**{name: np.zeros((6, 512), np.float16)[::-1]})


@pytest.mark.parametrize("make,name", [(make, name) for make, _, name in CASES] +
                         [(tree, "output"), (tree, "kPool"), (tree, "vPool"), (norm, "qWeight"), (norm_backward, "dQOut"), (norm_backward, "dKOut")])
def test_views_of_anything_but_rows_are_refused(make, name):
    """They have no stride in the request: every other element would be read in their place."""
    torch = pytest.importorskip("torch")
    kind = next((k for m, k, n in CASES if m is make and n == name), "float16")
    for value in (np.zeros((64, 64), kind)[:, 0], torch.zeros(64, 64, dtype=getattr(torch, kind))[:, 0]):
        with pytest.raises(ValueError, match=name):
            make(**{name: value})
