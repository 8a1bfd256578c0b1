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
