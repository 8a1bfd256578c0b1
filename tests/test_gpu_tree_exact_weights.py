"""The bits of bfloat16 weights in treeAttention: 16 for requests that see fewer than 256 keys, and for all where the caller
asks for them.  Half of the keys score zero and half a little more, with values that cancel, so that a weight rounded to 8
bits shows in full.  Tolerances as in test_gpu_tree_attention.py with 2^-16 for the rounding of a weight (what is left of
it after 8 bits, 2^-8 of it at most, rounded to 8 bits)."""
import numpy as np
import pytest

import test_gpu_tree_attention as base
from gpu_helpers import DT, from_io, to_storage

pytestmark = pytest.mark.gpu


def cancelling(lens, sizes, dim):
    case = base.TreeCase(95, lens, sizes, dtype=DT.bfloat16, dim=dim, kind="star", poison=False)
    bf16 = lambda x: from_io(to_storage(np.full(1, x, np.float32), DT.bfloat16), DT.bfloat16)[0]
    # the query whose weight lies farthest from a bfloat16 number
    queries = [bf16(x / dim ** 0.5) for x in np.linspace(0.05, 0.6, 200)]
    weight = lambda q: np.exp(-float(q) * dim ** 0.5)
    query = max(queries, key=lambda q: abs(bf16(weight(q)) / weight(q) - 1))
    assert abs(bf16(weight(query)) / weight(query) - 1) > 2.0 ** -9.5
    one = lambda x: to_storage(np.full(1, x, np.float32), DT.bfloat16)[0]
    case.q[:], case.k[:], case.v[:] = one(query), 0, 0
    case.k_pool[:, :, 0::2], case.k_pool[:, :, 1::2] = one(1), 0
    case.v_pool[:, :, 0::2], case.v_pool[:, :, 1::2] = one(1), one(-1 / weight(query))
    return case


# few rows and a short list: the mma kernel, as with head_dim 48; 20 and 40 rows: tcgen05 with one and two row tiles
@pytest.mark.parametrize("dim,sizes", [(128, [3]), (128, [20, 7]), (128, [40, 7]), (80, [20, 7]), (48, [3]), (48, [40, 9])])
def test_bits_of_bfloat16_weights(engine, monkeypatch, dim, sizes):
    monkeypatch.setitem(base.WEIGHT, DT.bfloat16, 2.0 ** -16)
    short, long = (cancelling([n] * len(sizes), sizes, dim) for n in (180, 1500))
    usual = short.check(engine)
    wide = long.run(engine)
    try:
        engine.setPrefillExactWeights(2)
        assert np.array_equal(short.run(engine), usual)
        exact = long.check(engine)
        engine.setPrefillExactWeights(0)
        rounded = short.run(engine)
        assert np.array_equal(long.run(engine), wide)
    finally:
        engine.setPrefillExactWeights(1)
    owned = slice(0, short.starts[-1])
    assert (rounded[owned] != usual[owned]).all() and (wide[owned] != exact[owned]).all()
