"""The weight gradients of normRotateBackward as exact sums: rows of ones and minus ones (their norm is one), whole numbers
as gradients, positions of zero.  Every product and partial sum is a whole number below 2^24, so that a row, a head or a
block's share that is lost or counted twice shows whatever the order of summation."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT, to_storage

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16, DT.bfloat16], ids=lambda d: d.name)
@pytest.mark.parametrize("rows", [1, 5, 1183, 5000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (32, 8, 128), (3, 1, 33), (40, 4, 128)])
@pytest.mark.parametrize("pages", [False, True])
def test_weight_gradients_count_every_row_once(engine, dtype, rows, heads, kv_heads, dim, pages):
    rng = np.random.default_rng(101)
    up, store = engine.makeBufferFrom, lambda a: to_storage(np.asarray(a, np.float32), dtype)
    sign = lambda *s: rng.integers(0, 2, s) * 2 - 1
    q, k = sign(rows, heads, dim), sign(rows, kv_heads, dim)
    dq, dk = rng.integers(-8, 9, (rows, heads, dim)), rng.integers(-8, 9, (rows, kv_heads, dim))
    positions = np.where(rng.random(rows) < 0.1, -1, 0).astype(np.int32)
    live = positions >= 0
    block = 16
    blocks = -(-rows // block) + 1
    slots = rng.permutation(blocks * block)[:rows].astype(np.int64)
    slots[rng.random(rows) < 0.1] = -1
    grads = dict(dKOut=up(store(dk)))
    if pages:
        pool = np.full((blocks, block, kv_heads, dim), 3)
        pool.reshape(-1, kv_heads, dim)[slots[slots >= 0]] = dk[slots >= 0]
        pool = store(pool.transpose(0, 2, 1, 3))
        dk = np.where((slots >= 0)[:, None, None], dk, 0)
        es = pool.itemsize
        grads = dict(dKPool=up(pool), dVPool=up(pool), slots=up(slots), dV=engine.makeBuffer(rows * kv_heads * dim * es))
    ones = up(store(np.ones(dim)))
    es = store(q).itemsize
    dwq, dwk = up(np.full(dim, 7, np.float32)), up(np.full(dim, 7, np.float32))
    rotary = dim // 2 // 16 * 32
    engine.normRotateBackward(pam.PagedNormRotateBackwardRequest(
        q=up(store(q)), k=up(store(k)), qWeight=ones, kWeight=ones, positions=up(positions), dQOut=up(store(dq)), **grads,
        dQ=engine.makeBuffer(rows * heads * dim * es), dK=engine.makeBuffer(rows * kv_heads * dim * es), dQWeight=dwq, dKWeight=dwk,
        invFreq=up(np.linspace(1, 0, rotary // 2, dtype=np.float32)), numRows=rows, rotaryDim=rotary, epsilon=0.0,
        layer=pam.PagedLayerSpec(dim, heads, kv_heads, block, dtype)))
    assert np.array_equal(dwq.download(np.float32, (dim,)), (q * dq)[live].sum((0, 1)))
    assert np.array_equal(dwk.download(np.float32, (dim,)), (k * dk)[live].sum((0, 1)))
