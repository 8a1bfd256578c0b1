"""treeAttention where the result comes from weights far below a row's largest: two tokens at the start of the cache with
a high score and values of zero, before hundreds that all score zero.  The weights that go into the second product as
float16 must not lose their bits to its small numbers (below 2^-14), above all since equal weights are all rounded the
same way.  Tolerances as in test_gpu_tree_attention.py: half a float16 step, relative, for each weight."""
import numpy as np
import pytest

from gpu_helpers import DT, to_storage
from test_gpu_tree_attention import TreeCase

pytestmark = pytest.mark.gpu

# head_dim -> queries (the keys are ones): scores of about 14.3, the weight of a token is then about 10.5 * 2^-24.
# 128: tcgen05, 48: mma, 40 behind float8 pages: the general kernel, whose weights are float32.
QUERIES = {128: 1.2627, 48: 2.062, 40: 2.2588}


@pytest.mark.parametrize("dim", QUERIES)
@pytest.mark.parametrize("dtype", [DT.float16, DT.float8, DT.bfloat16], ids=lambda d: d.name)
def test_many_small_weights_behind_two_large_ones(engine, dim, dtype):
    """(So many requests that a block has whole ones: a piece of a request without the large weights is exact anyway.)"""
    case = TreeCase(91, [900] * 40, [1, 2] * 20, heads=8, kv_heads=8, dtype=dtype, dim=dim, poison=False)
    one = lambda x: to_storage(np.full(1, x, np.float32), dtype)[0]
    case.q[:], case.k[:], case.v[:] = one(QUERIES[dim]), 0, one(0.125)
    case.k_pool[:] = 0
    if dtype == DT.float8:
        case.v_pool[:], case.v_scale[:], case.k_scale[:] = 0x70, 2.0 ** -10, 1       # (0x70: 128)
    else:
        case.v_pool[:] = one(0.125)
    for token in (0, 128):                               # (tiles of 128 keys alternate between two groups of threads)
        blk = case.tables[:, token // 16]
        case.k_pool[blk, :, token % 16] = 0x38 if dtype == DT.float8 else one(1.0)
        case.v_pool[blk, :, token % 16] = 0
    out = case.check(engine)
    assert (out[:case.starts[-1]] > 0).all()
