"""treeAttention over FP8 pages whose scales are not finite numbers: they reach the rows that see such a page, on
every kernel alike, and no others.  (A float16 key or value that is infinite gives its page an infinite scale when it
is appended.)  Tolerances as in test_gpu_tree_attention.py."""
import numpy as np
import pytest

from gpu_helpers import DT
from test_gpu_tree_attention import TreeCase

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:invalid value encountered")]

# head_dim -> kernel: 128 and 80 tcgen05, 48 mma, 40 and 256 the general one
DIMS = [128, 80, 48, 40, 256]
BAD = [np.inf, np.nan]


def wider(case, columns, entry):
    """The block tables with `columns` more entries, all `entry`."""
    case.tables = np.concatenate([case.tables, np.full((case.B, columns), entry, np.int32)], 1)
    case.width += columns
    return case


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("sizes", [[3, 1, 2], [40, 9, 33]])
def test_scales_of_pages_behind_the_last_token(engine, dim, what, sizes):
    """Unused table entries name a block that belongs to somebody else."""
    case = TreeCase(71, [200, 37, 0], sizes, dtype=DT.float8, dim=dim)
    free = np.setdiff1d(np.arange(case.n_pool), case.tables)[0]
    case.tables[case.tables < 0] = free
    wider(case, 9, free)
    case.k_scale[free] = case.v_scale[free] = what
    case.k_pool[free] = case.v_pool[free] = 0x7E
    case.check(engine)
    case.k_scale[free] = 1
    case.check(engine)
    case.k_scale[free], case.v_scale[free] = what, 1
    case.check(engine)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("where", ["k_scale", "v_scale"])
def test_scales_of_pages_before_and_at_the_edge_of_a_window(engine, dim, what, where):
    """A page that only the nodes near the root see, and the page before it, which nobody sees."""
    case = TreeCase(72, [300, 64], [40, 33], dtype=DT.float8, dim=dim, window=90, kind="chain")
    edge = (300 + 1 - 90) // 16                          # the root sees tokens from 211 on
    getattr(case, where)[case.tables[0, edge], 0] = what
    getattr(case, where)[case.tables[0, edge - 1]] = what
    out = case.check(engine, finite=False)
    first = case.starts[0]
    assert not np.isfinite(out[first, :4]).any()         # KV head 0's query heads
    assert np.isfinite(out[first:case.starts[2], 4:]).all() and np.isfinite(out[first + 13:case.starts[1]]).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("where", ["k_scale", "v_scale"])
@pytest.mark.parametrize("lens", [[130, 70], [5000, 40]])
def test_scales_of_pages_that_every_row_sees(engine, dim, what, where, lens):
    case = TreeCase(73, lens, [20, 40], dtype=DT.float8, dim=dim)
    blk = case.tables[0, 3]
    getattr(case, where)[blk, 1] = what
    case.v_pool[blk, :, :, ::7] = 0x38                   # one: all infinities of a column alike
    out = case.check(engine, finite=False)
    a, b, c = case.starts
    assert not np.isfinite(out[a:b, 4:]).any() and np.isfinite(out[a:b, :4]).all() and np.isfinite(out[b:c]).all()
    if where == "v_scale" and what == np.inf:
        assert (out[a:b, 4:, ::7] == np.inf).all()
