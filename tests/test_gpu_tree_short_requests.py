"""treeAttention over batches in which requests of several key tiles stand between runs of requests of one: a block then
walks from a part that both groups of its threads work on through many that only one of them does, longer runs than it
keeps parts in sight."""
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT
from test_gpu_tree_attention import TreeCase

pytestmark = pytest.mark.gpu


@pytest.fixture
def strict():
    """An engine that raises where a call would otherwise be tried again and end in zeros."""
    engine = pam.PagedAttentionEngine()
    engine.enableGracefulDegradation = False
    engine.maxRetries = 1
    yield engine
    engine.close()


@pytest.mark.parametrize("dtype", [DT.float16, DT.bfloat16, DT.float8], ids=lambda d: d.name)
@pytest.mark.parametrize("lens,sizes,kv_heads", [
    ([200, 0] * 100, [2, 1] * 100, 8), ([0] * 30 + [300] + [0] * 200, [1] * 231, 8), (([500] + [0] * 40) * 12, ([3] + [2] * 40) * 12, 2),
    ([130, 0, 0, 0] * 60, [4, 1, 0, 2] * 60, 8), ([0] * 400 + [5000, 0, 0], [33] * 403, 1)], ids=range(5))
def test_runs_of_requests_of_one_tile(strict, dtype, lens, sizes, kv_heads):
    TreeCase(121, lens, sizes, heads=kv_heads, kv_heads=kv_heads, dtype=dtype, dim=64).check(strict)
    assert strict.lastError is None


def test_wide_form_between_short_requests(strict):
    """More than 128 rows under a KV head somewhere in the batch: two query tiles for all of it."""
    lens, sizes = ([300, 700] + [0] * 30) * 8, ([20, 40] + [1] * 30) * 8
    TreeCase(122, lens, sizes, heads=32, kv_heads=8, dim=64).check(strict)
