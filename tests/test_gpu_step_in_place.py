"""acceptTree that adds to the lengths in place, as a recorded step does that is replayed again and again."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from oracle import step_oracle as so
from test_gpu_step_plan import make_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,batch", [(16, 8), (200, 40), (1024, 7)])
def test_new_lengths_over_lengths(engine, size, batch):
    rng = np.random.default_rng(111)
    rows, width = size * batch, 4096 // 16
    starts = (np.arange(batch + 1) * size).astype(np.int32)
    parents = np.concatenate([make_tree(rng, size, "chain" if b % 2 else "random") for b in range(batch)])
    draft, target = rng.integers(0, 2, rows).astype(np.int32), rng.integers(0, 2, rows).astype(np.int32)
    for b in range(1, batch, 2):                         # whole chains are accepted
        target[starts[b]:starts[b + 1] - 1] = draft[starts[b] + 1:starts[b + 1]]
    tables = rng.permutation(batch * width).reshape(batch, width).astype(np.int32)
    lens = rng.integers(0, 100, batch).astype(np.int32)
    up = engine.makeBufferFrom
    lengths, slots, counts = up(lens), up(np.zeros(rows, np.int64)), up(np.zeros(batch, np.int32))
    request = pam.PagedAcceptRequest(
        rowStarts=up(starts), parents=up(parents), draftTokens=up(draft), targetTokens=up(target), lengths=lengths, batchSize=batch,
        numRows=rows, maxTree=size, blockTables=up(tables), maxNumBlocks=width, blockSize=16, slots=slots, acceptedCounts=counts,
        newLengths=lengths)
    for _ in range(3):
        engine.acceptTree(request)
        want = so.accept_tree(starts, parents, draft, target, lens, rows, size, 1, tables, 16)
        assert np.array_equal(slots.download(np.int64, (rows,)), want["slots"])
        assert np.array_equal(counts.download(np.int32, (batch,)), want["counts"])
        lens = lengths.download(np.int32, (batch,))
        assert np.array_equal(lens, want["totals"].astype(np.int32))
