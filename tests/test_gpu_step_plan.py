"""planStep and acceptTree on the GPU against the plain restatements: whole numbers, equal."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from oracle import step_oracle as so

pytestmark = pytest.mark.gpu


def make_tree(rng, n, kind="random"):
    if kind == "chain":
        return np.arange(n, dtype=np.int32) - 1
    if kind == "star":
        return np.where(np.arange(n) == 0, -1, 0).astype(np.int32)
    if kind == "odd":                                   # several roots, parents behind or at the node, far below zero
        p = rng.integers(-3, n + 3, n).astype(np.int32)
        return p
    i = np.arange(n)
    return np.where(i == 0, -1, i - 1 - np.floor(rng.random(n) * np.minimum(i, 5)).astype(int)).astype(np.int32)


class PlanCase:
    def __init__(self, seed, lens, new, block, max_new, spare_rows=0, stride=None, num_lists=None, width=None, index=None,
                 tree=None, words=0, slots=True, negative_entries=False):
        rng = np.random.default_rng(seed)
        self.B = len(lens)
        self.lens, self.new = np.array(lens, np.int32), np.array(new, np.int32)
        self.block, self.max_new = block, max_new
        n = np.clip(self.new, 0, max_new)
        self.rows = max(1, int(n.sum()) + spare_rows)
        need = max(1, int(((np.maximum(self.lens, 0) + n + block - 1) // block).max()))
        self.stride = need if stride is None else stride
        self.num_lists = self.B if num_lists is None else num_lists
        self.lists = rng.integers(0, 10000, (self.num_lists, self.stride)).astype(np.int32)
        if negative_entries:
            self.lists[rng.random(self.lists.shape) < 0.2] = -1
        self.width = need + 1 if width is None else width
        self.index = None if index is None else np.array(index, np.int32)
        self.words = words
        self.parents = None
        self.slots = slots and tree is None
        if tree is not None:
            self.parents = np.full(self.rows, -1, np.int32)
            at = 0
            for c in n:
                c = min(int(c), self.rows - at)
                self.parents[at:at + c] = make_tree(rng, c, tree)
                at += c

    def run(self, engine, host=False):
        put = (lambda a: a) if host else engine.makeBufferFrom
        out = dict(tables=np.full((self.B, self.width), 77, np.int32), totals=np.full(self.B, 77, np.uint32),
                   starts=np.full(self.B + 1, 77, np.int32), positions=np.full(self.rows, 77, np.int32))
        if self.slots:
            out["slots"] = np.full(self.rows, 77, np.int64)
        if self.words:
            out["masks"] = np.full((self.rows, self.words), 77, np.uint32)
        bufs = {k: put(v) for k, v in out.items()}
        opt = lambda a: None if a is None else put(a)
        engine.planStep(pam.PagedStepPlanRequest(
            blockLists=put(self.lists), lengths=put(self.lens), newTokens=put(self.new), batchSize=self.B,
            numLists=self.num_lists, listStride=self.stride, blockSize=self.block, numRows=self.rows,
            maxNewTokens=self.max_new, listIndex=opt(self.index), parents=opt(self.parents), tables=bufs["tables"],
            maxNumBlocks=self.width, totalLengths=bufs["totals"], rowStarts=bufs["starts"], positions=bufs["positions"],
            slots=bufs.get("slots"), masks=bufs.get("masks"), maskWords=self.words))
        assert engine.lastStats.operation == pam.Operation.planStep
        return out if host else {k: bufs[k].download(v.dtype, v.shape) for k, v in out.items()}

    def check(self, engine, host=False):
        got = self.run(engine, host)
        want = so.plan_step(self.lists, self.lens, self.new, self.rows, self.max_new, self.block, self.index, self.parents,
                            self.width, self.words)
        for name, value in got.items():
            assert np.array_equal(value, want[name]), name


CASES = {
    "one token, one request": dict(lens=[0], new=[1], block=16, max_new=1),
    "decode step": dict(lens=[5, 0, 16, 15, 300], new=[1] * 5, block=16, max_new=1, spare_rows=3),
    "some idle": dict(lens=[5, 7, 9], new=[0, 4, 0], block=4, max_new=4, spare_rows=2, words=1),
    "all idle": dict(lens=[5, 7], new=[0, -3], block=4, max_new=4, spare_rows=5, words=1),
    "clamped": dict(lens=[-4, 7, 9], new=[9, -1, 3], block=24, max_new=5, words=2),
    "short lists": dict(lens=[100, 30], new=[9, 70], block=16, max_new=64, stride=4, words=2),
    "negative entries": dict(lens=[100, 30, 2], new=[9, 70, 33], block=8, max_new=70, words=3, negative_entries=True),
    "index": dict(lens=[10, 20, 30], new=[3, 4, 5], block=16, max_new=5, num_lists=7, index=[6, 0, 3]),
    "bad index": dict(lens=[10, 20, 30], new=[3, 4, 5], block=16, max_new=5, num_lists=7, index=[7, -1, 3]),
    "narrow table": dict(lens=[100, 130], new=[40, 1], block=16, max_new=40, width=3),
    "long prompts": dict(lens=[0, 3000, 17], new=[5000, 2049, 4096], block=16, max_new=5000, spare_rows=700),
    "wide table": dict(lens=[70000, 3], new=[1, 1], block=16, max_new=1, width=4500),
    "tree": dict(lens=[100, 0, 31], new=[17, 64, 1], block=16, max_new=64, tree="random", words=2, spare_rows=4),
    "tree without masks": dict(lens=[100, 31], new=[17, 20], block=16, max_new=20, tree="random"),
    "odd parents": dict(lens=[100, 0, 31], new=[17, 40, 1], block=16, max_new=40, tree="odd", words=2),
    "chain of 1024": dict(lens=[100, 12], new=[1024, 1000], block=16, max_new=1024, tree="chain", words=32),
    "star": dict(lens=[100, 12], new=[1000, 33], block=16, max_new=1024, tree="star", words=33),
}


@pytest.mark.parametrize("name", CASES)
def test_plan_matches_the_plain_form(engine, name):
    PlanCase(101, **CASES[name]).check(engine)


def test_plan_rows_cut_off_and_many_requests(engine):
    rng = np.random.default_rng(7)
    case = PlanCase(102, rng.integers(0, 400, 700), rng.integers(0, 9, 700), 16, 8, words=1)
    case.check(engine)
    case.rows -= 1000                                   # the last requests lose their rows
    case.check(engine)
    case.rows = 1
    case.check(engine)


def test_plan_takes_host_buffers(engine):
    PlanCase(103, **CASES["clamped"]).check(engine, host=True)
    PlanCase(103, **CASES["tree"]).check(engine, host=True)


def test_plan_without_outputs_but_one(engine):
    case = PlanCase(104, **CASES["decode step"])
    starts = engine.makeBufferFrom(np.zeros(case.B + 1, np.int32))
    engine.planStep(pam.PagedStepPlanRequest(
        blockLists=engine.makeBufferFrom(case.lists), lengths=engine.makeBufferFrom(case.lens),
        newTokens=engine.makeBufferFrom(case.new), batchSize=case.B, numLists=case.num_lists, listStride=case.stride,
        blockSize=16, numRows=case.rows, maxNewTokens=1, rowStarts=starts))
    assert list(starts.download(np.int32, (case.B + 1,))) == [0, 1, 2, 3, 4, 5]


def accept_case(engine, seed, sizes, kind="random", max_tree=None, max_path=None, width=40, agree=0.8, gap=0, first=0, host=False):
    rng = np.random.default_rng(seed)
    B, block = len(sizes), 16
    starts = (first + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)
    rows = max(1, int(starts[-1]) + gap)
    parents, draft, target = np.full(rows, -1, np.int32), rng.integers(0, 9, rows).astype(np.int32), rng.integers(0, 9, rows).astype(np.int32)
    for b, n in enumerate(sizes):
        s = starts[b]
        parents[s:s + n] = make_tree(rng, n, kind)
        for i in range(n):
            p = so.parent_of(parents[s + i], i)
            if p >= 0 and rng.random() < agree:
                target[s + p] = draft[s + i]
    lens = rng.integers(-1, 600, B).astype(np.int32)
    tables = rng.integers(-1, 5000, (B, width)).astype(np.int32)
    most = max(sizes) if max_tree is None else max_tree
    most = max(most, 1)
    depth = most if max_path is None else max_path
    put = (lambda a: a) if host else engine.makeBufferFrom
    out = dict(slots=np.full(rows, 77, np.int64), counts=np.full(B, 77, np.int32), path=np.full((B, depth), 77, np.int32),
               next=np.full(B, 77, np.int32), totals=np.full(B, 77, np.uint32))
    bufs = {k: put(v) for k, v in out.items()}
    engine.acceptTree(pam.PagedAcceptRequest(
        rowStarts=put(starts), parents=put(parents), draftTokens=put(draft), targetTokens=put(target), lengths=put(lens),
        batchSize=B, numRows=rows, maxTree=most, blockTables=put(tables), maxNumBlocks=width, blockSize=block,
        slots=bufs["slots"], acceptedCounts=bufs["counts"], acceptedRows=bufs["path"], maxPath=depth,
        nextTokens=bufs["next"], newLengths=bufs["totals"]))
    assert engine.lastStats.operation == pam.Operation.acceptTree
    got = out if host else {k: bufs[k].download(v.dtype, v.shape) for k, v in out.items()}
    want = so.accept_tree(starts, parents, draft, target, lens, rows, most, depth, tables, block)
    for name, value in got.items():
        assert np.array_equal(value, want[name]), name
    return want


@pytest.mark.parametrize("sizes,kw", [
    ([1], {}), ([5, 0, 16, 1], dict(gap=3)), ([64] * 9, {}), ([33, 64, 2], dict(kind="odd")), ([0, 0], dict(gap=2)),
    ([1024, 700, 3], dict(kind="chain", agree=1.0, width=110)), ([1000], dict(kind="star")),
    ([40, 50], dict(max_tree=20)), ([40, 50], dict(kind="chain", agree=1.0, max_path=7)),
    ([10, 12], dict(first=4, gap=1)), ([30, 30], dict(kind="chain", agree=1.0, width=2)), ([9, 9], dict(agree=0.0)),
])
def test_accept_matches_the_plain_form(engine, sizes, kw):
    accept_case(engine, 111, sizes, **kw)


def test_accept_many_requests_and_host_buffers(engine):
    rng = np.random.default_rng(3)
    want = accept_case(engine, 112, list(rng.integers(0, 65, 300)), width=50)
    assert want["counts"].max() > 3                     # paths of some length are among them
    accept_case(engine, 113, [5, 3, 0], host=True)
