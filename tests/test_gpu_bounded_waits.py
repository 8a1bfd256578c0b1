"""A wait inside a kernel that runs out is reported by pamc_synchronize wherever the launch came from: an asynchronous
call, a replayed graph, with other calls in between.  (A limit of one cycle makes the wait for the first tile run out;
the kernel then returns through its error exit.)"""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT
from test_gpu_step_plan import CASES, PlanCase
from test_gpu_tree_attention import TreeCase

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
RAN_OUT = "bounded wait ran out"


class Waits:
    def __init__(self):
        self.engine = pam.PagedAttentionEngine()
        self.engine.enableGracefulDegradation = False
        self.case = TreeCase(81, [3000, 500, 70], [40, 9, 3], dtype=DT.float16)
        self.out = self.engine.makeBufferFrom(np.zeros(self.case.q.shape, np.float16))
        self.request = self.case.request(self.engine, self.out)
        self.request.workspace = self.engine.makeBuffer(self.engine.treeAttentionWorkspace(self.request))
        self.engine.treeAttention(self.request)
        self.want = self.result()
        self.stream = torch.cuda.Stream()
        self.engine.setStream(self.stream.cuda_stream)

    def result(self):
        return self.out.download(np.float16, self.case.q.shape)

    def clear(self):
        self.out.upload(np.zeros(self.case.q.shape, np.float16))

    def record(self, limit):
        self.engine.setWaitLimit(limit)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=self.stream):
            self.engine.treeAttention(self.request)
        self.engine.setWaitLimit(0)
        return graph

    def replay(self, graph):
        with torch.cuda.stream(self.stream):
            graph.replay()
        torch.cuda.synchronize()

    def close(self):
        self.engine.setStream(None)
        self.engine.close()


@pytest.fixture
def waits():
    w = Waits()
    yield w
    w.close()


def test_replays_that_run_out_are_reported(waits):
    short, usual = waits.record(1), waits.record(0)
    waits.engine.synchronize()
    for _ in range(3):
        waits.replay(short)
        with pytest.raises(pam.PagedAttentionError, match=RAN_OUT):
            waits.engine.synchronize()
        waits.engine.synchronize()                      # (reported once)
        waits.clear()
        waits.replay(usual)
        waits.engine.synchronize()
        assert np.array_equal(waits.result(), waits.want)
    del short, usual


def test_other_calls_do_not_take_the_report(waits):
    graph = waits.record(1)
    plan = lambda: PlanCase(82, **CASES["tree"]).check(waits.engine)
    plan()                                              # after the recording
    waits.replay(graph)
    plan()                                              # after the replay
    with pytest.raises(pam.PagedAttentionError, match=RAN_OUT):
        waits.engine.synchronize()
    waits.replay(graph)
    waits.clear()
    waits.engine.treeAttention(waits.request)           # starts behind the expired one, and is right
    assert np.array_equal(waits.result(), waits.want)
    with pytest.raises(pam.PagedAttentionError, match=RAN_OUT):
        waits.engine.synchronize()
    waits.engine.synchronize()
    del graph


@pytest.mark.parametrize("between", ["nothing", "plan", "attention"])
def test_asynchronous_calls_that_run_out_are_reported(waits, between):
    waits.engine.setWaitLimit(1)
    waits.engine.setAsync(True)
    waits.engine.treeAttention(waits.request)
    waits.engine.setAsync(False)
    waits.engine.setWaitLimit(0)
    if between == "plan":
        PlanCase(83, **CASES["decode step"]).check(waits.engine)
    if between == "attention":
        waits.clear()
        waits.engine.treeAttention(waits.request)
        assert np.array_equal(waits.result(), waits.want)
    with pytest.raises(pam.PagedAttentionError, match=RAN_OUT):
        waits.engine.synchronize()
    waits.engine.synchronize()
    waits.clear()
    waits.engine.treeAttention(waits.request)
    assert np.array_equal(waits.result(), waits.want)


def test_calls_for_several_layers_do_not_take_the_report(waits):
    """They wait once at their end; a prefill on the tensor cores starts although an earlier wait ran out."""
    engine, rng = waits.engine, np.random.default_rng(84)
    up, rows = engine.makeBufferFrom, 40
    layer = pam.PagedLayerSpec(128, 4, 2, 16, DT.float16)
    q = up(rng.standard_normal((rows, 4, 128)).astype(np.float16))
    pools = [up(rng.standard_normal((3, 2, 16, 128)).astype(np.float16)) for _ in range(2)]
    table, outs = up(np.array([2, 0, 1], np.int32)), [up(np.zeros((rows, 4, 128), np.float16)) for _ in range(2)]
    prefill = lambda out: engine.prefillLayers([q, q], *pools, table, [out, out], rows, [layer, layer])
    prefill(outs[0])
    graph = waits.record(1)
    waits.replay(graph)
    prefill(outs[1])
    assert np.array_equal(*(x.download(np.float16, (rows, 4, 128)) for x in outs))
    with pytest.raises(pam.PagedAttentionError, match=RAN_OUT):
        engine.synchronize()
    prefill(outs[1])
    engine.synchronize()
    del graph
