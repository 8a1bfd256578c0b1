"""The calls of a speculative step together, as a serving loop runs them: a toy attention layer
decodes drafted trees, commits what is accepted, and the next step over the grown cache agrees with a
cache that was filled token by token.  Eagerly, recorded into a graph and replayed, on other streams."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT
from oracle import step_oracle as so
from test_gpu_step_plan import make_tree

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

H, KVH, D, BLOCK = 8, 2, 64, 16
TORCH = {DT.float16: torch.float16, DT.bfloat16: torch.bfloat16, DT.float8: torch.float16, DT.float32: torch.float32}


class Step:
    """Static buffers and requests of a step of up to `rows` rows over `batch` requests."""

    def __init__(self, engine, batch, rows, max_new, blocks, dtype, width=16, cache=None, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        io = TORCH[dtype]
        z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device="cuda")
        self.engine, self.dtype, self.cache, self.rows, self.batch, self.width = engine, dtype, cache, rows, batch, width
        self.lists, self.lengths, self.new, self.parents = z(batch, width), z(batch), z(batch), z(rows)
        self.totals, self.starts, self.positions = z(batch), z(batch + 1), z(rows)
        self.words = -(-max_new // 32)
        self.masks, self.tables = z(rows, self.words), z(batch, width)
        self.wide = (H + 2 * KVH) * D
        self.qkv = torch.randn(rows, self.wide, generator=g, device="cuda").to(io)
        self.wq, self.wk = torch.rand(D, generator=g, device="cuda").to(io) + 0.5, torch.rand(D, generator=g, device="cuda").to(io) + 0.5
        self.freq = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
        self.q, self.k, self.out = z(rows, H, D, t=io), z(rows, KVH, D, t=io), z(rows, H, D, t=io)
        self.draft, self.target, self.slots = z(rows), z(rows), z(rows, t=torch.int64)
        self.counts, self.path, self.next, self.grown = z(batch), z(batch, max_new), z(batch), z(batch)
        layer = pam.PagedLayerSpec(D, H, KVH, BLOCK, dtype)
        pools = dict(kPool=cache.kPoolBuffer, vPool=cache.vPoolBuffer)
        self.plan = pam.PagedStepPlanRequest(
            blockLists=self.lists, lengths=self.lengths, newTokens=self.new, batchSize=batch, numLists=batch, listStride=width,
            blockSize=BLOCK, numRows=rows, maxNewTokens=max_new, parents=self.parents, tables=self.tables, maxNumBlocks=width,
            totalLengths=self.totals, rowStarts=self.starts, positions=self.positions, masks=self.masks, maskWords=self.words)
        q, k, v = self.qkv[:, :H * D], self.qkv[:, H * D:(H + KVH) * D], self.qkv[:, (H + KVH) * D:]
        self.v = v
        self.norm = pam.PagedNormRotateRequest(q=q, k=k, qWeight=self.wq, kWeight=self.wk, invFreq=self.freq, positions=self.positions,
                                               qOut=self.q, kOut=self.k, numRows=rows, rotaryDim=D, layer=layer, qStride=self.wide,
                                               kStride=self.wide)
        self.attention = pam.PagedTreeAttentionRequest(
            q=self.q, k=self.k, v=v, vStride=self.wide, blockTables=self.tables, cacheLengths=self.lengths, rowStarts=self.starts,
            masks=self.masks, positions=self.positions, output=self.out, batchSize=batch, maxNumBlocks=width, numRows=rows,
            maxNewTokens=max_new, maskWords=self.words, layer=layer, kScaleBuffer=cache.kScaleBuffer, vScaleBuffer=cache.vScaleBuffer, **pools)
        self.attention.workspace = torch.zeros(engine.treeAttentionWorkspace(self.attention), dtype=torch.uint8, device="cuda")
        self.accept = pam.PagedAcceptRequest(
            rowStarts=self.starts, parents=self.parents, draftTokens=self.draft, targetTokens=self.target, lengths=self.lengths,
            batchSize=batch, numRows=rows, maxTree=max_new, blockTables=self.lists, maxNumBlocks=width, blockSize=BLOCK,
            slots=self.slots, acceptedCounts=self.counts, acceptedRows=self.path, maxPath=max_new, nextTokens=self.next,
            newLengths=self.grown)

    def fill(self, rng, lens, sizes, lists):
        """New inputs in the static buffers."""
        parents = np.full(self.rows, 5, np.int32)
        draft, target = rng.integers(0, 50, self.rows).astype(np.int32), rng.integers(0, 50, self.rows).astype(np.int32)
        at = 0
        for n in sizes:
            parents[at:at + n] = make_tree(rng, n)
            for i in range(n):
                p = so.parent_of(parents[at + i], i)
                if p >= 0 and rng.random() < 0.8:
                    target[at + p] = draft[at + i]
            at += n
        put = lambda t, a: t.copy_(torch.from_numpy(np.ascontiguousarray(a)).view(t.shape))
        put(self.lists, lists)
        put(self.lengths, np.array(lens, np.int32))
        put(self.new, np.array(sizes, np.int32))
        for t, a in ((self.parents, parents), (self.draft, draft), (self.target, target)):
            put(t, a)
        self.qkv.copy_(torch.from_numpy(rng.standard_normal((self.rows, self.wide), dtype=np.float32)).to(self.qkv.dtype))
        torch.cuda.synchronize()

    def calls(self):
        self.engine.planStep(self.plan)
        self.engine.normRotate(self.norm)
        self.engine.treeAttention(self.attention)
        self.engine.acceptTree(self.accept)

    def snapshot(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.tables, self.totals, self.starts, self.positions, self.masks, self.q, self.k, self.out,
                                    self.slots, self.counts, self.path, self.next, self.grown)]


def lists_of(cache, ids, width):
    out = np.full((len(ids), width), -1, np.int32)
    for i, s in enumerate(ids):
        t = cache.getBlockTable(s)
        out[i, :len(t)] = t
    return out


@pytest.mark.parametrize("dtype", [DT.float16, DT.bfloat16, DT.float8, DT.float32], ids=lambda d: d.name)
def test_speculative_steps_equal_a_cache_filled_row_by_row(engine, dtype):
    """Three steps; after each, the pages hold exactly the rows of the accepted path (bit for bit what
    reshapeAndCache writes of them), and a causal step without a tree over the last path sees the same."""
    rng = np.random.default_rng(51)
    ids, width, max_new = [3, 9, 4], 16, 20
    cache = pam.KVCacheManager(engine, 64, BLOCK, D, KVH, dtype)
    plain = pam.KVCacheManager(engine, 64, BLOCK, D, KVH, dtype)
    for s in ids:
        for c in (cache, plain):
            c.allocateSequence(s)
            c.appendTokens(s, 200)                       # pages reserved ahead
    lists = lists_of(cache, ids, width)
    assert np.array_equal(lists, lists_of(plain, ids, width))
    lens = [0, 37, 90]
    for s, n in zip(ids, lens):
        if n:
            k, v = (rng.standard_normal((n, KVH, D)).astype(np.float32) for _ in range(2))
            as_io = lambda a: torch.from_numpy(a).to(TORCH[dtype]).cuda()
            k, v = as_io(k), as_io(v)
            torch.cuda.synchronize()
            for c in (cache, plain):
                engine.appendKV(c, s, k, v, 0, n, H)
    step = Step(engine, 3, 48, max_new, 64, dtype, width, cache)
    for sizes in ([1, 20, 13], [7, 0, 20], [20, 5, 9]):
        step.fill(rng, lens, sizes, lists)
        step.calls()
        torch.cuda.synchronize()
        starts = step.starts.cpu().numpy()
        want = so.accept_tree(starts, step.parents.cpu().numpy(), step.draft.cpu().numpy(), step.target.cpu().numpy(), lens, 48,
                              max_new, max_new, lists, BLOCK)
        assert np.array_equal(step.slots.cpu().numpy(), want["slots"]) and np.array_equal(step.next.cpu().numpy(), want["next"])
        # every row of the tree attends what a causal pass over its own path would
        for b in range(3):
            for r in {int(x) for x in want["path"][b] if x >= 0}:
                d = int(step.positions[r].item()) - lens[b]
                rows = torch.tensor([int(x) for x in want["path"][b][:d + 1]], device="cuda")
                n = len(rows)
                q, k, v = step.q[rows].contiguous(), step.k[rows].contiguous(), step.v[rows].contiguous()
                out = torch.zeros_like(q)
                i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
                request = pam.PagedTreeAttentionRequest(
                    q=q, k=k, v=v, kPool=cache.kPoolBuffer, vPool=cache.vPoolBuffer, blockTables=step.tables[b].contiguous(),
                    cacheLengths=i32(lens[b]), rowStarts=i32(0, n), output=out, batchSize=1, maxNumBlocks=width, numRows=n,
                    maxNewTokens=n, layer=step.attention.layer, kScaleBuffer=cache.kScaleBuffer, vScaleBuffer=cache.vScaleBuffer)
                torch.cuda.synchronize()                 # (the engine has a stream of its own)
                engine.treeAttention(request)
                torch.cuda.synchronize()
                # the same keys in another order of summation: a rounding of the output and of the weights each
                eps = torch.finfo(step.out.dtype).eps
                assert (out[-1].double() - step.out[r].double()).abs().max() <= 4 * eps * v.double().abs().max().clamp(min=4)
        values = step.v.contiguous()
        torch.cuda.synchronize()
        engine.reshapeAndCache(cache, step.k, values, step.slots, 48)
        for b, s in enumerate(ids):
            rows = torch.tensor([int(x) for x in want["path"][b] if x >= 0], device="cuda", dtype=torch.long)
            if len(rows):
                if dtype == DT.float8:                   # the scale of a block goes by the call: all requests in one
                    continue
                k, v = step.k[rows].contiguous(), step.v[rows].contiguous()
                torch.cuda.synchronize()
                engine.appendKV(plain, s, k, v, lens[b], len(rows), H)
        if dtype != DT.float8:
            for a, c in zip(cache.readPools()[:2], plain.readPools()[:2]):
                assert np.array_equal(a, c)
        lens = [int(x) for x in step.grown.cpu()]
        assert lens == [int(x) for x in want["totals"]]
    cache.close()
    plain.close()


@pytest.mark.parametrize("dtype", [DT.float16, DT.float32], ids=lambda d: d.name)
def test_recorded_step_replays_with_other_inputs(dtype):
    """One capture; replays with other lengths, trees and fewer rows give the bits of the eager calls; two graphs
    with workspaces of their own run at the same time."""
    dev = torch.device("cuda", 0)
    engine = pam.PagedAttentionEngine(0)
    cache = pam.KVCacheManager(engine, 64, BLOCK, D, KVH, dtype)
    rng = np.random.default_rng(52)
    for t in (cache.kPoolBuffer, cache.vPoolBuffer):
        host = torch.randn(t.bytes // TORCH[dtype].itemsize).to(TORCH[dtype])
        from pagedattentionmetal_b200._cabi import lib
        assert lib.pamc_memcpy(engine._ctx, t.ptr, host.data_ptr(), t.bytes, 0) == 0
    lists = rng.permutation(64)[:48].reshape(3, 16).astype(np.int32)
    steps = [Step(engine, 3, 48, 20, 64, dtype, 16, cache, seed=i) for i in range(2)]
    inputs = [([0, 37, 190], [1, 20, 13]), ([5, 200, 90], [7, 0, 20]), ([0, 0, 0], [0, 0, 0]), ([100, 16, 15], [16, 16, 16])]
    streams, graphs = [torch.cuda.Stream(dev) for _ in steps], []
    for step, stream in zip(steps, streams):
        step.fill(rng, *inputs[0], lists)
        step.calls()                                      # (kernels are loaded by their first call)
        graph = torch.cuda.CUDAGraph()
        engine.setStream(stream.cuda_stream)
        launches = engine.kernelLaunches
        with torch.cuda.graph(graph, stream=stream):
            step.calls()
        assert engine.kernelLaunches > launches
        graphs.append(graph)
    engine.setStream(None)
    for a in range(len(inputs)):
        eager = []
        for i, step in enumerate(steps):
            step.fill(rng, *inputs[(a + i) % len(inputs)], lists)
            step.calls()
            eager.append(step.snapshot())
            for t in (step.out, step.slots, step.masks):
                t.fill_(3)
        # (rows of no request keep what they held: compare the eager pass with the same fill)
        for i, step in enumerate(steps):
            step.calls()
            eager[i] = step.snapshot()
            for t in (step.out, step.slots, step.masks):
                t.fill_(3)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for i, step in enumerate(steps):
            for x, y in zip(eager[i], step.snapshot()):
                assert torch.equal(x, y)
    del graphs
    cache.close()
    engine.close()


def test_capture_refuses_what_it_cannot_record():
    engine = pam.PagedAttentionEngine(0)
    cache = pam.KVCacheManager(engine, 64, BLOCK, D, KVH, DT.float8)
    step = Step(engine, 3, 48, 20, 64, DT.float8, 16, cache)
    step.fill(np.random.default_rng(1), [0, 0, 0], [1, 2, 3], np.zeros((3, 16), np.int32))
    step.calls()
    host = np.zeros(3, np.int32)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    engine.setStream(stream.cuda_stream)
    errors = []
    with torch.cuda.graph(graph, stream=stream):
        step.engine.planStep(step.plan)
        for change in (lambda: setattr(step.plan, "lengths", host), lambda: setattr(step.attention, "workspace", None),
                       lambda: (setattr(step.norm, "slots", step.slots), setattr(step.norm, "v", step.v), setattr(step.norm, "vStride", step.wide))):
            change()
            for call in (lambda: engine.planStep(step.plan), lambda: engine.treeAttention(step.attention),
                         lambda: engine.normRotate(step.norm, cache if step.norm.slots is not None else None)):
                try:
                    call()
                except pam.PagedAttentionError as e:
                    errors.append(str(e))
    assert any("host memory" in e for e in errors)
    assert any("workspace" in e for e in errors)
    assert any("cannot be captured" in e for e in errors)
    graph.replay()
    torch.cuda.synchronize()
    engine.setStream(None)
    del graph
    cache.close()
    engine.close()


def test_asynchronous_calls_on_the_callers_stream(engine):
    """Calls follow work on the engine's stream and return before it is done; two engines on two streams
    at once do not disturb one another."""
    dev = torch.device("cuda", 0)
    engines, steps, caches, want = [], [], [], []
    rng = np.random.default_rng(53)
    lists = rng.permutation(64)[:48].reshape(3, 16).astype(np.int32)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for i, stream in enumerate(streams):
        e = pam.PagedAttentionEngine(0)
        c = pam.KVCacheManager(e, 64, BLOCK, D, KVH, DT.bfloat16)
        s = Step(e, 3, 48, 20, 64, DT.bfloat16, 16, c, seed=i)
        s.attention.workspace = None                      # the engine's own
        s.fill(rng, [0, 37, 190], [1, 20, 13], lists)
        s.calls()
        want.append(s.snapshot())
        e.setStream(stream.cuda_stream)
        e.setAsync(True)
        engines.append(e), caches.append(c), steps.append(s)
    for step in steps:
        step.out.zero_()
        step.q.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for step in steps:
            step.calls()
    for e in engines:
        e.synchronize()
    for step, w in zip(steps, want):
        for x, y in zip(step.snapshot(), w):
            assert torch.equal(x, y)
    for e, c in zip(engines, caches):
        c.close()
        e.close()
