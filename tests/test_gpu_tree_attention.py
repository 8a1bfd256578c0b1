"""treeAttention on the GPU against float64, key by key.

Tolerance.  u = 2^-24.  A score is a float32 sum of dim products (error serr, from the oracle: (dim + 8) u times the
largest sum of magnitudes of any of the row's keys) and a weight is off by that and by its own rounding: w = half a step of
the type that carries it into the second product (float32 2^-24; float16 2^-11; bfloat16 carried as two
operands 2^-16; an exp2 of 2^-22 on top).  The sums over n keys add n u; numerator and denominator both carry the
score's error.  With A = the weighted mean of |v|: A (2 serr + w + 2^-22 + (n + 8) u), one rounding to the output type.
The tensor-core products of 16-bit operands keep at least the float32 sum's error per term.
"""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT, from_io, io_numpy_dtype, quantize_pool, to_storage
from oracle import step_oracle as so
from test_gpu_step_plan import make_tree

pytestmark = pytest.mark.gpu
HALF_STEP = {DT.float32: 2.0 ** -24, DT.float16: 2.0 ** -11, DT.bfloat16: 2.0 ** -8, DT.float8: 2.0 ** -11}
WEIGHT = {DT.float32: 2.0 ** -24, DT.float16: 2.0 ** -11, DT.bfloat16: 2.0 ** -8, DT.float8: 2.0 ** -11}


def dequantised(codes, scale):
    """Codes times scale."""
    import torch
    value = torch.from_numpy(codes).view(torch.float8_e4m3fn).to(torch.float16).numpy()
    return value.astype(np.float64) * scale.astype(np.float64)[:, :, None, None]


class TreeCase:
    def __init__(self, seed, lens, sizes, heads=8, kv_heads=2, dim=128, block=16, dtype=DT.bfloat16, window=0, kind="random",
                 spare_rows=2, masks=True, strided=False, poison=True, width=None, first=0, scale=1.0):
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.lens, self.H, self.KVH, self.D, self.block, self.dtype, self.window = np.array(lens, np.uint32), heads, kv_heads, dim, block, dtype, window
        self.B, self.sizes = len(lens), sizes
        self.starts = (first + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)
        self.rows = max(1, int(self.starts[-1]) + spare_rows)
        self.max_new = max(max(sizes), 1)
        self.words = -(-self.max_new // 32)
        need = [-(-int(l) // block) for l in lens]
        self.n_pool = sum(need) + 3
        perm = rng.permutation(self.n_pool).astype(np.int32)
        self.width = max(max(need), 1) if width is None else width
        self.tables = np.full((self.B, self.width), -7 if width is None else 0, np.int32)     # unused entries: anything
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = perm[at:at + n][:self.width]
            at += n
        rnd = lambda *s: rng.standard_normal(s, dtype=np.float32)
        shape = (self.n_pool, kv_heads, block, dim)
        k32, v32 = rnd(*shape), rnd(*shape)
        self.k_scale = self.v_scale = None
        if dtype == DT.float8:
            self.k_pool, self.k_scale = quantize_pool(k32)
            self.v_pool, self.v_scale = quantize_pool(v32)
        else:
            self.k_pool, self.v_pool = to_storage(k32, dtype), to_storage(v32, dtype)
            if poison:
                nan = to_storage(np.full(1, np.nan, np.float32), dtype)[0]
                for b in range(self.B):
                    L = int(self.lens[b])
                    if L % block and L // block < self.width:
                        blk = self.tables[b, L // block]
                        self.k_pool[blk, :, L % block:] = nan
                        self.v_pool[blk, :, L % block:] = nan
        self.q = to_storage(scale * rnd(self.rows, heads, dim), dtype)
        self.pad = 24 if strided else 0                  # strided: parts of wider rows
        self.k = to_storage(rnd(self.rows, kv_heads, dim), dtype)
        self.v = to_storage(rnd(self.rows, kv_heads, dim), dtype)
        self.masks = self.positions = None
        if masks:
            self.masks = rng.integers(0, 2 ** 32, (self.rows, self.words), dtype=np.uint32)    # rows of no request: anything
            self.positions = np.full(self.rows, -1, np.int32)
            for b, n in enumerate(sizes):
                s = self.starts[b]
                sees = so.ancestors(make_tree(rng, n, kind))
                self.masks[s:s + n] = so.pack_bits(sees, self.words)
                self.positions[s:s + n] = int(self.lens[b]) + sees.sum(1) - 1
        self.layer = pam.PagedLayerSpec(dim, heads, kv_heads, block, dtype, window)

    def _rows(self, engine, a):
        """Rows on the device: back to back, or parts of wider rows (stride in elements)."""
        flat = a.reshape(self.rows, -1)
        if not self.pad:
            return engine.makeBufferFrom(flat), 0
        wide = np.zeros((self.rows, flat.shape[1] + self.pad), flat.dtype)
        wide[:, 8:8 + flat.shape[1]] = flat
        base = engine.makeBufferFrom(wide)
        from pagedattentionmetal_b200 import _cabi
        self.kept.append(base)
        return _cabi.PamBuffer(base.ptr + 8 * flat.itemsize, base.nbytes - 8 * flat.itemsize), wide.shape[1]

    def request(self, engine, out):
        self.kept = []
        up = engine.makeBufferFrom
        (q, qs), (k, ks), (v, vs) = (self._rows(engine, a) for a in (self.q, self.k, self.v))
        opt = lambda a: None if a is None else up(a)
        return pam.PagedTreeAttentionRequest(
            q=q, k=k, v=v, qStride=qs, kStride=ks, vStride=vs, kPool=up(self.k_pool), vPool=up(self.v_pool),
            blockTables=up(self.tables), cacheLengths=up(self.lens), rowStarts=up(self.starts), masks=opt(self.masks),
            positions=opt(self.positions), output=out, kScaleBuffer=opt(self.k_scale), vScaleBuffer=opt(self.v_scale),
            batchSize=self.B, maxNumBlocks=self.width, numRows=self.rows, maxNewTokens=self.max_new,
            maskWords=self.words if self.masks is not None else 0, layer=self.layer)

    def run(self, engine):
        fill = to_storage(np.full(1, 7.0, np.float32), self.dtype)[0]
        out = engine.makeBufferFrom(np.full(self.q.shape, fill))
        engine.treeAttention(self.request(engine, out))
        assert engine.lastStats.operation == pam.Operation.treeAttention
        return from_io(out.download(io_numpy_dtype(self.dtype), self.q.shape), self.dtype)

    def oracle(self):
        f = lambda a: from_io(a, self.dtype).astype(np.float64)
        pools = [dequantised(p, s) if s is not None else f(p) for p, s in ((self.k_pool, self.k_scale), (self.v_pool, self.v_scale))]
        return so.tree_attention(f(self.q), f(self.k), f(self.v), *pools, self.tables, self.lens, self.starts, self.block,
                                 self.masks, self.positions, self.window, self.max_new)

    def check(self, engine, finite=True):
        out = self.run(engine)
        want, mag, serr, count = self.oracle()
        unowned = np.isnan(want).all((1, 2)) & (count == 0)
        assert (out[unowned] == 7).all()
        owned = ~unowned
        if finite:
            assert np.isfinite(want[owned]).all()
        tol = mag * (2 * serr[:, :, None] + WEIGHT[self.dtype] + 2.0 ** -22 + (count[:, None, None] + 8) * so.U)
        tol = tol + HALF_STEP[self.dtype] * (np.abs(want) + tol) + 2.0 ** -25 * (self.dtype in (DT.float16, DT.float8))
        with np.errstate(invalid="ignore"):
            err = np.abs(out - want)
        good = np.isfinite(want) & owned[:, None, None]
        assert (err[good] <= tol[good]).all(), f"worst error over tolerance: {np.nanmax(err[good] / tol[good])}"
        odd = ~np.isfinite(want) & owned[:, None, None]
        assert np.array_equal(np.isnan(out[odd]), np.isnan(want[odd]))
        assert np.array_equal(np.sign(out[odd]), np.sign(want[odd]), equal_nan=True)
        return out


TYPES = [DT.float32, DT.float16, DT.bfloat16, DT.float8]
SHAPES = {
    "one row, one key": dict(lens=[0], sizes=[1]),
    "one row, one token": dict(lens=[1], sizes=[1]),
    "empty contexts": dict(lens=[0, 0, 5], sizes=[3, 0, 1]),
    "no rows": dict(lens=[7, 9], sizes=[0, 0]),
    "ragged": dict(lens=[63, 64, 65, 127, 128, 129, 1, 500], sizes=[1, 2, 5, 17, 33, 64, 3, 7]),
    "long": dict(lens=[4097], sizes=[5]),
    "many rows": dict(lens=[130, 31], sizes=[100, 40]),
    "wide groups": dict(lens=[70, 300], sizes=[9, 4], heads=16, kv_heads=1),
    "seven heads a group": dict(lens=[70, 300], sizes=[9, 20], heads=14, kv_heads=2),
    "no groups": dict(lens=[70, 300], sizes=[9, 33], heads=4, kv_heads=4),
    "dim 64": dict(lens=[70, 300], sizes=[9, 33], dim=64),
    "dim 80": dict(lens=[70, 300], sizes=[9, 3], dim=80),
    "dim 64, long": dict(lens=[2100, 300, 0], sizes=[40, 9, 65], dim=64),
    "dim 80, seven heads a group": dict(lens=[270, 900], sizes=[9, 30], dim=80, heads=14, kv_heads=2),
    "dim 96": dict(lens=[270, 1000, 17], sizes=[33, 5, 40], dim=96),
    "dim 112, strided": dict(lens=[270, 1000, 17], sizes=[33, 5, 64], dim=112, strided=True),
    "dim 33": dict(lens=[70, 20], sizes=[9, 3], dim=33),
    "dim 256": dict(lens=[70, 200], sizes=[9, 3], dim=256),
    "blocks of 8": dict(lens=[70, 300], sizes=[9, 20], block=8),
    "blocks of 24": dict(lens=[70, 300], sizes=[9, 20], block=24),
    "blocks of 8, long": dict(lens=[700, 129, 2000], sizes=[40, 9, 64], block=8),
    "blocks of 24, long": dict(lens=[700, 129, 2000], sizes=[40, 9, 64], block=24, dim=64),
    "blocks of 32": dict(lens=[70, 300], sizes=[9, 20], block=32),
    "blocks of 128": dict(lens=[70, 300], sizes=[9, 20], block=128),
    "chain": dict(lens=[70, 300], sizes=[40, 64], kind="chain"),
    "star": dict(lens=[70, 300], sizes=[40, 64], kind="star"),
    "several roots": dict(lens=[70, 300], sizes=[40, 64], kind="odd"),
    "without masks": dict(lens=[70, 300], sizes=[40, 70], masks=False),
    "strided": dict(lens=[70, 300], sizes=[9, 33], strided=True),
    "rows before the first": dict(lens=[70, 300], sizes=[9, 3], first=4),
    "short table": dict(lens=[100, 300], sizes=[9, 3], width=4),
    "large scores": dict(lens=[200, 300], sizes=[9, 30], scale=6.0),
    "many requests": dict(lens=list(range(0, 300, 7)), sizes=[(3 * i) % 11 for i in range(43)]),
}


@pytest.mark.parametrize("dtype", TYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("name", SHAPES)
def test_matches_float64(engine, dtype, name):
    TreeCase(31, dtype=dtype, **SHAPES[name]).check(engine)


@pytest.mark.parametrize("dtype", [DT.float16, DT.float8, DT.float32], ids=lambda d: d.name)
def test_very_many_short_requests(engine, dtype):
    """Hundreds of pairs in every block's piece, most of one key tile, some of none of the cache."""
    lens = [0 if i % 3 else 5 + i % 40 for i in range(900)]
    TreeCase(44, lens, [5 + i % 2 for i in range(900)], heads=8, kv_heads=2, dtype=dtype).check(engine)
    TreeCase(45, [0] * 1500, [17] + [0, 1] * 749 + [3], heads=8, kv_heads=2, dtype=dtype).check(engine)
    # small ones beside one with more than 128 rows under a KV head, and beside its second row tile
    TreeCase(49, lens[:300] + [500, 30], [5 + i % 2 for i in range(300)] + [40, 70], heads=8, kv_heads=2, dtype=dtype).check(engine)


@pytest.mark.parametrize("dtype", TYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("window", [1, 5, 64, 200])
@pytest.mark.parametrize("masks", [True, False])
def test_windows(engine, dtype, window, masks):
    TreeCase(32, [0, 3, 130, 700], [5, 9, 70, 12], dtype=dtype, window=window, masks=masks).check(engine)
    TreeCase(33, [300, 40], [64, 33], dtype=dtype, window=window, masks=masks, kind="chain", heads=4, kv_heads=4, dim=64).check(engine)


def test_engine_default_window_and_positions(engine):
    case = TreeCase(34, [300, 40], [17, 33], window=50)
    case.layer = pam.PagedLayerSpec(case.D, case.H, case.KVH, case.block, case.dtype, 0)
    engine.defaultWindowSize = 50
    try:
        case.check(engine)
        case.positions[:] = 0                           # below the cache length: counts as the cache length
        case.check(engine)
    finally:
        engine.defaultWindowSize = 0


@pytest.mark.parametrize("dtype", TYPES, ids=lambda d: d.name)
def test_masks_that_leave_rows_empty(engine, dtype):
    case = TreeCase(35, [0, 40, 0], [20, 33, 64], dtype=dtype)
    case.masks[case.starts[0]:case.starts[0] + 20:3] = 0           # no cache and no node: zeros
    case.masks[case.starts[1]:case.starts[2]] = 0                  # the cache alone
    case.masks[case.starts[2]] = 0
    out = case.check(engine)
    assert (out[case.starts[0]] == 0).all() and (out[case.starts[2]] == 0).all()


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16, DT.bfloat16], ids=lambda d: d.name)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("lens", [[100, 0], [3000, 64]])
@pytest.mark.parametrize("dim", [128, 80, 64])
def test_values_a_row_does_not_see_do_not_reach_it(engine, dtype, what, window, lens, dim):
    """A node's values that are not finite reach the rows that see it and no others; so at the edge of a window."""
    case = TreeCase(36, lens, [40, 70], dtype=dtype, window=window, dim=dim)
    bad = to_storage(np.full(1, what, np.float32), dtype)[0]
    case.v[case.starts[0] + 7, :, 3::5] = bad
    case.v[case.starts[1] + 30, 1, :] = bad
    case.v[case.starts[1] + 69] = bad                  # a leaf: its own row alone
    if window:
        for t in range(lens[0] + 1 - window, lens[0] + 3 - window):      # seen by the root, not by deep nodes
            case.v_pool[case.tables[0, t // 16], 0, t % 16, ::7] = bad
    out = case.check(engine, finite=False)
    assert np.isfinite(out[case.starts[0]:case.starts[2]]).any() and not np.isfinite(out[case.starts[2] - 1]).any()


@pytest.mark.parametrize("dim", [128, 80, 64])
@pytest.mark.parametrize("window", [0, 90])
def test_values_a_row_does_not_see_behind_float8_pages(engine, dim, window):
    """The same for float16 rows behind a float8 cache, whose codes know NaN (0x7f) as well."""
    lens = [300, 64]
    case = TreeCase(46, lens, [40, 70], dtype=DT.float8, window=window, dim=dim)
    bad = to_storage(np.full(1, np.inf, np.float32), DT.float16)[0]
    case.v[case.starts[0] + 7, :, 3::5] = bad
    case.v[case.starts[1] + 69] = bad
    if window:
        for t in range(lens[0] + 1 - window, lens[0] + 3 - window):
            case.v_pool[case.tables[0, t // 16], 0, t % 16, ::7] = 0x7F
    out = case.check(engine, finite=False)
    assert np.isfinite(out[case.starts[0]:case.starts[2]]).any() and not np.isfinite(out[case.starts[2] - 1]).any()


def test_float8_scales_of_zero(engine):
    """Pages whose scale is zero: keys that all score alike, values that are zero."""
    case = TreeCase(47, [300, 64], [40, 9], dtype=DT.float8)
    case.k_scale[::3] = 0
    case.v_scale[1::3] = 0
    case.check(engine)


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16, DT.bfloat16], ids=lambda d: d.name)
def test_keys_a_row_does_not_see_do_not_reach_it(engine, dtype):
    case = TreeCase(37, [100, 3], [40, 7], dtype=dtype)
    bad = to_storage(np.full(1, np.nan, np.float32), dtype)[0]
    node = case.starts[0] + 39
    case.k[node] = bad
    out = case.check(engine, finite=False)
    assert np.isfinite(np.delete(out, node, 0)).all() and np.isnan(out[node]).all()


def test_bad_row_starts_and_lengths_stay_in_bounds(engine):
    case = TreeCase(38, [70, 300, 20], [9, 20, 5])
    case.starts = np.array([-5, 9, 1 << 30, 3], np.int32)          # cut into the rows that exist
    case.lens = np.array([70, 0xFFFFFFF0, 20], np.uint32)          # more tokens than the table has
    case.tables[1, :] = np.array([1 << 30, -(1 << 30)] * (case.width // 2 + 1), np.int32)[:case.width]
    case.check(engine, finite=False)                   # (clamped entries reach the unused slots, which hold NaN)


def test_equal_inputs_give_equal_bits(engine):
    case = TreeCase(39, [5000, 900, 33], [30, 64, 1], dtype=DT.float16)
    first, again = case.run(engine), case.run(engine)
    assert np.array_equal(first, again)


def test_large_pool(engine):
    """Pages whose element offsets pass 2^31: the last blocks of a pool of 2.4 G elements."""
    torch = pytest.importorskip("torch")
    case = TreeCase(40, [150, 70], [9, 33], dtype=DT.float16, heads=8, kv_heads=8)
    want = case.run(engine)
    blocks = 150000
    big = torch.zeros(blocks * case.KVH * 16 * 128, dtype=torch.float16, device="cuda")
    shift = blocks - case.n_pool
    per = case.KVH * 16 * 128
    pools = []
    for src in (case.k_pool, case.v_pool):
        t = big.clone() if pools else big
        t[shift * per:] = torch.from_numpy(src.reshape(-1)).cuda()
        pools.append(t)
    torch.cuda.synchronize()
    out = engine.makeBufferFrom(np.full(case.q.shape, 7, np.float16))
    case.tables = np.where(case.tables >= 0, case.tables + shift, case.tables)
    request = case.request(engine, out)
    request.kPool, request.vPool = pools
    engine.treeAttention(request)
    assert np.array_equal(out.download(np.float16, case.q.shape).astype(np.float32), want)


def test_host_buffers_and_workspace(engine):
    case = TreeCase(41, [150, 70], [9, 33], dtype=DT.float16)
    want = case.run(engine)
    out = np.full(case.q.shape, 7, np.float16)
    up = engine.makeBufferFrom
    request = pam.PagedTreeAttentionRequest(
        q=case.q, k=case.k, v=case.v, kPool=up(case.k_pool), vPool=up(case.v_pool), blockTables=case.tables,
        cacheLengths=case.lens, rowStarts=case.starts, masks=case.masks, output=out, batchSize=case.B,
        maxNumBlocks=case.width, numRows=case.rows, maxNewTokens=case.max_new, maskWords=case.words, layer=case.layer)
    engine.treeAttention(request)
    assert np.array_equal(out.astype(np.float32), want)
    need = engine.treeAttentionWorkspace(request)
    request.workspace = engine.makeBuffer(need)
    out[:] = 7
    engine.treeAttention(request)
    assert np.array_equal(out.astype(np.float32), want)
    request.workspace = engine.makeBuffer(need - 1)
    with pytest.raises(pam.PagedAttentionError, match="workspace"):
        engine.treeAttention(request)
    request.workspace = np.zeros(need + 256, np.uint8)
    with pytest.raises(pam.PagedAttentionError, match="workspace"):
        engine.treeAttention(request)
    request.workspace = None
    request.kPool = case.k_pool
    with pytest.raises(pam.PagedAttentionError, match="device memory"):
        engine.treeAttention(request)


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("dtype", [DT.float32, DT.float16], ids=lambda d: d.name)
@pytest.mark.parametrize("dim", [128, 40])
def test_inputs_from_copies_and_other_streams_are_complete(engine, dtype, dim, recorded):
    """The kernels are set up early, but read nothing before what precedes them: a copy on their stream, and a
    stream that theirs waits for, which writes the queries at the end of a long queue."""
    torch = pytest.importorskip("torch")
    case = TreeCase(51, [3000, 500, 70], [9, 20, 17], dtype=dtype, dim=dim)
    out = engine.makeBufferFrom(np.zeros(case.q.shape, case.q.dtype))
    request = case.request(engine, out)
    engine.treeAttention(request)
    want = out.download(io_numpy_dtype(dtype), case.q.shape)
    q, v = (torch.from_numpy(x.view(np.uint8).reshape(-1).copy()).pin_memory() for x in (case.q, case.v))
    device = [torch.zeros_like(x, device="cuda") for x in (q, v)]
    ready = q.cuda()
    request.q, request.v = device
    request.workspace = engine.makeBuffer(engine.treeAttentionWorkspace(request))
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")

    def work():
        other.wait_stream(mine)
        with torch.cuda.stream(other):
            x = busy
            for _ in range(10):
                x = x @ busy
            device[0].copy_(ready)
        mine.wait_stream(other)
        device[1].copy_(v, non_blocking=True)
        engine.treeAttention(request)

    engine.setAsync(True)
    engine.setStream(mine.cuda_stream)
    try:
        torch.cuda.synchronize()
        with torch.cuda.stream(mine):
            work()
        torch.cuda.synchronize()
        if recorded:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=mine):
                work()
            for _ in range(3):
                for t in device:
                    t.zero_()
                out.upload(np.zeros(case.q.shape, case.q.dtype))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
            del graph
    finally:
        engine.setStream(None)
        engine.setAsync(False)
    assert np.array_equal(out.download(io_numpy_dtype(dtype), case.q.shape), want)


@pytest.mark.parametrize("dtype", [DT.float16, DT.bfloat16, DT.float8], ids=lambda d: d.name)
@pytest.mark.parametrize("sizes", [[9, 20, 17], [40, 64, 3]])
def test_waits_that_run_out_leave_the_context_usable(dtype, sizes):
    """With a limit of one cycle the wait for the first key tile runs out while the copies are on their way: the
    kernel waits for those, returns, and the call fails like any failed launch."""
    engine = pam.PagedAttentionEngine()
    case = TreeCase(50, [3000, 500, 70], sizes, dtype=dtype)
    out = engine.makeBufferFrom(np.full(case.q.shape, 7, case.q.dtype))
    request = case.request(engine, out)
    engine.setWaitLimit(1)
    engine.enableGracefulDegradation = False
    with pytest.raises(pam.PagedAttentionError, match="bounded wait ran out"):
        engine.treeAttention(request)
    engine.enableGracefulDegradation = True
    engine.treeAttention(request)
    assert (from_io(out.download(io_numpy_dtype(dtype), case.q.shape), dtype) == 0).all()
    engine.setWaitLimit(0)
    case.check(engine)
    engine.close()


@pytest.mark.parametrize("dtype", TYPES, ids=lambda d: d.name)
@pytest.mark.parametrize("dim", [33, 64, 80, 96, 128, 256])
@pytest.mark.parametrize("size", [1, 12, 40, 70])
def test_workspace_is_as_large_as_it_says(engine, dtype, dim, size):
    """The bytes behind the workspace stay as they are.  (They are there: a kernel that wrote them would harm nobody.)"""
    case = TreeCase(48, [2100, 40, 3], [size, 1, size], dtype=dtype, dim=dim)
    out = engine.makeBufferFrom(np.zeros(case.q.shape, case.q.dtype))
    request = case.request(engine, out)
    need, behind = engine.treeAttentionWorkspace(request), 32 << 20
    memory = engine.makeBufferFrom(np.full(need + behind, 0x5A, np.uint8))
    from pagedattentionmetal_b200 import _cabi
    request.workspace = _cabi.PamBuffer(memory.ptr, need)
    engine.treeAttention(request)
    assert (memory.download(np.uint8, (behind,), need) == 0x5A).all()


def test_failed_launches_degrade_like_a_decode(engine):
    case = TreeCase(42, [150, 70], [9, 33], dtype=DT.float16)
    out = engine.makeBufferFrom(np.full(case.q.shape, 7, np.float16))
    request = case.request(engine, out)
    engine.injectLaunchFailures(3)
    engine.treeAttention(request)
    assert (out.download(np.float16, case.q.shape) == 0).all()
    engine.enableGracefulDegradation = False
    try:
        engine.injectLaunchFailures(3)
        with pytest.raises(pam.PagedAttentionError):
            engine.treeAttention(request)
    finally:
        engine.enableGracefulDegradation = True
        engine.injectLaunchFailures(0)
    case.check(engine)
