"""normRotate and normRotateBackward on the GPU against float64.

Tolerances.  u = 2^-24.  A normed element carries the error of the sum of squares (at most 16 sums
in a lane and 5 across lanes, all terms positive, halved by the root), of the root, two products and the
weight: below 16 u relative.  Its turn adds the error of cos and sin, 2^-23 each for the rounding of the
reduced angle (pi times half a step at 1) and 2^-23 for the function: 4 u + 4 u absolute per unit, and three
operations.  Together below 32 u of |a| + |b|.  The gradient sums two such terms: 64 u of the sum of their
magnitudes.  Then one rounding to the type of the rows.  Weight gradients are float32 sums of up to M terms,
each off by 32 u: (M + 64) u of the sum of magnitudes.
"""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT, from_io, io_numpy_dtype, to_storage
from oracle import paged_oracle as po
from oracle import step_oracle as so

pytestmark = pytest.mark.gpu
HALF_STEP = {DT.float32: 2.0 ** -24, DT.float16: 2.0 ** -11, DT.bfloat16: 2.0 ** -8, DT.float8: 2.0 ** -11}
TINY = {DT.float32: 2.0 ** -149, DT.float16: 2.0 ** -25, DT.bfloat16: 2.0 ** -134, DT.float8: 2.0 ** -25}   # half the smallest step


def near(got, want, tol, dtype):
    tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + TINY[dtype]
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), f"worst error over tolerance: {(err / tol).max()}"


class NormCase:
    def __init__(self, seed, rows, heads, kv_heads, dim, rotary=None, interleaved=False, dtype=DT.bfloat16, block=16, far=5000,
                 padded=True, fused=True, offset=0):
        rng = np.random.default_rng(seed)
        self.R, self.H, self.KVH, self.D, self.block, self.dtype = rows, heads, kv_heads, dim, block, dtype
        self.rotary, self.inter, self.eps = dim if rotary is None else rotary, interleaved, 1e-5
        rnd = lambda *s: to_storage(rng.standard_normal(s, dtype=np.float32), dtype)
        self.wide = (heads + 2 * kv_heads) * dim + offset
        self.fused = fused
        self.qkv = rnd(rows, self.wide)
        at = [0, heads * dim, (heads + kv_heads) * dim, (heads + 2 * kv_heads) * dim]
        self.at = at
        self.q, self.k, self.v = (self.qkv[:, a:b].reshape(rows, -1, dim) for a, b in zip(at, at[1:]))
        self.wq, self.wk = (to_storage(1 + 0.3 * rng.standard_normal(dim, dtype=np.float32), dtype) for _ in range(2))
        self.freq = (10000.0 ** (-np.arange(0, self.rotary, 2) / max(self.rotary, 1))).astype(np.float32)
        self.pos = rng.integers(0, far, rows).astype(np.int32)
        if rows > 1:
            self.pos[rows // 2] = far - 1
        if padded and rows > 2:
            self.pos[rng.integers(0, rows, max(1, rows // 7))] = -1
        self.blocks = -(-rows // block) + 3
        self.slots = rng.permutation(self.blocks * block)[:rows].astype(np.int64)
        if padded and rows > 4:
            self.slots[1], self.slots[3] = -1, self.blocks * block        # not written
        self.live = self.pos >= 0
        self.in_pool = (self.slots >= 0) & (self.slots < self.blocks * block)
        self.layer = pam.PagedLayerSpec(dim, heads, kv_heads, block, dtype)
        self.io = io_numpy_dtype(dtype)

    def f(self, a):
        return from_io(a, self.dtype)

    def want(self, x, w):
        return so.norm_rotate(self.f(x), self.f(w), np.maximum(self.pos, 0), self.freq, self.rotary, self.inter, self.eps)

    def inputs(self, engine):
        es = self.qkv.itemsize
        if self.fused:
            base = engine.makeBufferFrom(self.qkv)
            total = base.nbytes
            part = lambda i: pam_buffer(base, self.at[i] * es, total - self.at[i] * es)
            return dict(q=part(0), k=part(1), v=part(2), qStride=self.wide, kStride=self.wide, vStride=self.wide), base
        bufs = [engine.makeBufferFrom(np.ascontiguousarray(x)) for x in (self.q, self.k, self.v)]
        return dict(q=bufs[0], k=bufs[1], v=bufs[2]), bufs

    def common(self, engine):
        d = engine.makeBufferFrom
        return dict(qWeight=d(self.wq), kWeight=d(self.wk), invFreq=d(self.freq) if self.rotary else None, positions=d(self.pos),
                    numRows=self.R, rotaryDim=self.rotary, interleaved=int(self.inter), epsilon=self.eps, layer=self.layer)

    def check_forward(self, engine, k_out=True, pages=True):
        inputs, keep = self.inputs(engine)
        fill = to_storage(np.full(1, 7.0, np.float32), self.dtype)[0]
        q0, k0 = np.full((self.R, self.H, self.D), fill), np.full((self.R, self.KVH, self.D), fill)
        p0 = np.full((self.blocks, self.KVH, self.block, self.D), fill)
        qo, ko = engine.makeBufferFrom(q0), engine.makeBufferFrom(k0)
        kp, vp = engine.makeBufferFrom(p0), engine.makeBufferFrom(p0)
        extra = dict(kPool=kp, vPool=vp, slots=engine.makeBufferFrom(self.slots)) if pages else {}
        if k_out:
            extra["kOut"] = ko
        engine.normRotate(pam.PagedNormRotateRequest(**inputs, **self.common(engine), qOut=qo, **extra))
        assert engine.lastStats.operation == pam.Operation.normRotate
        got_q, got_k = qo.download(self.io, q0.shape), ko.download(self.io, k0.shape)
        yq, mq = self.want(self.q, self.wq)
        yk, mk = self.want(self.k, self.wk)
        live = self.live
        near(self.f(got_q)[live], yq[live], 32 * so.U * mq[live], self.dtype)
        assert np.array_equal(got_q[~live], q0[~live])
        if k_out:
            near(self.f(got_k)[live], yk[live], 32 * so.U * mk[live], self.dtype)
            assert np.array_equal(got_k[~live], k0[~live])
        else:
            assert np.array_equal(got_k, k0)
        if pages:
            flat = lambda p: p.transpose(0, 2, 1, 3).reshape(-1, self.KVH, self.D)
            gk, gv = flat(kp.download(self.io, p0.shape)), flat(vp.download(self.io, p0.shape))
            there = live & self.in_pool
            near(self.f(gk[self.slots[there]]), yk[there], 32 * so.U * mk[there], self.dtype)
            assert np.array_equal(gv[self.slots[there]], self.v[there])
            rest = np.setdiff1d(np.arange(len(gk)), self.slots[there])
            assert (gk[rest] == fill).all() and (gv[rest] == fill).all()

    def check_backward(self, engine, pages=False, weights=True, seed=9):
        rng = np.random.default_rng(seed)
        rnd = lambda *s: to_storage(0.5 * rng.standard_normal(s, dtype=np.float32), self.dtype)
        dyq, dyk = rnd(self.R, self.H, self.D), rnd(self.R, self.KVH, self.D)
        dkp, dvp = rnd(self.blocks, self.KVH, self.block, self.D), rnd(self.blocks, self.KVH, self.block, self.D)
        flat = lambda p: p.transpose(0, 2, 1, 3).reshape(-1, self.KVH, self.D)
        if pages:
            gather = lambda p: np.where(self.in_pool[:, None, None], flat(p)[np.where(self.in_pool, self.slots, 0)], to_storage(np.zeros(1, np.float32), self.dtype))
            dyk, dv = gather(dkp), gather(dvp)
        fill = to_storage(np.full(1, 7.0, np.float32), self.dtype)[0]
        d0 = np.full((self.R, self.wide), fill)
        es, base = d0.itemsize, engine.makeBufferFrom(d0)
        part = lambda i: pam_buffer(base, self.at[i] * es, base.nbytes - self.at[i] * es)
        inputs, keep = self.inputs(engine)
        inputs = {k: v for k, v in inputs.items() if k not in ("v", "vStride")}
        up = engine.makeBufferFrom
        grads = dict(dKPool=up(dkp), dVPool=up(dvp), slots=up(self.slots), dV=part(2), dVStride=self.wide) if pages else dict(dKOut=up(dyk))
        wq, wk = up(np.full(self.D, 7, np.float32)), up(np.full(self.D, 7, np.float32))
        if weights:
            grads.update(dQWeight=wq, dKWeight=wk)
        request = pam.PagedNormRotateBackwardRequest(**inputs, **self.common(engine), dQOut=up(dyq), dQ=part(0), dK=part(1),
                                                     dQStride=self.wide, dKStride=self.wide, **grads)
        engine.normRotateBackward(request)
        assert engine.lastStats.operation == pam.Operation.normRotateBackward
        got = base.download(self.io, d0.shape)
        live = self.live
        for i, (x, w, dy, dw) in enumerate(((self.q, self.wq, dyq, wq), (self.k, self.wk, dyk, wk))):
            pos = np.maximum(self.pos, 0)
            dx, _, size, _ = so.norm_rotate_backward(self.f(x), self.f(w), self.f(dy), pos, self.freq, self.rotary, self.inter, self.eps)
            mine = got[:, self.at[i]:self.at[i + 1]].reshape(dx.shape)
            near(self.f(mine)[live], dx[live], 64 * so.U * size[live], self.dtype)
            _, dweight, _, total = so.norm_rotate_backward(self.f(x)[live], self.f(w), self.f(dy)[live], self.pos[live], self.freq,
                                                           self.rotary, self.inter, self.eps)
            if weights:
                terms = int(live.sum()) * x.shape[1]
                err = np.abs(dw.download(np.float32, (self.D,)) - dweight)
                assert (err <= (terms + 64) * so.U * total + 1e-30).all()
            else:
                assert (dw.download(np.float32, (self.D,)) == 7).all()
        if pages:
            mine = got[:, self.at[2]:self.at[3]].reshape(self.R, self.KVH, self.D)
            assert np.array_equal(mine[live], dv[live])
        else:
            assert (got[:, self.at[2]:] == fill).all()
        assert (got[~live] == fill).all() and (got[:, self.at[3]:] == fill).all()
        return got, wq.download(np.float32, (self.D,))


def pam_buffer(base, offset, nbytes):
    from pagedattentionmetal_b200 import _cabi
    return _cabi.PamBuffer(base.ptr + offset, nbytes)


SHAPES = [
    dict(rows=1, heads=1, kv_heads=1, dim=64), dict(rows=33, heads=32, kv_heads=8, dim=128),
    dict(rows=7, heads=6, kv_heads=2, dim=80, rotary=40, interleaved=True), dict(rows=20, heads=8, kv_heads=8, dim=96, rotary=48),
    dict(rows=9, heads=64, kv_heads=8, dim=128, interleaved=True), dict(rows=5, heads=4, kv_heads=1, dim=256, rotary=64),
    dict(rows=300, heads=2, kv_heads=1, dim=64, rotary=32), dict(rows=6, heads=3, kv_heads=1, dim=256, interleaved=True),
    dict(rows=11, heads=4, kv_heads=2, dim=20), dict(rows=11, heads=4, kv_heads=2, dim=33, rotary=10),
    dict(rows=4, heads=2, kv_heads=2, dim=16, rotary=0), dict(rows=13, heads=4, kv_heads=2, dim=128, rotary=0),
    dict(rows=12, heads=4, kv_heads=2, dim=64, rotary=36, interleaved=True), dict(rows=12, heads=4, kv_heads=2, dim=8),
    dict(rows=17, heads=5, kv_heads=1, dim=128, offset=3), dict(rows=2000, heads=4, kv_heads=2, dim=64, block=24),
]


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16, DT.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_forward(engine, dtype, shape):
    case = NormCase(21, dtype=dtype, **shape)
    case.check_forward(engine)
    NormCase(22, dtype=dtype, fused=False, **shape).check_forward(engine, k_out=False)
    case.check_forward(engine, pages=False)


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16, DT.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_backward(engine, dtype, shape):
    case = NormCase(23, dtype=dtype, **shape)
    first = case.check_backward(engine)
    again = case.check_backward(engine)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    case.check_backward(engine, pages=True)
    NormCase(24, dtype=dtype, fused=False, **shape).check_backward(engine, pages=True, weights=False)


def test_far_positions(engine):
    # an angle of millions of radians: a float32 product would be off by a tenth of a radian
    case = NormCase(25, 64, 4, 2, 64, dtype=DT.float32, far=2 ** 31 - 1, padded=False)
    case.check_forward(engine)
    case.check_backward(engine)


def test_every_row_skipped(engine):
    case = NormCase(26, 9, 4, 2, 64)
    case.pos[:] = -1
    case.live[:] = False
    case.check_forward(engine)
    base = engine.makeBufferFrom(np.full((9, 4, 64), 7, np.uint16))
    dk = engine.makeBufferFrom(np.full((9, 2, 64), 7, np.uint16))
    wq, wk = engine.makeBufferFrom(np.full(64, 7, np.float32)), engine.makeBufferFrom(np.full(64, 7, np.float32))
    inputs, keep = case.inputs(engine)
    inputs = {k: v for k, v in inputs.items() if k not in ("v", "vStride")}
    zeros = lambda *s: engine.makeBufferFrom(np.zeros(s, np.uint16))
    engine.normRotateBackward(pam.PagedNormRotateBackwardRequest(**inputs, **case.common(engine), dQOut=zeros(9, 4, 64),
                                                                 dKOut=zeros(9, 2, 64), dQ=base, dK=dk, dQWeight=wq, dKWeight=wk))
    assert (base.download(np.uint16, (9, 4, 64)) == 7).all() and (dk.download(np.uint16, (9, 2, 64)) == 7).all()
    assert (wq.download(np.float32, (64,)) == 0).all() and (wk.download(np.float32, (64,)) == 0).all()


@pytest.mark.parametrize("shape", [dict(heads=32, kv_heads=8, dim=128), dict(heads=4, kv_heads=2, dim=33, rotary=32)])
def test_in_place_on_the_projection_rows(engine, shape):
    case = NormCase(27, rows=19, dtype=DT.float16, **shape)
    inputs, base = case.inputs(engine)
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **case.common(engine), qOut=inputs["q"], qOutStride=case.wide,
                                                 kOut=inputs["k"], kOutStride=case.wide))
    got = base.download(case.io, case.qkv.shape)
    for i, (x, w) in enumerate(((case.q, case.wq), (case.k, case.wk))):
        y, m = case.want(x, w)
        mine = got[:, case.at[i]:case.at[i + 1]].reshape(y.shape)
        near(case.f(mine)[case.live], y[case.live], 32 * so.U * m[case.live], case.dtype)
    assert np.array_equal(got[~case.live], case.qkv[~case.live]) and np.array_equal(got[:, case.at[2]:], case.qkv[:, case.at[2]:])


def test_host_buffers(engine):
    case = NormCase(28, 10, 4, 2, 64, dtype=DT.float16, fused=False)
    qo, ko = np.full((10, 4, 64), 7, np.float16), np.full((10, 2, 64), 7, np.float16)
    engine.normRotate(pam.PagedNormRotateRequest(
        q=case.q.copy(), k=case.k.copy(), qWeight=case.wq, kWeight=case.wk, invFreq=case.freq, positions=case.pos, qOut=qo,
        kOut=ko, numRows=10, rotaryDim=64, epsilon=case.eps, layer=case.layer))
    y, m = case.want(case.q, case.wq)
    near(qo[case.live], y[case.live], 32 * so.U * m[case.live], case.dtype)
    assert (qo[~case.live] == 7).all() and (ko[~case.live] == 7).all()
    pool = np.zeros((4, 2, 16, 64), np.float16)
    with pytest.raises(pam.PagedAttentionError, match="device memory"):
        engine.normRotate(pam.PagedNormRotateRequest(
            q=case.q.copy(), k=case.k.copy(), v=case.v.copy(), qWeight=case.wq, kWeight=case.wk, invFreq=case.freq,
            positions=case.pos, qOut=qo, kPool=pool, vPool=pool, slots=case.slots, numRows=10, rotaryDim=64, layer=case.layer))


@pytest.mark.parametrize("dtype", [DT.float16, DT.float8, DT.bfloat16])
@pytest.mark.parametrize("k_out", [None, "rows", "strided"])
def test_append_through_the_cache_handle(engine, dtype, k_out):
    """The pages equal those of reshapeAndCache over the call's own key rows, FP8 scales included."""
    case = NormCase(29, 50, 8, 2, 64, dtype=dtype)
    make = lambda: pam.KVCacheManager(engine, case.blocks, case.block, case.D, case.KVH, dtype)
    one, two = make(), make()
    inputs, keep = case.inputs(engine)
    common = case.common(engine)
    qo = engine.makeBuffer(case.R * case.H * case.D * 2)
    rows = engine.makeBufferFrom(np.zeros((case.R, case.KVH, case.D), np.uint16))
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **common, qOut=qo, kOut=rows))
    slots = np.where(case.live, case.slots, -1)
    engine.reshapeAndCache(two, rows, engine.makeBufferFrom(np.ascontiguousarray(case.v)), engine.makeBufferFrom(slots), case.R)
    wide = 3 * case.KVH * case.D
    extra = {}
    if k_out:
        extra = dict(kOut=engine.makeBufferFrom(np.zeros((case.R, wide), np.uint16)), kOutStride=wide if k_out == "strided" else 0)
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **common, qOut=qo, slots=engine.makeBufferFrom(case.slots), **extra), one)
    for a, b in zip(one.readPools(), two.readPools()):
        assert (a is None) == (b is None)
        if a is not None:
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    if k_out:
        got = extra["kOut"].download(np.uint16, (case.R, wide))
        want = rows.download(np.uint16, (case.R, case.KVH * case.D))
        mine = got[:, :case.KVH * case.D] if k_out == "strided" else got.reshape(-1)[:want.size].reshape(want.shape)
        assert np.array_equal(mine[case.live], want[case.live])
    with pytest.raises(pam.PagedAttentionError, match="does not describe the cache"):
        common["layer"] = pam.PagedLayerSpec(case.D, case.H, case.KVH, 32, dtype)
        engine.normRotate(pam.PagedNormRotateRequest(**inputs, **common, qOut=qo, slots=engine.makeBufferFrom(case.slots)), one)
    one.close()
    two.close()


def test_a_row_of_zeros_and_of_infinity(engine):
    case = NormCase(30, 4, 2, 1, 64, dtype=DT.float32, padded=False, fused=False)
    case.q[0] = 0                                       # rsqrt(eps) * 0
    case.q[1, 0, 5] = np.inf                            # mean square infinite: 0 and inf * 0
    inputs, keep = case.inputs(engine)
    qo, ko = engine.makeBuffer(4 * 2 * 64 * 4), engine.makeBuffer(4 * 64 * 4)
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **case.common(engine), qOut=qo, kOut=ko))
    got = qo.download(np.float32, (4, 2, 64))
    assert (got[0] == 0).all()
    assert np.isnan(got[1, 0, 5]) and np.isfinite(got[1, 1]).all() and np.isfinite(got[2:]).all()
