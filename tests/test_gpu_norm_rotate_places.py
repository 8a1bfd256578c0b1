"""normRotate and normRotateBackward where their buffers may lie: outputs over the inputs, columns of one array of
the host, addresses off the 16-byte grid.  The same call with every buffer on its own is held against float64 by
test_gpu_norm_rotate.py; here its bits are the reference."""
import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from gpu_helpers import DT
from test_gpu_norm_rotate import NormCase, pam_buffer

pytestmark = pytest.mark.gpu


def pools_equal(one, two):
    for a, b in zip(one.readPools(), two.readPools()):
        assert (a is None) == (b is None)
        if a is not None:
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("shape", [dict(heads=8, kv_heads=2, dim=64), dict(heads=32, kv_heads=8, dim=128, interleaved=True),
                                   dict(heads=4, kv_heads=2, dim=33, rotary=32)], ids=lambda s: f"dim{s['dim']}")
@pytest.mark.parametrize("dtype", [DT.float8, DT.float16, DT.bfloat16], ids=lambda d: d.name)
@pytest.mark.parametrize("over", ["q", "k", "both"])
def test_in_place_with_an_append(engine, dtype, shape, over):
    """Queries and keys over the projection's own rows while the keys and values go to the pages."""
    case = NormCase(61, rows=50, dtype=dtype, **shape)
    one, two = (pam.KVCacheManager(engine, case.blocks, case.block, case.D, case.KVH, dtype) for _ in range(2))
    slots = engine.makeBufferFrom(case.slots)
    apart, keep = case.inputs(engine)
    q, k = (engine.makeBufferFrom(np.zeros((case.R, n, case.D), np.uint16)) for n in (case.H, case.KVH))
    engine.normRotate(pam.PagedNormRotateRequest(**apart, **case.common(engine), qOut=q, kOut=k, slots=slots), two)
    q, k = q.download(np.uint16, (case.R, case.H * case.D)), k.download(np.uint16, (case.R, case.KVH * case.D))
    inputs, base = case.inputs(engine)
    side = engine.makeBufferFrom(np.zeros((case.R, case.wide), np.uint16))
    part = lambda b, i: pam_buffer(b, case.at[i] * 2, b.nbytes - case.at[i] * 2)
    q_base, k_base = (base if over in (x, "both") else side for x in "qk")
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **case.common(engine), qOut=part(q_base, 0), qOutStride=case.wide,
                                                 kOut=part(k_base, 1), kOutStride=case.wide, slots=slots), one)
    pools_equal(one, two)
    want = case.qkv.view(np.uint16).copy()
    rest = np.zeros_like(want)
    for i, (rows, target) in enumerate(((q, want if q_base is base else rest), (k, want if k_base is base else rest))):
        target[case.live, case.at[i]:case.at[i + 1]] = rows[case.live]
    assert np.array_equal(base.download(np.uint16, want.shape), want)
    assert np.array_equal(side.download(np.uint16, want.shape), rest)
    one.close()
    two.close()


def host_columns(case, values, dtype=None):
    """One array of the host and its columns: queries, keys, values."""
    torch = pytest.importorskip("torch")
    wide = torch.from_numpy(values.copy())
    return wide, [wide[:, a:b] for a, b in zip(case.at, case.at[1:])]


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16], ids=lambda d: d.name)
@pytest.mark.parametrize("in_place", [False, True])
def test_forward_into_columns_of_one_host_array(engine, dtype, in_place):
    case = NormCase(62, 13, 4, 2, 64, dtype=dtype, offset=8)
    inputs, keep = case.inputs(engine)
    q, k = (engine.makeBufferFrom(np.zeros((case.R, n, case.D), case.io)) for n in (case.H, case.KVH))
    engine.normRotate(pam.PagedNormRotateRequest(**inputs, **case.common(engine), qOut=q, kOut=k))
    want = case.qkv.copy() if in_place else np.full_like(case.qkv, 7)
    for i, (rows, n) in enumerate(((q, case.H), (k, case.KVH))):
        want[case.live, case.at[i]:case.at[i + 1]] = rows.download(case.io, (case.R, n * case.D))[case.live]
    source, columns = host_columns(case, case.qkv)
    target, outs = (source, columns) if in_place else host_columns(case, np.full_like(case.qkv, 7))
    common = case.common(engine)
    engine.normRotate(pam.PagedNormRotateRequest(q=columns[0], k=columns[1], qStride=case.wide, kStride=case.wide, **common,
                                                 qOut=outs[0], qOutStride=case.wide, kOut=outs[1], kOutStride=case.wide))
    assert np.array_equal(target.numpy(), want)
    if not in_place:
        assert np.array_equal(source.numpy(), case.qkv)


@pytest.mark.parametrize("dtype", [DT.float32, DT.float16], ids=lambda d: d.name)
@pytest.mark.parametrize("pages", [False, True])
def test_gradient_into_columns_of_one_host_array(engine, dtype, pages):
    case = NormCase(63, 13, 4, 2, 64, dtype=dtype, offset=8)
    rng = np.random.default_rng(64)
    up, rnd = engine.makeBufferFrom, lambda *s: rng.standard_normal(s, dtype=np.float32).astype(case.io)
    dq_out, pool = rnd(case.R, case.H, case.D), (case.blocks, case.KVH, case.block, case.D)
    keys = dict(dKPool=up(rnd(*pool)), dVPool=up(rnd(*pool)), slots=up(case.slots)) if pages else dict(dKOut=up(rnd(case.R, case.KVH, case.D)))
    inputs, keep = case.inputs(engine)
    inputs = {x: y for x, y in inputs.items() if x not in ("v", "vStride")}
    strides = dict(dQStride=case.wide, dKStride=case.wide, **(dict(dVStride=case.wide) if pages else {}))

    def run(target, weights):
        dv = dict(dV=target[2]) if pages else {}
        engine.normRotateBackward(pam.PagedNormRotateBackwardRequest(
            **inputs, **case.common(engine), dQOut=up(dq_out), **keys, **strides, dQ=target[0], dK=target[1], **dv,
            dQWeight=weights[0], dKWeight=weights[1]))

    fill = np.full_like(case.qkv, 7)
    base, es = up(fill), fill.itemsize
    weights = [up(np.zeros(case.D, np.float32)) for _ in range(2)]
    run([pam_buffer(base, a * es, base.nbytes - a * es) for a in case.at[:3]], weights)
    host, columns = host_columns(case, fill)
    host_weights = [np.zeros(case.D, np.float32) for _ in range(2)]
    run(columns, host_weights)
    assert np.array_equal(host.numpy(), base.download(case.io, fill.shape))
    for a, b in zip(weights, host_weights):
        assert np.array_equal(a.download(np.float32, (case.D,)), b)


@pytest.mark.parametrize("shape", [dict(heads=8, kv_heads=2, dim=64), dict(heads=4, kv_heads=2, dim=24, rotary=16)], ids=lambda s: f"dim{s['dim']}")
@pytest.mark.parametrize("off", ["v", "kOut", "both"])
def test_float8_append_of_rows_off_the_16_byte_grid(engine, shape, off):
    """Back-to-back values and key rows that start one element into their buffers: the pages equal those of
    reshapeAndCache over aligned copies of the same rows."""
    case = NormCase(65, rows=30, dtype=DT.float8, fused=False, **shape)
    one, two = (pam.KVCacheManager(engine, case.blocks, case.block, case.D, case.KVH, DT.float8) for _ in range(2))
    n = case.R * case.KVH * case.D
    shifted = lambda values, by: engine.makeBufferFrom(np.concatenate([np.zeros(by, np.float16), values.reshape(-1)]))
    v_by, k_by = int(off in ("v", "both")), int(off in ("kOut", "both"))
    inputs, keep = case.inputs(engine)
    v_base, k_base = shifted(case.v, v_by), shifted(np.zeros(n, np.float16), k_by)
    inputs["v"] = pam_buffer(v_base, 2 * v_by, 2 * n)
    engine.normRotate(pam.PagedNormRotateRequest(
        **inputs, **case.common(engine), qOut=engine.makeBuffer(case.R * case.H * case.D * 2), kOut=pam_buffer(k_base, 2 * k_by, 2 * n),
        slots=engine.makeBufferFrom(case.slots)), one)
    keys = engine.makeBufferFrom(k_base.download(np.float16, (n,), 2 * k_by))
    engine.reshapeAndCache(two, keys, engine.makeBufferFrom(np.ascontiguousarray(case.v)),
                           engine.makeBufferFrom(np.where(case.live, case.slots, -1)), case.R)
    pools_equal(one, two)
    one.close()
    two.close()
