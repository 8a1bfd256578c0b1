"""The calls of a speculative step without a GPU: every refusal that comes before the device is
needed, the requests' own behaviour, and the plain restatements against one another."""
import ctypes as C

import numpy as np
import pytest

import pagedattentionmetal_b200 as pam
from oracle import step_oracle as so
from pagedattentionmetal_b200._cabi import lib

DT = pam.PagedAttentionDataType
CALLS = {pam.PagedStepPlanRequest: lambda ctx, r: lib.pamc_plan_step(ctx, r._ref),
         pam.PagedNormRotateRequest: lambda ctx, r: lib.pamc_norm_rotate(ctx, r._ref, None),
         pam.PagedNormRotateBackwardRequest: lambda ctx, r: lib.pamc_norm_rotate_backward(ctx, r._ref),
         pam.PagedTreeAttentionRequest: lambda ctx, r: lib.pamc_tree_attention(ctx, r._ref),
         pam.PagedAcceptRequest: lambda ctx, r: lib.pamc_accept_tree(ctx, r._ref)}


@pytest.fixture
def ctx():
    c = lib.pamc_create_host_context()
    yield c
    lib.pam_destroy_context(c)


def i32(*shape):
    return np.zeros(shape, np.int32)


def plan(**change):
    B, R, stride = 3, 10, 4
    args = dict(blockLists=i32(B, stride), lengths=i32(B), newTokens=i32(B), batchSize=B, numLists=B, listStride=stride,
                blockSize=16, numRows=R, maxNewTokens=8, tables=i32(B, 4), maxNumBlocks=4, totalLengths=i32(B),
                rowStarts=i32(B + 1), positions=i32(R), masks=i32(R, 1), maskWords=1)
    args.update(change)
    return pam.PagedStepPlanRequest(**args)


def accept(**change):
    B, R = 3, 10
    args = dict(rowStarts=i32(B + 1), parents=i32(R), draftTokens=i32(R), targetTokens=i32(R), lengths=i32(B), batchSize=B,
                numRows=R, maxTree=8, blockTables=i32(B, 4), maxNumBlocks=4, blockSize=16, slots=np.zeros(R, np.int64),
                acceptedCounts=i32(B), acceptedRows=i32(B, 8), maxPath=8, nextTokens=i32(B), newLengths=i32(B))
    args.update(change)
    return pam.PagedAcceptRequest(**args)


def layer(dtype=DT.float16, dim=64, heads=4, kv=2, block=16, window=0):
    return pam.PagedLayerSpec(dim, heads, kv, block, dtype, window)


def f16(*shape):
    return np.zeros(shape, np.float16)


def norm(**change):
    R, H, KVH, D = 5, 4, 2, 64
    args = dict(q=f16(R, H, D), k=f16(R, KVH, D), v=f16(R, KVH, D), qWeight=f16(D), kWeight=f16(D),
                invFreq=np.zeros(D // 2, np.float32), positions=i32(R), qOut=f16(R, H, D), kOut=f16(R, KVH, D), numRows=R,
                rotaryDim=D, layer=layer(), kPool=f16(3, KVH, 16, D), vPool=f16(3, KVH, 16, D), slots=np.zeros(R, np.int64))
    args.update(change)
    return pam.PagedNormRotateRequest(**args)


def norm_backward(**change):
    R, H, KVH, D = 5, 4, 2, 64
    args = dict(q=f16(R, H, D), k=f16(R, KVH, D), qWeight=f16(D), kWeight=f16(D), invFreq=np.zeros(D // 2, np.float32),
                positions=i32(R), dQOut=f16(R, H, D), dKOut=f16(R, KVH, D), dQ=f16(R, H, D), dK=f16(R, KVH, D), numRows=R,
                rotaryDim=D, layer=layer(), dQWeight=np.zeros(D, np.float32), dKWeight=np.zeros(D, np.float32))
    args.update(change)
    return pam.PagedNormRotateBackwardRequest(**args)


def tree(**change):
    B, R, H, KVH, D = 2, 6, 4, 2, 64
    args = dict(q=f16(R, H, D), k=f16(R, KVH, D), v=f16(R, KVH, D), kPool=f16(3, KVH, 16, D), vPool=f16(3, KVH, 16, D),
                blockTables=i32(B, 4), cacheLengths=i32(B), rowStarts=i32(B + 1), masks=i32(R, 1), output=f16(R, H, D),
                batchSize=B, maxNumBlocks=4, numRows=R, maxNewTokens=6, maskWords=1, layer=layer())
    args.update(change)
    return pam.PagedTreeAttentionRequest(**args)


INVALID, TOO_SMALL, UNSUPPORTED, NO_GPU = 4, 5, 8, 1
REFUSALS = [
    (plan, dict(batchSize=0), INVALID, b"batchSize"), (plan, dict(batchSize=65537), INVALID, b"batchSize"),
    (plan, dict(blockSize=0), INVALID, b"blockSize"), (plan, dict(numRows=0), INVALID, b"numRows"),
    (plan, dict(maxNewTokens=0), INVALID, b"maxNewTokens"), (plan, dict(listStride=0), INVALID, b"listStride"),
    (plan, dict(maxNumBlocks=0), INVALID, b"maxNumBlocks"), (plan, dict(maskWords=0), INVALID, b"maskWords"),
    (plan, dict(maxNewTokens=33), INVALID, b"maskWords"),
    (plan, dict(parents=i32(10), maxNewTokens=1025, maskWords=64, masks=i32(10, 64)), INVALID, b"1024 nodes"),
    (plan, dict(parents=i32(10), slots=np.zeros(10, np.int64)), INVALID, b"no slots"),
    (plan, dict(lengths=i32(2)), TOO_SMALL, b"lengths"), (plan, dict(rowStarts=i32(3)), TOO_SMALL, b"rowStarts"),
    (plan, dict(positions=i32(9)), TOO_SMALL, b"positions"), (plan, dict(blockLists=i32(2, 4)), TOO_SMALL, b"blockLists"),
    (plan, dict(newTokens=None), TOO_SMALL, b"newTokens"), (plan, dict(slots=np.zeros(9, np.int64)), TOO_SMALL, b"slots"),
    (accept, dict(batchSize=0), INVALID, b"batchSize"), (accept, dict(maxTree=0), INVALID, b"maxTree"),
    (accept, dict(maxTree=1025), INVALID, b"maxTree"), (accept, dict(maxPath=0), INVALID, b"maxPath"),
    (accept, dict(blockTables=None), INVALID, b"slots need"), (accept, dict(numRows=0), INVALID, b"numRows"),
    (accept, dict(parents=i32(9)), TOO_SMALL, b"parents"), (accept, dict(acceptedRows=i32(3, 7)), TOO_SMALL, b"acceptedRows"),
    (norm, dict(rotaryDim=63), INVALID, b"rotaryDim"), (norm, dict(rotaryDim=66), INVALID, b"rotaryDim"),
    (norm, dict(numRows=0), INVALID, b"numRows"), (norm, dict(epsilon=-1.0), INVALID, b"epsilon"),
    (norm, dict(epsilon=float("nan")), INVALID, b"epsilon"), (norm, dict(qStride=255), INVALID, b"qStride"),
    (norm, dict(kOutStride=-5), INVALID, b"kOutStride"), (norm, dict(vPool=None), INVALID, b"both kPool and vPool"),
    (norm, dict(kPool=None, vPool=None, kOut=None), INVALID, b"kOut or pages"),
    (norm, dict(layer=layer(DT.float8)), INVALID, b"cache handle"),
    (norm, dict(layer=layer(dim=512), rotaryDim=64), UNSUPPORTED, b"headDim above 256"),
    (norm, dict(layer=layer(heads=3)), INVALID, b"divisible"),
    (norm, dict(q=f16(4, 4, 64)), TOO_SMALL, b"Q"), (norm, dict(slots=None), TOO_SMALL, b"slots"),
    (norm, dict(v=None), TOO_SMALL, b"V"), (norm, dict(invFreq=np.zeros(31, np.float32)), TOO_SMALL, b"invFreq"),
    (norm, dict(kPool=f16(1, 1, 16, 64)), TOO_SMALL, b"K pool"),
    (norm, dict(qStride=300), TOO_SMALL, b"Q"),
    (norm_backward, dict(layer=layer(DT.float8)), UNSUPPORTED, b"FP8"),
    (norm_backward, dict(dKPool=f16(3, 2, 16, 64)), INVALID, b"not from both"),
    (norm_backward, dict(dV=f16(5, 2, 64)), INVALID, b"dV"), (norm_backward, dict(dKOut=None), TOO_SMALL, b"dKOut"),
    (norm_backward, dict(dKOut=None, dKPool=f16(3, 2, 16, 64)), TOO_SMALL, b"slots"),
    (norm_backward, dict(dKOut=None, dKPool=f16(3, 2, 16, 64), slots=np.zeros(5, np.int64), dV=f16(5, 2, 64)), TOO_SMALL, b"dV pool"),
    (norm_backward, dict(dKWeight=np.zeros(63, np.float32)), TOO_SMALL, b"dKWeight"),
    (norm_backward, dict(workspace=np.zeros(4, np.float32)), TOO_SMALL, b"workspace"),
    (tree, dict(batchSize=0), INVALID, b"batchSize"), (tree, dict(batchSize=4097), INVALID, b"batchSize"),
    (tree, dict(maxNumBlocks=0), INVALID, b"maxNumBlocks"), (tree, dict(maxNewTokens=33), INVALID, b"maskWords"),
    (tree, dict(layer=layer(window=4)), INVALID, b"positions"),
    (tree, dict(layer=layer(DT.float8)), INVALID, b"kScaleBuffer"),
    (tree, dict(layer=layer(dim=260)), UNSUPPORTED, b"headDim above 256"),
    (tree, dict(vStride=100), INVALID, b"vStride"), (tree, dict(output=f16(5, 4, 64)), TOO_SMALL, b"output"),
    (tree, dict(cacheLengths=i32(1)), TOO_SMALL, b"cacheLengths"), (tree, dict(rowStarts=i32(2)), TOO_SMALL, b"rowStarts"),
    (tree, dict(workspace=np.zeros(4, np.float32)), TOO_SMALL, b"workspace"),
    (tree, dict(blockTables=i32(2, 1 << 20), maxNumBlocks=1 << 20, numRows=1 << 20, maxNewTokens=1 << 20, masks=None,
                q=None), INVALID, b"split the batch"),
]


@pytest.mark.parametrize("make,change,code,text", REFUSALS, ids=[f"{m.__name__}-{'-'.join(c)}-{i}" for i, (m, c, _, _) in enumerate(REFUSALS)])
def test_refusals_come_before_the_device(ctx, make, change, code, text):
    request = make(**change)
    assert CALLS[type(request)](ctx, request) == -1
    assert lib.pamc_last_error_code(ctx) == code
    assert text in lib.pam_last_error(ctx)


@pytest.mark.parametrize("make", [plan, accept, norm, norm_backward, tree])
def test_valid_requests_only_miss_the_device(ctx, make):
    request = make()
    assert CALLS[type(request)](ctx, request) == -1
    assert lib.pamc_last_error_code(ctx) == NO_GPU
    assert CALLS[type(request)](None, request) == -1


def test_workspace_queries_need_no_device(ctx):
    assert lib.pamc_tree_attention_workspace(ctx, tree()._ref) > 0
    assert lib.pamc_norm_rotate_backward_workspace(ctx, norm_backward()._ref) > 0
    assert lib.pamc_norm_rotate_backward_workspace(ctx, norm_backward(dQWeight=None, dKWeight=None)._ref) == 0
    assert lib.pamc_tree_attention_workspace(ctx, tree(batchSize=0)._ref) == -1
    assert lib.pamc_tree_attention_workspace(ctx, None) == -1


def test_request_fields():
    torch = pytest.importorskip("torch")
    r = tree(vStride=512)
    assert r.vStride == 512 and r._c.v_stride == 512 and r._c.layer.num_heads == 4
    wide = torch.zeros(6, 512, dtype=torch.float16)
    r.v = wide[:, 128:256]                                     # a strided view: first to last element
    assert r._c.v.ptr == wide.data_ptr() + 256 and r._c.v.bytes == (5 * 512 + 128) * 2
    r.masks = None
    assert r._c.masks.ptr is None and r._c.masks.bytes == 0
    with pytest.raises(AttributeError):
        r.window = 3
    with pytest.raises(AttributeError):
        r.nothing
    with pytest.raises(TypeError):
        tree(nothing=1)
    with pytest.raises(TypeError):
        pam.PagedAcceptRequest(batchSize=1)


def test_plain_forms_agree_with_hand_worked_cases():
    # a tree of five nodes: 0 - 1 - 3, 0 - 2, and a second root 4
    parents = np.array([-1, 0, 0, 1, 9], np.int32)
    sees = so.ancestors(parents)
    assert [list(np.nonzero(r)[0]) for r in sees] == [[0], [0, 1], [0, 2], [0, 1, 3], [4]]
    got = so.plan_step([[7, 3, 5]], [30], [5], 6, 8, 16, parents=parents, width=4, words=1)
    assert list(got["positions"]) == [30, 31, 31, 32, 30, -1]
    assert list(got["tables"][0]) == [7, 3, 5, 0] and list(got["masks"][:, 0]) == [1, 3, 5, 11, 16, 0]
    # node 1 is drafted right, node 3 is not; node 2 as well: the lower index wins
    a = so.accept_tree([0, 5], parents, [9, 4, 4, 6, 1], [4, 8, 2, 0, 3], [30], 6, 8, 3, np.array([[7, 3, 5]], np.int32), 16)
    assert list(a["path"][0]) == [0, 1, -1] and a["counts"][0] == 2 and a["next"][0] == 8 and a["totals"][0] == 32
    assert list(a["slots"]) == [3 * 16 + 14, 3 * 16 + 15, -1, -1, -1, -1]


def test_plain_gradient_matches_differences():
    rng = np.random.default_rng(5)
    for rotary, interleaved in ((8, False), (4, True), (0, False)):
        x, w, dy = rng.standard_normal((3, 2, 8)), rng.standard_normal(8), rng.standard_normal((3, 2, 8))
        pos, freq = np.array([0, 5, 100000]), 10.0 ** -np.arange(rotary // 2).astype(np.float64)
        f = lambda x_, w_: (so.norm_rotate(x_, w_, pos, freq, rotary, interleaved, 1e-5)[0] * dy).sum()
        dx, dw, _, _ = so.norm_rotate_backward(x, w, dy, pos, freq, rotary, interleaved, 1e-5)
        h = 1e-6
        for i in np.ndindex(x.shape):
            e = np.zeros_like(x)
            e[i] = h
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx[i]) < 1e-7
        for i in range(8):
            e = np.zeros_like(w)
            e[i] = h
            assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[i]) < 1e-7
