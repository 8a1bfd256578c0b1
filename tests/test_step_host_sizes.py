"""Refusals of the calls of a speculative step that come from arithmetic on large sizes, without a GPU."""
import pytest

import pagedattentionmetal_b200 as pam
from pagedattentionmetal_b200._cabi import lib
from test_step_host import CALLS, TOO_SMALL, ctx, norm, norm_backward, plan, tree      # noqa: F401

FAR = 1 << 40                     # the largest stride that is taken, in elements
ROWS = (1 << 24) + 1              # (ROWS - 1) * FAR = 2^64


@pytest.mark.parametrize("make,stride,text", [
    (norm, "qStride", b"Q"), (norm, "kStride", b"K"), (norm, "vStride", b"V"), (norm, "qOutStride", b"qOut"),
    (norm, "kOutStride", b"kOut"), (norm_backward, "dQStride", b"dQ"), (norm_backward, "dKStride", b"dK"),
    (tree, "qStride", b"Q"), (tree, "kStride", b"K"), (tree, "vStride", b"V")])
def test_rows_whose_extent_passes_64_bits(ctx, make, stride, text):     # noqa: F811
    """The extent of the strided rows must not wrap round to one that fits their buffer."""
    request = make(numRows=ROWS, **{stride: FAR})
    buffers = {norm: ("q", "k", "v", "qOut", "kOut", "slots", "positions"),
               norm_backward: ("q", "k", "dQOut", "dKOut", "dQ", "dK", "positions"), tree: ("q", "k", "v", "output", "masks")}[make]
    for name in buffers:
        getattr(request._c, request._fields[name][0]).bytes = 1 << (20 if name == stride.removesuffix("Stride") else 50)
    assert CALLS[type(request)](ctx, request) == -1
    assert lib.pamc_last_error_code(ctx) == TOO_SMALL
    assert lib.pam_last_error(ctx).startswith(text + b" buffer is too small")


def test_lists_of_tiles_that_a_blocks_share_would_push_past_31_bits(ctx):     # noqa: F811
    """A block's piece of the list ends at its begin plus its share; begin + share must not pass 2^31."""
    text = b"split the batch"
    for blocks, refused in ((1073741820, True), (1 << 30, True), ((1 << 30) - (1 << 23) - 16, False)):
        request = tree(batchSize=1, numRows=4, maxNewTokens=4, maxNumBlocks=blocks)
        request.layer = pam.PagedLayerSpec(64, 2, 2, 32, pam.PagedAttentionDataType.float16, 0)     # (a tile for each block and head)
        assert CALLS[type(request)](ctx, request) == -1
        assert (text in lib.pam_last_error(ctx)) == refused, blocks


def test_total_lengths_over_lengths_are_refused(ctx):     # noqa: F811
    request = plan()
    request.totalLengths = request.lengths
    assert CALLS[type(request)](ctx, request) == -1 and b"totalLengths" in lib.pam_last_error(ctx)


def test_pages_of_more_than_31_bits_of_tokens_are_refused(ctx):     # noqa: F811
    """numKVHeads * blockSize is counted in 32 bits: at 2^32 it was the zero that the launch divided by."""
    request = tree(batchSize=1, numRows=1, maxNewTokens=1, maxNumBlocks=1)
    for heads, block, refused in ((1 << 16, 1 << 16, True), (1 << 15, 1 << 16, True), (1 << 14, 1 << 16, False)):
        request.layer = pam.PagedLayerSpec(64, heads, heads, block, pam.PagedAttentionDataType.float16, 0)
        assert CALLS[type(request)](ctx, request) == -1
        assert (b"numKVHeads times blockSize" in lib.pam_last_error(ctx)) == refused
