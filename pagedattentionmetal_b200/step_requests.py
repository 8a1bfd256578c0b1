"""Requests of the calls of a speculative step (include/pam_cuda.h: pamc_plan_step,
pamc_norm_rotate, pamc_norm_rotate_backward, pamc_tree_attention, pamc_accept_tree).

A request is a live C struct: assigning a field writes it, so that a serving loop builds
a request once over its static buffers and passes it every step without any conversion.
The buffers assigned to a request are kept alive by it.
"""
from __future__ import annotations

import ctypes as C

from . import _cabi
from .api_types import PagedLayerSpec


# Buffers of rows that may start a stride apart.
_ROWS = {"q", "k", "v", "qOut", "kOut", "dQ", "dK", "dV"}


def _span(x, name: str) -> _cabi.PamBuffer:
    """A buffer argument with its length; a view of strided rows reaches from its first to its last element."""
    if x is None:
        return _cabi.PamBuffer(None, 0)
    if hasattr(x, "is_contiguous"):
        if x.is_contiguous():
            return _cabi.PamBuffer(x.data_ptr(), x.numel() * x.element_size())
        strides, size = x.stride(), x.element_size()
    elif hasattr(x, "flags") and hasattr(x, "strides") and not x.flags.c_contiguous:
        strides, size = [s // x.itemsize for s in x.strides], x.itemsize
    else:
        return _cabi.buffer(x)
    width, shape = 1, x.shape                        # (elements of a row)
    for n, stride in zip(shape[:0:-1], strides[:0:-1]):
        if stride != width and n != 1:
            width = -1
            break
        width *= n
    if name not in _ROWS or width < 0 or strides[0] < 0:
        raise ValueError(f"{name} must be contiguous" + (" within a row" if name in _ROWS else ""))
    return _cabi.PamBuffer(_cabi.address(x), ((shape[0] - 1) * strides[0] + width) * size)


# What the index, scale and frequency buffers hold; arrays and tensors of another type are refused (rows, pages and
# weights hold what the layer says).
_HOLDS = {**{name: "int32" for name in (
              "blockLists", "listIndex", "lengths", "newTokens", "parents", "tables", "totalLengths", "rowStarts", "positions",
              "masks", "draftTokens", "targetTokens", "blockTables", "cacheLengths", "acceptedCounts", "acceptedRows",
              "nextTokens", "newLengths")},
          "slots": "int64", "invFreq": "float32", "dQWeight": "float32", "dKWeight": "float32",
          "kScaleBuffer": "float16", "vScaleBuffer": "float16"}
_TAKEN = {"uint32": "int32", "uint64": "int64"}
_HELD: dict = {}                                     # dtype of an array or a tensor -> what it counts as


def _held(dtype) -> str:
    name = str(dtype).rpartition(".")[2]             # ("torch.int32")
    return _HELD.setdefault(dtype, _TAKEN.get(name, name))


class _Request:
    """Fields by their Python names; `_fields` maps them to the struct's, with the default of a plain number."""
    _struct: type
    _fields: dict
    _required: tuple

    def __init__(self, **values):
        object.__setattr__(self, "_c", self._struct())
        object.__setattr__(self, "_values", {})
        object.__setattr__(self, "_ref", C.byref(self._c))
        missing = [x for x in self._required if x not in values]
        if missing:
            raise TypeError(f"{type(self).__name__} needs {', '.join(missing)}")
        unknown = [x for x in values if x not in self._fields]
        if unknown:
            raise TypeError(f"{type(self).__name__} has no field {', '.join(unknown)}")
        for name, (field, default) in self._fields.items():
            if name in values or default:            # (a new struct is all zeros, as most fields are to begin with)
                setattr(self, name, values.get(name, default))
            else:
                self._values[name] = default

    def __setattr__(self, name, value):
        if name not in self._fields:
            raise AttributeError(f"{type(self).__name__} has no field {name}")
        field, default = self._fields[name]
        if default is None:
            dtype = getattr(value, "dtype", None)
            if dtype is not None and name in _HOLDS and (_HELD.get(dtype) or _held(dtype)) != _HOLDS[name]:
                raise TypeError(f"{type(self).__name__}.{name} holds {_HOLDS[name]}, not {_held(dtype)}")
            c = _span(value, name)
        elif isinstance(value, PagedLayerSpec):
            c = _cabi.PamLayerSpec(value.headDim, value.numHeads, value.numKVHeads, value.blockSize,
                                   int(value.dataType), value.windowSize)
        elif isinstance(default, float):
            c = float(value)
        else:
            c = int(value)
        setattr(self._c, field, c)
        self._values[name] = value

    def __getattr__(self, name):                     # (a name that is no field must not look for _values)
        if name in type(self)._fields and "_values" in self.__dict__:
            return self._values[name]
        raise AttributeError(f"{type(self).__name__} has no field {name}")


def _buffers(**names):
    return {name: (field, None) for name, field in names.items()}


def _numbers(**names):
    return {name: (field, 0) for name, field in names.items()}


class PagedStepPlanRequest(_Request):
    """PamStepPlanRequest: row starts, positions, slots, block tables and masks from the lengths of a batch."""
    _struct = _cabi.PamStepPlanRequest
    _fields = {**_buffers(blockLists="block_lists", listIndex="list_index", lengths="lengths", newTokens="new_tokens",
                          parents="parents", tables="tables", totalLengths="total_lengths", rowStarts="row_starts",
                          positions="positions", slots="slots", masks="masks"),
               **_numbers(batchSize="batch_size", numLists="num_lists", listStride="list_stride",
                          maxNumBlocks="max_num_blocks", blockSize="block_size", numRows="num_rows",
                          maxNewTokens="max_new_tokens", maskWords="mask_words")}
    _required = ("blockLists", "lengths", "newTokens", "batchSize", "numLists", "listStride", "blockSize", "numRows",
                 "maxNewTokens")


class PagedNormRotateRequest(_Request):
    """PamNormRotateRequest: norm and rotation of queries and keys, append to the pages."""
    _struct = _cabi.PamNormRotateRequest
    _fields = {**_buffers(q="q", k="k", v="v", qWeight="q_weight", kWeight="k_weight", invFreq="inv_freq",
                          positions="positions", qOut="q_out", kOut="k_out", kPool="k_pool", vPool="v_pool",
                          slots="slots"),
               **_numbers(qStride="q_stride", kStride="k_stride", vStride="v_stride", qOutStride="q_out_stride",
                          kOutStride="k_out_stride", numRows="num_rows", rotaryDim="rotary_dim",
                          interleaved="interleaved"),
               "epsilon": ("epsilon", 1e-6), "layer": ("layer", PagedLayerSpec(0, 0, 0))}
    _required = ("q", "k", "qWeight", "kWeight", "positions", "qOut", "numRows", "rotaryDim", "layer")


class PagedNormRotateBackwardRequest(_Request):
    """PamNormRotateBackwardRequest: the gradient of PagedNormRotateRequest."""
    _struct = _cabi.PamNormRotateBackwardRequest
    _fields = {**_buffers(q="q", k="k", qWeight="q_weight", kWeight="k_weight", invFreq="inv_freq",
                          positions="positions", dQOut="d_q_out", dKOut="d_k_out", dKPool="d_k_pool", dVPool="d_v_pool",
                          slots="slots", dQ="d_q", dK="d_k", dV="d_v", dQWeight="d_q_weight", dKWeight="d_k_weight",
                          workspace="workspace"),
               **_numbers(qStride="q_stride", kStride="k_stride", dQStride="d_q_stride", dKStride="d_k_stride",
                          dVStride="d_v_stride", numRows="num_rows", rotaryDim="rotary_dim",
                          interleaved="interleaved"),
               "epsilon": ("epsilon", 1e-6), "layer": ("layer", PagedLayerSpec(0, 0, 0))}
    _required = ("q", "k", "qWeight", "kWeight", "positions", "dQOut", "dQ", "dK", "numRows", "rotaryDim", "layer")


class PagedTreeAttentionRequest(_Request):
    """PamTreeAttentionRequest: attention of the rows of a step over the cache and their own trees."""
    _struct = _cabi.PamTreeAttentionRequest
    _fields = {**_buffers(q="q", k="k", v="v", kPool="k_pool", vPool="v_pool", blockTables="block_tables",
                          cacheLengths="cache_lengths", rowStarts="row_starts", masks="masks", positions="positions",
                          output="output", kScaleBuffer="k_scale", vScaleBuffer="v_scale", workspace="workspace"),
               **_numbers(qStride="q_stride", kStride="k_stride", vStride="v_stride", batchSize="batch_size",
                          maxNumBlocks="max_num_blocks", numRows="num_rows", maxNewTokens="max_new_tokens",
                          maskWords="mask_words"),
               "layer": ("layer", PagedLayerSpec(0, 0, 0))}
    _required = ("q", "k", "v", "kPool", "vPool", "blockTables", "cacheLengths", "rowStarts", "output", "batchSize",
                 "maxNumBlocks", "numRows", "maxNewTokens", "layer")


class PagedAcceptRequest(_Request):
    """PamAcceptRequest: the accepted path of every drafted tree, its slots and next token."""
    _struct = _cabi.PamAcceptRequest
    _fields = {**_buffers(rowStarts="row_starts", parents="parents", draftTokens="draft_tokens",
                          targetTokens="target_tokens", lengths="lengths", blockTables="block_tables", slots="slots",
                          acceptedCounts="accepted_counts", acceptedRows="accepted_rows", nextTokens="next_tokens",
                          newLengths="new_lengths"),
               **_numbers(batchSize="batch_size", numRows="num_rows", maxTree="max_tree", maxPath="max_path",
                          maxNumBlocks="max_num_blocks", blockSize="block_size")}
    _required = ("rowStarts", "parents", "draftTokens", "targetTokens", "lengths", "batchSize", "numRows", "maxTree")
