"""Serving entry points of include/tilemix_capi.h: attention of packed sequences
and the paged 4-bit key/value cache. Like the rest of the binding they take torch
device tensors (or raw addresses, ``None`` for NULL), of the current device and of the
types that the header names, and return the hipError_t code; sizes, layouts and errors
are those of the C header. Strides count elements, 0 = dense [tokens, heads, d]; what has
no stride in the call (starts, lengths, slots, positions, the table of angles, the cache,
the workspace) is contiguous, and the rows of a block table lie as far apart as the call
says. Other devices, types and layouts: InvalidValue.
"""
from __future__ import annotations

import ctypes
import struct
import sys
from dataclasses import dataclass
from operator import attrgetter
from typing import Any

from .api import DTYPE_BF16, DTYPE_F16, ERROR_INVALID_VALUE, _stream, library

_vp, _int, _i64, _sz, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float


def _structure(name: str, fields: list[tuple[str, Any]]):
    return type(name, (ctypes.Structure,), {"_fields_": fields})


def _fields(pointers="", sizes="", int64s="") -> list[tuple[str, Any]]:
    return ([(n, _vp) for n in pointers.split()] + [(n, _i64) for n in int64s.split()]
            + [(n, _int) for n in sizes.split()])


_PackedArgs = _structure("_PackedArgs", _fields(
    "Q K V O q_starts k_starts", "batch q_tokens k_tokens q_heads kv_heads d dtype causal") + [("score_scale", _f32)]
    + _fields(int64s="q_row_stride k_row_stride v_row_stride o_row_stride q_head_stride k_head_stride v_head_stride "
                     "o_head_stride"))

_AppendArgs = _structure("_AppendArgs", _fields("Q K V Q_out K_out cos_sin token_positions slots cache", int64s="pages")
    + _fields(sizes="page_size tokens q_heads kv_heads d dtype rotary_dim interleaved positions")
    + _fields(int64s="q_row_stride k_row_stride v_row_stride q_out_row_stride k_out_row_stride q_head_stride "
                     "k_head_stride v_head_stride q_out_head_stride k_out_head_stride"))

_GatherArgs = _structure("_GatherArgs", _fields("cache slots K_out V_out", int64s="pages")
    + _fields(sizes="page_size tokens kv_heads d dtype")
    + _fields(int64s="k_row_stride v_row_stride k_head_stride v_head_stride"))

_Cache4AttentionArgs = _structure("_Cache4AttentionArgs", _fields("Q O cache block_table lengths workspace")
    + [("workspace_bytes", _sz)] + _fields(int64s="pages table_stride")
    + _fields(sizes="page_size max_pages batch q_heads kv_heads d dtype") + [("score_scale", _f32)]
    + _fields(int64s="q_row_stride o_row_stride q_head_stride o_head_stride"))


class _Entry:
    """An entry point that takes a structure, packed from the fields of the same names of a
    dataclass. The fields are fetched in one call and the bound function is kept, as a decode
    step's kernels are not much longer than the call (of 31 fields: 4.4 us with a ctypes
    structure filled from them, 2.4 us so; the whole call with 9 tensors' devices, types and layouts 3.3)."""

    # Types of what is not a tensor of the call's `dtype`. A kernel takes a tensor of narrower values for as many
    # of its own, and would read past the end; the cache and the workspace are bytes, whatever holds them.
    _TYPES = {**dict.fromkeys(("q_starts", "k_starts", "token_positions", "block_table", "lengths"), "int32"),
              "slots": "int64", "cos_sin": "float32", "cache": None, "workspace": None}
    _DENSE = {"q_starts", "k_starts", "token_positions", "lengths", "slots", "cos_sin", "cache", "workspace"}

    _CODES = {_vp: "P", _int: "i", _i64: "q", _sz: "N", _f32: "f"}

    def __init__(self, name: str, structure):
        names = [n for n, _ in structure._fields_]
        self._names = names
        self._name, self._fetch, self._function = name, attrgetter(*names), None
        self._pointers = sum(1 for _, kind in structure._fields_ if kind is _vp)
        self._dtype, self._known = names.index("dtype"), set()
        self._dense = [i for i, n in enumerate(names) if n in self._DENSE]
        self._table = attrgetter("block_table", "table_stride", "max_pages", "batch") if "block_table" in names else None
        assert all(kind is _vp for _, kind in structure._fields_[:self._pointers])
        # Native sizes and alignment; a C structure also ends at a multiple of its alignment.
        packing = struct.Struct("@" + "".join(self._CODES[kind] for _, kind in structure._fields_) + "0P")
        assert packing.size == ctypes.sizeof(structure)
        self._pack = packing.pack

    def _types_ok(self, dtype, types) -> bool:
        """Whether a call of `dtype` takes tensors of these types (None: no tensor); 16-bit values also as bits."""
        if (dtype, types) not in self._known:
            torch = sys.modules["torch"]
            rows = {DTYPE_F16: (torch.float16,), DTYPE_BF16: (torch.bfloat16,)}.get(dtype, ()) + (torch.int16, torch.uint16)
            for name, found in zip(self._names, types):
                wanted = self._TYPES.get(name, rows)
                if found is not None and wanted is not None and found not in (wanted if wanted is rows else (getattr(torch, wanted),)):
                    return False
            self._known.add((dtype, types))
        return True

    def _layouts_ok(self, args, values) -> bool:
        for i in self._dense:
            x = values[i]
            if x is not None and x.__class__ is not int and not x.is_contiguous():
                return False
        if self._table is not None:
            table, row, pages, batch = self._table(args)
            if table is not None and table.__class__ is not int:
                if table.dim() != 2:
                    return table.is_contiguous()
                between, step = table.stride()
                return (step == 1 or pages == 1) and (between == (row or pages) or batch <= 1)
        return True

    def __call__(self, args, stream) -> int:
        if self._function is None:
            function = getattr(library(), self._name)
            function.argtypes, function.restype = [ctypes.c_char_p, _vp], _int
            self._function = function
        values = self._fetch(args)
        n = self._pointers
        # A kernel of the current device would fault on another's memory, or the host's (device -1).
        pointers, types, device = [], [], None
        for x in values[:n]:
            if x is None or x.__class__ is int:
                pointers.append(x or 0)
                types.append(None)
            else:
                if device is None:
                    device = x.get_device()
                    if device < 0 or device != sys.modules["torch"].cuda.current_device():
                        return ERROR_INVALID_VALUE
                elif x.get_device() != device:
                    return ERROR_INVALID_VALUE
                pointers.append(x.data_ptr())
                types.append(x.dtype)
        if device is not None and not (self._types_ok(values[self._dtype], tuple(types)) and self._layouts_ok(args, values)):
            return ERROR_INVALID_VALUE
        packed = self._pack(*pointers, *values[n:])
        if stream is None and device is not None:  # as _stream, with the device known
            return self._function(packed, sys.modules["torch"]._C._cuda_getCurrentRawStream(device))
        return self._function(packed, _stream(stream))


@dataclass
class PackedAttentionArgs:
    """TileMixPackedAttentionArgs: `batch` packed sequences, starts int32 [batch + 1] device tensors."""
    Q: Any
    K: Any
    V: Any
    O: Any
    q_starts: Any
    batch: int
    q_tokens: int
    k_tokens: int
    q_heads: int
    kv_heads: int
    d: int
    dtype: int  # DTYPE_F16 or DTYPE_BF16
    score_scale: float
    causal: bool = True
    k_starts: Any = None  # None: q_starts
    q_row_stride: int = 0
    k_row_stride: int = 0
    v_row_stride: int = 0
    o_row_stride: int = 0
    q_head_stride: int = 0
    k_head_stride: int = 0
    v_head_stride: int = 0
    o_head_stride: int = 0


@dataclass
class Cache4AppendArgs:
    """TileMixCache4AppendArgs: rotate Q and K, write K and V to the cache at `slots` (int64 [tokens])."""
    K: Any
    V: Any
    slots: Any
    cache: Any
    pages: int
    page_size: int
    tokens: int
    kv_heads: int
    d: int
    dtype: int
    Q: Any = None
    Q_out: Any = None
    q_heads: int = 0
    K_out: Any = None
    cos_sin: Any = None  # fp32 [positions, rotary_dim]: cosines, then sines
    token_positions: Any = None  # int32 [tokens]
    positions: int = 0
    rotary_dim: int = 0
    interleaved: bool = False
    q_row_stride: int = 0
    k_row_stride: int = 0
    v_row_stride: int = 0
    q_out_row_stride: int = 0
    k_out_row_stride: int = 0
    q_head_stride: int = 0
    k_head_stride: int = 0
    v_head_stride: int = 0
    q_out_head_stride: int = 0
    k_out_head_stride: int = 0


@dataclass
class Cache4GatherArgs:
    """TileMixCache4GatherArgs: cached rows at `slots` (int64 [tokens]) back in 16 bits."""
    cache: Any
    slots: Any
    pages: int
    page_size: int
    tokens: int
    kv_heads: int
    d: int
    dtype: int
    K_out: Any = None
    V_out: Any = None
    k_row_stride: int = 0
    v_row_stride: int = 0
    k_head_stride: int = 0
    v_head_stride: int = 0


@dataclass
class Cache4AttentionArgs:
    """TileMixCache4AttentionArgs: one query token per sequence over its pages (block_table int32
    [batch, max_pages], lengths int32 [batch]); `workspace` was set to zero once."""
    Q: Any
    O: Any
    cache: Any
    block_table: Any
    lengths: Any
    workspace: Any
    workspace_bytes: int
    pages: int
    page_size: int
    max_pages: int
    batch: int
    q_heads: int
    kv_heads: int
    d: int
    dtype: int
    score_scale: float
    table_stride: int = 0  # 0: max_pages
    q_row_stride: int = 0
    o_row_stride: int = 0
    q_head_stride: int = 0
    o_head_stride: int = 0


_attention_packed = _Entry("tilemix_attention_packed", _PackedArgs)
_cache4_append = _Entry("tilemix_cache4_append", _AppendArgs)
_cache4_gather = _Entry("tilemix_cache4_gather", _GatherArgs)
_attention_cache4 = _Entry("tilemix_attention_cache4", _Cache4AttentionArgs)


def attention_packed(args: PackedAttentionArgs, stream=None) -> int:
    return _attention_packed(args, stream)


def cache4_append(args: Cache4AppendArgs, stream=None) -> int:
    return _cache4_append(args, stream)


def cache4_gather(args: Cache4GatherArgs, stream=None) -> int:
    return _cache4_gather(args, stream)


def attention_cache4(args: Cache4AttentionArgs, stream=None) -> int:
    return _attention_cache4(args, stream)


def cache4_block_bytes(d: int) -> int:
    """Bytes of 32 tokens of one key head; 0 for a head dimension that is not supported."""
    function = library().tilemix_cache4_block_bytes
    function.argtypes, function.restype = [_int], _sz
    return int(function(d))


def cache4_bytes(pages: int, page_size: int, kv_heads: int, d: int) -> int:
    function = library().tilemix_cache4_bytes
    function.argtypes, function.restype = [_i64, _int, _int, _int], _sz
    return int(function(pages, page_size, kv_heads, d))


def attention_cache4_workspace_bytes() -> int:
    function = library().tilemix_attention_cache4_workspace_bytes
    function.argtypes, function.restype = [], _sz
    return int(function())
