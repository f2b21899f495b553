"""The serving entry points without a GPU: sizes of the cache, argument errors (all
reported before any HIP runtime call), and the ctypes structures against the header."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

import tilemix
from tilemix import api, serving

HEADER = Path(__file__).resolve().parent.parent / "include" / "tilemix_capi.h"
INVALID, NOT_SUPPORTED = api.ERROR_INVALID_VALUE, api.ERROR_NOT_SUPPORTED
CONFIGURATION = api.ERROR_INVALID_CONFIGURATION
NAN, INF = float("nan"), float("inf")

_memory = np.zeros(64, dtype=np.uint8)
X = (_memory.ctypes.data + 15) // 16 * 16  # a 16-byte aligned host address, never read


def packed(**options):
    return tilemix.PackedAttentionArgs(**{**dict(Q=X, K=X, V=X, O=X, q_starts=X, k_starts=X, batch=2, q_tokens=5, k_tokens=7,
                                                 q_heads=4, kv_heads=2, d=64, dtype=tilemix.DTYPE_F16, score_scale=1.0), **options})


def append(**options):
    return tilemix.Cache4AppendArgs(**{**dict(
        Q=X, K=X, V=X, Q_out=X, K_out=X, slots=X, cache=X, cos_sin=X, token_positions=X, positions=9, rotary_dim=64, pages=3,
        page_size=32, tokens=5, q_heads=4, kv_heads=2, d=64, dtype=tilemix.DTYPE_BF16), **options})


def gather(**options):
    return tilemix.Cache4GatherArgs(**{**dict(cache=X, slots=X, K_out=X, V_out=X, pages=3, page_size=32, tokens=5, kv_heads=2,
                                              d=64, dtype=tilemix.DTYPE_F16), **options})


def decode(**options):
    return tilemix.Cache4AttentionArgs(**{**dict(
        Q=X, O=X, cache=X, block_table=X, lengths=X, workspace=X,
        workspace_bytes=tilemix.attention_cache4_workspace_bytes(), pages=3, page_size=64, max_pages=2, batch=2, q_heads=4,
        kv_heads=2, d=64, dtype=tilemix.DTYPE_F16, score_scale=1.0), **options})


CALLS = {"packed": (tilemix.attention_packed, packed), "append": (tilemix.cache4_append, append),
         "gather": (tilemix.cache4_gather, gather), "decode": (tilemix.attention_cache4, decode)}


def code(kind, **options):
    call, args = CALLS[kind]
    return call(args(**options))


def test_cache_sizes(tm):
    # 32 tokens: codes of 64 or 128 features for keys and values, a scale and a minimum per 64.
    for d in (8, 40, 64):
        assert tm.cache4_block_bytes(d) == 32 * (32 + 32 + 4 + 4)
    for d in (72, 96, 128):
        assert tm.cache4_block_bytes(d) == 32 * (64 + 64 + 8 + 8)
    for d in (0, -8, 4, 100, 129, 136):
        assert tm.cache4_block_bytes(d) == 0
    assert tm.cache4_bytes(10, 64, 8, 128) == 10 * 2 * 8 * 4608
    assert tm.cache4_bytes(1 << 20, 256, 8, 128) == (1 << 20) * 8 * 8 * 4608  # past 2^32
    for pages, page_size, heads, d in ((0, 32, 1, 64), (1, 0, 1, 64), (1, 33, 1, 64), (1, 16, 1, 64), (1, 32, 0, 64),
                                       (1, 32, 1, 12), (-1, 32, 1, 64), (1 << 31, 32, 1, 64)):
        assert tm.cache4_bytes(pages, page_size, heads, d) == 0
    assert 0 < tm.attention_cache4_workspace_bytes() <= 16 << 20


@pytest.mark.parametrize("kind", CALLS)
def test_null_arguments(tm, kind):
    assert getattr(tm.library(), {"packed": "tilemix_attention_packed", "append": "tilemix_cache4_append",
                                  "gather": "tilemix_cache4_gather", "decode": "tilemix_attention_cache4"}[kind])(None, None) == INVALID
    required = {"packed": "Q K V O q_starts", "append": "K V slots cache cos_sin token_positions Q Q_out",
                "gather": "cache slots", "decode": "Q O cache block_table lengths workspace"}[kind]
    for name in required.split():
        assert code(kind, **{name: None}) == INVALID, name
    assert code("gather", K_out=None, V_out=None) == INVALID


@pytest.mark.parametrize("kind", CALLS)
def test_sizes_types_and_alignment(tm, kind):
    for d in (0, -8, 4, 60, 65, 127):
        assert code(kind, d=d, **({"rotary_dim": 0} if kind == "append" else {})) == INVALID, d
    for d in (129, 136, 2 ** 31 - 1):
        assert code(kind, d=d) == NOT_SUPPORTED, d
    for dtype in (tm.DTYPE_F32, 3, -1):
        assert code(kind, dtype=dtype) == INVALID
    assert code(kind, kv_heads=0) == INVALID and code(kind, kv_heads=-1) == INVALID
    if kind in ("packed", "decode"):
        assert code(kind, kv_heads=3) == INVALID and code(kind, q_heads=0) == INVALID
        assert code(kind, batch=-1) == INVALID
        for scale in (NAN, INF, -INF):
            assert code(kind, score_scale=scale) == INVALID
        assert code(kind, O=X + 4) == INVALID and code(kind, o_row_stride=4 * 64 + 2) == INVALID
    if kind in ("append", "gather"):
        assert code(kind, tokens=-1) == INVALID
    if kind != "packed":
        for bad in (dict(pages=0), dict(pages=-1), dict(pages=1 << 31), dict(page_size=0), dict(page_size=16),
                    dict(page_size=48), dict(page_size=-32), dict(cache=X + 8)):
            assert code(kind, **bad) == INVALID, bad
    tensors = {"packed": {"q": "Q", "k": "K", "v": "V"}, "append": {"q": "Q", "k": "K", "v": "V", "q_out": "Q_out", "k_out": "K_out"},
               "gather": {"k": "K_out", "v": "V_out"}, "decode": {"q": "Q"}}[kind]
    for name, tensor in tensors.items():
        heads = 2 if tensor[0] in "KV" else 4
        assert code(kind, **{tensor: X + 8}) == INVALID, tensor                                  # 16-byte rows
        assert code(kind, **{f"{name}_row_stride": heads * 64 + 4}) == INVALID, name             # whole pieces
        assert code(kind, **{f"{name}_row_stride": heads * 64 - 8}) == INVALID, name             # rows overlap
        assert code(kind, **{f"{name}_head_stride": 56}) == INVALID, name                        # heads overlap
        assert code(kind, **{f"{name}_row_stride": -heads * 64}) == INVALID, name
        assert code(kind, **{f"{name}_head_stride": -64}) == INVALID, name
        assert code(kind, **{f"{name}_row_stride": 1 << 41}) == INVALID, name


def test_refusals_of_one_operator(tm):
    for rotary in (-2, 3, 66, 128):
        assert code("append", rotary_dim=rotary) == INVALID
    assert code("append", positions=0) == INVALID and code("append", q_heads=0) == INVALID
    assert code("decode", max_pages=0) == INVALID and code("decode", table_stride=1) == INVALID
    assert code("decode", table_stride=-2) == INVALID
    assert code("decode", workspace=X + 4) == INVALID
    assert code("decode", workspace_bytes=tm.attention_cache4_workspace_bytes() - 1) == INVALID
    for stride in ("k_row_stride", "v_row_stride"):
        assert code("packed", **{stride: (1 << 24) + 8}) == NOT_SUPPORTED
    assert code("packed", q_tokens=-1) == INVALID and code("packed", k_tokens=-1) == INVALID


def test_calls_too_large_for_a_launch(tm):
    """Fewer than 2^32 threads and, for the decode step, 2^30 places of blocks."""
    large = dict(kv_heads=1, d=128, tokens=1 << 28)
    assert code("append", **large, q_heads=1) == CONFIGURATION and code("gather", **large) == CONFIGURATION
    for tokens in (1 << 29, 2 ** 31 - 1):
        assert code("append", **{**large, "d": 64, "tokens": tokens}, q_heads=1) == CONFIGURATION
        assert code("gather", **{**large, "d": 64, "tokens": tokens}) == CONFIGURATION
    assert code("packed", q_tokens=2 ** 31 - 1, q_heads=2) == CONFIGURATION
    assert code("packed", q_tokens=1 << 27, q_heads=16, batch=1) == CONFIGURATION
    assert code("decode", batch=1 << 20, max_pages=1 << 20) == CONFIGURATION
    assert code("decode", batch=2 ** 31 - 1, max_pages=2 ** 31 - 1) == CONFIGURATION


def test_rows_in_place_have_one_layout(tm):
    for other in (dict(q_row_stride=512), dict(q_out_row_stride=512), dict(k_out_row_stride=256), dict(k_head_stride=128, k_row_stride=256)):
        assert code("append", **other) == INVALID, other


def test_host_tensors_are_refused(tm):
    import torch

    host = torch.zeros(64, dtype=torch.float16)
    for kind, names in (("packed", ("Q", "q_starts")), ("append", ("K", "slots", "cos_sin")), ("gather", ("K_out", "cache")),
                        ("decode", ("lengths", "workspace", "O"))):
        for name in names:
            assert code(kind, **{name: host}) == INVALID, (kind, name)


def test_calls_with_nothing_to_do(tm):
    """No device is asked for: they succeed on a machine without a GPU."""
    assert code("packed", batch=0) == 0 and code("packed", q_tokens=0, Q=None, O=None) == 0
    assert code("append", tokens=0, K=None, V=None, Q=None, Q_out=None, K_out=None, slots=None) == 0
    assert code("gather", tokens=0, K_out=None, V_out=None, slots=None) == 0
    assert code("decode", batch=0, Q=None, O=None, block_table=None, lengths=None) == 0


def test_structures_match_the_header():
    text = HEADER.read_text()
    for structure, name in ((serving._PackedArgs, "TileMixPackedAttentionArgs"), (serving._AppendArgs, "TileMixCache4AppendArgs"),
                            (serving._GatherArgs, "TileMixCache4GatherArgs"), (serving._Cache4AttentionArgs, "TileMixCache4AttentionArgs")):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        kinds = {"int": ctypes.c_int, "float": ctypes.c_float, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t}
        fields = []
        for line in filter(None, (x.strip() for x in body.split(";"))):
            kind, field = line.rsplit(None, 1) if "*" not in line else ("pointer", line.split("*")[1].strip())
            fields.append((field, ctypes.c_void_p if kind == "pointer" else kinds[kind]))
        assert [tuple(f) for f in structure._fields_] == fields, name


class _DeviceTensor:
    """What the binding asks of a tensor, as one of device 0 answers; its memory is never read."""

    def __init__(self, dtype, contiguous=True, shape=(64,), strides=(1,)):
        self.dtype, self._contiguous, self.shape, self._strides = dtype, contiguous, shape, strides

    def get_device(self):
        return 0

    def data_ptr(self):
        return X

    def is_contiguous(self):
        return self._contiguous

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def dim(self):
        return len(self.shape)


ROWS = "Q K V O Q_out K_out V_out".split()
INDEX_TYPES = dict(q_starts="int32", k_starts="int32", token_positions="int32", block_table="int32", lengths="int32", slots="int64",
                   cos_sin="float32")
TENSORS = {"packed": "Q K V O q_starts k_starts", "append": "Q K V Q_out K_out cos_sin token_positions slots",
           "gather": "slots K_out V_out", "decode": "Q O block_table lengths"}
TENSORS = {kind: names.split() for kind, names in TENSORS.items()}


def _with_tensors(monkeypatch, kind, **changed):
    """The code of a call of device tensors of the right types but for `changed`."""
    import torch

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    call, args = CALLS[kind]
    dtype = torch.bfloat16 if kind == "append" else torch.float16
    tensors = {n: _DeviceTensor(getattr(torch, INDEX_TYPES[n]) if n in INDEX_TYPES else dtype) for n in TENSORS[kind]}
    return call(args(**{**tensors, **changed}), stream=0)


@pytest.mark.parametrize("kind", CALLS)
def test_tensors_of_other_types_are_refused(tm, monkeypatch, kind):
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls that pass the checks are stopped by the missing GPU")
    for name in TENSORS[kind]:
        right = {INDEX_TYPES[name]} if name in INDEX_TYPES else {"bfloat16" if kind == "append" else "float16", "int16", "uint16"}
        for other in ("uint8", "int16", "uint16", "int32", "int64", "float16", "bfloat16", "float32", "float64"):
            got = _with_tensors(monkeypatch, kind, **{name: _DeviceTensor(getattr(torch, other))})
            assert (got != INVALID) == (other in right), (name, other, got)
    if kind != "packed":
        assert _with_tensors(monkeypatch, kind, cache=_DeviceTensor(torch.int32)) != INVALID  # bytes, whatever holds them


@pytest.mark.parametrize("kind", CALLS)
def test_tensors_of_other_layouts_are_refused(tm, monkeypatch, kind):
    """What a call has no stride for is read as it lies: a view with gaps would be other values."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls that pass the checks are stopped by the missing GPU")
    types = {**{n: t for n, t in INDEX_TYPES.items() if n != "block_table"}, "cache": "uint8", "workspace": "uint8"}
    for name in [n for n in TENSORS[kind] if n in types] + {"packed": [], "decode": ["cache", "workspace"]}.get(kind, ["cache"]):
        for contiguous in (True, False):
            got = _with_tensors(monkeypatch, kind, **{name: _DeviceTensor(getattr(torch, types[name]), contiguous=contiguous)})
            assert (got != INVALID) == contiguous, (name, contiguous)
    for name in set(TENSORS[kind]) & set(ROWS):  # these have strides of their own
        dtype = torch.bfloat16 if kind == "append" else torch.float16
        assert _with_tensors(monkeypatch, kind, **{name: _DeviceTensor(dtype, contiguous=False)}) != INVALID


def test_rows_of_a_block_table_are_as_far_apart_as_the_call_says(tm, monkeypatch):
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls that pass the checks are stopped by the missing GPU")

    def table(strides, **options):
        tensor = _DeviceTensor(torch.int32, contiguous=False, shape=(2,) * len(strides), strides=strides)
        return _with_tensors(monkeypatch, "decode", block_table=tensor, **options) != INVALID  # batch 2, max_pages 2

    assert table((2, 1)) and table((7, 1), table_stride=7) and table((7, 1), batch=1)
    assert not table((7, 1)) and not table((2, 1), table_stride=7) and not table((1, 2)) and not table((14, 2), table_stride=14)
    assert table((1, 5), max_pages=1) and table((5, 5), max_pages=1, table_stride=5) and not table((2,))


@pytest.mark.parametrize("kind,rows,heads", [("packed", "q_tokens", 4), ("packed", "k_tokens", 2), ("append", "tokens", 2),
                                             ("gather", "tokens", 2), ("decode", "batch", 4)])
def test_strides_whose_reach_passes_63_bits_are_refused(tm, kind, rows, heads):
    """2^23 rows 2^40 elements apart: their extent is 2^63, which as a signed product looks like
    none, and heads that lie inside one another's rows like heads that follow one another."""
    for name in "qo" if heads == 4 else "kv":
        for head in (1 << 40, 128):
            options = {rows: (1 << 23) + 1, f"{name}_row_stride": 1 << 40, f"{name}_head_stride": head}
            assert code(kind, **options) == INVALID, options
    import torch

    if not torch.cuda.is_available() and (kind != "packed" or rows == "q_tokens"):  # (key rows at most 2^24 apart) a few rows may lie as far apart
        assert code(kind, **{f"{name}_row_stride": 1 << 40, f"{name}_head_stride": 128}) != INVALID
