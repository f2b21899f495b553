"""The paged 4-bit cache: tilemix_cache4_append, tilemix_cache4_gather and
tilemix_attention_cache4 against tests/serving_reference.py.

Cached bytes are compared exactly (the codes are defined in fp32), everything else
of the cache with what it held before. Bounds of the attention: probabilities enter
as two bf16 parts (2^-16 of each, beside codes offset by 16: up to 31 scales of a
value's group), fp32 sums, and the output's half step.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _code(tm, dtype):
    return tm.DTYPE_F16 if dtype == "f16" else tm.DTYPE_BF16


def _cache(pages, page_size, heads, d, seed=0):
    """A host cache of random bytes: what nobody wrote may be anything."""
    rng = np.random.default_rng(seed)
    return rng.integers(0, 256, (pages, heads, page_size // 32, ref.block_bytes(d)), dtype=np.uint8)


def _table(positions, rotary):
    angles = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))
    return np.concatenate([np.cos(angles), np.sin(angles)], 1).astype(np.float32)


# ------------------------------------------------------------------ append

def _append(tokens=5, heads=(4, 2), d=64, dtype="f16", rotary=None, interleaved=False, page_size=32, in_place=False,
            layout="thd", special=False, query=True, key_out=True):
    return dict(tokens=tokens, heads=heads, d=d, dtype=dtype, rotary=d if rotary is None else rotary, interleaved=interleaved,
                page_size=page_size, in_place=in_place, layout=layout, special=special, query=query, key_out=key_out)


APPENDS = [
    _append(tokens=1, heads=(1, 1)), _append(tokens=1, heads=(8, 1), d=128, dtype="bf16"), _append(tokens=33, d=8, rotary=8),
    _append(tokens=70, heads=(12, 3), d=128, page_size=64), _append(tokens=40, d=72, rotary=72),  # half of 36: no whole pieces
    _append(tokens=17, d=72, rotary=18, interleaved=True, dtype="bf16"), _append(tokens=9, d=128, rotary=64, dtype="bf16"),
    _append(tokens=9, d=96, rotary=48, page_size=96), _append(tokens=30, d=80, rotary=20), _append(tokens=6, d=128, rotary=2),
    _append(tokens=12, d=64, rotary=0), _append(tokens=12, d=104, rotary=104, interleaved=True), _append(tokens=50, d=40, dtype="bf16"),
    _append(tokens=21, d=128, in_place=True), _append(tokens=21, d=72, rotary=36, in_place=True, dtype="bf16"),
    _append(tokens=19, d=64, layout="fused", dtype="bf16"), _append(tokens=19, d=128, layout="htd"),
    _append(tokens=25, d=64, special=True), _append(tokens=25, d=128, special=True, dtype="bf16"),
    _append(tokens=11, d=128, query=False, key_out=False), _append(tokens=11, d=64, query=False), _append(tokens=11, d=64, key_out=False),
    _append(tokens=300, heads=(16, 8), d=128, page_size=128, dtype="bf16"),
]


def _place_rows(values, layout):
    t, h, d = values.shape
    if layout == "htd":
        return values.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    if layout == "fused":
        row = torch.zeros(t, h + 2, d, dtype=values.dtype)
        row[:, 1:h + 1] = values
        return row.cuda()[:, 1:h + 1]
    return values.cuda()


@pytest.mark.parametrize("c", APPENDS, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_append(tm, cuda, c):
    tokens, (hq, hk), d, size = c["tokens"], c["heads"], c["d"], c["page_size"]
    gen = torch.Generator().manual_seed(tokens * 31 + d)
    dtype = DT[c["dtype"]]
    q, k, v = (torch.randn(tokens, h, d, generator=gen) for h in (hq, hk, hk))
    k[..., ::16] *= 6.0
    if c["special"]:
        k[1, 0, 3], k[2, 1, d - 1], v[3, 0, 0], v[4, 1, 5] = math.nan, math.inf, -math.inf, math.nan
        k[5], v[5] = 0.0, 2.0                      # constant groups
        k[6], v[6] = 1e-7 * k[6], 6e4 * v[6].sign()  # tiny and very large values
        v[7, :, :] = 1.0
        v[7, :, 0] = 1.0078125                     # one step apart
    q, k, v = (x.to(dtype) for x in (q, k, v))
    pages = tokens // size + 4
    rng = np.random.default_rng(5)
    slots = rng.permutation(pages * size)[:tokens].astype(np.int64)
    run = min(tokens, size)
    slots[:run] = 2 * size + np.arange(run)  # a run of consecutive ones
    taken = set(range(2 * size, 2 * size + run))
    free = [s for s in rng.permutation(pages * size) if s not in taken]
    slots[run:] = free[:tokens - run]
    if tokens > 8:
        slots[[4, 8]] = (-1, pages * size)  # padding and one past the last: not cached
    positions = 50
    table = _table(positions, c["rotary"])
    at = rng.integers(0, positions, tokens).astype(np.int32)
    if tokens > 16 and c["rotary"]:
        at[[9, 15]] = (-1, positions)  # outside the table: passed over
    skipped = (at < 0) | (at >= positions) if c["rotary"] else np.zeros(tokens, bool)

    cache = _cache(pages, size, hk, d)
    device_cache = torch.from_numpy(cache).cuda()
    tensors = {x: _place_rows(y, c["layout"]) for x, y in (("q", q), ("k", k), ("v", v))}
    guard = 9.0
    outs = {x: tensors[x] if c["in_place"] else _place_rows(torch.full_like(y, guard), c["layout"]) for x, y in (("q", q), ("k", k))}
    fields = dict(K=tensors["k"], V=tensors["v"], slots=torch.from_numpy(slots).cuda(), cache=device_cache, pages=pages,
                  page_size=size, tokens=tokens, kv_heads=hk, d=d, dtype=_code(tm, c["dtype"]), rotary_dim=c["rotary"],
                  interleaved=c["interleaved"], k_row_stride=tensors["k"].stride(0), k_head_stride=tensors["k"].stride(1),
                  v_row_stride=tensors["v"].stride(0), v_head_stride=tensors["v"].stride(1))
    if c["rotary"]:
        fields.update(cos_sin=torch.from_numpy(table).cuda(), token_positions=torch.from_numpy(at).cuda(), positions=positions)
    if c["query"]:
        fields.update(Q=tensors["q"], Q_out=outs["q"], q_heads=hq, q_row_stride=tensors["q"].stride(0),
                      q_head_stride=tensors["q"].stride(1), q_out_row_stride=outs["q"].stride(0), q_out_head_stride=outs["q"].stride(1))
    if c["key_out"]:
        fields.update(K_out=outs["k"], k_out_row_stride=outs["k"].stride(0), k_out_head_stride=outs["k"].stride(1))
    tm.check(tm.cache4_append(tm.Cache4AppendArgs(**fields)), "append")
    torch.cuda.synchronize()

    turn = np.zeros((tokens, c["rotary"]), np.float32)
    turn[~skipped] = table[at[~skipped]] if c["rotary"] else turn[~skipped]
    with np.errstate(all="ignore"):
        turned = {x: ref.rotate(y.float().numpy(), turn, c["interleaved"]) for x, y in (("q", q), ("k", k))}
    for x, wanted in (("q", c["query"]), ("k", c["key_out"])):
        expected = torch.from_numpy(turned[x]).to(dtype)
        before = {"q": q, "k": k}[x] if c["in_place"] else torch.full_like(expected, guard)
        expected[torch.from_numpy(skipped)] = before[torch.from_numpy(skipped)]
        got = outs[x].cpu()
        if wanted:
            assert torch.equal(torch.nan_to_num(got.float(), nan=1e9), torch.nan_to_num(expected.float(), nan=1e9)), x
        elif not c["in_place"]:
            assert torch.equal(got, torch.full_like(got, guard))
    for t in range(tokens):
        if not skipped[t] and 0 <= slots[t] < pages * size:
            for h in range(hk):
                ref.write_token(cache, size, int(slots[t]), h, turned["k"][t, h], v[t, h].float().numpy())
    got = device_cache.cpu().numpy()
    wrong = np.argwhere(got != cache)
    assert len(wrong) == 0, f"{len(wrong)} bytes differ, first at {wrong[0]}"


# ------------------------------------------------------------------ gather

@pytest.mark.parametrize("tokens,heads,d,dtype,size,outs,layout", [
    (1, 1, 64, "f16", 32, "kv", "thd"), (40, 2, 128, "bf16", 64, "kv", "thd"), (33, 3, 72, "f16", 32, "kv", "fused"),
    (65, 2, 40, "bf16", 96, "k", "thd"), (20, 4, 104, "f16", 32, "v", "htd"), (200, 8, 128, "f16", 128, "kv", "htd"),
    (70, 2, 8, "bf16", 32, "kv", "fused")])
def test_gather(tm, cuda, tokens, heads, d, dtype, size, outs, layout):
    pages = tokens // size + 3
    cache = _cache(pages, size, heads, d)
    rng = np.random.default_rng(tokens)
    gen = torch.Generator().manual_seed(tokens)
    for page in range(pages):  # parameters as appended rows have them
        for t in range(size):
            for h in range(heads):
                if rng.random() < 0.9 or tokens < 80:
                    x = torch.randn(2, d, generator=gen).numpy()
                    ref.write_token(cache, size, page * size + t, h, x[0], x[1])
        if page * size > 2 * tokens:
            break
    slots = rng.integers(0, pages * size, tokens).astype(np.int64)  # some twice
    if tokens > 10:
        slots[[3, 7, 9]] = (-1, pages * size, 2 ** 60)
    expected = ref.read_tokens(cache, size, np.where((slots < 0) | (slots >= pages * size), 0, slots), d)
    guard = torch.full((tokens, heads, d), 9.0, dtype=DT[dtype])
    got = {x: _place_rows(guard, layout) for x in "kv"}
    fields = dict(cache=torch.from_numpy(cache).cuda(), slots=torch.from_numpy(slots).cuda(), pages=pages, page_size=size, tokens=tokens,
                  kv_heads=heads, d=d, dtype=_code(tm, dtype))
    for x in outs:
        fields.update({f"{x.upper()}_out": got[x], f"{x}_row_stride": got[x].stride(0), f"{x}_head_stride": got[x].stride(1)})
    tm.check(tm.cache4_gather(tm.Cache4GatherArgs(**fields)), "gather")
    torch.cuda.synchronize()
    outside = torch.from_numpy((slots < 0) | (slots >= pages * size))
    for x, y in zip("kv", expected):
        rows = torch.from_numpy(y).float().to(DT[dtype])  # the value in fp32, rounded once more
        rows[outside] = guard[outside]
        if x not in outs:
            rows = guard
        assert torch.equal(torch.nan_to_num(got[x].cpu().float(), nan=1e9), torch.nan_to_num(rows.float(), nan=1e9)), x


# --------------------------------------------------------------- attention

def _decode(lengths, heads=(4, 2), d=64, dtype="f16", size=32, scale=None, layout="thd", bad_pages=(), table_pad=0):
    return dict(lengths=lengths, heads=heads, d=d, dtype=dtype, size=size, scale=1.0 / math.sqrt(d) if scale is None else scale,
                layout=layout, bad_pages=bad_pages, table_pad=table_pad)


DECODES = [
    _decode([1]), _decode([0]), _decode([1, 2, 31, 32, 33], d=128, dtype="bf16"), _decode([64, 0, 65, -3], heads=(1, 1), d=8),
    _decode([100, 257], heads=(8, 1), d=72), _decode([95, 96, 97], heads=(16, 1), d=128, size=96, dtype="bf16"),
    _decode([200], heads=(17, 1), d=64), _decode([130, 40], heads=(40, 1), d=128), _decode([300, 7], heads=(6, 2), d=40, dtype="bf16"),
    _decode([255, 256, 257, 511, 513], heads=(4, 4), d=128, size=64), _decode([1000, 3], heads=(8, 2), d=104, size=128),
    _decode([2000], heads=(4, 1), d=128, size=64, dtype="bf16"), _decode([90, 150], scale=-0.3), _decode([90, 150], scale=0.0, d=128),
    _decode([300], heads=(2, 1), scale=4.0, d=128), _decode([70, 140], heads=(4, 2), d=128, layout="fused"),
    _decode([70, 140], heads=(8, 4), d=64, layout="htd", dtype="bf16"),
    _decode([200, 90], heads=(4, 2), d=128, bad_pages=((0, 1, -1), (0, 3, 10 ** 6), (1, 0, -2 ** 31)), table_pad=3),
    _decode([(5 * i) % 70 for i in range(100)], heads=(2, 1), d=64), _decode([40] * 70, heads=(8, 8), d=64, dtype="bf16"),
    _decode([5000, 1, 0, 700], heads=(2, 1), d=64, table_pad=1),
]


def _decode_problem(c, seed=0):
    """A cache whose bytes past every length are random, block table, slots of each sequence's tokens."""
    (hq, hk), d, size = c["heads"], c["d"], c["size"]
    lengths = [max(0, n) for n in c["lengths"]]
    need = [(n + size - 1) // size for n in lengths]
    pages = sum(need) + 2
    cache = _cache(pages, size, hk, d, seed)
    rng = np.random.default_rng(seed + 1)
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(1, max(need)) + c["table_pad"]), 10 ** 9, dtype=np.int32)
    slots, at = [], 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        t = np.arange(lengths[b])
        slots.append(table[b, t // size].astype(np.int64) * size + t % size)
    # Rows written by the formula, many at once: parameters and codes straight into the blocks.
    k = [rng.standard_normal((len(s), hk, d)).astype(np.float32) for s in slots]
    v = [rng.standard_normal((len(s), hk, d)).astype(np.float32) for s in slots]
    for b, s in enumerate(slots):
        _write_rows(cache, size, s, k[b], v[b])
    return cache, table, slots, pages


def _write_rows(cache, size, slots, k, v):
    """ref.write_token for many tokens (one pass per place of a block)."""
    d, heads = k.shape[-1], k.shape[1]
    whole = 64 * ((d + 63) // 64)
    for t in range(32):
        here = np.nonzero(slots % size % 32 == t)[0]
        if len(here) == 0:
            continue
        key, value, key_params, value_params = ref.addresses(d, t)
        page, block = slots[here] // size, slots[here] % size // 32
        for rows, (at, shift), params in ((k, key, key_params), (v, value, value_params)):
            codes, words = ref.quantize(rows[here])
            padded = np.zeros(codes.shape[:2] + (whole,), np.uint8)
            padded[..., :d] = codes
            for a in np.unique(at):
                byte = np.zeros(codes.shape[:2], np.uint8)
                for f in np.nonzero(at == a)[0]:
                    byte |= padded[..., f] << np.uint8(shift[f])
                cache[page[:, None], np.arange(heads), block[:, None], a] = byte
            for m, a in enumerate(params):
                for i in range(4):
                    cache[page[:, None], np.arange(heads), block[:, None], a + i] = (words[..., m] >> (8 * i)) & 255


def _read_rows(cache, size, slots, d):
    """ref.read_tokens for many tokens."""
    heads = cache.shape[1]
    out = np.zeros((2, len(slots), heads, d))
    for t in range(32):
        here = np.nonzero(slots % size % 32 == t)[0]
        if len(here) == 0:
            continue
        key, value, key_params, value_params = ref.addresses(d, t)
        blocks = cache[slots[here] // size, :, slots[here] % size // 32]  # [n, heads, bytes]
        for i, ((at, shift), params) in enumerate(((key, key_params), (value, value_params))):
            codes = (blocks[..., at] >> shift.astype(np.uint8)) & 15
            words = np.ascontiguousarray(np.stack([blocks[..., a:a + 4] for a in params], -2)).view(np.uint32)[..., 0]
            scale, low = ref.bf16_value((words & 0xFFFF).astype(np.uint16)), ref.bf16_value((words >> 16).astype(np.uint16))
            group = np.arange(codes.shape[-1]) // 64
            out[i, here] = (low.astype(np.float64)[..., group] + scale.astype(np.float64)[..., group] * codes)[..., :d]
    return out


def _decode_expected(c, q, cache, slots):
    (hq, hk), d, size = c["heads"], c["d"], c["size"]
    half = ref.HALF_STEP[DT[c["dtype"]]]
    o = torch.zeros(len(slots), hq, d, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for b, s in enumerate(slots):
        s = s[[not any(b == x and t // size == i for x, i, _ in c["bad_pages"]) for t in range(len(s))]] if len(s) else s
        if len(s) == 0:
            continue
        k, v = (torch.from_numpy(x) for x in _read_rows(cache, size, s, d))
        for h in range(hq):
            g = h * hk // hq
            row, off = ref.attention(q[b, h:h + 1].double(), k[:, g], v[:, g], c["scale"], torch.ones(1, len(s), dtype=torch.bool), 2.0 ** -24)
            # Two bf16 parts of p scale, times 16 + code <= 31; the scale is at most the group's range / 15 (and its rounding).
            span = torch.zeros(d, dtype=torch.float64)
            for m in range(0, d, 64):
                group = v[:, g, m:m + 64]
                span[m:m + 64] = (group.amax(-1) - group.amin(-1)).amax()
            off = off + 2 * 31 / 15 * span * (2.0 ** -16 + (len(s) + 64) * ref.FP32)
            # Scores: fp32 sums over codes offset by 16 as well.
            size_k = (q[b, h].double().abs().sum() * 31 / 15 * (k[:, g].amax() - k[:, g].amin()) * abs(c["scale"]))
            off = off + 2 * v[:, g].abs().amax(0) * (d + 8) * ref.FP32 * size_k
            o[b, h], bound[b, h] = row[0], (off + half * (row.abs() + off))[0] + 2.0 ** -25
    return o, bound


def _decode_args(tm, c, q, o, cache, table, pages, workspace, **options):
    hq, hk = c["heads"]
    for b, i, value in c["bad_pages"]:
        table[b, i] = value
    fields = dict(Q=q, O=o, cache=torch.from_numpy(cache).cuda(), block_table=torch.from_numpy(table).cuda(),
                  lengths=torch.tensor(c["lengths"], dtype=torch.int32, device="cuda"), workspace=workspace,
                  workspace_bytes=workspace.numel(), pages=pages, page_size=c["size"], max_pages=table.shape[1], batch=len(c["lengths"]),
                  q_heads=hq, kv_heads=hk, d=c["d"], dtype=_code(tm, c["dtype"]), score_scale=c["scale"],
                  q_row_stride=q.stride(0), q_head_stride=q.stride(1), o_row_stride=o.stride(0), o_head_stride=o.stride(1))
    fields.update(options)
    return tm.Cache4AttentionArgs(**fields)


@pytest.fixture(scope="module")
def workspace(tm, cuda):
    """One workspace for every call here, whatever its shape."""
    return torch.zeros(tm.attention_cache4_workspace_bytes(), dtype=torch.uint8, device="cuda")


def _queries(c, seed=3):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(len(c["lengths"]), c["heads"][0], c["d"], generator=gen).to(DT[c["dtype"]])


def _check(o, expected, bound, label):
    error = (o.cpu().double() - expected).abs()
    bad = ~(error <= bound)
    assert not bad.any(), f"{label}: {int(bad.sum())} of {bad.numel()} outside, worst {float((error / bound.clamp(min=1e-300)).max()):.3g}"


@pytest.mark.parametrize("c", DECODES, ids=lambda c: "-".join(f"{k}{v if k != 'lengths' else 'x'.join(map(str, v[:6]))}" for k, v in c.items()))
def test_attention_matches_float64(tm, cuda, workspace, c):
    cache, table, slots, pages = _decode_problem(c)
    q = _queries(c)
    expected, bound = _decode_expected(c, q, cache, slots)
    o = _place_rows(torch.full_like(q, 9.0), c["layout"])
    args = _decode_args(tm, c, _place_rows(q, c["layout"]), o, cache, table, pages, workspace)
    for turn in range(2):
        o.fill_(9.0)
        tm.check(tm.attention_cache4(args), "attention_cache4")
        torch.cuda.synchronize()
        _check(o, expected, bound, f"call {turn}")
        if turn == 0:
            first = o.clone()
    assert torch.equal(o, first), "the same call, other bits"
    if c["layout"] == "fused":
        assert (o._base[:, 0] == 0).all() and (o._base[:, -1] == 0).all()


@pytest.mark.parametrize("d,dtype,size", [(128, "bf16", 64), (64, "f16", 32), (72, "f16", 96)])
def test_every_token_can_be_the_one_attended(tm, cuda, workspace, d, dtype, size):
    """Sequence b of many that share the same pages asks for token b: its query is that
    token's key, long enough that no other token has weight (scores 60 apart or more)."""
    tokens = 131
    one = _decode([tokens], heads=(1, 1), d=d, dtype=dtype, size=size)
    cache, table, slots, pages = _decode_problem(one)
    k, v = (x[:, 0] for x in _read_rows(cache, size, slots[0], d))
    q = torch.from_numpy(k / np.linalg.norm(k, axis=1, keepdims=True) ** 2).to(DT[dtype])
    alike = (q.double() @ torch.from_numpy(k).T).numpy()
    others = np.where(np.eye(tokens, dtype=bool), -np.inf, alike).max(1)
    scale = float(60.0 / (np.diag(alike) - others).min())
    assert scale > 0
    c = dict(one, lengths=[tokens] * tokens, scale=scale)
    o = torch.empty(tokens, 1, d, dtype=DT[dtype], device="cuda")
    args = _decode_args(tm, c, q[:, None].contiguous().cuda(), o, cache, np.repeat(table, tokens, 0), pages, workspace)
    tm.check(tm.attention_cache4(args))
    torch.cuda.synchronize()
    expected = torch.from_numpy(v)
    # The one value, in two bf16 parts beside its group's minimum, and the output's rounding.
    bound = 31 / 15 * 2.0 ** -15 * (expected.amax(-1, keepdim=True) - expected.amin(-1, keepdim=True)) * 2 + ref.HALF_STEP[DT[dtype]] * expected.abs() + 2.0 ** -24
    _check(o[:, 0], expected, bound, "the token attended")


def test_not_finite_rows_reach_their_sequence_only(tm, cuda, workspace):
    c = _decode([80, 80, 80], heads=(2, 1), d=128)
    cache, table, slots, pages = _decode_problem(c)
    row = np.ones((1, 128), np.float32)
    nan = row.copy()
    nan[0, 70] = np.nan
    ref.write_token(cache, c["size"], int(slots[1][50]), 0, row[0], nan[0])
    ref.write_token(cache, c["size"], int(slots[2][3]), 0, nan[0], row[0])
    q = _queries(c)
    expected, bound = _decode_expected(c, q, cache, slots)
    o = torch.full_like(q, 9.0).cuda()
    tm.check(tm.attention_cache4(_decode_args(tm, c, q.cuda(), o, cache, table, pages, workspace)))
    torch.cuda.synchronize()
    got = o.cpu()
    _check(got[0], expected[0], bound[0], "the sequence without")
    _check(got[1, :, :64], expected[1, :, :64], bound[1, :, :64], "the group without")
    assert torch.isnan(got[1, :, 64:]).all() and torch.isnan(got[2]).all()


def test_lengths_past_the_table_end_there(tm, cuda, workspace):
    c = _decode([96, 64], heads=(4, 2), d=64)
    cache, table, slots, pages = _decode_problem(c)
    q = _queries(c)
    expected, bound = _decode_expected(c, q, cache, slots)
    o = torch.empty_like(q).cuda()
    lengths = torch.tensor([2 ** 31 - 1, 64], dtype=torch.int32, device="cuda")
    tm.check(tm.attention_cache4(_decode_args(tm, c, q.cuda(), o, cache, table, pages, workspace, lengths=lengths)))
    torch.cuda.synchronize()
    _check(o, expected, bound, "length past the table")


def test_cache_past_4_gib(tm, cuda, workspace):
    """Append, gather and attention on the last pages of a cache of 4.8 GB."""
    heads, d, size, tokens = 2, 128, 64, 90
    page = tm.cache4_bytes(1, size, heads, d)
    pages = 4_800_000_000 // page
    cache = torch.empty(pages * page, dtype=torch.uint8, device="cuda").view(pages, heads, size // 32, -1)
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(tokens, heads, d, generator=gen).half() for _ in "kv")
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    t = torch.arange(tokens, device="cuda")
    slots = table[0, t // size].long() * size + t % size
    shape = dict(cache=cache, pages=pages, page_size=size, kv_heads=heads, d=d, dtype=tm.DTYPE_F16)
    tm.check(tm.cache4_append(tm.Cache4AppendArgs(K=k.cuda(), V=v.cuda(), slots=slots, tokens=tokens, **shape)))
    back = [torch.empty(tokens, heads, d, dtype=torch.float16, device="cuda") for _ in "kv"]
    tm.check(tm.cache4_gather(tm.Cache4GatherArgs(slots=slots, tokens=tokens, K_out=back[0], V_out=back[1], **shape)))
    small = _cache(2, size, heads, d)
    places = np.arange(tokens)
    _write_rows(small, size, places, k.float().numpy(), v.float().numpy())
    for got, rows in zip(back, _read_rows(small, size, places, d)):
        assert torch.equal(got.cpu(), torch.from_numpy(rows).float().half())
    c = _decode([tokens], heads=(4, heads), d=d, size=size)
    q = _queries(c)
    expected, bound = _decode_expected(c, q, small, [places])
    o = torch.empty_like(q).cuda()
    tm.check(tm.attention_cache4(tm.Cache4AttentionArgs(
        Q=q.cuda(), O=o, block_table=table, lengths=torch.tensor([tokens], dtype=torch.int32, device="cuda"), workspace=workspace,
        workspace_bytes=workspace.numel(), max_pages=2, batch=1, q_heads=4, score_scale=c["scale"], **shape)))
    torch.cuda.synchronize()
    _check(o, expected, bound, "the last pages")


def test_captured_step_takes_lengths_and_slots_at_replay(tm, cuda):
    """append + attention of one decode step in a graph: each replay adds a token."""
    heads, d, size, batch, dtype = (8, 2), 128, 32, 3, torch.bfloat16
    pages, table = 12, torch.arange(12, dtype=torch.int32).view(3, 4)
    cache = torch.zeros(pages, heads[1], size // 32, ref.block_bytes(d), dtype=torch.uint8, device="cuda")
    gen = torch.Generator().manual_seed(1)
    rotation = _table(200, d)
    device = dict(table=table.cuda(), lengths=torch.zeros(batch, dtype=torch.int32, device="cuda"),
                  slots=torch.zeros(batch, dtype=torch.int64, device="cuda"), at=torch.zeros(batch, dtype=torch.int32, device="cuda"),
                  rotation=torch.from_numpy(rotation).cuda(), ws=torch.zeros(tm.attention_cache4_workspace_bytes(), dtype=torch.uint8, device="cuda"))
    q, k, v = (torch.zeros(batch, h, d, dtype=dtype, device="cuda") for h in (heads[0], heads[1], heads[1]))
    q_out, o = torch.zeros_like(q), torch.zeros_like(q)
    shape = dict(cache=cache, pages=pages, page_size=size, kv_heads=heads[1], d=d, dtype=tm.DTYPE_BF16)
    step = tm.Cache4AppendArgs(Q=q, K=k, V=v, Q_out=q_out, q_heads=heads[0], slots=device["slots"], token_positions=device["at"],
                               cos_sin=device["rotation"], positions=200, rotary_dim=d, tokens=batch, **shape)
    attend = tm.Cache4AttentionArgs(Q=q_out, O=o, block_table=device["table"], lengths=device["lengths"], workspace=device["ws"],
                                    workspace_bytes=device["ws"].numel(), max_pages=4, batch=batch, q_heads=heads[0],
                                    score_scale=d ** -0.5, **shape)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        tm.check(tm.cache4_append(step))
        tm.check(tm.attention_cache4(attend))
    first = [0, 31, 60]  # tokens before the first step: zeros, as the cache starts
    host = np.zeros(cache.shape, np.uint8)
    for turn in range(40):
        lengths = [n + turn + 1 for n in first]
        where = [int(table[b, (n - 1) // size]) * size + (n - 1) % size for b, n in enumerate(lengths)]
        rows = [torch.randn(batch, h, d, generator=gen).to(dtype) for h in (heads[0], heads[1], heads[1])]
        for x, y in zip((q, k, v), rows):
            x.copy_(y)
        device["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
        device["slots"].copy_(torch.tensor(where))
        device["at"].copy_(torch.tensor(lengths, dtype=torch.int32) - 1)
        graph.replay()
        torch.cuda.synchronize()
        turned = [ref.rotate(y.float().numpy(), rotation[[n - 1 for n in lengths]], False) for y in rows[:2]]
        _write_rows(host, size, np.array(where), turned[1], rows[2].float().numpy())
        if turn % 8 and turn != 39:
            continue
        assert np.array_equal(cache.cpu().numpy(), host), turn
        c = _decode(lengths, heads=heads, d=d, dtype="bf16", size=size)
        slots = [table[b, np.arange(n) // size].numpy().astype(np.int64) * size + np.arange(n) % size for b, n in enumerate(lengths)]
        expected, bound = _decode_expected(c, torch.from_numpy(turned[0]).to(dtype), host, slots)
        _check(o, expected, bound, f"replay {turn}")
        eager = torch.zeros_like(o)
        attend_now = tm.Cache4AttentionArgs(**{**attend.__dict__, "O": eager})
        tm.check(tm.attention_cache4(attend_now))
        torch.cuda.synchronize()
        assert torch.equal(eager, o)


# Enough blocks that workgroups share sequences and have parts of two, with 8 and 16 rows
# a workgroup, and one sequence in as many parts as there are.
LARGE_DECODES = [
    _decode([(37 * i * i) % 2500 for i in range(80)], heads=(8, 2), size=64), _decode([3000, 1, 0, 900, 2047], heads=(32, 2), d=128, size=128, dtype="bf16"),
    _decode([9000], heads=(1, 1), d=128, size=32), _decode([1024] * 6, heads=(4, 4), d=72, size=64, dtype="bf16"),
    _decode([200] * 400, heads=(4, 4), dtype="bf16"), _decode([100] * 200, heads=(4, 4), d=128), _decode([700] * 100, heads=(12, 4)),
    _decode([300 + 7 * i for i in range(40)], heads=(20, 1), size=96, table_pad=2), _decode([31] * 300, heads=(2, 2), d=128),
]


def _run(tm, c, problem, workspace):
    cache, table, _, pages = problem
    o = torch.empty(len(c["lengths"]), c["heads"][0], c["d"], dtype=DT[c["dtype"]], device="cuda")
    tm.check(tm.attention_cache4(_decode_args(tm, c, _queries(c).cuda(), o, cache, table, pages, workspace)))
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("c", LARGE_DECODES, ids=lambda c: f"{len(c['lengths'])}x{max(c['lengths'])}-h{c['heads'][0]}x{c['heads'][1]}-d{c['d']}-{c['dtype']}")
def test_large_batches_match_float64(tm, cuda, workspace, c):
    problem = _decode_problem(c)
    expected, bound = _decode_expected(c, _queries(c), problem[0], problem[2])
    _check(_run(tm, c, problem, workspace), expected, bound, "large")


def test_a_workspace_serves_any_shape(tm, cuda):
    """The same bits from one workspace after calls of other shapes as from a new one each."""
    def new():
        return torch.zeros(tm.attention_cache4_workspace_bytes(), dtype=torch.uint8, device="cuda")

    one = new()
    problems = [(c, _decode_problem(c)) for c in (LARGE_DECODES[3], DECODES[0], LARGE_DECODES[5], DECODES[11], LARGE_DECODES[4])]
    for c, problem in problems + problems[::-1]:
        assert torch.equal(_run(tm, c, problem, one), _run(tm, c, problem, new()))


def test_queries_of_zeros_under_the_largest_scale(tm, cuda, workspace):
    """Scores of 0 whatever the scale: the mean of the values."""
    c = _decode([100, 33], heads=(4, 2), d=64, scale=3.4e38)
    cache, table, slots, pages = _decode_problem(c)
    q = torch.zeros_like(_queries(c))
    expected, bound = _decode_expected(c, q, cache, slots)
    o = torch.empty_like(q).cuda()
    tm.check(tm.attention_cache4(_decode_args(tm, c, q.cuda(), o, cache, table, pages, workspace)))
    torch.cuda.synchronize()
    _check(o, expected, bound, "mean")


def test_two_streams_with_their_own_workspaces(tm, cuda):
    c = _decode([4000, 900], heads=(4, 1), d=64, size=64)
    cache, table, slots, pages = _decode_problem(c)
    q = _queries(c)
    expected, bound = _decode_expected(c, q, cache, slots)
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.zeros(tm.attention_cache4_workspace_bytes(), dtype=torch.uint8, device="cuda") for _ in streams]
    outs = [torch.empty_like(q).cuda() for _ in streams]
    args = [_decode_args(tm, c, q.cuda(), o, cache, table, pages, w) for o, w in zip(outs, spaces)]
    torch.cuda.synchronize()
    for _ in range(5):
        for a, s in zip(args, streams):
            tm.check(tm.attention_cache4(a, stream=s))
    torch.cuda.synchronize()
    for o in outs:
        _check(o, expected, bound, "streams")


# ------------------------------------------------- the operators as a server has them

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompts_chunks_and_decode_steps(tm, cuda, workspace, dtype):
    """Prompts packed, rotated, attended and cached; a second chunk against the gathered
    context; then decode steps: every output against float64 on the same 16-bit or cached rows."""
    (hq, hk), d, size, batch = (6, 2), 72, 32, 3
    real = DT[dtype]
    pages, most = 20, 6
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table = order[:batch * most].view(batch, most)
    cache = torch.zeros(pages, hk, size // 32, ref.block_bytes(d), dtype=torch.uint8, device="cuda")
    rotation = _table(400, d)
    gen = torch.Generator().manual_seed(4)
    shape = dict(kv_heads=hk, d=d, dtype=_code(tm, dtype))
    paged = dict(cache=cache, pages=pages, page_size=size)
    lengths = [0] * batch

    def take(counts):
        """`counts` new tokens per sequence through append; their rotated queries, keys and values."""
        tokens = sum(counts)
        rows = [torch.randn(tokens, h, d, generator=gen).to(real).cuda() for h in (hq, hk, hk)]
        at = [lengths[b] + i for b, n in enumerate(counts) for i in range(n)]
        where = [int(table[b, t // size]) * size + t % size for b, n in enumerate(counts) for t in range(lengths[b], lengths[b] + n)]
        q, k = torch.empty_like(rows[0]), torch.empty_like(rows[1])
        tm.check(tm.cache4_append(tm.Cache4AppendArgs(
            Q=rows[0], K=rows[1], V=rows[2], Q_out=q, K_out=k, q_heads=hq, slots=torch.tensor(where, device="cuda"),
            token_positions=torch.tensor(at, dtype=torch.int32, device="cuda"), cos_sin=torch.from_numpy(rotation).cuda(),
            positions=400, rotary_dim=d, tokens=tokens, **shape, **paged)))
        for b, n in enumerate(counts):
            lengths[b] += n
        return q, k, rows[2]

    def check(o, q, k, v, q_lens, k_lens):
        from test_packed_attention_gpu import _compare, _expected

        c = dict(q_lens=q_lens, k_lens=k_lens, heads=(hq, hk), d=d, dtype=dtype, causal=True, scale=d ** -0.5)
        starts = [[sum(x[:i]) for i in range(len(x) + 1)] for x in (q_lens, k_lens)]
        p = dict(q=q.cpu(), k=k.cpu(), v=v.cpu(), q_starts=starts[0], k_starts=starts[1])
        expected, bound = _expected(c, p)
        _compare(o, expected, bound, "prompt")

    def attend(q, k, v, q_lens, k_lens):
        o = torch.empty_like(q)
        starts = [torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32, device="cuda") for x in (q_lens, k_lens)]
        tm.check(tm.attention_packed(tm.PackedAttentionArgs(
            Q=q, K=k, V=v, O=o, q_starts=starts[0], k_starts=starts[1], batch=batch, q_tokens=q.shape[0], k_tokens=k.shape[0], q_heads=hq,
            score_scale=d ** -0.5, **shape)))
        torch.cuda.synchronize()
        return o

    first = [40, 1, 0]
    q, k, v = take(first)
    check(attend(q, k, v, first, first), q, k, v, first, first)
    # The next chunk: its own rows exactly, the context as cached.
    before, chunk = list(lengths), [30, 64, 5]
    q, k, v = take(chunk)
    context = torch.tensor([int(table[b, t // size]) * size + t % size for b in range(batch) for t in range(before[b])], device="cuda")
    old = [torch.empty(len(context), hk, d, dtype=real, device="cuda") for _ in "kv"]
    tm.check(tm.cache4_gather(tm.Cache4GatherArgs(K_out=old[0], V_out=old[1], slots=context, tokens=len(context), **shape, **paged)))
    whole = [torch.cat([x for b in range(batch) for x in (past[sum(before[:b]):sum(before[:b + 1])], new[sum(chunk[:b]):sum(chunk[:b + 1])])])
             for past, new in zip(old, (k, v))]
    k_lens = [n + m for n, m in zip(before, chunk)]
    check(attend(q, *whole, chunk, k_lens), q, *whole, chunk, k_lens)
    for _ in range(3):
        q, k, v = take([1] * batch)
        o = torch.empty_like(q)
        tm.check(tm.attention_cache4(tm.Cache4AttentionArgs(
            Q=q, O=o, block_table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), workspace=workspace,
            workspace_bytes=workspace.numel(), max_pages=most, batch=batch, q_heads=hq, score_scale=d ** -0.5, **shape, **paged)))
        torch.cuda.synchronize()
        c = _decode(lengths, heads=(hq, hk), d=d, dtype=dtype, size=size)
        slots = [table[b, np.arange(n) // size].numpy().astype(np.int64) * size + np.arange(n) % size for b, n in enumerate(lengths)]
        expected, bound = _decode_expected(c, q.cpu(), cache.cpu().numpy(), slots)
        _check(o, expected, bound, "decode step")
