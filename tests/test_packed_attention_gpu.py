"""Attention of packed sequences (tilemix_attention_packed) against the formula in
float64: lengths at the edges of blocks and tiles, empty sequences, keys before and
missing rows, every number of heads a workgroup may hold, odd head dimensions, strided
tensors, masks that leave a row empty, values that are not finite in places a row
does not see, starts that make no sense, many sequences, tensors past 2 GiB,
captured calls.

Every tensor has NaN rows around what the sequences cover, and the rows of O
outside every sequence have to stay as they were. Bounds: serving_reference
(probabilities rounded to the type; of fp16, those under 2^-14 of the largest are
off by up to 2^-25 each), then the output's own half step.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
GUARD = 3.0


def _case(q_lens, k_lens=None, heads=(4, 2), d=64, dtype="f16", causal=True, layout="thd", scale=None, pad=(3, 5)):
    return dict(q_lens=q_lens, k_lens=k_lens or q_lens, heads=heads, d=d, dtype=dtype, causal=causal, layout=layout,
                scale=1.0 / math.sqrt(d) if scale is None else scale, pad=pad)


CASES = [
    _case([1]), _case([1, 1, 1], heads=(1, 1), d=8), _case([2, 31, 32, 33], heads=(8, 2), dtype="bf16"),
    _case([63, 64, 65], heads=(3, 1), d=128), _case([127, 1, 128, 129], heads=(4, 4), d=128, dtype="bf16"),
    _case([0, 5, 0, 0, 70, 0], heads=(12, 2), d=72), _case([257], heads=(5, 1), d=96, dtype="bf16"),
    _case([200, 3], heads=(16, 2), d=40), _case([100, 61], heads=(6, 3), d=24, causal=False),
    _case([64, 128], heads=(2, 1), d=128, causal=False, dtype="bf16"), _case([333, 190], heads=(4, 1), d=104),
    # Keys before the rows (chunks), and fewer keys than rows: the first rows see none.
    _case([1, 5, 40], [100, 5, 300], heads=(4, 2), d=128), _case([33, 64], [97, 640], heads=(8, 1), dtype="bf16"),
    _case([50, 20, 7], [30, 0, 1], heads=(4, 2)), _case([50, 20], [30, 0], heads=(2, 2), d=128, causal=False),
    _case([130], [64], heads=(1, 1), d=80, dtype="bf16"), _case([9, 0], [9, 50], heads=(4, 4), d=56),
    # Fused projections, heads first, wide rows.
    _case([70, 33], heads=(4, 2), d=128, layout="fused"), _case([70, 33], heads=(8, 4), d=72, layout="htd", dtype="bf16"),
    _case([45, 90], heads=(4, 2), layout="wide"),
    _case([80, 17], heads=(4, 2), scale=-0.2), _case([80, 17], heads=(4, 2), scale=0.0, dtype="bf16"),
    _case([60, 40], heads=(2, 1), d=128, scale=3.0),  # a few keys take nearly all of the weight
    # More sequences than a wave has lanes.
    _case([(7 * i) % 45 for i in range(70)], heads=(2, 2)), _case([(11 * i) % 37 for i in range(150)], heads=(4, 1), dtype="bf16"),
]


def _id(c):
    lens = "x".join(map(str, c["q_lens"][:6])) + ("" if c["k_lens"] == c["q_lens"] else "-k" + "x".join(map(str, c["k_lens"])))
    return f"{lens}-h{c['heads'][0]}x{c['heads'][1]}-d{c['d']}-{c['dtype']}-{c['layout']}-{'causal' if c['causal'] else 'full'}-s{c['scale']:.2g}"


def _starts(lens, first):
    return [first + sum(lens[:i]) for i in range(len(lens) + 1)]


def _tensor(values, layout, extra):
    """Device tensor viewed [tokens, heads, d] in a layout; `extra` heads lie beside it in "fused" rows."""
    t, h, d = values.shape
    if layout == "htd":
        return values.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    if layout in ("fused", "wide"):
        row = torch.full((t, h + extra, d + (8 if layout == "wide" else 0)), float("nan"), dtype=values.dtype)
        row[:, :h, :d] = values
        return row.cuda()[:, :h, :d]
    return values.cuda()


def _problem(c, seed=0):
    gen = torch.Generator().manual_seed(1000 + seed)
    hq, hk = c["heads"]
    q_starts, k_starts = _starts(c["q_lens"], c["pad"][0]), _starts(c["k_lens"], c["pad"][0])
    out = dict(q_starts=q_starts, k_starts=k_starts)
    for name, heads, starts in (("q", hq, q_starts), ("k", hk, k_starts), ("v", hk, k_starts)):
        x = torch.full((starts[-1] + c["pad"][1], heads, c["d"]), float("nan"))
        x[starts[0]:starts[-1]] = torch.randn(starts[-1] - starts[0], heads, c["d"], generator=gen)
        out[name] = x.to(DT[c["dtype"]])
    return out


def _expected(c, p):
    """Float64 output and bound of every row of O (rows outside the sequences: the guard, no error)."""
    hq, hk = c["heads"]
    dtype = DT[c["dtype"]]
    o = torch.full((p["q"].shape[0], hq, c["d"]), GUARD, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for b in range(len(c["q_lens"])):
        q0, q1, k0, k1 = p["q_starts"][b], p["q_starts"][b + 1], p["k_starts"][b], p["k_starts"][b + 1]
        n, m = q1 - q0, k1 - k0
        visible = torch.ones(n, m, dtype=torch.bool)
        if c["causal"]:
            visible = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
        for h in range(hq):
            k, v = (p[x][k0:k1, h * hk // hq].double() for x in "kv")
            row, off = ref.attention(p["q"][q0:q1, h].double(), k, v, c["scale"], visible, ref.HALF_STEP[dtype])
            if dtype == torch.float16 and m:
                off = off + m * 2.0 ** -25 * v.abs().amax(0)
            o[q0:q1, h], bound[q0:q1, h] = row, off + ref.HALF_STEP[dtype] * (row.abs() + off) + 2.0 ** -25
    return o, bound


def _args(tm, c, p, o, **options):
    hq, hk = c["heads"]
    t = {x: _tensor(p[x], c["layout"], extra) for x, extra in (("q", 3), ("k", 2), ("v", 1))}
    fields = dict(Q=t["q"], K=t["k"], V=t["v"], O=o, q_starts=torch.tensor(p["q_starts"], dtype=torch.int32, device="cuda"),
                  k_starts=torch.tensor(p["k_starts"], dtype=torch.int32, device="cuda"), batch=len(c["q_lens"]),
                  q_tokens=t["q"].shape[0], k_tokens=t["k"].shape[0], q_heads=hq, kv_heads=hk, d=c["d"],
                  dtype=tm.DTYPE_F16 if c["dtype"] == "f16" else tm.DTYPE_BF16, causal=c["causal"], score_scale=c["scale"])
    for x, tensor in (("q", t["q"]), ("k", t["k"]), ("v", t["v"]), ("o", o)):
        fields[f"{x}_row_stride"], fields[f"{x}_head_stride"] = tensor.stride(0), tensor.stride(1)
    fields.update(options)
    return tm.PackedAttentionArgs(**fields)


def _output(c, p):
    return _tensor(torch.full((p["q"].shape[0], c["heads"][0], c["d"]), GUARD, dtype=DT[c["dtype"]]), c["layout"], 1)


def _compare(o, expected, bound, label):
    got = o.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(expected)), f"{label}: NaN in other places"
    infinite = torch.isinf(expected)
    assert torch.equal(got[infinite], expected[infinite]) and not torch.isinf(got[~infinite]).any(), f"{label}: infinities"
    fine = torch.isfinite(expected)
    error = (got - expected).abs()[fine]
    bad = error > bound[fine]
    assert not bad.any(), f"{label}: {int(bad.sum())} of {bad.numel()} outside, worst {float((error / bound[fine].clamp(min=1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("c", CASES, ids=_id)
def test_matches_float64(tm, cuda, c):
    p = _problem(c)
    expected, bound = _expected(c, p)
    o = _output(c, p)
    whole = o._base if o._base is not None else o
    before = whole.clone()
    tm.check(tm.attention_packed(_args(tm, c, p, o)), "packed")
    torch.cuda.synchronize()
    _compare(o, expected, bound, _id(c))
    # What lies beside the heads of O is untouched.
    o.copy_(torch.full_like(o, GUARD))
    assert torch.equal(torch.nan_to_num(whole, nan=-7.0), torch.nan_to_num(before, nan=-7.0))


def test_k_starts_default_to_q_starts_and_calls_repeat(tm, cuda):
    c = _case([77, 130, 1], heads=(8, 2), d=128, dtype="bf16")
    p = _problem(c)
    first, second = _output(c, p), _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, first)))
    tm.check(tm.attention_packed(_args(tm, c, p, second, k_starts=None)))
    torch.cuda.synchronize()
    assert torch.equal(first, second)


@pytest.mark.parametrize("what", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_values_not_finite_reach_only_rows_that_see_them(tm, cuda, what, dtype):
    c = _case([100, 40], [130, 40], heads=(4, 2), d=128, dtype=dtype)
    p = _problem(c)
    first, second = p["k_starts"][0], p["k_starts"][1]
    for at, feature in ((first + 60, 5), (first + 127, 64), (second + 20, 0), (second + 39, 127)):
        p["v"][at, 0, feature] = what
    p["v"][first + 100, 1, 7] = what
    p["v"][first + 101, 1, 7] = -what  # +inf and -inf: NaN for rows that see both
    expected, bound = _expected(c, p)
    # In float64 too a hidden key's 0 times infinity is NaN: those rows are taken from finite values.
    clean = {**p, "v": torch.nan_to_num(p["v"], nan=0.0, posinf=0.0, neginf=0.0)}
    finite, finite_bound = _expected(c, clean)
    for b in range(2):
        q0, k0 = p["q_starts"][b], p["k_starts"][b]
        n, m = c["q_lens"][b], c["k_lens"][b]
        for h in range(4):
            v = p["v"][k0:k0 + m, h // 2].double()
            visible = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
            seen = [(visible.double() @ hit.double()) > 0 for hit in (v == math.inf, v == -math.inf, torch.isnan(v))]
            row = finite[q0:q0 + n, h].clone()
            row[seen[0]], row[seen[1]] = math.inf, -math.inf
            row[seen[2] | (seen[0] & seen[1])] = math.nan
            expected[q0:q0 + n, h], bound[q0:q0 + n, h] = row, finite_bound[q0:q0 + n, h]
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)))
    torch.cuda.synchronize()
    _compare(o, expected, bound, str(what))


def test_keys_not_finite_reach_only_rows_that_see_them(tm, cuda):
    c = _case([90], heads=(2, 1), d=64, dtype="bf16")
    p = _problem(c)
    clean = {**p, "k": p["k"].clone()}
    p["k"][p["k_starts"][0] + 70] = float("nan")
    expected, bound = _expected(c, clean)
    first = p["q_starts"][0]
    expected[first + 70:first + 90] = math.nan
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)))
    torch.cuda.synchronize()
    _compare(o, expected, bound, "NaN key")


def test_starts_that_make_no_sense_stay_inside(tm, cuda):
    """Clamped to the tensors, empty where they decrease; the sequences between are computed."""
    c = _case([40, 30, 25], heads=(4, 2), d=64)
    p = _problem(c)
    total = p["q"].shape[0]
    starts = [-5, 43, 20, 2 ** 31 - 1]  # 0 .. 43, none, 20 .. total
    for x in "qkv":
        p[x] = torch.randn(total, p[x].shape[1], 64, generator=torch.Generator().manual_seed(3)).half()
    o = _output(c, p)
    args = _args(tm, c, p, o, q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), k_starts=None)
    tm.check(tm.attention_packed(args))
    torch.cuda.synchronize()
    one = {**c, "q_lens": [43], "k_lens": [43]}
    expected, bound = _expected(one, {**p, "q_starts": [0, 43], "k_starts": [0, 43]})
    _compare(o[:20], expected[:20], bound[:20], "rows of the first sequence alone")
    tail = {**c, "q_lens": [total - 20], "k_lens": [total - 20]}
    expected, bound = _expected(tail, {**p, "q_starts": [20, total], "k_starts": [20, total]})
    _compare(o[43:], expected[43:], bound[43:], "rows of the last sequence alone")


def test_keys_and_values_past_2_gib(tm, cuda):
    """Rows 4 MiB apart: the last keys of the sequence lie 2.5 GB from its first."""
    c = _case([40], [600], heads=(2, 1), d=64, pad=(0, 0))
    p = _problem(c)
    expected, bound = _expected(c, p)
    row = 1 << 21
    k, v = (torch.empty(600 * row, dtype=torch.float16, device="cuda").view(600, row) for _ in "kv")
    k[:, :64], v[:, :64] = p["k"][:, 0].cuda(), p["v"][:, 0].cuda()
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o, K=k, V=v, k_row_stride=row, v_row_stride=row)))
    torch.cuda.synchronize()
    _compare(o, expected, bound, "rows 4 MiB apart")


def test_captured_calls_take_the_lengths_at_replay(tm, cuda):
    cases = [_case([64, 10, 30], heads=(8, 2), d=128, dtype="bf16", pad=(0, 0)),
             _case([3, 100, 1], heads=(8, 2), d=128, dtype="bf16", pad=(0, 0))]
    c = cases[0]
    p = _problem(c)
    o = _output(c, p)
    args = _args(tm, c, p, o, k_starts=None)
    starts = args.q_starts
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tm.check(tm.attention_packed(args))
    for turn in range(4):
        lens = cases[turn % 2]["q_lens"]
        now = {**c, "q_lens": lens, "k_lens": lens}
        at = _starts(lens, 0)
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        o.fill_(GUARD)
        graph.replay()
        torch.cuda.synchronize()
        expected, bound = _expected(now, {**p, "q_starts": at, "k_starts": at})
        _compare(o, expected, bound, f"replay {turn}")
        eager = torch.full_like(o, GUARD)
        tm.check(tm.attention_packed(_args(tm, c, p, eager, q_starts=starts, k_starts=None)))
        torch.cuda.synchronize()
        assert torch.equal(o, eager)


def test_two_streams_at_once(tm, cuda):
    c = _case([300, 50, 200], heads=(8, 2), d=128)
    p = _problem(c)
    expected, bound = _expected(c, p)
    outputs = [_output(c, p) for _ in range(2)]
    args = [_args(tm, c, p, o) for o in outputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for a, s in zip(args, streams):
            tm.check(tm.attention_packed(a, stream=s))
    torch.cuda.synchronize()
    for o in outputs:
        _compare(o, expected, bound, "streams")


# Few blocks of long walks: their key tiles are walked by several workgroups.
SPLIT_CASES = [
    _case([1], [1500], heads=(2, 1), d=128), _case([40], [1029], heads=(8, 2), d=128, dtype="bf16"),
    _case([129, 64], [900, 1100], heads=(2, 2), d=64), _case([1, 0, 33, 0], [2000, 900, 1211, 3], heads=(4, 1), d=72, dtype="bf16"),
    _case([300], [1700], heads=(3, 1), d=96), _case([70, 30], [1300, 1290], heads=(6, 3), d=128, causal=False),
    _case([50, 20, 2000], [3000, 0, 40], heads=(1, 1), d=40), _case([1700], heads=(4, 2), d=128, dtype="bf16"),
    _case([5, 6, 7, 8], [800, 900, 1000, 4000], heads=(16, 8), d=128), _case([64], [5000], heads=(1, 1), d=8, layout="wide"),
    _case([40], [1500], heads=(4, 2), d=128, scale=3.0), _case([30], [1200], heads=(2, 1), d=64, scale=-0.3, layout="htd"),
]


@pytest.mark.parametrize("c", SPLIT_CASES, ids=_id)
def test_split_calls_match_float64(tm, cuda, c):
    p = _problem(c)
    expected, bound = _expected(c, p)
    o, again = _output(c, p), _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)), "packed")
    tm.check(tm.attention_packed(_args(tm, c, p, again)), "packed")
    torch.cuda.synchronize()
    _compare(o, expected, bound, _id(c))
    assert torch.equal(o, again)  # parts are merged in their order, whichever is done first


@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_split_rows_of_values_not_finite(tm, cuda, what):
    """In the first range, in a diagonal tile of the last one, and behind what the first rows see."""
    c = _case([40], [1200], heads=(4, 2), d=128, dtype="bf16")
    p = _problem(c)
    expected, bound = _expected(c, p)
    q0, k0 = p["q_starts"][0], p["k_starts"][0]
    for key, head, feature in ((10, 0, 3), (1165, 0, 70), (1199, 1, 127)):
        p["v"][k0 + key, head, feature] = what
        expected[q0 + max(key - 1160, 0):q0 + 40, 2 * head:2 * head + 2, feature] = what
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)))
    torch.cuda.synchronize()
    _compare(o, expected, bound, str(what))


def test_split_calls_on_more_streams_than_workspaces_and_replayed(tm, cuda):
    cases = [_case([40], [1500], heads=(4, 2), d=128, dtype="bf16"), _case([200, 10], [1100, 900], heads=(8, 2)),
             _case([64], [3000], heads=(1, 1), d=128)]
    problems = [_problem(c, 7 + i) for i, c in enumerate(cases)]
    expected = [_expected(c, p) for c, p in zip(cases, problems)]
    outputs = [_output(cases[i % 3], problems[i % 3]) for i in range(7)]
    calls = [_args(tm, cases[i % 3], problems[i % 3], o) for i, o in enumerate(outputs)]
    streams = [torch.cuda.Stream() for _ in range(6)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):  # takes no workspace, and the same ranges in turn
        tm.check(tm.attention_packed(calls[6]))
    for turn in range(4):
        for o in outputs:
            o.fill_(GUARD)
        torch.cuda.synchronize()
        graph.replay()
        for a, s in zip(calls, streams):
            for _ in range(3):
                tm.check(tm.attention_packed(a, stream=s))
        torch.cuda.synchronize()
        for i, o in enumerate(outputs):
            _compare(o, *expected[i % 3], f"turn {turn} call {i}")


def test_queries_of_zeros_under_the_largest_scale(tm, cuda):
    """Scores of 0 whatever the scale: the mean of the values."""
    c = _case([70, 5], heads=(2, 1), scale=3.4e38)
    p = _problem(c)
    p["q"].zero_()
    expected, bound = _expected({**c, "scale": 1.0}, p)
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)))
    torch.cuda.synchronize()
    _compare(o, expected, bound, "mean")


@pytest.mark.parametrize("c", SPLIT_CASES, ids=_id)
def test_split_calls_replay_with_the_same_bits(tm, cuda, c):
    """A captured call has no workspace: one workgroup takes a block's ranges in turn."""
    p = _problem(c)
    eager, o = _output(c, p), _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, eager)), "packed")
    args = _args(tm, c, p, o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        tm.check(tm.attention_packed(args))
    for turn in range(3):
        o.fill_(GUARD)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o.nan_to_num(nan=77.0), eager.nan_to_num(nan=77.0)), turn
        eager.mul_(1)  # work of its own between the replays


def test_replays_keep_values_not_finite(tm, cuda):
    c = _case([40], [1200], heads=(4, 2), d=128)
    p = _problem(c)
    for key, what in ((10, math.inf), (1170, math.nan), (1190, -math.inf), (1199, math.inf)):
        p["v"][p["k_starts"][0] + key, 0, key % 128] = what
    eager, o = _output(c, p), _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, eager)))
    args = _args(tm, c, p, o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        tm.check(tm.attention_packed(args))
    for _ in range(3):
        o.fill_(GUARD)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o.nan_to_num(nan=77.0), eager.nan_to_num(nan=77.0))
    assert torch.isinf(eager[:, :2]).any() and torch.isnan(eager[:, :2]).any() and torch.isfinite(eager[p["q_starts"][0]:p["q_starts"][1], 2:]).all()


# More sequences than a wave has lanes are found by their starts.
MANY = [
    _case([(3 * i) % 5 for i in range(1000)], heads=(2, 1)), _case([0] * 200 + [130, 0, 1] + [0] * 90, heads=(4, 2), dtype="bf16"),
    _case([33] * 65, heads=(1, 1), d=128, pad=(700, 300)), _case([1] * 129, [(17 * i) % 90 for i in range(129)], heads=(8, 2), d=128),
    _case([64] * 70, heads=(3, 3), d=40, causal=False), _case([200] + [1] * 80 + [300], heads=(4, 4), dtype="bf16"),
    # Split: few rows each, many keys.
    _case([1 + i % 3 for i in range(70)], [700 + 11 * i for i in range(70)], heads=(1, 1)),
    _case([0, 40] * 40, [0, 1500] * 40, heads=(2, 1), dtype="bf16"),
]


@pytest.mark.parametrize("c", MANY, ids=_id)
def test_many_sequences(tm, cuda, c):
    p = _problem(c)
    expected, bound = _expected(c, p)
    o = _output(c, p)
    tm.check(tm.attention_packed(_args(tm, c, p, o)), "packed")
    torch.cuda.synchronize()
    _compare(o, expected, bound, _id(c))


def test_many_starts_that_make_no_sense_stay_inside(tm, cuda):
    """Rows outside the tensor are neither read nor written, whatever the starts hold."""
    c = _case([4] * 100, heads=(4, 2), d=64)
    p = _problem(c)
    gen = torch.Generator().manual_seed(5)
    o = _output(c, p)
    whole = torch.full((o.numel() + 2 * 4096,), GUARD, dtype=o.dtype, device="cuda")
    inside = whole[4096:-4096].view(o.shape)
    for _ in range(4):
        starts = torch.randint(-2 ** 31, 2 ** 31 - 1, (101,), generator=gen).to(torch.int32)
        starts[::3] = torch.randint(0, p["q"].shape[0], (34,), generator=gen).to(torch.int32)
        tm.check(tm.attention_packed(_args(tm, c, p, inside, q_starts=starts.cuda(), k_starts=starts.flip(0).cuda())))
        torch.cuda.synchronize()
    assert (whole[:4096] == GUARD).all() and (whole[-4096:] == GUARD).all()
