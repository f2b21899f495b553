"""The serving operators at the edges of what their entry points take: pages past
2 GiB, wide page tables, sequences of nearly 2^31 keys, values near the ends of
their types.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import serving_reference as ref
from test_cache4_gpu import DT, _check, _code, _decode, _decode_args, _decode_expected, _decode_problem, _queries, _read_rows, _write_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def workspace(tm, cuda):
    return torch.zeros(tm.attention_cache4_workspace_bytes(), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("d,blocks,dtype", [(128, 470_000, "f16"), (40, 940_000, "bf16")])
def test_one_page_past_2_gib(tm, cuda, workspace, d, blocks, dtype):
    """A contiguous cache of one page a sequence: its last blocks lie 2.17 GB from its first.
    All tokens before the last 90 are zeros, whose scores of 0 have no weight beside 50 and more."""
    size, tokens = 32 * blocks, 90
    cache = torch.zeros(tm.cache4_bytes(2, size, 1, d), dtype=torch.uint8, device="cuda")
    assert cache.numel() // 2 > 2 ** 31
    gen = torch.Generator().manual_seed(d)
    base = torch.randn(1, 1, d, generator=gen)
    k = (base + 0.1 * torch.randn(tokens, 1, d, generator=gen)).to(DT[dtype])
    v = torch.randn(tokens, 1, d, generator=gen).to(DT[dtype])
    q = (base + 0.1 * torch.randn(1, 2, d, generator=gen)).to(DT[dtype])
    scale = 60.0 / float((base ** 2).sum())
    slots = torch.arange(2 * size - tokens, 2 * size, device="cuda")  # the end of page 1
    shape = dict(cache=cache, pages=2, page_size=size, kv_heads=1, d=d, dtype=_code(tm, dtype))
    tm.check(tm.cache4_append(tm.Cache4AppendArgs(K=k.cuda(), V=v.cuda(), slots=slots, tokens=tokens, **shape)))
    back = [torch.empty(tokens, 1, d, dtype=DT[dtype], device="cuda") for _ in "kv"]
    tm.check(tm.cache4_gather(tm.Cache4GatherArgs(slots=slots, tokens=tokens, K_out=back[0], V_out=back[1], **shape)))
    o = torch.full((1, 2, d), 9.0, dtype=DT[dtype], device="cuda")
    tm.check(tm.attention_cache4(tm.Cache4AttentionArgs(
        Q=q.cuda(), O=o, block_table=torch.tensor([[1]], dtype=torch.int32, device="cuda"),
        lengths=torch.tensor([size], dtype=torch.int32, device="cuda"), workspace=workspace, workspace_bytes=workspace.numel(),
        max_pages=1, batch=1, q_heads=2, score_scale=scale, **shape)))
    torch.cuda.synchronize()
    small, places = np.zeros((2, 1, 2, ref.block_bytes(d)), np.uint8), np.arange(tokens)
    _write_rows(small, 64, places, k.float().numpy(), v.float().numpy())
    for got, rows in zip(back, _read_rows(small, 64, places, d)):
        assert torch.equal(got.cpu(), torch.from_numpy(rows).float().to(DT[dtype]))
    c = _decode([tokens], heads=(2, 1), d=d, dtype=dtype, size=64, scale=scale)
    scores = _read_rows(small, 64, places, d)[0][:, 0] @ q[0].double().numpy().T * scale
    assert scores.max(0).min() > 50  # 3e7 zeros weigh under 3e7 e^-50 < 2^-46 of the row
    expected, bound = _decode_expected(c, q, small, [places])
    _check(o, expected, bound, "the end of the page")


@pytest.mark.parametrize("last", [8.0, float("nan"), float("inf")])
@pytest.mark.parametrize("heads", [1, 4])
def test_a_sequence_of_nearly_2_31_keys(tm, cuda, last, heads):
    """Row 1 of two sees the last of 2^31 - 1 keys, row 0 does not. All other keys and
    values are zeros; the last key's score is 64, beside which 2^31 zeros weigh 2^-61."""
    keys, d = 2 ** 31 - 1, 8
    x = torch.zeros(keys, d, dtype=torch.float16, device="cuda")  # K and V alike
    x[-1] = last
    q = torch.ones(2, heads, d, dtype=torch.float16, device="cuda")
    o = torch.full_like(q, 9.0)
    starts = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (2, keys)]
    tm.check(tm.attention_packed(tm.PackedAttentionArgs(
        Q=q, K=x, V=x, O=o, q_starts=starts[0], k_starts=starts[1], batch=1, q_tokens=2, k_tokens=keys, q_heads=heads, kv_heads=1,
        d=d, dtype=tm.DTYPE_F16, score_scale=1.0)))
    torch.cuda.synchronize()
    assert (o[0] == 0).all()
    assert (o[1] == last).all() if last == 8.0 else torch.isnan(o[1]).all()


def test_tensors_of_other_types_are_refused(tm, cuda, workspace):
    """Index tensors above all: a kernel takes narrower ones for as many values of its own."""
    d, size = 64, 32
    cache = torch.zeros(tm.cache4_bytes(2, size, 1, d), dtype=torch.uint8, device="cuda")
    rows = {n: torch.ones(4, 1, d, dtype=torch.float16, device="cuda") for n in ("Q", "K", "V", "O")}
    shape = dict(kv_heads=1, d=d, dtype=tm.DTYPE_F16)
    paged = dict(cache=cache, pages=2, page_size=size)
    int32 = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda")
    append = dict(K=rows["K"], V=rows["V"], slots=int32[:4].long(), tokens=4, **paged, **shape)
    gather = dict(slots=int32[:4].long(), K_out=rows["K"], V_out=rows["V"], tokens=4, **paged, **shape)
    decode = dict(Q=rows["Q"], O=rows["O"], block_table=int32[:4].view(4, 1), lengths=int32[1:], workspace=workspace,
                  workspace_bytes=workspace.numel(), max_pages=1, batch=4, q_heads=1, score_scale=1.0, **paged, **shape)
    packed = dict(Q=rows["Q"], K=rows["K"], V=rows["V"], O=rows["O"], q_starts=int32, k_starts=int32, batch=4, q_tokens=4, k_tokens=4,
                  q_heads=1, score_scale=1.0, **shape)
    for call, args, fields, names in (
            (tm.cache4_append, tm.Cache4AppendArgs, append, "K V slots"), (tm.cache4_gather, tm.Cache4GatherArgs, gather, "K_out V_out slots"),
            (tm.attention_cache4, tm.Cache4AttentionArgs, decode, "Q O block_table lengths"),
            (tm.attention_packed, tm.PackedAttentionArgs, packed, "Q K V O q_starts k_starts")):
        tm.check(call(args(**fields)))
        for name in names.split():
            for other in (torch.uint8, torch.bfloat16, torch.float32, torch.int32 if name == "slots" else torch.int64):
                assert call(args(**{**fields, name: fields[name].to(other)})) == 1, (name, other)
    torch.cuda.synchronize()


def test_index_tensors_with_gaps_are_refused(tm, cuda, workspace):
    c = _decode([40, 70], heads=(2, 1), d=64)
    cache, table, _, pages = _decode_problem(c)
    q = _queries(c).cuda()
    args = _decode_args(tm, c, q, torch.empty_like(q), cache, table, pages, workspace)
    tm.check(tm.attention_cache4(args))

    def refused(**changed):
        return tm.attention_cache4(tm.Cache4AttentionArgs(**{**args.__dict__, **changed})) == 1

    assert refused(lengths=args.lengths.repeat_interleave(2)[::2])
    wide = torch.zeros(2, table.shape[1] + 2, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = args.block_table
    assert refused(block_table=wide[:, :table.shape[1]]) and refused(block_table=wide.t().contiguous().t()[:, :table.shape[1]])
    assert not refused(block_table=wide[:, :table.shape[1]], table_stride=wide.shape[1])
    torch.cuda.synchronize()


@pytest.mark.parametrize("c,past", [
    (_decode([5000, 3, 0, 2300, 64], heads=(2, 1), d=64), 0), (_decode([2400] * 3 + [2399], heads=(8, 2), d=128, dtype="bf16"), 500),
    (_decode([(13 * i) % 190 for i in range(90)], heads=(4, 2), d=72, size=64), 0), (_decode([4096, 100], heads=(20, 1), d=128, size=64), 1),
    (_decode([160] * 70, heads=(4, 4), d=64, dtype="bf16"), 40)],
    ids=lambda x: f"{len(x['lengths'])}x{max(x['lengths'])}" if isinstance(x, dict) else str(x))
def test_block_tables_with_more_columns_than_the_call_has_pages(tm, cuda, workspace, c, past):
    """A resident table of which a call uses the first max_pages columns: the others hold pages
    of other sequences, which lengths `past` the call's pages must not reach."""
    cache, table, slots, pages = _decode_problem(c)
    max_pages = table.shape[1]
    rng = np.random.default_rng(7)
    wide = rng.integers(0, pages, (len(c["lengths"]), max_pages + 9)).astype(np.int32)
    for b, n in enumerate(c["lengths"]):
        need = (n + c["size"] - 1) // c["size"]
        wide[b, :need] = table[b, :need]
    q = _queries(c)
    expected, bound = _decode_expected(c, q, cache, slots)
    lengths = torch.tensor([n + past if n == max_pages * c["size"] else n for n in c["lengths"]], dtype=torch.int32, device="cuda")
    assert past == 0 or int(lengths.max()) > max_pages * c["size"]
    o = torch.full_like(q, 9.0).cuda()
    args = _decode_args(tm, c, q.cuda(), o, cache, wide, pages, workspace, max_pages=max_pages, table_stride=wide.shape[1], lengths=lengths)
    tm.check(tm.attention_cache4(args))
    torch.cuda.synchronize()
    _check(o, expected, bound, "wide table")


def test_a_group_past_bf16_is_held_as_nan(tm, cuda):
    """Rotated keys between bf16's largest value and fp32's: their minimum rounds to infinity."""
    d, size, tokens = 8, 32, 3
    k = torch.full((tokens, 1, d), 3.3895e38, dtype=torch.bfloat16)
    k[1] *= -1
    k[2, 0, 0] = 1.0
    table = np.concatenate([np.full((1, 4), 1.003), np.zeros((1, 4))], 1).astype(np.float32)
    with np.errstate(all="ignore"):
        turned = ref.rotate(k.float().numpy(), np.repeat(table, tokens, 0), False)
    assert np.isfinite(turned).all() and (np.abs(turned[:2]) > 3.396e38).all()
    cache = np.zeros((1, 1, 1, ref.block_bytes(d)), np.uint8)
    device = torch.from_numpy(cache).cuda()
    paged = dict(cache=device, pages=1, page_size=size, kv_heads=1, d=d, dtype=tm.DTYPE_BF16)
    slots = torch.arange(tokens, device="cuda")
    tm.check(tm.cache4_append(tm.Cache4AppendArgs(
        K=k.cuda(), V=torch.ones_like(k).cuda(), slots=slots, cos_sin=torch.from_numpy(table).cuda(), positions=1, rotary_dim=d,
        token_positions=torch.zeros(tokens, dtype=torch.int32, device="cuda"), tokens=tokens, **paged)))
    back = torch.empty_like(k).cuda()
    tm.check(tm.cache4_gather(tm.Cache4GatherArgs(slots=slots, tokens=tokens, K_out=back, **paged)))
    torch.cuda.synchronize()
    for t in range(tokens):
        ref.write_token(cache, size, t, 0, turned[t, 0], np.ones(d, np.float32))
    assert np.array_equal(device.cpu().numpy(), cache)
    assert torch.isnan(back[:2]).all() and torch.isfinite(back[2]).all()


@pytest.mark.parametrize("d,heads,keys", [(8, 1, 700), (64, 4, 700), (128, 2, 500), (96, 1, 3000)])
def test_many_keys_far_below_the_first_keep_their_weight(tm, cuda, d, heads, keys):
    """One key of value 0 and many of value 1000 with 2^-25.2 of its weight each, which is under
    half of fp16's smallest step: their sum is the output. (3000 keys are split.) Bound: fp16
    probabilities of up to 2^15 are off by 2^-25 each, of the first key's 2^7 or more, beside the
    bounds of serving_reference.attention, which are relative to the mean |v|."""
    gap = 25.2 * np.log(2.0)
    q = torch.ones(1, heads, d, dtype=torch.float16)
    k = torch.zeros(keys, 1, d, dtype=torch.float16)
    k[0] = 1.0
    v = torch.full((keys, 1, d), 1000.0, dtype=torch.float16)
    v[0] = 0.0
    expected, bound = ref.attention(q[0].double(), k[:, 0].double(), v[:, 0].double(), gap / d, torch.ones(heads, keys, dtype=torch.bool),
                                    ref.HALF_STEP[torch.float16])
    assert (expected > 0.01).all()
    bound = bound + keys * 2.0 ** -32 * 1000.0 + ref.HALF_STEP[torch.float16] * expected + 2.0 ** -25
    assert (bound < 0.02 * expected).all()
    o = torch.full_like(q, 9.0).cuda()
    starts = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (1, keys)]
    tm.check(tm.attention_packed(tm.PackedAttentionArgs(
        Q=q.cuda(), K=k.cuda(), V=v.cuda(), O=o, q_starts=starts[0], k_starts=starts[1], batch=1, q_tokens=1, k_tokens=keys, q_heads=heads,
        kv_heads=1, d=d, dtype=tm.DTYPE_F16, score_scale=gap / d)))
    torch.cuda.synchronize()
    _check(o[0], expected, bound, "the tail")


@pytest.mark.parametrize("dtype,below", [("f16", 20.7), ("f16", 25.2), ("f16", 30.5), ("bf16", 25.2)])
def test_values_that_agree_come_out_as_they_are(tm, cuda, dtype, below):
    """The row sums take the probabilities that P.V uses, also those below fp16's normal numbers:
    of 60000 keys `below` bits under the first one, which weigh up to 3 % together, the average of
    ones is 1. (As many rows as not to be split.) O is summed in steps of 8 keys or more and the row
    sum in one per tile and lane, each off by up to half an fp32 step of a sum that hardly grows:
    (keys / 8 + keys / 64 + 64) 2^-24 = 5.1e-4 in all, and the output's half step; a sum that had
    left out the keys 25.2 bits under the first would be 1.6e-3 off."""
    d, heads, rows, keys = 8, 8, 4160, 60000
    q = torch.ones(rows, heads, d, dtype=DT[dtype], device="cuda")
    k = torch.zeros(keys, heads, d, dtype=DT[dtype], device="cuda")
    k[0] = 1.0
    v = torch.ones_like(k)
    o = torch.full_like(q, 9.0)
    starts = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (rows, keys)]
    tm.check(tm.attention_packed(tm.PackedAttentionArgs(
        Q=q, K=k, V=v, O=o, q_starts=starts[0], k_starts=starts[1], batch=1, q_tokens=rows, k_tokens=keys, q_heads=heads, kv_heads=heads,
        d=d, dtype=_code(tm, dtype), score_scale=float(below * np.log(2.0) / d), causal=False)))
    torch.cuda.synchronize()
    assert float((o.double() - 1.0).abs().max()) <= (keys / 8 + keys / 64 + 64) * ref.FP32 + ref.HALF_STEP[DT[dtype]]
