"""Serving a model over a 4-bit key/value cache, as timed cases.

Four operators, each in its plain form here and, where ``own`` is true, through ``tilemix``:

* ``prompt``: ``attention_packed`` - attention of packed sequences of different lengths with
  grouped query heads; causal rows are aligned at the end of their sequence's keys;
* ``append``: ``cache4_append`` - keys and queries rotated by their positions, keys and values
  written to pages of 4-bit codes; the cached rows are read back, as the values they stand for;
* ``gather``: ``cache4_gather`` - cached rows back in 16 bits;
* ``decode``: ``attention_cache4`` - one query token per sequence over its pages.

The cache: pages of ``page_size`` tokens, [pages][kv heads][page_size / 32] blocks of 32 tokens.
With B = ceil(d / 64) groups of 64 features a block is

* key codes, 32 B bytes a token: features 64 m + 16 g + 8 w + e in the 32-bit word
  2 B g + 2 m + w, feature e at bits 4 (e / 2) + 16 (e % 2);
* value codes, [16 B quarters of 4 features][32 places] of 16 bits, feature f at bits 4 f;
* key, then value parameters, [B][32 places] of two bf16: scale (low half), minimum (high half).

Token t of a block has the place 8 ((t % 16) / 4) + 4 (t / 16) + t % 4. A value is
minimum + scale * code, with minimum = bf16(least of the group), scale = bf16((largest - minimum) / 15)
and code = (x - minimum) / scale rounded to even.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
WORKSPACE = 16 << 20  # bytes a serving program keeps for its decode calls
KEYS = 32  # tokens of a cache block


def _tilemix():
    package = str(Path.cwd() / "tilemix-cuda_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import tilemix

    return tilemix


# ------------------------------------------------------------------ cases


def listed():
    return [
        # A handful of short prompts, one of them a single token: latency.
        dict(name="prompt-short", kind="prompt", batch=4, longest=61, spread="ragged", context=0, q_heads=16, kv_heads=4,
             d=64, dtype="f16", causal=True),
        # A batch of chat prompts of very different lengths, 4 query heads to a key head.
        dict(name="prompt-ragged", kind="prompt", batch=16, longest=4096, spread="ragged", context=0, q_heads=32,
             kv_heads=8, d=128, dtype="bf16", causal=True),
        # One long document; the largest work.
        dict(name="prompt-long", kind="prompt", batch=1, longest=16384, spread="equal", context=0, q_heads=32, kv_heads=8,
             d=128, dtype="bf16", causal=True),
        # A chunk of two long prompts against the keys so far, one key head per query head.
        dict(name="prompt-chunk", kind="prompt", batch=2, longest=512, spread="equal", context=7680, q_heads=16,
             kv_heads=16, d=128, dtype="f16", causal=True),
        # One decode step's tokens, 32 sequences.
        dict(name="append-step", kind="append", batch=32, longest=1, spread="equal", q_heads=32, kv_heads=8, d=128,
             dtype="bf16", rotary=128, interleaved=False, page_size=64),
        # Prompts being cached: 8192 tokens of two sequences.
        dict(name="append-prompt", kind="append", batch=2, longest=4096, spread="equal", q_heads=32, kv_heads=8, d=128,
             dtype="bf16", rotary=128, interleaved=False, page_size=64),
        # Odd sizes: a quarter of the features rotated in neighbouring pairs, a head of 72.
        dict(name="append-odd", kind="append", batch=5, longest=1003, spread="ragged", q_heads=12, kv_heads=12, d=72,
             dtype="f16", rotary=18, interleaved=True, page_size=32),
        # The context of one chunked prompt back in 16 bits.
        dict(name="gather-context", kind="gather", batch=1, longest=16384, spread="equal", kv_heads=8, d=128,
             dtype="bf16", page_size=64),
        # A short shared prefix.
        dict(name="gather-prefix", kind="gather", batch=1, longest=250, spread="equal", kv_heads=4, d=64, dtype="f16",
             page_size=32),
        # One user, a short conversation: latency.
        dict(name="decode-one", kind="decode", batch=1, longest=1003, spread="equal", q_heads=16, kv_heads=4, d=64,
             dtype="f16", page_size=32),
        # A serving batch of very different lengths.
        dict(name="decode-ragged", kind="decode", batch=64, longest=16384, spread="ragged", q_heads=32, kv_heads=8,
             d=128, dtype="bf16", page_size=64),
        # Two long contexts, one key head per query head.
        dict(name="decode-long", kind="decode", batch=2, longest=32768, spread="equal", q_heads=16, kv_heads=16, d=128,
             dtype="f16", page_size=128),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random):
    kind = rng.choice(["prompt", "prompt", "append", "gather", "decode", "decode"])
    d = rng.choice([128, 128, 128, 64, 64, 96, 80, 72, 40])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    case = dict(kind=kind, kv_heads=kv_heads, d=d, dtype=rng.choice(["f16", "bf16"]),
                spread=rng.choice(["ragged", "ragged", "equal"]))
    q_heads = kv_heads * rng.choice([1, 2, 4, 4, 8] if kv_heads <= 4 else [1, 2, 4])
    if kind == "prompt":
        longest, batch = _log_int(rng, 16, 8192), _log_int(rng, 1, 32)
        context = rng.choice([0, 0, _log_int(rng, 1, 8192)])
        while batch * longest * (longest + context) > 16384 * 16384 // 2 or batch * longest > 16384:
            batch, longest = (batch // 2, longest) if batch > 1 else (1, longest // 2)
        case.update(batch=batch, longest=longest, q_heads=min(q_heads, 32), causal=rng.random() < 0.85, context=context)
    elif kind == "append":
        longest, batch = _log_int(rng, 1, 4096), _log_int(rng, 1, 64)
        while batch > 1 and batch * longest > 8192:
            batch //= 2
        rotary = rng.choice([d, d, d // 2, d // 4])
        case.update(batch=batch, longest=longest, q_heads=q_heads, rotary=rotary - rotary % 2,
                    interleaved=rng.random() < 0.3, page_size=rng.choice([32, 64, 128]))
    elif kind == "gather":
        case.update(batch=rng.choice([1, 1, 2]), longest=_log_int(rng, 32, 8192), page_size=rng.choice([32, 64, 128]))
    else:
        longest, batch = _log_int(rng, 32, 32768), _log_int(rng, 1, 128)
        while batch > 1 and batch * longest * kv_heads > 20 * 16384 * 8:
            batch //= 2
        case.update(batch=batch, longest=longest, q_heads=q_heads, page_size=rng.choice([32, 64, 128]))
    return case


def _lengths(case):
    """Tokens of each sequence: all alike, or from the longest down to a single one, one of them empty."""
    n, longest = case["batch"], case["longest"]
    if case["spread"] == "equal":
        return [longest] * n
    lengths = [longest] + [max(1, int(longest * ((i * 0.6180339887498949) % 1.0) ** 2)) for i in range(1, n)]
    if n > 2:
        lengths[2] = 0
    return lengths


def _starts(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return starts


def _visible(case):
    """(query rows, keys, visible pairs) of a prompt case, over its sequences."""
    pairs = rows = keys = 0
    for n in _lengths(case):
        k = n + case["context"]
        rows, keys = rows + n, keys + k
        pairs += n * case["context"] + n * (n + 1) // 2 if case["causal"] else n * k
    return rows, keys, pairs


def work(case):
    d, tokens = case["d"], sum(_lengths(case))
    groups = (d + 63) // 64
    row4 = d // 2 + 4 * groups  # bytes of a cached row of one head: codes, scale and minimum
    if case["kind"] == "prompt":
        rows, keys, pairs = _visible(case)
        return {"bytes": 2 * d * (2 * rows * case["q_heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * d * case["q_heads"] * pairs}
    kv = case["kv_heads"]
    if case["kind"] == "append":
        rotated = 2 * 2 * d * (case["q_heads"] + kv)  # Q and K, in and out
        cached = 2 * d * kv + 2 * row4 * kv           # V in, both written
        back = 2 * row4 * kv + 2 * 2 * d * kv         # read back
        return {"bytes": tokens * (rotated + cached + back + 4 * case["rotary"] + 12),
                "flops": 3 * tokens * case["rotary"] * (case["q_heads"] + kv) + 8 * tokens * d * 2 * kv}
    if case["kind"] == "gather":
        return {"bytes": tokens * (2 * kv * (row4 + 2 * d) + 8), "flops": 4 * tokens * kv * d}
    return {"bytes": 2 * tokens * kv * row4 + 4 * case["batch"] * case["q_heads"] * d,
            "flops": 4 * tokens * case["q_heads"] * d}


# ----------------------------------------------------------------- inputs


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _keys(gen, *shape):
    """Keys as models have them: a few features, the same for every token, larger than the others."""
    x = _normal(gen, *shape)
    x[..., 3::32] *= 4.0
    return x


def _place(t):
    return 8 * ((t % 16) // 4) + 4 * (t // 16) + t % 4


def _quantize(x, group):
    """Codes (fp32), scale and minimum (fp32 holding bf16 values) of x [..., d] in groups of `group` features."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    minimum = low.to(torch.bfloat16).float()
    # Quotients in 64 bits: differences of 16-bit values often lie half way between two codes.
    scale = ((high - minimum).double() / 15.0).to(torch.bfloat16).float()
    codes = torch.clamp(torch.round((x - minimum).double() / scale), 0.0, 15.0).float()
    return torch.where(scale > 0, codes, torch.zeros_like(codes)), scale, minimum


def _pack(k, v, d):
    """Blocks [n, block bytes] (uint8) of rows k, v [n, 32, d] (fp32)."""
    n, groups = k.shape[0], (d + 63) // 64
    place = torch.tensor([_place(t) for t in range(KEYS)], device=k.device)
    codes, params = [], []
    for x in (k, v):
        whole = torch.zeros(n, KEYS, 64 * groups, dtype=torch.int64, device=k.device)
        words = torch.empty(n, groups, KEYS, dtype=torch.int64, device=k.device)
        for m in range(groups):
            part = x[..., 64 * m:min(64 * m + 64, d)]
            c, s, low = _quantize(part, 64)
            whole[..., 64 * m:64 * m + part.shape[-1]] = c.long()
            bits = lambda y: y.to(torch.bfloat16).view(torch.int16).long() & 0xFFFF  # noqa: E731
            words[:, m, place] = (bits(s) | (bits(low) << 16))[..., 0]
        codes.append(whole)
        params.append(words.to(torch.int32).contiguous().view(torch.uint8).reshape(n, -1))
    e = torch.arange(8, device=k.device)
    key = codes[0].view(n, KEYS, groups, 4, 2, 8)  # [.., m, g, w, e]
    key = (key << (4 * (e // 2) + 16 * (e % 2))).sum(-1).permute(0, 1, 3, 2, 4)  # [.., g, m, w]
    key = key.to(torch.int32).contiguous().view(torch.uint8).reshape(n, -1)
    value = (codes[1].view(n, KEYS, 16 * groups, 4) << (4 * torch.arange(4, device=k.device))).sum(-1)
    placed = torch.empty(n, 16 * groups, KEYS, dtype=torch.int64, device=k.device)
    placed[:, :, place] = value.permute(0, 2, 1)
    value = placed.to(torch.int16).contiguous().view(torch.uint8).reshape(n, -1)
    return torch.cat([key, value, params[0], params[1]], dim=1)


def _block_bytes(d):
    return KEYS * 72 * ((d + 63) // 64)


def _filled_cache(gen, pages, page_size, kv_heads, d):
    """A cache of random keys and values, [pages, kv_heads, page_size / 32, block bytes]."""
    blocks = pages * kv_heads * (page_size // KEYS)
    cache = torch.empty(blocks, _block_bytes(d), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (KEYS * d))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        cache[at:at + n] = _pack(_keys(gen, n, KEYS, d), _normal(gen, n, KEYS, d), d)
    return cache.view(pages, kv_heads, page_size // KEYS, -1)


def _tables(gen, lengths, page_size):
    """Pages of each sequence [batch, most pages], in random order among a tenth more, and how many there are."""
    counts = [(n + page_size - 1) // page_size for n in lengths]
    pages = sum(counts) + sum(counts) // 10 + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _slots(table, lengths, page_size):
    """Slots (page * page_size + place in it) of every token, packed."""
    rows = []
    for b, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        rows.append(table[b, t // page_size].long() * page_size + t % page_size)
    return torch.cat(rows)


def prepare(case, seed):
    gen = _generator(seed)
    dtype, d, lengths = DTYPES[case["dtype"]], case["d"], _lengths(case)
    tokens, kv = sum(lengths), case["kv_heads"]
    state = dict(case, tokens=tokens, lengths=lengths)
    if case["kind"] == "prompt":
        q_starts = _starts(lengths)
        k_starts = _starts([n + case["context"] for n in lengths])
        state.update(
            Q=_normal(gen, tokens, case["q_heads"], d).to(dtype), K=_keys(gen, k_starts[-1], kv, d).to(dtype),
            V=_normal(gen, k_starts[-1], kv, d).to(dtype), O=torch.empty(tokens, case["q_heads"], d, dtype=dtype, device="cuda"),
            q_starts=torch.tensor(q_starts, dtype=torch.int32, device="cuda"),
            k_starts=torch.tensor(k_starts, dtype=torch.int32, device="cuda"), q_at=q_starts, k_at=k_starts)
        return state
    table, pages = _tables(gen, lengths, case["page_size"])
    state.update(table=table, pages=pages)
    if case["kind"] == "append":
        # One projection's output, as models make it: Q, K and V of a token side by side.
        heads = case["q_heads"] + 2 * kv
        qkv = _normal(gen, tokens, heads, d)
        qkv[:, case["q_heads"]:case["q_heads"] + kv, 3::32] *= 4.0
        qkv = qkv.to(dtype)
        # Prompts start at position 0; a decode step's token follows what its sequence has.
        first = torch.randint(0, 16384, (len(lengths),), generator=gen, device="cuda") if case["longest"] == 1 else \
            torch.zeros(len(lengths), dtype=torch.int64, device="cuda")
        positions = torch.cat([first[b] + torch.arange(n, device="cuda") for b, n in enumerate(lengths)])
        at = torch.arange(16384 + case["longest"], device="cuda", dtype=torch.float64)
        half = case["rotary"] // 2
        angles = at[:, None] * (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(1, half)))
        state.update(
            Q=qkv[:, :case["q_heads"]], K=qkv[:, case["q_heads"]:case["q_heads"] + kv], V=qkv[:, case["q_heads"] + kv:],
            cos_sin=torch.cat([angles.cos(), angles.sin()], 1).float().contiguous(), positions=positions.to(torch.int32),
            slots=_slots(table, lengths, case["page_size"]),
            cache=torch.zeros(pages, kv, case["page_size"] // KEYS, _block_bytes(d), dtype=torch.uint8, device="cuda"),
            Q_out=torch.empty(tokens, case["q_heads"], d, dtype=dtype, device="cuda"),
            **{x: torch.empty(tokens, kv, d, dtype=dtype, device="cuda") for x in ("K_out", "K_back", "V_back")})
        return state
    state.update(cache=_filled_cache(gen, pages, case["page_size"], kv, d))
    if case["kind"] == "gather":
        state.update(slots=_slots(table, lengths, case["page_size"]),
                     **{x: torch.empty(tokens, kv, d, dtype=dtype, device="cuda") for x in ("K_back", "V_back")})
        return state
    state.update(Q=_normal(gen, case["batch"], case["q_heads"], d).to(dtype),
                 O=torch.empty(case["batch"], case["q_heads"], d, dtype=dtype, device="cuda"),
                 context=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                 workspace=torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda"))
    return state


# ------------------------------------------------------------ plain forms


def _rotate(x, cos, sin, rotary, interleaved):
    """x [tokens, heads, d] (fp32) rotated by cos, sin [tokens, 1, rotary / 2]."""
    if rotary == 0:
        return x
    turned, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        both = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned.chunk(2, dim=-1)
        both = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([both, rest], dim=-1)


def _as_cached(x):
    """The values that the cache holds for x [tokens, heads, d] (fp32)."""
    out = torch.empty_like(x)
    for m in range(0, x.shape[-1], 64):
        codes, scale, minimum = _quantize(x[..., m:m + 64], 64)
        out[..., m:m + 64] = codes * scale + minimum
    return out


def _unpack(blocks, d, real):
    """Keys and values [n, 32, d] (type `real`) of blocks [n, block bytes]."""
    n, groups = blocks.shape[0], (d + 63) // 64
    place = torch.tensor([_place(t) for t in range(KEYS)], device=blocks.device)
    codes, params = blocks[:, :KEYS * 64 * groups], blocks[:, KEYS * 64 * groups:]
    e = torch.arange(8, device=blocks.device, dtype=torch.int32)
    key = codes[:, :KEYS * 32 * groups].contiguous().view(torch.int32).view(n, KEYS, 4, groups, 2, 1)
    key = ((key >> (4 * (e // 2) + 16 * (e % 2))) & 15).permute(0, 1, 3, 2, 4, 5).reshape(n, KEYS, groups, 64)
    value = codes[:, KEYS * 32 * groups:].contiguous().view(torch.int16).view(n, 16 * groups, KEYS, 1).int()
    value = (value >> (4 * torch.arange(4, device=blocks.device, dtype=torch.int32))) & 15
    value = value[:, :, place].permute(0, 2, 1, 3).reshape(n, KEYS, groups, 64)
    pairs = params.contiguous().view(torch.bfloat16).view(n, 2, groups, KEYS, 2)[:, :, :, place].to(real)
    out = []
    for i, x in enumerate((key, value)):
        scale, minimum = (pairs[:, i, :, :, j].permute(0, 2, 1).unsqueeze(-1) for j in (0, 1))
        out.append((x.to(real) * scale + minimum).reshape(n, KEYS, 64 * groups)[..., :d])
    return out


def _plain_prompt(state):
    q_heads, kv, d = state["q_heads"], state["kv_heads"], state["d"]
    group, scale = q_heads // kv, 1.0 / math.sqrt(d)
    out = torch.empty(state["tokens"], q_heads, d, dtype=torch.float32, device="cuda")
    for q0, q1, k0, k1 in zip(state["q_at"], state["q_at"][1:], state["k_at"], state["k_at"][1:]):
        n, keys = q1 - q0, k1 - k0
        if n == 0 or keys == 0:
            continue
        q = state["Q"][q0:q1].float().view(n, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * n, d)
        k = state["K"][k0:k1].float().permute(1, 2, 0).contiguous()
        v = state["V"][k0:k1].float().permute(1, 0, 2).contiguous()
        s = torch.bmm(q, k).mul_(scale).view(kv, group, n, keys)
        if state["causal"]:
            hidden = torch.arange(keys, device="cuda") > torch.arange(n, device="cuda")[:, None] + (keys - n)
            s.masked_fill_(hidden, -math.inf)
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = s.sum(-1)
        o = torch.bmm(s.view(kv, group * n, keys), v).view(kv, group, n, d) / total.unsqueeze(-1)
        out[q0:q1] = o.permute(2, 0, 1, 3).reshape(n, q_heads, d)
    return out.to(DTYPES[state["dtype"]])


def _plain_append(state):
    dtype, half = DTYPES[state["dtype"]], state["rotary"] // 2
    turns = state["cos_sin"][state["positions"].long()].unsqueeze(1)
    cos, sin = turns[..., :half], turns[..., half:]
    q = _rotate(state["Q"].float(), cos, sin, state["rotary"], state["interleaved"])
    k = _rotate(state["K"].float(), cos, sin, state["rotary"], state["interleaved"])
    return q.to(dtype), k.to(dtype), _as_cached(k).to(dtype), _as_cached(state["V"].float()).to(dtype)


def _plain_pages(state, pages, real):
    """Keys and values [pages, heads, page_size, d] of the pages named."""
    blocks = state["cache"][pages]  # [n, heads, page_size / 32, bytes]
    n, heads, per_page, size = blocks.shape
    k, v = _unpack(blocks.reshape(-1, size), state["d"], real)
    return tuple(x.view(n, heads, per_page * KEYS, state["d"]) for x in (k, v))


def _plain_gather(state):
    dtype, size = DTYPES[state["dtype"]], state["page_size"]
    pages, where = torch.unique(state["slots"] // size, return_inverse=True)
    k, v = _plain_pages(state, pages, torch.float32)
    inside = state["slots"] % size
    return k[where, :, inside].to(dtype), v[where, :, inside].to(dtype)


def _plain_decode(state):
    q_heads, kv, d, size = state["q_heads"], state["kv_heads"], state["d"], state["page_size"]
    table, batch = state["table"], state["batch"]
    n, most = table.shape[1] * size, table.shape[1]
    k, v = _plain_pages(state, table.clamp(min=0).long().view(-1), torch.float32)
    k, v = (x.view(batch, most, kv, size, d).transpose(1, 2).reshape(batch * kv, n, d) for x in (k, v))
    q = state["Q"].float().view(batch * kv, q_heads // kv, d)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(d)).view(batch, q_heads, n)
    seen = torch.arange(n, device="cuda") < state["context"][:, None, None]
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, (s - torch.where(seen.any(-1, keepdim=True), top, torch.zeros_like(top))).exp(), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(batch * kv, q_heads // kv, n), v).view(batch, q_heads, d)
    return torch.where(total > 0, o / total.clamp(min=1e-30), torch.zeros_like(o)).to(DTYPES[state["dtype"]])


# ------------------------------------------------------------- one pass


def run(state):
    kind = state["kind"]
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "gather": _plain_gather, "decode": _plain_decode}[kind](state)
    tm = _tilemix()
    dtype = tm.DTYPE_F16 if state["dtype"] == "f16" else tm.DTYPE_BF16
    shape = dict(kv_heads=state["kv_heads"], d=state["d"], dtype=dtype)
    if kind == "prompt":
        args = tm.PackedAttentionArgs(
            Q=state["Q"], K=state["K"], V=state["V"], O=state["O"], q_starts=state["q_starts"], k_starts=state["k_starts"],
            batch=state["batch"], q_tokens=state["tokens"], k_tokens=state["k_at"][-1], q_heads=state["q_heads"],
            score_scale=1.0 / math.sqrt(state["d"]), causal=state["causal"], **shape)
        tm.check(tm.attention_packed(args), "attention_packed")
        return state["O"]
    shape.update(cache=state["cache"], pages=state["pages"], page_size=state["page_size"])
    if kind == "decode":
        args = tm.Cache4AttentionArgs(
            Q=state["Q"], O=state["O"], lengths=state["context"], block_table=state["table"],
            max_pages=state["table"].shape[1], batch=state["batch"], q_heads=state["q_heads"],
            score_scale=1.0 / math.sqrt(state["d"]), workspace=state["workspace"], workspace_bytes=WORKSPACE, **shape)
        tm.check(tm.attention_cache4(args), "attention_cache4")
        return state["O"]
    if kind == "append":
        row = (state["q_heads"] + 2 * state["kv_heads"]) * state["d"]
        args = tm.Cache4AppendArgs(
            Q=state["Q"], K=state["K"], V=state["V"], Q_out=state["Q_out"], K_out=state["K_out"], slots=state["slots"],
            token_positions=state["positions"], cos_sin=state["cos_sin"], positions=state["cos_sin"].shape[0],
            rotary_dim=state["rotary"], interleaved=state["interleaved"], tokens=state["tokens"],
            q_heads=state["q_heads"], q_row_stride=row, k_row_stride=row, v_row_stride=row, **shape)
        tm.check(tm.cache4_append(args), "cache4_append")
    args = tm.Cache4GatherArgs(K_out=state["K_back"], V_out=state["V_back"], slots=state["slots"], tokens=state["tokens"], **shape)
    tm.check(tm.cache4_gather(args), "cache4_gather")
    if kind == "append":
        return state["Q_out"], state["K_out"], state["K_back"], state["V_back"]
    return state["K_back"], state["V_back"]


# ------------------------------------------------------------- in 64 bits


def _exact_rows(q, k, v, first):
    """Softmax attention of rows q [n, d] over k, v [keys, d] in 64 bits; row i sees keys up to first + i (None: all)."""
    s = q @ k.t().contiguous() / math.sqrt(q.shape[-1])
    if first is not None:
        at = torch.arange(k.shape[0], device=q.device)
        s[at[None, :] - torch.arange(q.shape[0], device=q.device)[:, None] > first] = -math.inf
    return torch.softmax(s, dim=-1) @ v


def _exact_rotated(x, angles, rotary, interleaved):
    """x [tokens, heads, d] as complex numbers times exp(i angle), in 64 bits."""
    if rotary == 0:
        return x
    half = rotary // 2
    first = list(range(0, rotary, 2)) if interleaved else list(range(half))
    second = list(range(1, rotary, 2)) if interleaved else list(range(half, rotary))
    z = torch.complex(x[..., first], x[..., second]) * angles.unsqueeze(1)
    y = x.clone()
    y[..., first], y[..., second] = z.real.contiguous(), z.imag.contiguous()
    return y


def _exact_cached(x):
    out = x.clone()
    for m in range(0, x.shape[-1], 64):
        part = x[..., m:m + 64]
        low = part.min(-1, keepdim=True).values.to(torch.bfloat16).double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).to(torch.bfloat16).double()
        code = torch.where(step > 0, ((part - low) / step).round().clamp(0, 15), torch.zeros_like(part))
        out[..., m:m + 64] = low + step * code
    return out


def _exact_values(state, slots, which):
    """Cached rows [slots, heads, d] in 64 bits, every value looked up where the format has it."""
    d, heads, size = state["d"], state["kv_heads"], state["page_size"]
    groups, flat = (d + 63) // 64, state["cache"].view(-1)
    f = torch.arange(d, device="cuda")
    m, g, w, e = f // 64, f % 64 // 16, f % 16 // 8, f % 8
    out = torch.empty(len(slots), heads, d, dtype=torch.float64, device="cuda")
    for at in range(0, len(slots), 4096):
        slot = slots[at:at + 4096, None, None]
        head, t = torch.arange(heads, device="cuda")[:, None], slot % size % KEYS
        base = (((slot // size) * heads + head) * (size // KEYS) + slot % size // KEYS) * _block_bytes(d)
        if which == "K":
            code = flat[base + 4 * (t * 8 * groups + 2 * groups * g + 2 * m + w) + (e // 2 + 4 * (e % 2)) // 2]
            code = code.int() >> (4 * (e // 2 % 2)).int()
        else:
            code = flat[base + 1024 * groups + 64 * (f // 4) + 2 * _place(t) + f % 4 // 2]
            code = code.int() >> (4 * (f % 2)).int()
        pair = base + 2048 * groups + (128 * groups if which == "V" else 0) + 128 * m + 4 * _place(t)
        scale, low = (((flat[pair + i + 1].int() << 24) | (flat[pair + i].int() << 16)).view(torch.float32).double() for i in (0, 2))
        out[at:at + 4096] = low + scale * (code & 15)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    d, kv = case["d"], case["kv_heads"]
    if case["kind"] == "prompt":
        group = case["q_heads"] // kv
        out = torch.empty(state["tokens"], case["q_heads"], d, dtype=torch.float64, device="cuda")
        for q0, q1, k0, k1 in zip(state["q_at"], state["q_at"][1:], state["k_at"], state["k_at"][1:]):
            for h in range(case["q_heads"]):
                k, v = state["K"][k0:k1, h // group].double(), state["V"][k0:k1, h // group].double()
                for at in range(q0, q1, 4096):
                    end = min(q1, at + 4096)
                    first = (k1 - k0) - (q1 - q0) + (at - q0) if case["causal"] else None
                    out[at:end, h] = _exact_rows(state["Q"][at:end, h].double(), k, v, first)
        return out
    if case["kind"] == "append":
        half = case["rotary"] // 2
        turns = state["cos_sin"][state["positions"].long()].double()
        angles = torch.complex(turns[:, :half].contiguous(), turns[:, half:].contiguous())
        q, k = (_exact_rotated(state[x].double(), angles, case["rotary"], case["interleaved"]) for x in ("Q", "K"))
        return q, k, _exact_cached(k), _exact_cached(state["V"].double())
    if case["kind"] == "gather":
        return _exact_values(state, state["slots"], "K"), _exact_values(state, state["slots"], "V")
    out = torch.zeros(case["batch"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(state["lengths"]):
        if n == 0:
            continue
        slots = _slots(state["table"][b:b + 1], [n], case["page_size"])
        k, v = (_exact_values(state, slots, x).transpose(0, 1).contiguous() for x in ("K", "V"))
        for h in range(case["q_heads"]):
            g = h * kv // case["q_heads"]
            out[b, h] = _exact_rows(state["Q"][b, h:h + 1].double(), k[g], v[g], None)[0]
    return out
