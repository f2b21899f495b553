"""Plain implementations of the serving operators (tilemix_attention_packed,
tilemix_cache4_*, tilemix_attention_cache4) on the CPU, from the formulas of
include/tilemix_capi.h: the cache format value by value in float32 where its codes
are defined there, everything else in float64, with the error that an output of
the type may have beside each result.

Half a rounding step, relative to the value: bf16 2^-8, fp16 2^-11, fp32 2^-24.
"""
from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FP32 = 2.0 ** -24


# ------------------------------------------------------------- the format


def place(t):
    return 8 * ((t % 16) // 4) + 4 * (t // 16) + t % 4


def bf16_bits(x: np.ndarray) -> np.ndarray:
    """bf16 bits of float32 values, rounded to nearest even."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


def bf16_value(bits: np.ndarray) -> np.ndarray:
    return (bits.astype(np.uint32) << 16).view(np.float32)


def quantize(x: np.ndarray):
    """float32 [..., d] -> codes uint8 [..., d], parameter words uint32 [..., groups]."""
    d = x.shape[-1]
    groups = (d + 63) // 64
    codes = np.zeros(x.shape, np.uint8)
    words = np.zeros(x.shape[:-1] + (groups,), np.uint32)
    with np.errstate(all="ignore"):
        for m in range(groups):
            part = x[..., 64 * m:64 * m + 64].astype(np.float32)
            low = bf16_value(bf16_bits(part.min(-1))) + np.float32(0)  # a zero without its sign
            low_bits = bf16_bits(low)
            span = part.max(-1) - low  # float32
            scale_bits = bf16_bits((span.astype(np.float64) / 15.0).astype(np.float32))
            scale = bf16_value(scale_bits)
            finite = np.isfinite(part).all(-1) & np.isfinite(scale)
            coded = finite & (scale >= 2.0 ** -100)
            steps = (part - low[..., None]).astype(np.float64) / scale[..., None].astype(np.float64)
            steps = np.clip(np.rint(steps.astype(np.float32)), 0, 15)
            codes[..., 64 * m:64 * m + 64] = np.where(coded[..., None], np.nan_to_num(steps), 0)
            word = np.where(coded, scale_bits, 0).astype(np.uint32) | (low_bits.astype(np.uint32) << 16)
            words[..., m] = np.where(finite, word, 0x7FC07FC0)
    return codes, words


def block_bytes(d: int) -> int:
    return 32 * 72 * ((d + 63) // 64)


def addresses(d: int, t: int):
    """Byte and shift of every feature's key and value code of token t in a block, byte of its parameter words."""
    B = (d + 63) // 64
    f = np.arange(64 * B)
    m, g, w, e = f // 64, f % 64 // 16, f % 16 // 8, f % 8
    bit = 4 * (e // 2) + 16 * (e % 2)
    key = (4 * (8 * B * t + 2 * B * g + 2 * m + w) + bit // 8, bit % 8)
    value = (1024 * B + 64 * (f // 4) + 2 * place(t) + (f % 4) // 2, 4 * (f % 2))
    params = 2048 * B + 128 * np.arange(B) + 4 * place(t)
    return key, value, params, params + 128 * B


def block_of(cache: np.ndarray, page_size: int, slot: int, head: int) -> np.ndarray:
    """View of the block of `slot` in a cache [pages, heads, page_size / 32, block bytes]."""
    return cache[slot // page_size, head, slot % page_size // 32]


def write_token(cache, page_size, slot, head, k, v):
    """Key and value rows (float32 [d]) of one token and head into a host cache."""
    d = len(k)
    block = block_of(cache, page_size, slot, head)
    key, value, key_params, value_params = addresses(d, slot % page_size % 32)
    for row, (at, shift), params in ((k, key, key_params), (v, value, value_params)):
        codes, words = quantize(row)
        whole = np.zeros(64 * ((d + 63) // 64), np.uint8)
        whole[:d] = codes
        for a, s, c in zip(at, shift, whole):
            block[a] = (block[a] & ~np.uint8(15 << s)) | np.uint8(c << s)
        for a, word in zip(params, words):
            block[a:a + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)


def read_token(cache, page_size, slot, head, d):
    """(key, value) float64 [d] of one token and head."""
    block = block_of(cache, page_size, slot, head)
    key, value, key_params, value_params = addresses(d, slot % page_size % 32)
    out = []
    for (at, shift), params in ((key, key_params), (value, value_params)):
        codes = (block[at] >> shift) & 15
        words = np.stack([block[a:a + 4].copy().view(np.uint32)[0] for a in params])
        scale, low = bf16_value((words & 0xFFFF).astype(np.uint16)), bf16_value((words >> 16).astype(np.uint16))
        group = np.arange(len(codes)) // 64
        out.append((low.astype(np.float64)[group] + scale.astype(np.float64)[group] * codes)[:d])
    return out


def read_tokens(cache, page_size, slots, d):
    """Keys and values float64 [slots, heads, d] of a host cache."""
    heads = cache.shape[1]
    rows = [[read_token(cache, page_size, int(s), h, d) for h in range(heads)] for s in slots]
    array = np.array(rows, np.float64).reshape(len(slots), heads, 2, d)
    return array[:, :, 0], array[:, :, 1]


# ------------------------------------------------------------ the rotation


def rotate(x: np.ndarray, table: np.ndarray, interleaved: bool) -> np.ndarray:
    """x float32 [tokens, heads, d] turned by table float32 [tokens, rotary]; products and sums in float32."""
    rotary = table.shape[1]
    half = rotary // 2
    cos, sin = table[:, None, :half], table[:, None, half:]
    out = x.astype(np.float32).copy()
    first = slice(0, rotary, 2) if interleaved else slice(0, half)
    second = slice(1, rotary, 2) if interleaved else slice(half, rotary)
    a, b = x[..., first].astype(np.float32), x[..., second].astype(np.float32)
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


# ----------------------------------------------------------- the attention


def attention(q, k, v, scale, visible, rounded):
    """One head in float64: q [n, d], k, v [m, d], visible [n, m] bool.

    Returns (o, bound): bound is how far an output of a kernel may be whose
    probabilities have a relative error of `rounded` each (in sums and products
    alike: it moves o by at most 2 rounded times the mean |v|), whose scores are
    fp32 sums of exact products (d + 8 roundings of sum |q k|, in the exponent),
    and whose fp32 sums over keys have an error of (m + 64) half steps. The
    rounding of the output itself comes on top.
    """
    n, m = len(q), len(k)
    o, bound = torch.zeros(n, v.shape[-1], dtype=torch.float64), torch.zeros(n, v.shape[-1], dtype=torch.float64)
    if m == 0:
        return o, bound
    s = (q @ k.T) * scale
    size = (q.abs() @ k.abs().T) * abs(scale)
    s = torch.where(visible, s, torch.tensor(-math.inf, dtype=torch.float64))
    size = torch.where(visible, size, torch.zeros_like(size))
    some = visible.any(-1)
    top = torch.where(some, s.amax(-1), torch.zeros(n, dtype=torch.float64))
    p = torch.where(visible, (s - top[:, None]).exp(), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True).clamp(min=1e-300)
    w = p / total
    clean = torch.where(visible.any(0)[:, None], v, torch.zeros_like(v))  # keys that nobody sees
    o = w @ clean
    mean = w @ clean.abs()
    score = (q.shape[-1] + 8) * FP32 * size.amax(-1, keepdim=True) + 8 * FP32 * (1 + s.abs().where(visible, torch.zeros_like(s)).amax(-1, keepdim=True))
    bound = mean * (2 * rounded + 2 * score + 2 * (m + 64) * FP32)
    return o, bound
