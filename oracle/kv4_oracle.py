"""CPU oracle of the 4-bit K/V cache and the operators around it, in numpy and 64-bit arithmetic:
the page format channel by channel, quantization, rotary positions, softmax attention and eviction
as include/busfill.h defines them."""
from __future__ import annotations

import numpy as np

PAGE = 64
MAX_SCALE = 896.0


def quantize(x):
    """x [..., D] -> (codes uint8 [..., D], scales fp64 [..., D/32])."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=65504.0, neginf=-65504.0)
    x = np.clip(x, -65504.0, 65504.0)
    b = x.reshape(*x.shape[:-1], -1, 32)
    first = np.abs(b).argmax(-1)          # the first of equals
    step = np.take_along_axis(b, first[..., None], -1)[..., 0] / -8.0
    mant, exp = np.frexp(step)
    step = np.ldexp(np.rint(mant * 128.0), exp - 7)     # 7 significant bits, ties to even
    step = np.clip(step, -MAX_SCALE, MAX_SCALE).astype(np.float16).astype(np.float64)
    safe = np.where(step == 0, 1.0, step)[..., None]
    code = np.clip(np.floor(b / safe + 8.5), 0, 15)
    code = np.where(step[..., None] == 0, 8, code)
    return code.reshape(x.shape).astype(np.uint8), step


def values(codes, scales):
    c = codes.reshape(*codes.shape[:-1], -1, 32).astype(np.float64)
    return ((c - 8.0) * scales[..., None]).reshape(codes.shape)


def put_token(page, t, k, v):
    """Write keys and values [D] of one token into slot t of a page uint8 [72 D] (in place)."""
    dim = k.shape[0]
    n = dim // 32
    swz = {64: 0, 128: 4 * (t // 4 % 2), 256: 2 * (t // 2 % 4)}[dim]
    kc, kd = quantize(k)
    vc, vd = quantize(v)
    for ch in range(dim):
        b, j, m = ch // 32, ch % 32 // 8, ch % 8
        for base, nib, code in ((0, 8 * (j * n + b) + m // 2 + 4 * (m % 2), kc[ch]),
                                (36 * dim, 4 * (((2 * j + m % 2) ^ swz) * n + b) + m // 2, vc[ch])):
            at = base + t * dim // 2 + nib // 2
            keep = 0x0F if nib % 2 else 0xF0
            page[at] = (int(page[at]) & keep) | (int(code) << (4 * (nib % 2)))
    page[32 * dim + 2 * t * n:32 * dim + 2 * (t + 1) * n] = kd.astype(np.float16).view(np.uint8)
    for b in range(n):
        at = 68 * dim + 2 * (b * PAGE + (t ^ (t // 2 % 2)))
        page[at:at + 2] = vd[b:b + 1].astype(np.float16).view(np.uint8)


def get_token(page, t, dim):
    """(k, v) fp64 [D] that slot t of a page uint8 [72 D] stands for."""
    n = dim // 32
    swz = {64: 0, 128: 4 * (t // 4 % 2), 256: 2 * (t // 2 % 4)}[dim]
    out = np.empty((2, dim))
    kd = page[32 * dim + 2 * t * n:32 * dim + 2 * (t + 1) * n].copy().view(np.float16).astype(np.float64)
    for ch in range(dim):
        b, j, m = ch // 32, ch % 32 // 8, ch % 8
        nib = 8 * (j * n + b) + m // 2 + 4 * (m % 2)
        out[0, ch] = ((int(page[t * dim // 2 + nib // 2]) >> (4 * (nib % 2)) & 15) - 8) * kd[b]
        nib = 4 * (((2 * j + m % 2) ^ swz) * n + b) + m // 2
        at = 68 * dim + 2 * (b * PAGE + (t ^ (t // 2 % 2)))
        vd = float(page[at:at + 2].copy().view(np.float16)[0])
        out[1, ch] = ((int(page[36 * dim + t * dim // 2 + nib // 2]) >> (4 * (nib % 2)) & 15) - 8) * vd
    return out[0], out[1]


def rope(x, positions, cos, sin, axis, adjacent=False, inverse=False):
    """x [tokens, heads, D] fp64, positions [axes, tokens], cos/sin [max_pos, half]."""
    half = cos.shape[1]
    col = np.arange(half)
    pos = np.asarray(positions)[np.asarray(axis)]               # [half, tokens]
    c = cos[pos, col[:, None]].T[:, None].astype(np.float64)
    s = sin[pos, col[:, None]].T[:, None].astype(np.float64) * (-1.0 if inverse else 1.0)
    y = np.array(x, np.float64)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if adjacent else (slice(0, half), slice(half, 2 * half))
    x0, x1 = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def attention(q, k, v, scale, seen):
    """q [n, D], k and v [L, D], seen bool [n, L] -> (out, lse, p); a row that sees nothing: 0, -inf, 0."""
    s = np.where(seen, q @ k.T * scale, -np.inf) if k.shape[0] else np.zeros((q.shape[0], 0))
    top = s.max(-1, initial=-np.inf, keepdims=True)
    e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = e.sum(-1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = np.where(total == 0, -np.inf, np.log(total) + np.where(np.isfinite(top), top, 0.0))
    return p @ v, lse[:, 0], p


def seen(n, length, causal=True, window=0):
    """Which of `length` slots each of a sequence's n newest rows sees, bool [n, length]."""
    last = length - n + np.arange(n)[:, None]
    slot = np.arange(length)[None]
    ok = slot <= last if causal else np.ones((n, length), bool)
    return ok & (slot > last - window) if window else ok


def kept(weights, length, keep, recent):
    """Slots of one sequence and head that stay, ascending."""
    keep = min(length, keep)
    recent = min(recent, keep)
    old = np.asarray(weights[:length - recent], np.float64)
    nan = np.isnan(old)                       # below every number, -inf too
    order = np.lexsort((-np.where(nan, 0.0, old), nan))[:keep - recent]
    return np.concatenate([np.sort(order), np.arange(length - recent, length)]).astype(np.int64)
