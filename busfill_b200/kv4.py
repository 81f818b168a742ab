"""Rotary positions, the paged 4-bit K/V cache, attention over it and eviction:
the operators of a decoder layer between its QKV and its O projection.

Shapes and terms (include/busfill.h has the format and the exact rules):

* ``pages`` uint8 [num_pages, kv_heads, 72 * D]: the pool; a page holds 64 tokens of a head.
* ``table`` int32 [batch, cols]: the pages of each sequence; ``kv_len`` int32 [batch]: its cached
  tokens, the ones of the current step included.
* ``q_start`` int32 [batch + 1]: where each sequence's rows begin in the step's tensors
  [tokens, heads, D]; None: one row per sequence.

All tensors are CUDA tensors of one device; queries, keys and values are fp16 or bf16 with
contiguous channels and free token and head strides, e.g. slices of a fused QKV output. Calls are
asynchronous on ``stream`` (default: the current one); what they return is made on that stream.
Out-of-range device indices are not followed and show in ``stream_status()``.
"""
from __future__ import annotations

import contextlib
import ctypes

from . import _check, _lib, _ptr, _stream, _torch

KV4_PAGE = 64

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64


class Cache(ctypes.Structure):
    """busfill_kv4"""
    _fields_ = [("pages", _P), ("table", _P), ("kv_len", _P), ("num_pages", _I), ("table_cols", _I), ("batch", _I),
                ("heads", _I), ("head_dim", _I)]


class Rope(ctypes.Structure):
    """busfill_rope"""
    _fields_ = [("q", _P), ("k", _P), ("q_out", _P), ("k_out", _P), ("positions", _P), ("cos", _P), ("sin", _P),
                ("axis", _P), ("q_token", _L), ("q_head", _L), ("k_token", _L), ("k_head", _L), ("q_out_token", _L),
                ("q_out_head", _L), ("k_out_token", _L), ("k_out_head", _L), ("tokens", _I), ("q_heads", _I),
                ("k_heads", _I), ("head_dim", _I), ("rot", _I), ("axes", _I), ("max_pos", _I), ("adjacent", _I),
                ("inverse", _I), ("dtype", _I)]


class Rows(ctypes.Structure):
    """busfill_kv4_rows"""
    _fields_ = [("k", _P), ("v", _P), ("q_start", _P), ("k_token", _L), ("k_head", _L), ("v_token", _L),
                ("v_head", _L), ("tokens", _I), ("dtype", _I)]


class Attn(ctypes.Structure):
    """busfill_attn"""
    _fields_ = [("q", _P), ("out", _P), ("lse", _P), ("weights", _P), ("q_start", _P), ("q_token", _L),
                ("q_head", _L), ("out_token", _L), ("out_head", _L), ("weights_cols", _L), ("scale", ctypes.c_float),
                ("tokens", _I), ("q_heads", _I), ("max_q", _I), ("causal", _I), ("window", _I), ("dtype", _I)]


class Eviction(ctypes.Structure):
    """busfill_kv4_eviction"""
    _fields_ = [("weights", _P), ("weights_out", _P), ("weights_cols", _L), ("index", _P), ("kv_len_out", _P),
                ("out_table", _P), ("out_cols", _I), ("keep", _I), ("recent", _I)]


def _dtype(t):
    torch = _torch()
    return {torch.float16: 1, torch.bfloat16: 30}[t.dtype]


def _need_heads(t, name, like=None):
    """A step's tensor [tokens, heads, D], fp16 or bf16, channels contiguous."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in (torch.float16, torch.bfloat16) or (like is not None and t.dtype != like.dtype):
        raise TypeError(f"{name} must be {'fp16 or bf16' if like is None else like.dtype}, got {t.dtype}")
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be [tokens, heads, D] with contiguous channels")


def _need_array(t, dtype, name, ndim):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {ndim}-D tensor")


def _cache(pages, table, kv_len):
    torch = _torch()
    _need_array(pages, torch.uint8, "pages", 3)
    _need_array(table, torch.int32, "table", 2)
    _need_array(kv_len, torch.int32, "kv_len", 1)
    dim, rest = divmod(pages.shape[2], 72)
    if rest or dim not in (64, 128, 256):
        raise ValueError(f"pages must be [num_pages, kv_heads, 72 * D] with D 64, 128 or 256, got {tuple(pages.shape)}")
    if table.shape[0] != kv_len.shape[0]:
        raise ValueError(f"table {tuple(table.shape)} and kv_len {tuple(kv_len.shape)} differ in batch")
    return Cache(pages.data_ptr(), table.data_ptr(), kv_len.data_ptr(), pages.shape[0], table.shape[1],
                 table.shape[0], pages.shape[1], dim)


def _need_start(q_start, cache, tokens):
    if q_start is None:
        if tokens != cache.batch:
            raise ValueError(f"{tokens} rows for {cache.batch} sequences: give q_start")
        return None
    _need_array(q_start, _torch().int32, "q_start", 1)
    if q_start.shape[0] != cache.batch + 1:
        raise ValueError(f"q_start must have {cache.batch + 1} entries, got {q_start.shape[0]}")
    return q_start.data_ptr()


def _on(stream):
    """Allocations inside belong to the call's stream."""
    return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)


def kv4_page_bytes(head_dim: int) -> int:
    """Bytes of a page (64 tokens, keys and values) of one head."""
    n = _lib().busfill_kv4_page_bytes(int(head_dim))
    _check(min(n, 0), "busfill_kv4_page_bytes")
    return n


def kv4_pool(num_pages: int, kv_heads: int, head_dim: int, device="cuda"):
    """A zeroed pool of pages, uint8 [num_pages, kv_heads, 72 * head_dim]."""
    torch = _torch()
    return torch.zeros((num_pages, kv_heads, kv4_page_bytes(head_dim)), dtype=torch.uint8, device=device)


def rope_table(max_pos: int, rot: int, base: float = 10000.0, inv_freq=None, device="cuda"):
    """(cos, sin) fp32 [max_pos, rot / 2] of the angles pos * inv_freq, computed in fp64; inv_freq
    defaults to base ** (-2i / rot)."""
    torch = _torch()
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv_freq.to(device).double()
    return angle.cos().float(), angle.sin().float()


def rope_axes(q, k, positions, cos, sin, axis=None, adjacent=False, inverse=False, q_out=None, k_out=None,
              stream=None):
    """Rotary positions with several axes on queries and keys [tokens, heads, D] (k may be None).

    positions int32 [axes, tokens] (or [tokens] for one axis); cos, sin fp32 [max_pos, rot / 2]
    (:func:`rope_table`); ``axis``: for each of the rot / 2 frequencies the axis whose position turns
    it (default: axis 0). Frequency i turns channels (i, i + rot/2), or (2i, 2i + 1) with
    ``adjacent``; channels from rot on are copied. ``inverse`` turns back, which is also the gradient.
    q_out, k_out may be q, k. Returns (q_out, k_out)."""
    torch = _torch()
    _need_heads(q, "q")
    if positions.dim() == 1:
        positions = positions[None]
    _need_array(positions, torch.int32, "positions", 2)
    _need_array(cos, torch.float32, "cos", 2)
    _need_array(sin, torch.float32, "sin", 2)
    tokens, heads, dim = q.shape
    half = cos.shape[1]
    axis = [0] * half if axis is None else [int(a) for a in axis]
    if cos.shape != sin.shape or len(axis) != half or positions.shape[1] != tokens:
        raise ValueError(f"shape mismatch: cos {tuple(cos.shape)}, sin {tuple(sin.shape)}, axis {len(axis)}, "
                         f"positions {tuple(positions.shape)}, q {tuple(q.shape)}")
    if any(not 0 <= a < positions.shape[0] for a in axis):
        raise ValueError(f"axis entries must be in 0..{positions.shape[0] - 1}")
    if k is not None:
        _need_heads(k, "k", like=q)
        if k.shape[0] != tokens or k.shape[2] != dim:
            raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}")
    with _on(stream):
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if k is not None and k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    for t, like, name in ((q_out, q, "q_out"), (k_out, k, "k_out")):
        if like is not None:
            _need_heads(t, name, like=like)
            if t.shape != like.shape:
                raise ValueError(f"{name} must be {tuple(like.shape)}, got {tuple(t.shape)}")
    table = (ctypes.c_uint8 * half)(*axis)
    r = Rope(q.data_ptr(), None if k is None else k.data_ptr(), q_out.data_ptr(),
             None if k is None else k_out.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
             ctypes.cast(table, _P), q.stride(0), q.stride(1), 0 if k is None else k.stride(0),
             0 if k is None else k.stride(1), q_out.stride(0), q_out.stride(1), 0 if k is None else k_out.stride(0),
             0 if k is None else k_out.stride(1), tokens, heads, 0 if k is None else k.shape[1], dim, 2 * half,
             positions.shape[0], cos.shape[0], int(adjacent), int(inverse), _dtype(q))
    _check(_lib().busfill_rope_axes(ctypes.byref(r), _stream(stream)), "busfill_rope_axes")
    return q_out, k_out


def kv4_append(pages, table, kv_len, k, v, q_start=None, stream=None):
    """Quantize the step's keys and values [tokens, kv_heads, D] into the slots of their sequences'
    newest tokens (row r of a sequence's n rows goes to slot kv_len - n + r)."""
    c = _cache(pages, table, kv_len)
    _need_heads(k, "k")
    _need_heads(v, "v", like=k)
    if k.shape != v.shape or k.shape[1] != c.heads or k.shape[2] != c.head_dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {c.heads}, {c.head_dim}]")
    r = Rows(k.data_ptr(), v.data_ptr(), _need_start(q_start, c, k.shape[0]), k.stride(0), k.stride(1), v.stride(0),
             v.stride(1), k.shape[0], _dtype(k))
    _check(_lib().busfill_kv4_append(ctypes.byref(c), ctypes.byref(r), _stream(stream)), "busfill_kv4_append")


def kv4_read(pages, table, kv_len, q_start=None, tokens=None, stream=None):
    """The exact fp16 values (k, v) [tokens, kv_heads, D] that the cache holds for the newest tokens
    of every sequence; for whole sequences let q_start be the running sum of kv_len."""
    torch = _torch()
    c = _cache(pages, table, kv_len)
    tokens = c.batch if tokens is None else int(tokens)
    start = _need_start(q_start, c, tokens)
    with _on(stream):
        k = torch.empty((tokens, c.heads, c.head_dim), dtype=torch.float16, device=pages.device)
        v = torch.empty_like(k)
    _check(_lib().busfill_kv4_read(ctypes.byref(c), start, tokens, _ptr(k), _ptr(v), _stream(stream)),
           "busfill_kv4_read")
    return k, v


def attn_kv4(q, pages, table, kv_len, q_start=None, max_q=None, scale=None, causal=True, window=0, out=None, lse=None,
             weights=None, stream=None):
    """Attention of q [tokens, q_heads, D] over the cache; q_heads is a multiple of the cache's heads.

    A row sees its whole sequence, with ``causal`` the slots up to its own, with window > 0 the last
    ``window`` of these; a row that sees nothing gives 0. ``max_q`` bounds the rows of one sequence
    (default: all rows); a sequence with more is cut and reported. scale defaults to D ** -0.5.
    ``lse`` fp32 [tokens, q_heads] gets each row's log-sum-exp (-inf for a row that sees nothing).
    To ``weights`` fp32 [batch, kv_heads, cols >= 64 * table columns] the attention weight of every
    cached token, summed over the call's rows and the group's heads, is added."""
    torch = _torch()
    c = _cache(pages, table, kv_len)
    _need_heads(q, "q")
    tokens, heads, dim = q.shape
    if dim != c.head_dim or heads % c.heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {c.heads} heads of {c.head_dim}")
    start = _need_start(q_start, c, tokens)
    if weights is not None:
        _need_array(weights, torch.float32, "weights", 3)
        if weights.shape[:2] != (c.batch, c.heads) or weights.shape[2] < KV4_PAGE * c.table_cols:
            raise ValueError(f"weights must be [{c.batch}, {c.heads}, >= {KV4_PAGE * c.table_cols}], got "
                             f"{tuple(weights.shape)}")
    with _on(stream):
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if lse is None and weights is not None:
            lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device)
    _need_heads(out, "out", like=q)
    if out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    if lse is not None:
        _need_array(lse, torch.float32, "lse", 2)
        if lse.shape != (tokens, heads):
            raise ValueError(f"lse must be [{tokens}, {heads}], got {tuple(lse.shape)}")
    a = Attn(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
             None if weights is None else weights.data_ptr(), start, q.stride(0), q.stride(1), out.stride(0),
             out.stride(1), 0 if weights is None else weights.shape[2], dim ** -0.5 if scale is None else float(scale),
             tokens, heads, max(1, tokens if max_q is None else int(max_q)) if start else 1, int(bool(causal)),
             int(window), _dtype(q))
    _check(_lib().busfill_attn_kv4(ctypes.byref(c), ctypes.byref(a), _stream(stream)), "busfill_attn_kv4")
    return out


def kv4_evict(pages, table, kv_len, weights, keep, recent, out_table=None, weights_out=None, stream=None):
    """Bring every sequence longer than ``keep`` down to ``keep`` tokens, head by head: the last
    ``recent`` stay, and of the others those with the largest accumulated weights (the lower slot of
    equals), in their order. ``out_table`` int32 [batch, cols] names the pages they move to (default:
    the same table, in place). Returns (index, weights_out, new kv_len): index int32 [batch,
    kv_heads, keep] holds the slots they came from (-1 behind a shorter sequence's)."""
    torch = _torch()
    c = _cache(pages, table, kv_len)
    _need_array(weights, torch.float32, "weights", 3)
    if weights.shape[:2] != (c.batch, c.heads) or weights.shape[2] < KV4_PAGE * c.table_cols:
        raise ValueError(f"weights must be [{c.batch}, {c.heads}, >= {KV4_PAGE * c.table_cols}], got "
                         f"{tuple(weights.shape)}")
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"need 1 <= keep and 0 <= recent <= keep, got keep {keep}, recent {recent}")
    out_table = table if out_table is None else out_table
    _need_array(out_table, torch.int32, "out_table", 2)
    if out_table.shape[0] != c.batch or out_table.shape[1] * KV4_PAGE < keep:
        raise ValueError(f"out_table must be [{c.batch}, >= {-(-keep // KV4_PAGE)}], got {tuple(out_table.shape)}")
    with _on(stream):
        index = torch.empty((c.batch, c.heads, keep), dtype=torch.int32, device=pages.device)
        kv_len_out = torch.empty_like(kv_len)
        if weights_out is None:
            weights_out = torch.empty_like(weights)
    _need_array(weights_out, torch.float32, "weights_out", 3)
    if weights_out.shape != weights.shape:
        raise ValueError(f"weights_out must be {tuple(weights.shape)}, got {tuple(weights_out.shape)}")
    e = Eviction(weights.data_ptr(), weights_out.data_ptr(), weights.shape[2], index.data_ptr(),
                 kv_len_out.data_ptr(), out_table.data_ptr(), out_table.shape[1], keep, recent)
    _check(_lib().busfill_kv4_evict(ctypes.byref(c), ctypes.byref(e), _stream(stream)), "busfill_kv4_evict")
    return index, weights_out, kv_len_out
