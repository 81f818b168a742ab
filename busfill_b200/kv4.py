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

import ctypes
import struct

from . import _check, _lib, _torch

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


def _packer(cls):
    """cls's fields as native bytes: several times cheaper to make per call than the ctypes object."""
    code = {_P: "P", _L: "q", _I: "i", ctypes.c_float: "f"}
    return struct.Struct("@" + "".join(code[t] for _, t in cls._fields_) + "0q").pack


_pack_cache, _pack_rope, _pack_rows, _pack_attn, _pack_eviction = map(_packer, (Cache, Rope, Rows, Attn, Eviction))
_TYPE = {}   # torch dtype -> BUSFILL_TYPE_*; filled with torch's dtypes at the first call
_U8 = _I32 = _F32 = _F16 = _raw_stream = _empty_like = _contiguous = None


def _init():
    global _U8, _I32, _F32, _F16, _raw_stream, _empty_like, _contiguous
    torch = _torch()
    _empty_like, _contiguous = torch.empty_like, torch.contiguous_format
    _U8, _I32, _F32, _F16 = torch.uint8, torch.int32, torch.float32, torch.float16
    _raw_stream = torch._C._cuda_getCurrentRawStream
    _TYPE.update({torch.float16: 1, torch.bfloat16: 30})


def _refuse_heads(t, name, like):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPE or (like is not None and t.dtype != like.dtype):
        raise TypeError(f"{name} must be {'fp16 or bf16' if like is None else like.dtype}, got {t.dtype}")
    raise ValueError(f"{name} must be [tokens, heads, D] with contiguous channels, got {tuple(t.shape)} with strides "
                     f"{t.stride()}")


def _heads(t, name, like=None):
    """(token, head) strides of a step's tensor [tokens, heads, D]: fp16 or bf16, channels contiguous."""
    if not _TYPE:
        _init()
    try:
        if t.is_cuda and (t.dtype in _TYPE if like is None else t.dtype is like.dtype):
            token, head, channel = t.stride()
            if channel == 1 or t.shape[2] == 1:
                return token, head
    except (AttributeError, ValueError):
        pass
    _refuse_heads(t, name, like)


def _array(t, dtype, name, ndim):
    """The address of a contiguous CUDA tensor of that type and rank."""
    try:
        if t.is_cuda and t.dtype is dtype and t.dim() == ndim and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    raise ValueError(f"{name} must be a contiguous {ndim}-D tensor")


def _cache(pages, table, kv_len):
    """(busfill_kv4 as bytes, batch, heads, head_dim, table columns)"""
    if not _TYPE:
        _init()
    pages_ptr, table_ptr, len_ptr = (_array(pages, _U8, "pages", 3), _array(table, _I32, "table", 2),
                                     _array(kv_len, _I32, "kv_len", 1))
    num_pages, heads, width = pages.shape
    batch, cols = table.shape
    dim, rest = divmod(width, 72)
    if rest or dim not in (64, 128, 256):
        raise ValueError(f"pages must be [num_pages, kv_heads, 72 * D] with D 64, 128 or 256, got {tuple(pages.shape)}")
    if batch != kv_len.shape[0]:
        raise ValueError(f"table {tuple(table.shape)} and kv_len {tuple(kv_len.shape)} differ in batch")
    return _pack_cache(pages_ptr, table_ptr, len_ptr, num_pages, cols, batch, heads, dim), batch, heads, dim, cols


def _need_start(q_start, batch, tokens):
    if q_start is None:
        if tokens != batch:
            raise ValueError(f"{tokens} rows for {batch} sequences: give q_start")
        return 0
    ptr = _array(q_start, _I32, "q_start", 1)
    if q_start.shape[0] != batch + 1:
        raise ValueError(f"q_start must have {batch + 1} entries, got {q_start.shape[0]}")
    return ptr


def _weights(weights, name, batch, heads, cols):
    """(address, columns)"""
    ptr = _array(weights, _F32, name, 3)
    b, h, n = weights.shape
    if b != batch or h != heads or n < KV4_PAGE * cols:
        raise ValueError(f"{name} must be [{batch}, {heads}, >= {KV4_PAGE * cols}], got {tuple(weights.shape)}")
    return ptr, n


def _raw(stream, like):
    """The cudaStream_t of the call."""
    if stream is None:
        return _raw_stream(like.get_device())
    return stream.cuda_stream


def _another(stream, like):
    """A contiguous tensor of like's shape and type that belongs to the call's stream."""
    if stream is None:
        return _empty_like(like, memory_format=_contiguous)
    with _torch().cuda.stream(stream):
        return _empty_like(like, memory_format=_contiguous)


def _empty(stream, like, shape, dtype):
    """A tensor on like's device that belongs to the call's stream."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


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
    q_token, q_head = _heads(q, "q")
    if getattr(positions, "ndim", 0) == 1:
        positions = positions[None]
    pos_ptr, cos_ptr, sin_ptr = (_array(positions, _I32, "positions", 2), _array(cos, _F32, "cos", 2),
                                 _array(sin, _F32, "sin", 2))
    shape = q.shape
    tokens, heads, dim = shape
    max_pos, half = cos.shape
    axes, n = positions.shape
    axis = bytes(half) if axis is None else bytes(axis)
    if sin.shape != cos.shape or len(axis) != half or n != tokens:
        raise ValueError(f"shape mismatch: cos {tuple(cos.shape)}, sin {tuple(sin.shape)}, axis {len(axis)}, "
                         f"positions {tuple(positions.shape)}, q {tuple(shape)}")
    if half and max(axis) >= axes:
        raise ValueError(f"axis entries must be in 0..{axes - 1}")
    if q_out is None:
        q_out = _another(stream, q)
        qo_token, qo_head = heads * dim, dim
    else:
        qo_token, qo_head = _heads(q_out, "q_out", like=q)
        if q_out.shape != shape:
            raise ValueError(f"q_out must be {tuple(shape)}, got {tuple(q_out.shape)}")
    k_ptr = ko_ptr = k_heads = k_token = k_head = ko_token = ko_head = 0
    if k is not None:
        k_token, k_head = _heads(k, "k", like=q)
        n, k_heads, k_dim = k.shape
        if n != tokens or k_dim != dim:
            raise ValueError(f"shape mismatch: q {tuple(shape)}, k {tuple(k.shape)}")
        if k_out is None:
            k_out = _another(stream, k)
            ko_token, ko_head = k_heads * dim, dim
        else:
            ko_token, ko_head = _heads(k_out, "k_out", like=q)
            if k_out.shape != k.shape:
                raise ValueError(f"k_out must be {tuple(k.shape)}, got {tuple(k_out.shape)}")
        k_ptr, ko_ptr = k.data_ptr(), k_out.data_ptr()
    table = ctypes.create_string_buffer(axis, half)
    r = _pack_rope(q.data_ptr(), k_ptr, q_out.data_ptr(), ko_ptr, pos_ptr, cos_ptr, sin_ptr, ctypes.addressof(table),
                   q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head, tokens, heads, k_heads, dim,
                   2 * half, axes, max_pos, bool(adjacent), bool(inverse), _TYPE[q.dtype])
    _check(_lib().busfill_rope_axes(r, _raw(stream, q)), "busfill_rope_axes")
    return q_out, k_out


def kv4_append(pages, table, kv_len, k, v, q_start=None, stream=None):
    """Quantize the step's keys and values [tokens, kv_heads, D] into the slots of their sequences'
    newest tokens (row r of a sequence's n rows goes to slot kv_len - n + r)."""
    c, batch, heads, dim, _ = _cache(pages, table, kv_len)
    k_token, k_head = _heads(k, "k")
    v_token, v_head = _heads(v, "v", like=k)
    tokens, k_heads, k_dim = k.shape
    if k.shape != v.shape or k_heads != heads or k_dim != dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {heads}, {dim}]")
    r = _pack_rows(k.data_ptr(), v.data_ptr(), _need_start(q_start, batch, tokens), k_token, k_head, v_token, v_head,
                   tokens, _TYPE[k.dtype])
    _check(_lib().busfill_kv4_append(c, r, _raw(stream, pages)), "busfill_kv4_append")


def kv4_read(pages, table, kv_len, q_start=None, tokens=None, stream=None):
    """The exact fp16 values (k, v) [tokens, kv_heads, D] that the cache holds for the newest tokens
    of every sequence; for whole sequences let q_start be the running sum of kv_len."""
    c, batch, heads, dim, _ = _cache(pages, table, kv_len)
    tokens = batch if tokens is None else int(tokens)
    start = _need_start(q_start, batch, tokens)
    k = _empty(stream, pages, (tokens, heads, dim), _F16)
    v = _another(stream, k)
    _check(_lib().busfill_kv4_read(c, start, tokens, k.data_ptr(), v.data_ptr(), _raw(stream, pages)),
           "busfill_kv4_read")
    return k, v


def attn_kv4(q, pages, table, kv_len, q_start=None, max_q=None, scale=None, causal=True, window=0, out=None, lse=None,
             weights=None, stream=None):
    """Attention of q [tokens, q_heads, D] over the cache; q_heads is a multiple of the cache's heads.

    A row sees its whole sequence, with ``causal`` the slots up to its own, with window > 0 the last
    ``window`` of these; a row that sees nothing gives 0. ``max_q`` bounds the rows of one sequence
    (default: all rows, which for a ragged step of few rows a sequence chooses the slower kernel:
    give it); a sequence with more is cut and reported. scale defaults to D ** -0.5.
    ``lse`` fp32 [tokens, q_heads] gets each row's log-sum-exp (-inf for a row that sees nothing).
    To ``weights`` fp32 [batch, kv_heads, cols >= 64 * table columns] the attention weight of every
    cached token, summed over the call's rows and the group's heads, is added."""
    c, batch, kv_heads, head_dim, cols = _cache(pages, table, kv_len)
    q_token, q_head = _heads(q, "q")
    shape = q.shape
    tokens, heads, dim = shape
    if dim != head_dim or heads % kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {kv_heads} heads of {head_dim}")
    start = _need_start(q_start, batch, tokens)
    w_ptr = w_cols = lse_ptr = 0
    if weights is not None:
        w_ptr, w_cols = _weights(weights, "weights", batch, kv_heads, cols)
        if lse is None:
            lse = _empty(stream, q, (tokens, heads), _F32)
    if lse is not None:
        lse_ptr = _array(lse, _F32, "lse", 2)
        if lse.shape != (tokens, heads):
            raise ValueError(f"lse must be [{tokens}, {heads}], got {tuple(lse.shape)}")
    if out is None:
        out = _another(stream, q)
        o_token, o_head = heads * dim, dim
    else:
        o_token, o_head = _heads(out, "out", like=q)
        if out.shape != shape:
            raise ValueError(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    a = _pack_attn(q.data_ptr(), out.data_ptr(), lse_ptr, w_ptr, start, q_token, q_head, o_token, o_head, w_cols,
                   dim ** -0.5 if scale is None else scale, tokens, heads,
                   max(1, tokens if max_q is None else int(max_q)) if start else 1, bool(causal), int(window),
                   _TYPE[q.dtype])
    _check(_lib().busfill_attn_kv4(c, a, _raw(stream, q)), "busfill_attn_kv4")
    return out


def attn_kv4_kernel(tokens: int, q_heads: int, kv_heads: int, head_dim: int, max_q: int) -> tuple:
    """(row tiles of a warp, or 0 for the kernel of many rows; whether the kernel of many rows sums the
    weights) of an :func:`attn_kv4` call of that shape (busfill_attn_kv4_kernel_for)."""
    n = _lib().busfill_attn_kv4_kernel_for(int(tokens), int(q_heads), int(kv_heads), int(head_dim), int(max_q))
    _check(min(n, 0), "busfill_attn_kv4_kernel_for")
    return (1, 2, 0)[n & 3], bool(n & 4)


def kv4_evict(pages, table, kv_len, weights, keep, recent, out_table=None, weights_out=None, stream=None):
    """Bring every sequence longer than ``keep`` down to ``keep`` tokens, head by head: the last
    ``recent`` stay, and of the others those with the largest accumulated weights (the lower slot of
    equals), in their order. ``out_table`` int32 [batch, cols] names the pages they move to (default:
    the same table, in place; then no page may be shared between sequences). Returns (index, weights_out, new kv_len): index int32 [batch,
    kv_heads, keep] holds the slots they came from (-1 behind a shorter sequence's)."""
    c, batch, heads, _, cols = _cache(pages, table, kv_len)
    w_ptr, w_cols = _weights(weights, "weights", batch, heads, cols)
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"need 1 <= keep and 0 <= recent <= keep, got keep {keep}, recent {recent}")
    out_table = table if out_table is None else out_table
    out_ptr = _array(out_table, _I32, "out_table", 2)
    rows, out_cols = out_table.shape
    if rows != batch or out_cols * KV4_PAGE < keep:
        raise ValueError(f"out_table must be [{batch}, >= {-(-keep // KV4_PAGE)}], got {tuple(out_table.shape)}")
    index = _empty(stream, kv_len, (batch, heads, keep), _I32)
    kv_len_out = _another(stream, kv_len)
    if weights_out is None:
        weights_out = _another(stream, weights)
        wo_ptr = weights_out.data_ptr()
    else:
        wo_ptr = _array(weights_out, _F32, "weights_out", 3)
        if weights_out.shape != weights.shape:
            raise ValueError(f"weights_out must be {tuple(weights.shape)}, got {tuple(weights_out.shape)}")
    e = _pack_eviction(w_ptr, wo_ptr, w_cols, index.data_ptr(), kv_len_out.data_ptr(), out_ptr, out_cols, keep, recent)
    _check(_lib().busfill_kv4_evict(c, e, _raw(stream, pages)), "busfill_kv4_evict")
    return index, weights_out, kv_len_out
