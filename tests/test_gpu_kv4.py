"""The 4-bit K/V cache, attention over it, rotary positions and eviction on the GPU against the
64-bit oracle. The pool starts as 0xFF bytes (every unused scale is a NaN), tables are scattered.

Tolerances, derived: the cache's values are exact, so append and read are compared for equality.
Rotary: two fp32 products and a sum, then one rounding. Attention: `_bounds` adds up the roundings
of the kernels (scores in fp32 block by block; p and p d in fp16; the output's own rounding)."""
import numpy as np
import pytest

import busfill_b200 as bf
from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu

UNIT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}     # half a step, relative
DEV = "cuda"


def _torch():
    import torch
    return torch


def _dt(name):
    torch = _torch()
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[name]


def _np(t):
    return t.detach().double().cpu().numpy()


class Batch:
    """Sequences of given lengths in a scattered cache, filled through kv4_append in one call."""

    def __init__(self, lens, heads, dim, dtype="fp16", seed=0, cols=None, spare=3, big=1.0):
        torch = _torch()
        rng = np.random.default_rng(seed)
        self.lens, self.heads, self.dim = list(lens), heads, dim
        pages = [-(-n // 64) for n in lens]
        self.cols = cols or max(1, max(pages))
        self.num_pages = sum(pages) + spare
        order = rng.permutation(self.num_pages)
        table = np.full((len(lens), self.cols), 1 << 20, np.int32)    # unused entries: out of range
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        self.table = torch.from_numpy(table).to(DEV)
        self.kv_len = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.pages = torch.full((self.num_pages, heads, 72 * dim), 0xFF, dtype=torch.uint8, device=DEV)
        total = sum(lens)
        gen = torch.Generator().manual_seed(seed)
        k = torch.randn((total, heads, dim), generator=gen) * (1 + 4 * (torch.rand((1, heads, dim), generator=gen) > 0.9))
        v = torch.randn((total, heads, dim), generator=gen) * big
        self.start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.k_in, self.v_in = k.to(_dt(dtype)).to(DEV), v.to(_dt(dtype)).to(DEV)
        if total:
            bf.kv4_append(self.pages, self.table, self.kv_len, self.k_in, self.v_in, q_start=self.starts(lens))
        self.k = orc.values(*orc.quantize(_np(self.k_in)))
        self.v = orc.values(*orc.quantize(_np(self.v_in)))

    def starts(self, n):
        torch = _torch()
        return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).to(DEV)

    def seq(self, i, h):
        a, b = self.start[i], self.start[i + 1]
        return self.k[a:b, h], self.v[a:b, h]


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim,heads,dtype,lens", [
    (64, 1, "fp16", [1]), (128, 8, "fp16", [65, 0, 64, 130]), (256, 3, "bf16", [200, 63]),
    (128, 2, "bf16", [1] * 70), (64, 5, "bf16", [129, 1, 0, 0, 300]),
])
def test_append_fills_pages_and_reads_back_exactly(dim, heads, dtype, lens):
    b = Batch(lens, heads, dim, dtype, seed=dim + heads)
    k, v = bf.kv4_read(b.pages, b.table, b.kv_len, b.starts(lens), sum(lens))
    assert np.array_equal(_np(k), b.k) and np.array_equal(_np(v), b.v)
    pages = b.pages.cpu().numpy()
    table = b.table.cpu().numpy()
    used = np.zeros((b.num_pages, heads, 64), bool)
    for i, n in enumerate(lens):
        for t in range(0, n, max(1, n // 7)):
            h = t % heads
            kk, vv = orc.get_token(pages[table[i, t // 64], h], t % 64, dim)
            assert np.array_equal(kk, b.seq(i, h)[0][t]) and np.array_equal(vv, b.seq(i, h)[1][t])
        for t in range(n):
            used[table[i, t // 64], :, t % 64] = True
    for pg in range(b.num_pages):      # unused pages are untouched
        if not used[pg].any():
            assert np.all(pages[pg] == 0xFF)
    assert bf.stream_status() == 0


def test_append_special_values_strides_and_ties():
    torch = _torch()
    heads, dim, n = 2, 128, 6
    fused = torch.randn((n, 3 * heads + 1, dim), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    fused[0, :, 5] = float("inf")
    fused[1, :, 7] = float("nan")
    fused[2, :, 40], fused[2, :, 41] = 9.0, -9.0
    fused[3] = 0
    fused[4] *= 2.0 ** -18
    fused[5, :, 3] = -65504.0
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:3 * heads]
    pages = bf.kv4_pool(1, heads, dim)
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([n + 3], dtype=torch.int32, device=DEV)
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    bf.kv4_append(pages, table, kv_len, k, v, q_start=start)
    kk, vv = bf.kv4_read(pages, table, kv_len, start, n)
    assert np.array_equal(_np(kk), orc.values(*orc.quantize(_np(k))))
    assert np.array_equal(_np(vv), orc.values(*orc.quantize(_np(v))))
    # rows that are not 16-byte aligned take the element loads
    odd = torch.empty(n * (2 * heads * dim + 1) + 1, dtype=torch.float16, device=DEV)[1:]
    odd = torch.as_strided(odd, (n, 2 * heads, dim), (2 * heads * dim + 1, dim, 1))
    odd.copy_(fused[:, :2 * heads])
    bf.kv4_append(pages, table, kv_len, odd[:, :heads], odd[:, heads:], q_start=start)
    kk, vv = bf.kv4_read(pages, table, kv_len, start, n)
    assert np.array_equal(_np(kk), orc.values(*orc.quantize(_np(fused[:, :heads]))))
    assert np.array_equal(_np(vv), orc.values(*orc.quantize(_np(fused[:, heads:2 * heads]))))
    assert bf.stream_status() == 0


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,axes,adjacent,dtype", [
    (1, 4, 1, 128, 128, 1, False, "fp16"), (37, 8, 8, 128, 112, 3, False, "bf16"), (300, 6, 2, 64, 64, 2, True, "fp16"),
    (5, 3, 1, 256, 48, 4, False, "fp16"), (9, 2, 1, 64, 34, 2, True, "bf16"), (9, 2, 1, 64, 34, 2, False, "fp16"),
    (4000, 16, 2, 128, 96, 3, True, "fp16"), (3, 2, 0, 80, 80, 1, False, "bf16"),
])
def test_rope(tokens, heads, kv, dim, rot, axes, adjacent, dtype):
    torch = _torch()
    gen = torch.Generator().manual_seed(tokens)
    qkv = torch.randn((tokens, heads + 2 * kv + 1, dim), generator=gen).to(_dt(dtype)).to(DEV)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv] if kv else None
    pos = torch.randint(0, 5000, (axes, tokens), generator=gen).int().to(DEV)
    cos, sin = bf.rope_table(5000, rot, base=1e6)
    axis = [(i * 7) % axes for i in range(rot // 2)]
    qo, ko = bf.rope_axes(q, k, pos, cos, sin, axis, adjacent=adjacent)
    c, s, u = _np(cos), _np(sin), UNIT[dtype]
    for x, y in ((q, qo), (k, ko)):
        if x is None:
            continue
        x = _np(x)
        ref = orc.rope(x, pos.cpu().numpy(), c, s, axis, adjacent)
        pair = np.abs(x[..., :rot]).max(-1, keepdims=True) * 2 if x.size else 0
        assert np.all(np.abs(_np(y) - ref) <= u * np.abs(ref) + 2.0 ** -23 * 2 * pair + 2.0 ** -25)
        assert np.array_equal(_np(y)[..., rot:], x[..., rot:])
    # in place, and back: the inverse of the rounded result is within its rounding
    back = qkv.clone()
    bq = back[:, :heads]
    bf.rope_axes(bq, None, pos, cos, sin, axis, adjacent=adjacent, q_out=bq)
    assert torch.equal(bq, qo) and torch.equal(back[:, heads:], qkv[:, heads:])
    bf.rope_axes(bq, None, pos, cos, sin, axis, adjacent=adjacent, inverse=True, q_out=bq)
    ref = orc.rope(_np(qo), pos.cpu().numpy(), c, s, axis, adjacent, inverse=True)
    assert np.all(np.abs(_np(bq) - ref) <= u * np.abs(ref) + 2.0 ** -20 * np.abs(_np(qo)).max() + 2.0 ** -25)
    assert bf.stream_status() == 0


def test_rope_inverse_is_the_gradient():
    """d/dx of <g, rope(x)> is rope^-1(g): against central differences of the 64-bit formula."""
    torch = _torch()
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((4, 2, 64), generator=gen).double().numpy()
    g = torch.randn((4, 2, 64), generator=gen).half()
    pos = torch.randint(0, 100, (2, 4), generator=gen).int().to(DEV)
    cos, sin = bf.rope_table(100, 64)
    axis = [i % 2 for i in range(32)]
    got, _ = bf.rope_axes(g.to(DEV), None, pos, cos, sin, axis, inverse=True)

    def f(y):
        return (orc.rope(y, pos.cpu().numpy(), _np(cos), _np(sin), axis) * g.double().numpy()).sum()

    rng = np.random.default_rng(0)
    for _ in range(40):
        at = tuple(rng.integers(0, d) for d in x.shape)
        e = np.zeros_like(x)
        e[at] = 0.5
        diff = f(x + e) - f(x - e)       # linear: exact up to fp64
        assert abs(_np(got)[at] - diff) <= 2.0 ** -11 * abs(diff) + 1e-5


def test_rope_position_out_of_range_is_nan_and_reported():
    torch = _torch()
    q = torch.ones((3, 1, 64), dtype=torch.float16, device=DEV)
    cos, sin = bf.rope_table(10, 32)
    pos = torch.tensor([[0, 10, -1]], dtype=torch.int32, device=DEV)
    out, _ = bf.rope_axes(q, None, pos, cos, sin)
    assert bf.stream_status_bits() == (-9, 256)
    assert bf.stream_status() == 0
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:, :, :32]).all() and (out[:, :, 32:] == 1).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _bounds(q, k, v, scale, p, lse, u):
    """Bounds of the output error, of the relative error of p, and of lse, for one head's rows."""
    blocks = np.abs(k).reshape(len(k), k.shape[1] // 32, 32).max(-1) / 7.0          # >= the block's scale
    size = np.abs(q).reshape(len(q), q.shape[1] // 32, 32).sum(-1) @ blocks.T       # sum over blocks of |d| sum |q|
    top = np.abs(q).max(-1, keepdims=True)
    # score: a block's sum starts at 8 sum|q| and adds 32 products up to 15 |q|: 34 roundings of at
    # most 2^-23 x 23 sum|q|; the cast of q / 16 below fp16's range (2^-31 of the row's maximum); the
    # blocks' sum and the factor (16 roundings of the score)
    ds = scale * size * (23 * 34 * 2.0 ** -23) + scale * top * 2.0 ** -26 * blocks.sum(-1)[None] * 32
    ds = ds + 16 * 2.0 ** -24 * scale * size * 8
    smax = ds.max(-1, keepdims=True) if ds.shape[1] else np.zeros((q.shape[0], 1))
    dp = 2 * smax + 2.0 ** -20                  # relative error of p: the score's, the sum's, exp2's
    # p d: two fp16 roundings, relative or, below fp16's normal range, 2^-24 of the largest p's scale;
    # codes weigh up to 8, sums in fp32
    n = k.shape[0]
    pmax = p.max(-1, keepdims=True, initial=0.0)
    vblock = np.repeat(np.abs(v).reshape(n, v.shape[1] // 32, 32).max(-1) / 7.0, 32, axis=-1) if n else v   # >= |d|
    sub = 2.0 ** -24 * 8 * 2 * pmax * (n + (vblock.sum(0)[None] if n else 0.0))
    # sum p d (c - 8) is the difference of sum p d c and 8 sum p d: fp32 sums of up to 15 p d
    out = (p @ np.abs(v)) * (2.0 ** -10 + dp) + (p @ vblock) * 32 * 2.0 ** -19 + sub
    return out, dp, smax[:, 0] + 2.0 ** -20 * (1 + np.abs(np.where(np.isfinite(lse), lse, 0.0)))


def _check(b, q, new, out, lse, weights, w0, causal, window, scale, dtype, sample=None):
    """Compare with the oracle, all heads or a sample of (sequence, kv head)."""
    group = q.shape[1] // b.heads
    qn, on, ln = _np(q), _np(out), None if lse is None else _np(lse)
    starts = np.concatenate([[0], np.cumsum(new)])
    pairs = [(i, h) for i in range(len(new)) for h in range(b.heads)]
    for i, h in (pairs if sample is None else sample):
        n, length = new[i], b.lens[i]
        k, v = b.seq(i, h)
        seen = orc.seen(n, length, causal, window)
        wsum, wtol = np.zeros(length), np.zeros(length)
        for g in range(group):
            rows = slice(starts[i], starts[i] + n)
            x = qn[rows, h * group + g]
            ref, rl, p = orc.attention(x, k, v, scale, seen)
            tol, dp, tl = _bounds(x, k, v, scale, p, rl, UNIT[dtype])
            err = np.abs(on[rows, h * group + g] - ref)
            assert np.all(err <= tol + UNIT[dtype] * (np.abs(ref) + tol) + 2.0 ** -25), (i, h, g, (err / (tol + 1e-30)).max())
            if ln is not None:
                got = ln[rows, h * group + g]
                assert np.array_equal(np.isneginf(got), np.isneginf(rl))
                fin = np.isfinite(rl)
                assert np.all(np.abs(got[fin] - rl[fin]) <= tl[fin])
            wsum += p.sum(0)
            wtol += (p * (2 * dp + 2.0 ** -20)).sum(0) if n else 0.0
        if weights is not None:
            base = _np(w0)[i, h]
            got = _np(weights)[i, h]
            lim = wtol + 2.0 ** -22 * (1 + group * n / 8) * (wsum + np.abs(base[:length]))
            assert np.all(np.abs(got[:length] - base[:length] - wsum) <= lim), (i, h)
            assert np.array_equal(got[length:], base[length:])


def _attend(lens, new, heads, kv, dim, dtype="fp16", causal=True, window=0, weights=True, seed=0, sample=None,
            qscale=1.0, **kw):
    torch = _torch()
    b = Batch(lens, kv, dim, "bf16" if seed % 2 else "fp16", seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    wide = torch.randn((sum(new), heads + 2, dim), generator=gen).mul(qscale).to(_dt(dtype)).to(DEV)
    q = wide[:, 1:heads + 1]                     # a strided view
    lse = torch.full((sum(new), heads), 7.0, device=DEV)
    w = torch.rand((len(lens), kv, 64 * b.cols), generator=gen).to(DEV) if weights else None
    w0 = w.clone() if weights else None
    out = torch.full((sum(new), heads, dim), float("nan"), dtype=q.dtype, device=DEV)
    scale = dim ** -0.5
    bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts(new), max_q=max(new), causal=causal, window=window,
                out=out, lse=lse, weights=w, **kw)
    assert bf.stream_status() == 0
    _check(b, q, new, out, lse, w, w0, causal, window, scale, dtype, sample)
    return b, q, out, lse, w


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_decode_lengths_that_end_anywhere_in_a_page(dim, dtype):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 200, 700]
    _attend(lens, [1] * len(lens), 8, 1, dim, dtype, seed=dim)


@pytest.mark.parametrize("group", [1, 3, 4, 8, 16])
@pytest.mark.parametrize("new", [1, 2, 5])
def test_groups_and_speculated_tokens(group, new):
    lens = [new, 70, 333]
    _attend(lens, [new] * 3, 2 * group, 2, 128, "fp16", seed=10 * group + new)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 50), (True, 200)])
def test_ragged_rows_masks_and_empty_rows(dim, causal, window):
    # no rows; rows but nothing cached; more rows than slots (the first see nothing); whole prompts
    lens = [40, 0, 5, 150, 0, 77, 200]
    new = [0, 3, 9, 150, 0, 1, 33]
    _attend(lens, new, 6, 2, dim, "bf16" if window else "fp16", causal, window, seed=window + dim)


@pytest.mark.parametrize("dim,group,new,length,window", [
    (128, 8, 300, 300, 0), (128, 8, 129, 1000, 0), (128, 1, 257, 700, 300), (64, 4, 200, 513, 0), (256, 2, 90, 400, 0),
    (128, 5, 64, 64, 0), (64, 16, 33, 2000, 100), (256, 7, 130, 130, 64),
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_prompts(dim, group, new, length, window, dtype):
    _attend([length, new, 3 * length // 4 + new], [new, new, new // 2 + 1], 2 * group, 2, dim, dtype, window=window,
            seed=new + (dtype == "bf16"))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 50), (True, 300)])
def test_prompts_ragged_masks_and_empty_rows(dim, causal, window):
    # the first case's masks, with rows enough for the kernel of many rows
    lens = [0, 300, 31, 190, 65, 400]
    new = [70, 0, 64, 190, 64, 20]
    _attend(lens, new, 12, 2, dim, "bf16" if window else "fp16", causal, window, seed=7 * window + dim)


@pytest.mark.parametrize("dim,new,lens,window", [
    (128, 100, [9000], 0), (128, 40, [5000, 300, 7000], 0), (64, 70, [12000], 3000), (256, 60, [4000, 4100], 0),
])
def test_rows_on_a_long_cache_are_split_and_joined(dim, new, lens, window):
    sample = [(0, 0), (len(lens) - 1, 1)]
    _attend(lens, [new] * len(lens), 8, 2, dim, "bf16", window=window, seed=dim + new, sample=sample)


def test_long_cache_is_split_and_joined():
    sample = [(0, 0), (0, 3), (1, 1)]
    _attend([70001, 33000], [1, 1], 32, 4, 128, "fp16", seed=4, sample=sample)
    _attend([20011, 64], [6, 1], 8, 2, 64, "bf16", seed=5, sample=[(0, 0), (1, 1)])


def test_many_short_sequences():
    rng = np.random.default_rng(0)
    lens = rng.integers(1, 140, 300).tolist()
    _attend(lens, [1] * 300, 16, 2, 128, "fp16", seed=6, sample=[(i, i % 2) for i in range(0, 300, 13)])


@pytest.mark.parametrize("new", [1, 70])
def test_a_window_longer_than_the_cache_is_none(new):
    b, q, out, lse, w = _attend([200, 90], [new] * 2, 16, 2, 128, "fp16", window=0, seed=30 + new)
    w2, w3 = _torch().zeros_like(w), _torch().zeros_like(w)
    y = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts([new] * 2), max_q=new, weights=w2)
    z = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts([new] * 2), max_q=new, weights=w3, window=2**31 - 1)
    t = _torch()
    assert t.equal(y, out) and t.equal(z, out) and t.equal(w2, w3) and float(w3.sum()) > 0.99 * new * 32


@pytest.mark.parametrize("qscale", [2.0 ** -12, 30.0, 3000.0])
def test_query_magnitudes(qscale):
    # tiny (all tokens nearly alike), sharp, and one-hot rows
    _attend([190, 64], [1, 3], 8, 2, 128, "bf16", seed=8, qscale=qscale)
    _attend([190, 64], [1, 30], 8, 2, 128, "fp16", seed=8, qscale=min(qscale, 30.0))


def test_results_repeat_and_ignore_the_stream_and_a_graph():
    torch = _torch()
    lens, new = [3000, 17, 640], [2, 1, 2]
    b, q, out, lse, w = _attend(lens, new, 16, 2, 128, "fp16", seed=20)
    q = q.contiguous()
    start = b.starts(new)
    again = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, max_q=2)
    assert torch.equal(again, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w1, w2 = torch.zeros_like(w), torch.zeros_like(w)
    one = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, max_q=2, weights=w1, stream=side)
    two = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, max_q=2, weights=w2, stream=side)
    assert bf.stream_status(side) == 0
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, out) and torch.equal(two, out) and torch.equal(w1, w2)
    # captured: the lengths are read when the graph runs
    graph_out = torch.zeros_like(q)
    kv_len = b.kv_len.clone()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            bf.attn_kv4(q, b.pages, b.table, kv_len, q_start=start, max_q=2, out=graph_out, stream=side)
        g.replay()
    side.synchronize()
    assert torch.equal(graph_out, out)
    kv_len.copy_(torch.tensor([2900, 17, 500], dtype=torch.int32))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        g.replay()
    side.synchronize()
    want = bf.attn_kv4(q, b.pages, b.table, kv_len, q_start=start, max_q=2)
    assert torch.equal(graph_out, want) and not torch.equal(want, out)


def test_decode_without_starts_equals_starts():
    torch = _torch()
    b = Batch([100, 260, 5], 2, 128, seed=3)
    q = torch.randn((3, 8, 128), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    x = bf.attn_kv4(q, b.pages, b.table, b.kv_len)
    y = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts([1, 1, 1]), max_q=1)
    assert torch.equal(x, y)
    k, v = bf.kv4_read(b.pages, b.table, b.kv_len)
    assert np.array_equal(_np(k), b.k[[99, 359, 364]])


def test_out_of_range_indices_are_reported_and_not_followed():
    torch = _torch()
    b = Batch([100, 60], 2, 128, seed=3)
    q = torch.randn((2, 4, 128), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    table = b.table.clone()
    table[0, 1] = b.num_pages
    out = bf.attn_kv4(q, b.pages, table, b.kv_len)
    assert bf.stream_status() == -9
    assert torch.equal(out[1], bf.attn_kv4(q, b.pages, b.table, b.kv_len)[1])
    bf.attn_kv4(q, b.pages, b.table, torch.tensor([100000, -5], dtype=torch.int32, device=DEV))
    assert bf.stream_status() == -9
    bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=torch.tensor([0, 5, 2], dtype=torch.int32, device=DEV), max_q=2)
    assert bf.stream_status() == -9
    before = b.pages.clone()
    kv = torch.randn((2, 2, 128)).half().to(DEV)
    bf.kv4_append(b.pages, table, torch.tensor([100, 0], dtype=torch.int32, device=DEV), kv, kv)
    assert bf.stream_status() == -9 and torch.equal(before, b.pages)
    ok = bf.attn_kv4(q, b.pages, b.table, b.kv_len)
    assert bf.stream_status() == 0 and torch.isfinite(ok).all()


def test_refusals():
    torch = _torch()
    b = Batch([10, 20], 2, 128)
    q = torch.zeros((2, 4, 128), dtype=torch.float16, device=DEV)
    args = (b.pages, b.table, b.kv_len)
    with pytest.raises(TypeError):
        bf.attn_kv4(q.float(), *args)
    with pytest.raises(TypeError):
        bf.attn_kv4(q.cpu(), *args)
    with pytest.raises(ValueError):
        bf.attn_kv4(q[:, :3], *args)
    with pytest.raises(ValueError):
        bf.attn_kv4(q[..., :64], *args)
    with pytest.raises(ValueError):
        bf.attn_kv4(q[:1], *args)
    with pytest.raises(ValueError):
        bf.attn_kv4(q, b.pages[..., :-1].contiguous(), b.table, b.kv_len)
    with pytest.raises(ValueError):
        bf.attn_kv4(q, *args, weights=torch.zeros((2, 2, 10), device=DEV))
    with pytest.raises(bf.BusfillError):
        bf.attn_kv4(q, *args, window=5, causal=False)
    with pytest.raises(TypeError):
        bf.kv4_append(*args, q[:, :2], q[:, :2].bfloat16())
    with pytest.raises(ValueError):
        bf.kv4_append(*args, q, q)
    with pytest.raises(ValueError):
        bf.kv4_evict(*args, torch.zeros((2, 2, 64), device=DEV), keep=4, recent=5)
    cos, sin = bf.rope_table(8, 64)
    with pytest.raises(ValueError):
        bf.rope_axes(q, None, torch.zeros((1, 2), dtype=torch.int32, device=DEV), cos, sin, axis=[1] * 32)
    with pytest.raises(TypeError):
        bf.rope_axes(q, None, torch.zeros((1, 2), dtype=torch.int64, device=DEV), cos, sin)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,keep,recent,kind", [
    ([200, 64, 3, 0, 65], 64, 10, "random"), ([1000, 999], 300, 0, "ties"), ([500], 129, 129, "random"),
    ([130, 700], 1, 0, "zeros"), ([5000, 2600], 2500, 100, "special"), ([50], 80, 5, "random"),
])
def test_evict(dim, in_place, lens, keep, recent, kind):
    torch = _torch()
    heads = 2
    need = sum(-(-min(n, keep) // 64) for n in lens)
    b = Batch(lens, heads, dim, seed=len(lens) + keep, cols=max(-(-max(lens) // 64), -(-keep // 64)), spare=need + 1)
    rng = np.random.default_rng(keep)
    shape = (len(lens), heads, 64 * b.cols + 5)
    w = {"random": lambda: rng.random(shape), "ties": lambda: rng.integers(0, 4, shape) / 2.0,
         "zeros": lambda: np.zeros(shape), "special": lambda: rng.standard_normal(shape) * 10.0 ** rng.integers(-40, 30, shape)}[kind]()
    w = w.astype(np.float32)
    if kind == "special":
        w[..., ::7], w[..., 1::11], w[..., 2::13], w[..., 3::17] = np.nan, -0.0, np.inf, -np.inf
    weights = torch.from_numpy(w).to(DEV)
    table = b.table
    if not in_place:
        t = np.zeros((len(lens), -(-keep // 64)), np.int32)
        at = 0
        for i, n in enumerate(lens):
            m = -(-min(n, keep) // 64)
            t[i, :m] = b.free[at:at + m]
            at += m
        table = torch.from_numpy(t).to(DEV)
    before = b.pages.clone()
    index, wout, kv_len = bf.kv4_evict(b.pages, b.table, b.kv_len, weights, keep, recent,
                                       out_table=None if in_place else table, weights_out=weights if in_place else None)
    assert bf.stream_status() == 0
    assert (wout is weights) == in_place
    new = [min(n, keep) for n in lens]
    assert kv_len.tolist() == new
    start = b.starts(new)
    k, v = bf.kv4_read(b.pages, table, kv_len, start, sum(new))
    k, v, index, wout = _np(k), _np(v), index.cpu().numpy(), wout.cpu().numpy()
    s = start.cpu().numpy()
    for i, n in enumerate(lens):
        for h in range(heads):
            stay = orc.kept(w[i, h], n, keep, recent)
            assert np.array_equal(index[i, h, :new[i]], stay) and np.all(index[i, h, new[i]:] == -1)
            assert np.array_equal(wout[i, h, :new[i]], w[i, h][stay], equal_nan=True) and np.all(wout[i, h, new[i]:] == 0)
            kk, vv = b.seq(i, h)
            assert np.array_equal(k[s[i]:s[i + 1], h], kk[stay]) and np.array_equal(v[s[i]:s[i + 1], h], vv[stay])
    if not in_place:   # the source pages are as they were
        used = torch.unique(b.table[b.table < b.num_pages]).long()
        assert torch.equal(before[used], b.pages[used])


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_of_sequences_beyond_shared_memory(in_place):
    torch = _torch()
    lens, keep, recent, heads, dim = [90000, 41000], 30001, 77, 1, 64
    need = sum(-(-min(n, keep) // 64) for n in lens)
    b = Batch(lens, heads, dim, seed=5, spare=need)
    gen = torch.Generator().manual_seed(5)
    weights = (torch.rand((2, heads, 64 * b.cols), generator=gen) * 1000).round().to(DEV)    # many equals
    w = weights.cpu().numpy().copy()
    table = b.table
    if not in_place:
        t = np.zeros((2, -(-keep // 64)), np.int32)
        t[:] = b.free[:t.size].reshape(t.shape)
        table = torch.from_numpy(t).to(DEV)
    index, wout, kv_len = bf.kv4_evict(b.pages, b.table, b.kv_len, weights, keep, recent,
                                       out_table=None if in_place else table, weights_out=weights if in_place else None)
    k, v = bf.kv4_read(b.pages, table, kv_len, b.starts([keep, keep]), 2 * keep)
    assert bf.stream_status() == 0 and kv_len.tolist() == [keep, keep]
    for i, n in enumerate(lens):
        stay = orc.kept(w[i, 0], n, keep, recent)
        assert np.array_equal(index[i, 0].cpu().numpy(), stay)
        assert np.array_equal(wout[i, 0, :keep].cpu().numpy(), w[i, 0][stay])
        kk, vv = b.seq(i, 0)
        assert np.array_equal(_np(k)[i * keep:(i + 1) * keep, 0], kk[stay])
        assert np.array_equal(_np(v)[i * keep:(i + 1) * keep, 0], vv[stay])


def test_weights_then_evict_then_attend_runs_a_sequence_under_budget():
    """Steps of append, attention with weights and eviction in place, against the oracle's own run."""
    torch = _torch()
    heads, group, dim, keep, recent = 2, 4, 128, 96, 32
    gen = torch.Generator().manual_seed(9)
    pages = torch.full((4, heads, 72 * dim), 0xFF, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    weights = torch.zeros((1, heads, 192), device=DEV)
    kv_len = torch.zeros(1, dtype=torch.int32, device=DEV)
    ks, vs = [np.zeros((0, dim)) for _ in range(heads)], [np.zeros((0, dim)) for _ in range(heads)]
    for n in (120, 1, 1, 30, 1, 50):
        k = torch.randn((n, heads, dim), generator=gen).half()
        v = torch.randn((n, heads, dim), generator=gen).half()
        q = torch.randn((n, heads * group, dim), generator=gen).half()
        kv_len += n
        start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        bf.kv4_append(pages, table, kv_len, k.to(DEV), v.to(DEV), q_start=start)
        out = bf.attn_kv4(q.to(DEV), pages, table, kv_len, q_start=start, max_q=n, weights=weights)
        for h in range(heads):
            ks[h] = np.concatenate([ks[h], orc.values(*orc.quantize(k[:, h].double().numpy()))])
            vs[h] = np.concatenate([vs[h], orc.values(*orc.quantize(v[:, h].double().numpy()))])
            for g in range(group):
                x = q[:, h * group + g].double().numpy()
                ref, rl, p = orc.attention(x, ks[h], vs[h], dim ** -0.5, orc.seen(n, len(ks[h])))
                tol, _, _ = _bounds(x, ks[h], vs[h], dim ** -0.5, p, rl, UNIT["fp16"])
                err = np.abs(_np(out)[:, h * group + g] - ref)
                assert np.all(err <= tol + 2.0 ** -11 * (np.abs(ref) + tol))
        index, weights, kv_len = bf.kv4_evict(pages, table, kv_len, weights, keep, recent)
        stay = index.cpu().numpy()[0]
        for h in range(heads):
            at = stay[h][stay[h] >= 0]
            ks[h], vs[h] = ks[h][at], vs[h][at]
    assert bf.stream_status() == 0
