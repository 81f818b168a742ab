"""Attention over the 4-bit cache at any magnitude of the values, with a token that most rows look
at (a sink) and with the rest of the weight spread over a long cache, against the 64-bit oracle.
Batches are wide (sequences that share their pages), so that one warp sees a sink and thousands of
tokens behind it.

Tolerance, derived: every product p v carries a few relative roundings that differ from token to
token: p to fp16 and (single rows) p d to fp16 again, at most 2^-11 each, and the error of the
score. Over the tokens they add up like the root of the sum of squares, and all of it scales with
the values; then the output's own rounding. Nothing in it depends on the number of tokens alone."""
import numpy as np
import pytest

import busfill_b200 as bf
from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu

DEV = "cuda"
HEADS = 8          # query heads of the one key/value head


def _sequence(n, dim, rows, sink, vexp, seed, spikes=0, empty_sink=False):
    """One cached sequence whose token 0 scores about `sink` above the others for every row.
    Returns (q, pages, table, kv_len, k, v): k, v are the cached values in 64 bits."""
    import torch
    gen = torch.Generator().manual_seed(seed)
    base = torch.randn((1, 1, dim), generator=gen)
    q = (base + 0.2 * torch.randn((rows, HEADS, dim), generator=gen)).half()
    k = torch.randn((n, 1, dim), generator=gen)
    k[0] = base[0] * (sink / dim ** 0.5)
    v = torch.randn((n, 1, dim), generator=gen) * 2.0 ** vexp
    if empty_sink:
        v[0] = 0
    for i in range(spikes):        # tokens of much larger values that no row looks at
        k[7 + 13 * i], v[7 + 13 * i] = -base[0], v[7 + 13 * i] * 2.0 ** 12
    k, v = k.half(), v.half()
    cols = -(-n // 64)
    pages = torch.full((cols + 1, 1, 72 * dim), 0xFF, dtype=torch.uint8, device=DEV)
    table = torch.randperm(cols + 1, generator=gen)[:cols].int().view(1, cols).to(DEV)
    kv_len = torch.tensor([n], dtype=torch.int32, device=DEV)
    bf.kv4_append(pages, table, kv_len, k.to(DEV), v.to(DEV),
                  q_start=torch.tensor([0, n], dtype=torch.int32, device=DEV))
    return q, pages, table, kv_len, *(orc.values(*orc.quantize(t[:, 0].double().numpy())) for t in (k, v))


def _check(q, out, k, v, causal):
    """Every row and head: the norm of the error against the bound above."""
    rows, heads, dim = q.shape
    x, o = q.double().numpy(), out.double().cpu().numpy()
    blocks = np.abs(k).reshape(len(k), dim // 32, 32).max(-1) / 7.0
    scale, seen = dim ** -0.5, orc.seen(rows, len(k), causal)
    for h in range(heads):
        ref, _, p = orc.attention(x[:, h], k, v, scale, seen)
        size = np.abs(x[:, h]).reshape(rows, dim // 32, 32).sum(-1) @ blocks.T
        ds = scale * size.max(-1) * (23 * 34 + 64) * 2.0 ** -23       # fp32 sums of a block's 32 products
        spread = np.sqrt((p * p) @ (v * v).sum(-1))                   # root of the sum of (p |v|)^2
        bound = spread * (2.0 ** -10 + 2 * ds) + np.linalg.norm(ref, axis=-1) * 2.0 ** -11
        bound = bound + np.abs(p @ v).sum(-1) * 2.0 ** -19 + dim ** 0.5 * 2.0 ** -25
        err = np.linalg.norm(o[:, h] - ref, axis=-1)
        assert np.all(err <= bound), (h, (err / bound).max(), (err / np.linalg.norm(ref, axis=-1)).max())


def _wide(q, table, kv_len, batch):
    """The same rows for `batch` sequences over the same pages: (q, table, kv_len, q_start)."""
    import torch
    rows = q.shape[0]
    return (q.repeat(batch, 1, 1).to(DEV), table.expand(batch, -1).contiguous(), kv_len.repeat(batch),
            torch.arange(0, batch * rows + 1, rows, dtype=torch.int32, device=DEV))


def _check_wide(q, out, k, v, causal, batch):
    """All sequences of _wide; the oracle's work is done once."""
    rows = q.shape[0]
    o = out.view(batch, rows, HEADS, -1)
    first = o[0].double()
    far = (o.double() - first).norm(dim=-1).flatten(1).amax(1).argmax()    # the one farthest from the first
    for i in {0, int(far), batch // 2, batch - 1}:
        _check(q, o[i], k, v, causal)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,batch,sink,vexp", [(16000, 900, 8, -6), (16000, 900, 8, -10), (16000, 900, 8, -13),
                                               (131071, 700, 10, -8), (700, 5, 0, -14), (16000, 900, 8, 0),
                                               (16000, 900, 8, 9)])
def test_single_rows_follow_the_values_magnitude(dim, n, batch, sink, vexp):
    q, pages, table, kv_len, k, v = _sequence(n, dim, 1, sink, vexp, seed=dim + n - vexp)
    wide, table, kv_len, _ = _wide(q, table, kv_len, batch)
    out = bf.attn_kv4(wide, pages, table, kv_len)
    assert bf.stream_status() == 0
    _check_wide(q, out, k, v, True, batch)


@pytest.mark.parametrize("dim,rows", [(64, 1), (64, 4), (128, 1), (256, 2)])
def test_unseen_large_values_take_nothing_from_small_ones(dim, rows):
    # heads of 64, 4 rows of 8 heads: the kernel's form of two row tiles
    q, pages, table, kv_len, k, v = _sequence(5000, dim, rows, 9, -3, seed=dim, spikes=40)
    wide, table, kv_len, start = _wide(q, table, kv_len, 500)
    out = bf.attn_kv4(wide, pages, table, kv_len, q_start=start, max_q=rows)
    assert bf.stream_status() == 0
    _check_wide(q, out, k, v, True, 500)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,n,causal", [(100, 6000, True), (330, 1000, False), (1, 6000, True), (4, 6000, True)])
def test_rows_keep_what_lies_far_below_a_sink_without_value(dim, rows, n, causal):
    """The sink takes all but e^-14 of every weight and has no value: the output is the other
    tokens', whose weights are 2^-20 of the largest. 100 rows of 8 heads take the kernel of many rows."""
    q, pages, table, kv_len, k, v = _sequence(n, dim, rows, 14, 8, seed=dim + rows, empty_sink=True)
    wide, table, kv_len, start = _wide(q, table, kv_len, 100 if rows < 8 else 3)
    out = bf.attn_kv4(wide, pages, table, kv_len, q_start=start, max_q=rows, causal=causal)
    assert bf.stream_status() == 0
    _check_wide(q, out, k, v, causal, 100 if rows < 8 else 3)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 100])
def test_products_are_rounded_once(dim, rows):
    """Where the sum of p v nearly cancels, the output's own rounding is small and the rms error against
    the root of the sum of (p v)^2 is that of p v's roundings. One to fp16, of log-uniform mantissas m
    in [1, 2): 2^-10 / sqrt(12) * sqrt(E[1 / m^2]) with E = 3 / (8 ln 2), 2.07e-4; two: sqrt(2) more."""
    import torch
    n, batch = 400, 600 // rows
    one = 2.0 ** -10 / 12 ** 0.5 * (3 / (8 * np.log(2))) ** 0.5
    _, pages, table, kv_len, k, v = _sequence(n, dim, 1, 1, 0, seed=dim + rows)
    q = torch.randn((batch * rows, HEADS, dim), generator=torch.Generator().manual_seed(rows)).half()
    _, table, kv_len, start = _wide(q[:rows], table, kv_len, batch)
    out = bf.attn_kv4(q.to(DEV), pages, table, kv_len, q_start=start, max_q=rows, causal=False).double().cpu().numpy()
    assert bf.stream_status() == 0
    x = q.double().numpy().reshape(-1, dim)
    ref, _, p = orc.attention(x, k, v, dim ** -0.5, orc.seen(len(x), n, False))
    spread = np.sqrt((p * p) @ (v * v))
    near = np.abs(ref) < spread / 16
    assert near.sum() > 5000
    rms = np.sqrt(np.mean(((out.reshape(-1, dim) - ref) / spread)[near] ** 2))
    assert 0.5 * one < rms < 1.2 * one, rms / one
