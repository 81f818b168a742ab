"""The cache oracle against the format's own claims, on the CPU, and the bit tricks that the
kernels build on: exact fp16 products, the code's fp16 subnormal, the tile orders."""
import ctypes

import numpy as np
import pytest

import busfill_b200 as bf
from busfill_b200 import kv4
from oracle import kv4_oracle as orc


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_round_trip_uses_every_byte_once(dim):
    rng = np.random.default_rng(dim)
    page = np.zeros(72 * dim, np.uint8)
    k = rng.standard_normal((64, dim)) * 3
    v = rng.standard_normal((64, dim))
    for t in range(64):
        orc.put_token(page, t, k[t], v[t])
    for t in range(64):
        kk, vv = orc.get_token(page, t, dim)
        assert np.array_equal(kk, orc.values(*orc.quantize(k[t])))
        assert np.array_equal(vv, orc.values(*orc.quantize(v[t])))


def test_quantize_edges():
    x = np.zeros((8, 32))
    x[1] = 1e6                                  # saturates
    x[2, 3], x[2, 9] = np.inf, -1.0
    x[3, 5] = np.nan
    x[4, 4], x[4, 8] = 2.0, -2.0                # equals: the first decides the sign of the scale
    x[5, 4], x[5, 8] = -2.0, 2.0
    x[6] = np.arange(32) - 16.0
    x[7, 0] = 2.0 ** -20
    c, d = orc.quantize(x)
    v = orc.values(c, d[..., :])
    assert np.all(c[0] == 8) and d[0] == 0
    assert np.all(v[1] == 7168.0) and np.all(np.abs(v) <= 7168.0)
    assert v[2, 3] == 7168.0 and np.all(v[3] == 0)
    assert d[4, 0] == -0.25 and d[5, 0] == 0.25
    assert v[4, 4] == 2.0 and v[4, 8] == -1.75
    assert np.array_equal(v[6], np.minimum(np.floor(x[6] / 2.0 + 0.5) * 2.0, 14.0))   # codes end at +7


def test_code_times_scale_is_exact_in_fp16():
    # every scale of 7 significant bits up to 896: (64 + c) d - 72 d has one rounding, and 72 d and
    # (c - 8) d need none
    m = np.arange(64, 128)
    for e in range(-24 - 6, 4):
        d = np.ldexp(m.astype(np.float64), e)
        d = d[(d <= 896) & (d == d.astype(np.float16))]
        for c in range(16):
            for x in (72 * d, (c - 8) * d):
                assert np.array_equal(x, x.astype(np.float16).astype(np.float64))


def test_code_bits_are_subnormals():
    c = np.arange(16, dtype=np.uint16)
    assert np.array_equal(c.view(np.float16).astype(np.float64), c * 2.0 ** -24)
    assert np.array_equal((c << 4).view(np.float16).astype(np.float64), c * 2.0 ** -20)
    assert np.array_equal((c << 4 | 0x5400).view(np.float16).astype(np.float64), 64.0 + c)


@pytest.mark.parametrize("dim", [128, 256])
def test_value_words_of_one_load_lie_on_different_banks(dim):
    """A load's lanes (c, j) of one phase read the words of 4 tokens: no two on one bank."""
    n = dim // 32
    for rows in ([0, 2, 4, 6], [1, 3, 5, 7]):
        tokens = [r ^ (r >> 1 & 1) for r in rows]
        lanes = [(c, t) for c in range(8) for t in tokens]
        per = 32 * 4 // (2 * n)                 # lanes of a 128-byte phase
        for at in range(0, 32, per):
            banks = set()
            for c, t in lanes[at:at + per]:
                swz = 4 * (t >> 2 & 1) if dim == 128 else 2 * (t >> 1 & 3)
                byte = t * dim // 2 + (c ^ swz) * 2 * n
                banks |= {byte // 4 % 32 + i for i in range(2 * n // 4)}
            assert len(banks) == 32


def test_null_and_bad_arguments_are_refused_before_any_device_work():
    lib = bf.load_library()
    assert lib.busfill_kv4_page_bytes(128) == 9216 and lib.busfill_kv4_page_bytes(96) == -2
    assert lib.busfill_rope_axes(None, None) == -1
    assert lib.busfill_kv4_append(None, None, None) == -1
    assert lib.busfill_kv4_read(None, None, 1, None, None, None) == -1
    assert lib.busfill_attn_kv4(None, None, None) == -1
    assert lib.busfill_kv4_evict(None, None, None) == -1

    def cache(**kw):
        args = dict(pages=4096, table=4096, kv_len=8192, num_pages=4, table_cols=2, batch=2, heads=2, head_dim=128)
        args.update(kw)
        return kv4.Cache(**args)

    def attn(c=None, **kw):
        args = dict(q=4096, out=4096, q_token=512, q_head=128, out_token=512, out_head=128, scale=1.0, tokens=2,
                    q_heads=4, max_q=1, causal=1, window=0, dtype=1)
        args.update(kw)
        return lib.busfill_attn_kv4(ctypes.byref(c or cache()), ctypes.byref(kv4.Attn(**args)), None)

    assert attn(cache(head_dim=96)) == -2 and attn(cache(batch=0)) == -2 and attn(cache(batch=1025)) == -2
    assert attn(cache(pages=4100)) == -3 and attn(cache(table=None)) == -1
    assert attn(q=None) == -1 and attn(dtype=0) == -1 and attn(window=-1) == -1 and attn(window=4, causal=0) == -1
    assert attn(weights=4096) == -1                                     # weights need lse
    assert attn(weights=4096, lse=4096, weights_cols=127) == -2
    assert attn(q_heads=3) == -2 and attn(tokens=3) == -2 and attn(max_q=0) == -2
    assert attn(q=4104) == -3 and attn(q_head=132) == -3

    def append(**kw):
        args = dict(k=4096, v=4096, tokens=2, dtype=30)
        args.update(kw)
        return lib.busfill_kv4_append(ctypes.byref(cache()), ctypes.byref(kv4.Rows(**args)), None)

    assert append(k=None) == -1 and append(dtype=2) == -1 and append(tokens=5) == -2 and append(v=4097) == -3

    def evict(**kw):
        args = dict(weights=4096, weights_out=4096, weights_cols=128, index=4096, kv_len_out=4096, out_table=4096,
                    out_cols=2, keep=64, recent=8)
        args.update(kw)
        return lib.busfill_kv4_evict(ctypes.byref(cache()), ctypes.byref(kv4.Eviction(**args)), None)

    assert evict(index=None) == -1 and evict(kv_len_out=8192) == -1
    assert evict(keep=0) == -2 and evict(recent=65) == -2 and evict(weights_cols=100) == -2 and evict(keep=129) == -2
    assert evict(out_cols=3) == -2                                      # in place: the same shape
    assert evict(weights=4098) == -3

    def rope(axis=(0, 0), **kw):
        table = (ctypes.c_uint8 * 2)(*axis)
        args = dict(q=4096, q_out=4096, positions=4096, cos=4096, sin=4096, axis=ctypes.addressof(table), tokens=1,
                    q_heads=1, head_dim=8, rot=4, axes=1, max_pos=1, dtype=1)
        args.update(kw)
        return lib.busfill_rope_axes(ctypes.byref(kv4.Rope(**args)), None)

    assert rope(cos=None) == -1 and rope(axis=(0, 1)) == -1 and rope(k_heads=1) == -1 and rope(dtype=3) == -1
    assert rope(rot=3) == -2 and rope(rot=10) == -2 and rope(axes=5) == -2 and rope(max_pos=0) == -2
    assert rope(q=4097) == -3


def test_kept_slots():
    w = np.array([5.0, 1.0, 5.0, np.nan, 0.0, -0.0, 7.0, 2.0])
    assert orc.kept(w, 8, 4, 2).tolist() == [0, 2, 6, 7]
    assert orc.kept(w, 8, 4, 0).tolist() == [0, 2, 6, 7]
    assert orc.kept(w, 6, 5, 0).tolist() == [0, 1, 2, 4, 5]
    assert orc.kept(w, 3, 8, 2).tolist() == [0, 1, 2]
    assert orc.kept(w, 8, 2, 2).tolist() == [6, 7]
