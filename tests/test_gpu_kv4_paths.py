"""Forms of the attention kernels that ordinary calls do not reach: queries of any magnitude, scales of
any sign, outputs that do not start on 32 bytes, rows that are not finite, two row tiles. Each case
states the kernel that it is there for; the tolerances are those of test_gpu_kv4."""
import numpy as np
import pytest

import busfill_b200 as bf
from oracle import kv4_oracle as orc
from test_gpu_kv4 import DEV, UNIT, Batch, _attend, _check, _dt, _np

pytestmark = pytest.mark.gpu


def _kernel(new, heads, kv, dim):
    return bf.attn_kv4_kernel(sum(new), heads, kv, dim, max(new))


# lens, new, query heads, key/value heads, dim -> row tiles (0: many rows), weights of many rows
FEW = ([190, 64, 700], [1, 3, 2], 8, 2)
MANY = ([300, 190, 700], [100, 3, 90], 16, 2)


def _shape(many, dim):
    lens, new, heads, kv = MANY if many else FEW
    assert _kernel(new, heads, kv, dim) == ((0, True) if many else (1, False))
    return lens, new, heads, kv


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype,scale,qscale", [("fp16", -0.11, 1.0), ("bf16", -0.11, 1.0), ("fp16", 0.0, 1.0), ("bf16", 0.0, 1.0),
                                                ("bf16", 0.0, 2.0 ** -60), ("bf16", 2.0 ** -70, 2.0 ** -60),
                                                ("bf16", 2.0 ** 57, 2.0 ** -60)])
def test_scales_of_any_sign_and_size(dim, many, dtype, scale, qscale):
    import torch
    lens, new, heads, kv = _shape(many, dim)
    b = Batch(lens, kv, dim, seed=3)
    gen = torch.Generator().manual_seed(4)
    q = torch.randn((sum(new), heads, dim), generator=gen).mul(qscale).to(_dt(dtype)).to(DEV)
    lse = torch.zeros((sum(new), heads), device=DEV)
    w = torch.zeros((len(lens), kv, 64 * b.cols), device=DEV)
    out = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts(new), max_q=max(new), scale=scale, lse=lse, weights=w)
    assert bf.stream_status() == 0
    # a negative scale is the negated queries'
    _check(b, -q if scale < 0 else q, new, out, lse, w, torch.zeros_like(w), True, 0, abs(scale), dtype)
