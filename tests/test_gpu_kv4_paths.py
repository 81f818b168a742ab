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
@pytest.mark.parametrize("dtype,qscale", [("bf16", 2.0 ** -100), ("bf16", 2.0 ** -12), ("bf16", 3000.0), ("fp16", 2.0 ** -12),
                                          ("fp16", 30.0)])
def test_prompt_query_magnitudes(dim, dtype, qscale):
    lens, new, heads, kv = _shape(True, dim)
    _attend(lens, new, heads, kv, dim, dtype, seed=8, qscale=qscale)


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


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_outputs_on_sixteen_bytes(dim, many, dtype):
    """Rows of dim + 8 elements and an odd start: 16-byte aligned, not 32."""
    import torch
    lens, new, heads, kv = _shape(many, dim)
    lens, new = [*lens, 9000], [*new, new[0]]        # and an item that is cut and joined
    b = Batch(lens, kv, dim, seed=5)
    gen = torch.Generator().manual_seed(6)
    q = torch.randn((sum(new), heads, dim), generator=gen).to(_dt(dtype)).to(DEV)
    wide = torch.full((sum(new) * heads * (dim + 8) + 8,), 9.0, dtype=q.dtype, device=DEV)
    out = torch.as_strided(wide, (sum(new), heads, dim), (heads * (dim + 8), dim + 8, 1), 8)
    assert out.data_ptr() % 32 == 16
    lse = torch.zeros((sum(new), heads), device=DEV)
    bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts(new), max_q=max(new), out=out, lse=lse)
    assert bf.stream_status() == 0
    plain = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=b.starts(new), max_q=max(new))
    assert torch.equal(out, plain)
    gaps = torch.as_strided(wide, (sum(new) * heads, 8), (dim + 8, 1), 0)
    assert bool((gaps == 9.0).all())
    _check(b, q, new, out, lse, None, None, True, 0, dim ** -0.5, dtype, sample=[(0, 0), (2, 1), (3, 1)])


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 90)])
@pytest.mark.parametrize("new", [[7, 7, 7], [8, 1, 14], [9, 0, 13]])
def test_two_row_tiles(causal, window, new):
    lens, heads, kv, dim = [500, 77, 64 * 90 + 5], 32, 8, 64
    assert _kernel(new, heads, kv, dim)[0] == 2
    _attend(lens, new, heads, kv, dim, "bf16" if window else "fp16", causal, window, seed=window + new[0])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_that_are_not_finite_stay_alone(dim, many, dtype):
    import torch
    lens, new, heads, kv = _shape(many, dim)
    b = Batch(lens, kv, dim, seed=7)
    gen = torch.Generator().manual_seed(8)
    q = torch.randn((sum(new), heads, dim), generator=gen).to(_dt(dtype)).to(DEV)
    args = (b.pages, b.table, b.kv_len)
    kw = dict(q_start=b.starts(new), max_q=max(new))
    lse, w = torch.zeros((sum(new), heads), device=DEV), torch.zeros((3, kv, 64 * b.cols), device=DEV)
    want = bf.attn_kv4(q, *args, **kw, lse=lse, weights=w)
    bad = q.clone()
    bad[0, 1, 3] = float("nan")
    bad[new[0], 0, dim - 1] = float("inf")
    bad[new[0] + 1, heads - 1, :] = float("-inf")
    lse2, w2 = torch.zeros_like(lse), torch.zeros_like(w)
    out = bf.attn_kv4(bad, *args, **kw, lse=lse2, weights=w2)
    assert bf.stream_status() == 0
    whole = torch.ones((sum(new), heads), dtype=torch.bool, device=DEV)
    whole[0, 1] = whole[new[0], 0] = whole[new[0] + 1, heads - 1] = False
    assert torch.equal(out[whole], want[whole]) and torch.equal(lse[whole], lse2[whole])
    assert not bool(torch.isfinite(out[~whole]).any()) and bool(torch.isnan(lse2[0, 1]))
    assert torch.equal(w[2], w2[2])                  # sequences without such a row
    assert bool(torch.isnan(w2[0, 0, :lens[0] - new[0] + 1]).all())
    assert torch.equal(w[0, 1], w2[0, 1])            # and heads without one


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,rot,pad", [(128, 96, 0), (64, 64, 3), (80, 34, 8)])
def test_rope_into_strided_outputs(adjacent, dim, rot, pad):
    """Queries and keys turned into slices of wider tensors, and a key output in place."""
    import torch
    tokens, heads, kv = 33, 6, 2
    gen = torch.Generator().manual_seed(dim)
    q, k = (torch.randn((tokens, h, dim), generator=gen).half().to(DEV) for h in (heads, kv))
    pos = torch.randint(0, 900, (2, tokens), generator=gen).int().to(DEV)
    cos, sin = bf.rope_table(900, rot)
    axis = [i % 2 for i in range(rot // 2)]
    want = [orc.rope(_np(x), pos.cpu().numpy(), _np(cos), _np(sin), axis, adjacent) for x in (q, k)]
    pair = [np.abs(_np(x)).max(-1, keepdims=True) * 2 for x in (q, k)]

    def close(y, i):
        return np.all(np.abs(_np(y) - want[i]) <= UNIT["fp16"] * np.abs(want[i]) + 2.0 ** -22 * pair[i] + 2.0 ** -25)

    wide = torch.full((tokens, heads + kv + 1, dim + pad), 7.0, dtype=torch.float16, device=DEV)
    qo, ko = wide[:, :heads, :dim], wide[:, heads + 1:, :dim]
    got = bf.rope_axes(q, k, pos, cos, sin, axis, adjacent=adjacent, q_out=qo, k_out=ko)
    assert got[0] is qo and got[1] is ko and close(qo, 0) and close(ko, 1)
    assert bool((wide[:, heads] == 7.0).all()) and bool((wide[..., dim:] == 7.0).all())
    bf.rope_axes(q, k, pos, cos, sin, axis, adjacent=adjacent, q_out=qo, k_out=k)
    assert torch.equal(k, ko) and bf.stream_status() == 0
