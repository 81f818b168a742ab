"""The example layer (examples/decode_layer.py) against the same layer in torch and the oracle: Q4_K
projections on dequantized weights, rotary positions, the quantized cache, attention and eviction."""
import importlib.util
import os

import numpy as np
import pytest

import busfill_b200 as bf
from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("decode_layer", os.path.join(ROOT, "examples", "decode_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_lengths_stay_under_the_budget_and_runs_repeat():
    import torch
    ex = _example()
    x, lengths, layer = ex.run(steps=40, budget=64, prompts=(150, 40))
    assert lengths[0] == [65, 41] and lengths[15] == [80, 56] and lengths[16] == [65, 57] and lengths[39] == [72, 72]
    assert torch.isfinite(x).all()
    again, _, _ = ex.run(steps=40, budget=64, prompts=(150, 40))
    assert torch.equal(x, again)


def test_first_tokens_match_the_layer_in_torch():
    """A prompt without eviction: every stage from the kernels' own previous stage, so that each
    comparison has one operator in it."""
    import torch
    ex = _example()
    dev = torch.device("cuda")
    n = 37
    layer = ex.Layer(1, 64, dev, seed=3)
    x = torch.randn((n, ex.HIDDEN), generator=torch.Generator().manual_seed(4)).half().to(dev)
    pos = ex.image_positions(n, dev)
    y = layer(x, pos, [n])
    assert bf.stream_status() == 0
    h = torch.nn.functional.rms_norm(x.float(), (ex.HIDDEN,)).half()
    qkv = bf.gemm_q4k(layer.w_qkv, h).view(n, -1, ex.DIM)
    w = bf.dequant_q4k(layer.w_qkv, ex.HIDDEN)
    ref = h.double() @ w.double().t()
    assert (qkv.view(n, -1).double() - ref).norm() <= 1e-3 * ref.norm()
    c, s = layer.cos.double().cpu().numpy(), layer.sin.double().cpu().numpy()
    p = pos.cpu().numpy()
    q = orc.rope(qkv[:, :64].double().cpu().numpy(), p, c, s, layer.axis).astype(np.float16).astype(np.float64)
    k = orc.rope(qkv[:, 64:72].double().cpu().numpy(), p, c, s, layer.axis).astype(np.float16).astype(np.float64)
    k = orc.values(*orc.quantize(k))
    v = orc.values(*orc.quantize(qkv[:, 72:].double().cpu().numpy()))
    o = np.zeros((n, 64, 128))
    for g in range(64):
        o[:, g], _, _ = orc.attention(q[:, g], k[:, g // 8], v[:, g // 8], 128 ** -0.5, orc.seen(n, n))
    wo = bf.dequant_q4k(layer.w_o, 64 * 128).double().cpu().numpy()
    want = x.double().cpu().numpy() + o.reshape(n, -1) @ wo.T
    # fp16 rounding of q and k can move a code by a step (1/8 of its block's largest value)
    err = np.linalg.norm(y.double().cpu().numpy() - want) / np.linalg.norm(want - x.double().cpu().numpy())
    assert err <= 5e-3, err
