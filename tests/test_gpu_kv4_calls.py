"""Calls that a server makes of the cache operators besides the plain ones: pages given back, padded
batches, empty steps, captured steps, and calls that are refused on the device."""
import numpy as np
import pytest

import busfill_b200 as bf
from test_gpu_kv4 import DEV, Batch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype="float16"):
    import torch
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(getattr(torch, dtype)).to(DEV)


# ---------------------------------------------------------------------------
# pages before every row's window may have been given back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 6, 70, 200])
def test_pages_before_the_window_are_not_looked_up(dim, new):
    import torch
    lens, window, heads = [64 * 9 + new, 1000, 64 * 5 + 30 + new], 50, 12
    b = Batch(lens, 2, dim, seed=dim + new)
    # page 0 belongs to nobody and holds NaN scales
    pages = torch.cat([torch.full_like(b.pages[:1], 0xFF), b.pages])
    table = torch.where(b.table < b.num_pages, b.table + 1, b.table)
    gone = table.clone()
    for i, n in enumerate(lens):
        first = max(0, n - new + 1 - window) // 64
        assert first > 0
        gone[i, :first] = torch.tensor([-1, b.num_pages + 1], dtype=torch.int32, device=DEV).repeat(first)[:first]
    q, start = _rand((3 * new, heads, dim), 1), b.starts([new] * 3)
    results = []
    for t in (table, gone):
        lse = torch.zeros((3 * new, heads), device=DEV)
        weights = torch.zeros((3, 2, 64 * b.cols), device=DEV)
        out = bf.attn_kv4(q, pages, t, b.kv_len, q_start=start, max_q=new, window=window, lse=lse, weights=weights)
        assert bf.stream_status() == 0
        results.append((out, lse, weights))
    assert torch.isfinite(results[0][0]).all()
    for x, y in zip(*results):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------
# steps without tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_steps_of_no_tokens_do_nothing(dtype):
    import torch
    b = Batch([70, 5], 2, 128, seed=2)
    pages, start = b.pages.clone(), b.starts([0, 0])
    cache = (b.pages, b.table, b.kv_len)
    q, k = _rand((0, 8, 128), 0, dtype), _rand((0, 2, 128), 0, dtype)
    cos, sin = bf.rope_table(16, 128)
    qo, ko = bf.rope_axes(q, k, torch.zeros((3, 0), dtype=torch.int32, device=DEV), cos, sin, [i % 3 for i in range(64)])
    assert qo.shape == q.shape and ko.shape == k.shape
    bf.kv4_append(*cache, k, k, q_start=start)
    kk, vv = bf.kv4_read(*cache, q_start=start, tokens=0)
    assert kk.shape == vv.shape == (0, 2, 128)
    weights = torch.rand((2, 2, 64 * b.cols), device=DEV)
    before = weights.clone()
    assert bf.attn_kv4(q, *cache, q_start=start, weights=weights).shape == q.shape
    assert torch.equal(weights, before) and torch.equal(b.pages, pages) and bf.stream_status() == 0


@pytest.mark.parametrize("new", [(0, 0, 1), (0, 90, 0)])
def test_steps_of_some_sequences_leave_the_others_alone(new):
    import torch
    b = Batch([70, 100, 5], 2, 128, seed=2)
    q, start = _rand((sum(new), 16, 128), 3), b.starts(new)
    weights = torch.zeros((3, 2, 64 * b.cols), device=DEV)
    out = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, weights=weights)
    assert bf.stream_status() == 0 and torch.isfinite(out).all()
    for i, n in enumerate(new):
        assert bool(weights[i].any()) == (n > 0)


# ---------------------------------------------------------------------------
# calls of more work than is counted
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cols", [(1 << 18, 1), (1 << 17, 2)])
def test_a_call_of_too_much_work_does_nothing_and_is_reported(cols):
    """2^23 query rows against 2^24 tokens, in one sequence or two: a sequence has 2^32 or 2^31 units
    and a few, which in 32 bits are a small or a negative number."""
    import torch
    cols, batch = cols
    new, heads, dim = (1 << 19) // batch, 16, 64
    pages = torch.zeros((1, 1, 72 * dim), dtype=torch.uint8, device=DEV)
    table = torch.zeros((batch, cols * batch), dtype=torch.int32, device=DEV)     # all of page 0
    kv_len = torch.full((batch,), 64 * cols * batch, dtype=torch.int32, device=DEV)
    start = torch.arange(0, (batch + 1) * new, new, dtype=torch.int32, device=DEV)
    q = torch.zeros((batch * new, heads, dim), dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 5.0)
    bf.attn_kv4(q, pages, table, kv_len, q_start=start, max_q=new, causal=False, out=out)
    assert bf.stream_status_bits() == (-9, 256)
    assert bool((out == 5.0).all())
    # what comes after is right
    b = Batch([3000], 1, dim, seed=1)
    x = _rand((64, heads, dim), 4)
    s = b.starts([64])
    one = bf.attn_kv4(x, b.pages, b.table, b.kv_len, q_start=s, max_q=64)
    two = bf.attn_kv4(x, b.pages, b.table, b.kv_len, q_start=s, max_q=64)
    assert bf.stream_status() == 0 and torch.equal(one, two) and float(one.float().abs().max()) > 0


@pytest.mark.parametrize("new,heads,batch,cols", [(632, 1, 1, 1 << 24), (1 << 15, 16, 1, 1 << 22)])
def test_a_refused_call_adds_no_weights(new, heads, batch, cols):
    """The attention kernel refuses (2^24 pages x 79 row groups; 2^21 tiles x 2^11 row groups), where
    the weights' pass of the first call counts far fewer units and would go on."""
    import torch
    dim = 128
    pages = torch.zeros((1, 1, 72 * dim), dtype=torch.uint8, device=DEV)
    table = torch.zeros((batch, cols), dtype=torch.int32, device=DEV)
    kv_len = torch.full((batch,), 64 * cols, dtype=torch.int32, device=DEV)
    start = torch.tensor([0, new], dtype=torch.int32, device=DEV)
    q = torch.zeros((new, heads, dim), dtype=torch.float16, device=DEV)
    weights = torch.zeros((batch, 1, 64 * cols), device=DEV)
    lse = torch.zeros((new, heads), device=DEV)
    bf.attn_kv4(q, pages, table, kv_len, q_start=start, max_q=new, lse=lse, weights=weights)
    assert bf.stream_status_bits() == (-9, 256)
    assert not bool(weights.any()) and not bool(lse.any())
    # the refusal is the call's own
    b = Batch([3000, 70], 2, dim, seed=1)
    x, w = _rand((2, 8, dim), 4), torch.zeros((2, 2, 64 * b.cols), device=DEV)
    bf.attn_kv4(x, b.pages, b.table, b.kv_len, weights=w)
    assert bf.stream_status() == 0
    assert torch.allclose(w.sum(-1), torch.full((2, 2), 4.0, device=DEV), rtol=1e-4)


# ---------------------------------------------------------------------------
# starts that do not rise
# ---------------------------------------------------------------------------
def test_rows_in_front_of_their_sequence_are_not_cached():
    """Starts 0, 4, 6, 0, 8: the search for rows 0 to 3 ends at sequence 1, whose own start, 4, is
    behind them. They are left out; what its older 28 tokens hold stays."""
    import torch
    b = Batch([20, 30, 9, 8], 2, 128, seed=4)
    start = torch.tensor([0, 4, 6, 0, 8], dtype=torch.int32, device=DEV)
    k = _rand((8, 2, 128), 5)
    older = (b.pages, b.table[1:2].contiguous(), torch.tensor([28], dtype=torch.int32, device=DEV))
    whole = torch.tensor([0, 28], dtype=torch.int32, device=DEV)
    before = bf.kv4_read(*older, q_start=whole, tokens=28)
    bf.kv4_append(b.pages, b.table, b.kv_len, k, k, q_start=start)
    assert bf.stream_status_bits() == (-9, 256)
    after = bf.kv4_read(*older, q_start=whole, tokens=28)
    assert bf.stream_status() == 0
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])


# ---------------------------------------------------------------------------
# batches padded with empty sequences
# ---------------------------------------------------------------------------
def _event_us(f, n=15):
    import torch
    times = []
    for _ in range(n):
        a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        z.record()
        z.synchronize()
        times.append(a.elapsed_time(z) * 1e3)
    return sorted(times)[n // 2]


@pytest.mark.parametrize("dim,new,dtype", [(64, 1, "float16"), (128, 1, "bfloat16"), (256, 4, "float16"),
                                           (128, 40, "float16"), (128, 700, "bfloat16")])
def test_rows_of_empty_sequences_are_zero_and_cost_little(dim, new, dtype):
    """The rows of empty sequences, whole and in strided outputs; 31 of 32 sequences of one token
    cost no more than as many sequences of a page each."""
    import torch
    batch, heads = (32, 64) if new < 100 else (3, 64)
    lens = [64 + new] + [0] * (batch - 1)
    b = Batch(lens, 8, dim, seed=new)
    q, start = _rand((batch * new, heads, dim), 1, dtype), b.starts([new] * batch)
    wide = torch.full((batch * new, heads + 1, dim), 3.0, dtype=q.dtype, device=DEV)
    lse = torch.full((batch * new, heads), 3.0, device=DEV)
    args = dict(q_start=start, max_q=new)
    bf.attn_kv4(q, b.pages, b.table, b.kv_len, out=wide[:, 1:], lse=lse, **args)
    assert bf.stream_status() == 0
    assert not bool(wide[new:, 1:].any()) and bool((wide[:, 0] == 3.0).all()) and bool((lse[new:] == -float("inf")).all())
    alone = bf.attn_kv4(q[:new], b.pages, b.table[:1].contiguous(), b.kv_len[:1].contiguous(), q_start=start[:2].contiguous(),
                        max_q=new)
    assert bool(wide[:new, 1:].any()) and torch.allclose(wide[:new, 1:].float(), alone.float(), rtol=2e-2, atol=2e-3)
    full = Batch([64 + new] * batch, 8, dim, seed=new)
    out = torch.empty_like(q)
    padded = _event_us(lambda: bf.attn_kv4(q, b.pages, b.table, b.kv_len, out=out, **args))
    whole = _event_us(lambda: bf.attn_kv4(q, full.pages, full.table, full.kv_len, out=out, **args))
    assert padded <= 1.5 * whole + 10.0, (padded, whole)


# ---------------------------------------------------------------------------
# graphs and streams side by side
# ---------------------------------------------------------------------------
def _captured(stream, calls):
    import torch
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(g, stream=stream):
            for f in calls:
                f()
    return g


def test_every_capture_has_a_workspace_of_its_own_and_gives_it_back():
    import gc
    import time
    import torch
    b = Batch([5000], 2, 128, seed=1)
    q, out = _rand((1, 16, 128), 2), torch.empty((1, 16, 128), dtype=torch.float16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = [lambda: bf.attn_kv4(q, b.pages, b.table, b.kv_len, out=out, stream=side)]
    call[0]()
    side.synchronize()
    want = out.clone()
    gc.collect()
    time.sleep(0.5)
    count, held = bf.internal_allocations(), []
    while bf.internal_allocations() == count and len(held) < 100:    # what earlier graphs gave back
        held.append(_captured(side, call))
    count = bf.internal_allocations()
    one = _captured(side, call * 3)          # one for all of a capture's calls
    two = _captured(side, call)
    assert bf.internal_allocations() == count + 2
    for g in (one, two):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del one, g
    gc.collect()
    torch.cuda.synchronize()
    count = bf.internal_allocations()
    for _ in range(50):                      # the driver gives it back from a thread of its own
        time.sleep(0.1)
        three = _captured(side, call)
        if bf.internal_allocations() == count:
            break
        held.append(three)
        count = bf.internal_allocations()
    else:
        pytest.fail("no workspace came back")
    out.zero_()
    torch.cuda.synchronize()
    three.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and bf.stream_status(side) == 0


@pytest.mark.parametrize("new", [1, 80])
def test_graphs_of_one_stream_run_beside_each_other_and_beside_its_calls(new):
    import torch
    side, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    b = [Batch([9000 + 700 * i, 40 + new, 3000], 2, 128, seed=i) for i in range(3)]
    q = [_rand((3 * new, 16, 128), 5 + i) for i in range(3)]
    start = b[0].starts([new] * 3)
    out = [torch.empty_like(x) for x in q]
    lse = [torch.zeros((3 * new, 16), device=DEV) for _ in q]
    w = [torch.zeros((3, 2, 64 * x.cols), device=DEV) for x in b]
    torch.cuda.synchronize()

    def call(i):
        return lambda: bf.attn_kv4(q[i], b[i].pages, b[i].table, b[i].kv_len, q_start=start, max_q=new, out=out[i],
                                   lse=lse[i], weights=w[i], stream=side)

    want, total = [], []          # of the same calls one after another
    for i in range(3):
        for _ in range(80):
            call(i)()
        side.synchronize()
        want.append(out[i].clone())
        total.append(w[i].clone())
        w[i].zero_()
    torch.cuda.synchronize()
    graphs = [_captured(side, [call(0)] * 4), _captured(side, [call(1)] * 4)]
    for _ in range(20):
        for s, g in zip(others, graphs):
            with torch.cuda.stream(s):
                g.replay()
        for _ in range(4):
            call(2)()
    torch.cuda.synchronize()
    assert bf.stream_status(side) == 0
    for i in range(3):
        assert torch.equal(out[i], want[i]) and torch.equal(w[i], total[i])


def test_threads_on_their_own_default_streams_share_no_workspace():
    """cudaStreamPerThread is one handle and a stream in every thread."""
    import threading
    import torch
    b = [Batch([9000 + 700 * i, 3000], 2, 128, seed=i) for i in range(2)]
    q = [_rand((2, 16, 128), 5 + i) for i in range(2)]
    out = [torch.empty_like(x) for x in q]
    want = [bf.attn_kv4(q[i], b[i].pages, b[i].table, b[i].kv_len) for i in range(2)]
    torch.cuda.synchronize()
    per_thread = torch.cuda.ExternalStream(2)
    wrong = []

    def work(i):
        for _ in range(60):
            for _ in range(5):
                bf.attn_kv4(q[i], b[i].pages, b[i].table, b[i].kv_len, out=out[i], stream=per_thread)
            per_thread.synchronize()
            if not torch.equal(out[i], want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    before = bf.internal_allocations()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and bf.stream_status(per_thread) == 0
    assert bf.internal_allocations() == before + 3      # two workspaces and the handle's error words


# ---------------------------------------------------------------------------
# more rows than the caller's bound
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("new,max_q,many", [([2, 7, 1], 3, False), ([60, 150, 31], 80, True)])
def test_rows_beyond_max_q_are_left_out_and_the_others_stay_in_place(dim, window, new, max_q, many):
    import torch
    lens, heads = [300, 400, 90], 16
    b = Batch(lens, 2, dim, seed=dim)
    assert (bf.attn_kv4_kernel(sum(new), heads, 2, dim, max_q)[0] == 0) == many
    q, start = _rand((sum(new), heads, dim), 3), b.starts(new)
    cut = list(range(new[0])) + list(range(new[0], new[0] + max_q)) + list(range(new[0] + new[1], sum(new)))
    gone = list(range(new[0] + max_q, new[0] + new[1]))
    want = bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, max_q=max(new), window=window).float()
    assert bf.stream_status() == 0
    out, lse = torch.full_like(q, 5.0), torch.full((sum(new), heads), 5.0, device=DEV)
    w = torch.zeros((3, 2, 64 * b.cols), device=DEV)
    bf.attn_kv4(q, b.pages, b.table, b.kv_len, q_start=start, max_q=max_q, window=window, out=out, lse=lse, weights=w)
    assert bf.stream_status_bits() == (-9, 256)
    assert bool((out[gone] == 5.0).all()) and bool((lse[gone] == 5.0).all())
    # another bound may choose another kernel: fp16 roundings apart
    assert torch.allclose(out[cut].float(), want[cut], rtol=4e-3, atol=2e-3)
    # every row that is there gives each of its heads a weight of 1, up to its own slot
    rows = torch.tensor([new[0], max_q, new[2]], device=DEV)
    assert torch.allclose(w.sum(-1), (rows * (heads // 2)).float()[:, None].expand(3, 2), rtol=1e-4)
    assert not bool(w[1, :, lens[1] - new[1] + max_q:].any())
