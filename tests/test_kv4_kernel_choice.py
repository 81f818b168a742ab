"""Which attention kernel a call takes, and that what means to run a kernel has a shape that does. CPU."""
import os
import sys

import pytest

import busfill_b200 as bf

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_choice_by_rows():
    assert bf.attn_kv4_kernel(32, 64, 8, 128, 1) == (1, False)
    assert bf.attn_kv4_kernel(8000, 64, 8, 128, 8000) == (0, True)
    assert bf.attn_kv4_kernel(80, 8, 2, 128, 80) == (0, True) and bf.attn_kv4_kernel(79, 8, 2, 128, 79) == (1, True)
    assert bf.attn_kv4_kernel(48, 32, 8, 64, 6) == (1, False) and bf.attn_kv4_kernel(56, 32, 8, 64, 7) == (2, False)
    assert bf.attn_kv4_kernel(90, 32, 8, 64, 14) == (2, True) and bf.attn_kv4_kernel(90, 32, 8, 64, 15) == (0, True)


@pytest.mark.parametrize("bad", [(1, 4, 1, 96, 1), (-1, 4, 1, 64, 1), (1, 3, 2, 64, 1), (1, 4, 0, 64, 1), (1, 4, 1, 64, 0)])
def test_shapes_that_attention_refuses(bad):
    with pytest.raises(bf.BusfillError):
        bf.attn_kv4_kernel(*bad)


def test_smoke_runs_both_attention_kernels():
    import __graft_entry__ as entry
    s = entry.SMOKE_ATTENTION
    taken = [bf.attn_kv4_kernel(n, s["kv_heads"] * s["group"], s["kv_heads"], s["dim"], n)[0] for n in s["rows"]]
    assert taken == [1, 0]
