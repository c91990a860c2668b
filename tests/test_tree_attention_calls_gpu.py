"""Attention of several new tokens as programs call it: batches with places that no sequence has, and the like."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402
from test_tree_attention_gpu import BF16, E4M3, INT8, Batch, dev, run  # noqa: E402

FORMATS = [BF16, E4M3, INT8]


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def microseconds(call, n=15):
    times = []
    for i in range(n + 3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times[3:])[n // 2]


def padded(where, new, slots, live=8):
    n, ctx = np.zeros(slots, int), np.zeros(slots, int)
    at = {"before": slots - live + np.arange(live), "behind": np.arange(live), "between": np.arange(live) * (slots // live)}[where]
    n[at], ctx[at] = new, 150
    return at, ctx.tolist(), n.tolist()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new,slots", [(1, 37), (1, 900), (30, 50), (64, 300)])
@pytest.mark.parametrize("where", ["before", "behind", "between"])
def test_sequences_without_rows(L, fmt, new, slots, where):
    at, ctx, n = padded(where, new, slots)
    b = Batch(8, 2, 64, fmt, ctx, n, seed=40)
    run(L, b)
    b.check()
    assert b.status.item() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_without_rows_cost_little_wherever_they_are(L, fmt, new):
    """A batch with room for 20000 sequences: those that lie before the live ones are looked at by all threads of a CTA, and those behind them took 65 times as long, one after the other."""
    at, ctx, n = padded("before", new, 20000)
    b = Batch(32, 8, 128, fmt, ctx, n, seed=41)
    before = microseconds(lambda: b.call(L))
    for where in ("behind", "between"):
        at, ctx, n = padded(where, new, 20000)
        b = Batch(32, 8, 128, fmt, ctx, n, seed=41)
        took = microseconds(lambda: b.call(L))
        assert took < 4 * before, (where, took, before)
        b.check(only=at)
