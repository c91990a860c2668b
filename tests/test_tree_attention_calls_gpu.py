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


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ctx,new", [(0, 300), (77, 129), (200, 64)])
def test_a_prompt_in_pieces_of_64(L, fmt, ctx, new):
    """A prompt's pieces are sequences over the same pages, each with the ones before as cached tokens: held to a chain of one token at a time of the same cache, by the definition."""
    starts = list(range(0, new, 64)) + [new]
    lens = [b - a for a, b in zip(starts, starts[1:])]
    whole = Batch(8, 2, 128, fmt, [ctx + new - lens[-1]], [lens[-1]], seed=42, chain=True)      # its pages hold all of the prompt
    pieces = Batch(8, 2, 128, fmt, [0] * len(lens), lens, seed=43, chain=True)                 # queries and rows
    pieces.cache, pieces.values, pieces.pages, pieces.ctx = whole.cache, whole.values, whole.pages, [ctx + a for a in starts[:-1]]
    pieces.tables = np.repeat(whole.tables, len(lens), 0)
    pieces.need = [-(-(c + n) // 64) for c, n in zip(pieces.ctx, lens)]
    pieces.d.update(tables=dev(pieces.tables), ctx=dev(pieces.ctx))
    run(L, pieces)
    pieces.check()
    assert pieces.status.item() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 30])
def test_two_captured_calls_at_once(L, fmt, new):
    """Scratch of a captured call is its own: two graphs run beside each other, again and again."""
    bs = [Batch(8, 2, 128, fmt, [2000, 30], [new, 2], seed=44 + i) for i in range(2)]
    want, graphs, streams = [], [], [torch.cuda.Stream() for _ in bs]
    for b in bs:
        run(L, b)
        b.check()
        want.append(b.out.clone())
        b.out.fill_(5.0)
    for b, st in zip(bs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(3):
                assert b.call(L, stream=C.c_void_p(st.cuda_stream)) == 0
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for b, w in zip(bs, want):
        assert torch.equal(b.out.view(torch.int16), w.view(torch.int16)) and b.status.item() == 0
