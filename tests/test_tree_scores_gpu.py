"""Attention of several new tokens over caches of 8 bits: scores of any size, against the plain implementation in 64 bits of test_tree_attention_gpu.py and its tolerances."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402
from test_tree_attention_gpu import BF16, E4M3, INT8, PAGE, Batch, run  # noqa: E402

FORMATS = [BF16, E4M3, INT8]


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def key_scales(b):
    """[page, head, place] of the keys, in the cache itself."""
    return b.cache[0, :, :, PAGE * b.dim:].view(torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,n_kv,dim", [(8, 1, 64), (16, 2, 128)])
@pytest.mark.parametrize("size,scale", [(0.25, 0.0), (1e-6, 0.0), (1e-37, 0.0), (0.0, 0.0), (1.0, 1 / 128), (1.0, 1e-6)])
@pytest.mark.parametrize("window,chain", [(0, True), (70, False)])
def test_small_scores_beside_keys_that_a_row_tile_does_not_see(L, fmt, heads, n_kv, dim, size, scale, window, chain):
    """64 new tokens are four tiles of rows: the first ones' last keys are all drafts that none of their rows sees."""
    b = Batch(heads, n_kv, dim, fmt, [0, 64, 100, 128], [64] * 4, seed=31, chain=chain, window=window, sinks=2 if window else 0)
    q = (b.q.float() * size).bfloat16()
    run(L, b, q=q, scale=scale)
    b.check(q=q, scale=scale)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("size", [0.25, 0.0])
@pytest.mark.parametrize("new", [2, 40])
def test_keys_of_zeros(L, fmt, size, new):
    """Tiles of keys whose scales are all 0, at the end and before it."""
    b = Batch(8, 2, 128, fmt, [300, 100, 0], [new, new, new], seed=32)
    q = (b.q.float() * size).bfloat16()
    pages = torch.tensor([int(p) for i, cut in ((0, range(0, 4)), (1, range(0, 3)), (2, range(0, 1))) for p in b.tables[i, :b.need[i]][list(cut)[0]:list(cut)[-1] + 1]], device="cuda")
    scales = key_scales(b)
    scales[pages] = torch.where(scales[pages].isfinite(), 0.0, scales[pages])
    b.values[0, pages] = 0.0
    run(L, b, q=q)
    b.check(q=q)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_see_nothing_beside_small_scores(L, fmt):
    """Blind rows get zeros where the other rows' queries are small, or zeros themselves."""
    seen = [[0 if t % 5 == 2 else (1 << t) | 1 for t in range(64)]]
    for size in (0.1, 0.0):
        b = Batch(16, 1, 128, fmt, [0], [64], seen=seen, seed=33)
        q = (b.q.float() * size).bfloat16()
        run(L, b, q=q)
        b.check(q=q)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("new", [1, 30])
def test_largest_keys_under_small_queries(L, fmt, new):
    """Keys up to 2^127 and queries that bring their scores to ordinary sizes."""
    def factors(shape):
        f = torch.ones(shape, device="cuda")
        f[0] = 2.0 ** 125
        return f
    b = Batch(8, 2, 128, fmt, [300, 20], [new, 1], seed=34, scales=factors)
    q = (b.q.double() * 2.0 ** -125).bfloat16()
    assert key_scales(b)[key_scales(b).isfinite()].max() > 2.0 ** 118
    run(L, b, q=q)
    b.check(q=q)
