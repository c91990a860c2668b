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


def expected_error(b, q, many):
    """The norm of the error that roundings leave, and of the output, by the formula: a rounding is off by a step over sqrt(12) in the mean, independently of the others.  bf16 steps of the output; a weight's
    steps, of bf16 or fp16, taken as 2 half-steps of the weight; over 8 bits and tiles of 128 rows fp16 steps of keys and values, where a key's move its score s_j and that moves the
    output by p_j ds_j (v_j - o).  Few rows over 8 bits have values' scales in their weights."""
    def step(x, bits):
        return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -200))) - bits)
    width, scale, total, size, err = b.heads * b.dim, b.dim ** -0.5, 0.0, 0.0, 0.0
    for i in range(len(b.ctx)):
        pages = torch.tensor(b.tables[i, : b.need[i]].astype(np.int64), device="cuda")
        k, v = (b.values[j, pages].transpose(1, 2).reshape(-1, b.n_kv, b.dim) for j in (0, 1))
        for t in range(b.new[i]):
            r = int(b.starts[i]) + t
            see = torch.tensor(sorted(b.places(i, t)), device="cuda", dtype=torch.long)
            x, ks, vs = q[r, :width].double().view(b.n_kv, -1, b.dim), k[see], v[see]
            p = torch.softmax(torch.einsum("khd,pkd->khp", x, ks) * scale, -1)
            o = torch.einsum("khp,pkd->khd", p, vs)
            weight = (2.0 ** -7 if b.fmt == BF16 else 2.0 ** -10) / 12 ** 0.5
            var = step(o, 7).square().sum() / 12 + weight ** 2 * torch.einsum("khp,pkd->", p.square(), vs.square())
            if many:
                var += torch.einsum("khp,pkd->", p.square(), step(vs, 10).square()) / 12
                score = scale ** 2 / 12 * torch.einsum("khd,pkd->khp", x.square(), step(ks, 10).square())
                away = torch.einsum("pkd,pkd->kp", vs, vs)[:, None] - 2 * torch.einsum("khd,pkd->khp", o, vs) + o.square().sum(-1, keepdim=True)
                var += (p.square() * score * away).sum()
            total += var.item()
            size += o.square().sum().item()
            err += (b.out[r, :width].double().view(b.n_kv, -1, b.dim) - o).square().sum().item()
    return err ** 0.5 / size ** 0.5, total ** 0.5 / size ** 0.5


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1, 4, 8, 16])
@pytest.mark.parametrize("new", [1, 3, 20])
def test_errors_of_large_scores(L, fmt, dim, size, new):
    """The error's norm is what independent roundings make it, for scores up to about 80: a quarter is left for a sum over some thousand rows of heads.  4 and 12 rows of a sequence, and 80."""
    b = Batch(32, 8, dim, fmt, [700 + 13 * i for i in range(64 // new)] if new < 20 else [2500, 900, 40], [new] * (64 // new if new < 20 else 3), seed=35)
    q = (b.q.float() * size).bfloat16()
    run(L, b, q=q)
    b.check(q=q)
    err, want = expected_error(b, q, b.fmt != BF16 and new == 20)
    assert err <= 1.25 * want, (err, want)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("new", [1, 30])
def test_values_under_an_infinite_scale(L, fmt, new):
    """A value under a scale of infinity is infinite, of its own sign, and 0 times infinity none."""
    b = Batch(4, 1, 128, fmt, [200], [new], seed=36, chain=True)
    run(L, b)
    page = int(b.tables[0, 1])
    b.cache[1, page, 0, PAGE * 128:].view(torch.float32)[9] = float("inf")
    b.values[1, page, 0, 9] *= float("inf")
    run(L, b)
    want, got = b.values[1, page, 0, 9], b.out[:new, :512].view(new, 4, 128).double()
    finite_zero = torch.isnan(want)
    assert torch.isnan(got[..., finite_zero]).all() and (got[..., ~finite_zero] == want[~finite_zero]).all()
