"""Attention of several new tokens of each sequence on the B200, through the C ABI, against a plain implementation in 64 bits: chains and trees over caches of
bf16, e4m3 and int8, windows with first tokens that stay visible, rows that see nothing.

Tolerances come from arithmetic.  `U` is 2^-24.  A weight is rounded to bf16 (2^-8) or, over 8 bits, to fp16 (2^-11, and 2^-25 of a unit that is 2^-15 of a power of two above the largest scale)
for the second product; scores are sums of D products in fp32 and three more factors ((D + 8) U of the sum of |q k|, scaled), which moves a weight by twice that at most (its own, and l's), 2^x by
2^-21; joining parts rounds a dozen times in fp32; the output rounds once (2^-8).
Over 8 bits, for sequences of more than 16 rows, scales are rounded to fp16 and so are keys and values times them: twice 2^-11 of a value, and of each product of a score; the products' own floor
is 2^-24 beside a largest scaled key of 2^-3 or more, half a tile's largest: 2^-20 of a score's sum under the largest key."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402

PAGE, U = 64, 2.0 ** -24
BF16, E4M3, INT8 = 0, 1, 2
FORMATS = [BF16, E4M3, INT8]


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def now():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.array(a, dtype)).cuda()


def randn(seed, shape, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * std


def a_tree(n, rng, chain=False):
    rows = []
    for t in range(n):
        parent = t - 1 if chain or t == 0 else int(rng.integers(0, t))
        rows.append((rows[parent] if t else 0) | 1 << t)
    return rows


class Batch:
    """Sequences whose pages lie anywhere in a cache; what no row sees holds NaN (bf16), or any byte under a scale that is not finite."""

    def __init__(self, heads, n_kv, dim, fmt, ctx, new, seed=0, window=0, sinks=0, chain=False, seen=None, pad=0, std=1.0, wide=0, before=0, scales=None):
        self.heads, self.n_kv, self.dim, self.fmt, self.ctx, self.new, self.window, self.sinks, self.pad = heads, n_kv, dim, fmt, list(ctx), list(new), window, sinks, pad
        rng = np.random.default_rng(seed)
        n = len(self.ctx)
        self.chain = chain
        self.seen = [list(x) for x in seen] if seen else [a_tree(k, rng, chain) for k in self.new]
        self.need = [-(-(c + k) // PAGE) for c, k in zip(self.ctx, self.new)]
        self.pages = sum(self.need) + 3
        order, at = rng.permutation(self.pages), 0
        self.tables = np.full((n, max(self.need + [1]) + wide), 10 ** 9, np.int32)
        for i, k in enumerate(self.need):
            self.tables[i, :k] = order[at:at + k]
            at += k
        used = torch.zeros(self.pages, PAGE, dtype=torch.bool)
        for i in range(n):
            for place in set().union(*[self.places(i, t) for t in range(self.new[i])]) if self.new[i] else ():
                used[self.tables[i, place // PAGE], place % PAGE] = True
        unused = ~used.cuda()
        self.values = torch.empty((2, self.pages, n_kv, PAGE, dim), dtype=torch.float64, device="cuda")       # what places stand for
        x = randn(seed + 1, (2, self.pages, n_kv, PAGE, dim), std)
        if fmt == BF16:
            self.cache = x.bfloat16().masked_fill(unused[None, :, None, :, None], math.nan)
            self.values.copy_(self.cache)
        else:
            self.cache = torch.empty((2, self.pages, n_kv, PAGE * (dim + 4)), dtype=torch.uint8, device="cuda")
            scale = x.abs().amax(-1) / (448.0 if fmt == E4M3 else 127.0)
            y = x / scale[..., None]
            y = y.clamp(-448, 448).to(torch.float8_e4m3fn) if fmt == E4M3 else y.round().clamp(-127, 127).to(torch.int8)
            if scales is not None:
                scale = scale * scales(scale.shape)
            self.values.copy_(y.double() * scale.double()[..., None])
            junk = torch.randint(0, 256, y.shape, dtype=torch.uint8, device="cuda")
            bad = torch.where(torch.arange(PAGE, device="cuda") % 3 == 0, math.inf, math.nan).expand_as(scale)
            self.cache[..., : PAGE * dim] = torch.where(unused[None, :, None, :, None], junk, y.view(torch.uint8)).flatten(-2)
            self.cache[..., PAGE * dim:] = torch.where(unused[None, :, None, :], bad, scale).view(torch.uint8)
        self.before = before
        self.rows = sum(self.new)
        pitch = heads * dim + pad
        self.q = randn(seed + 2, (before + self.rows + 2, pitch), std).bfloat16()
        self.out = torch.full((before + self.rows + 2, pitch), 5.0, dtype=torch.bfloat16, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.starts = (before + np.concatenate([[0], np.cumsum(self.new)])).astype(np.int32)
        bits = [0] * before + [b for s in self.seen for b in s] + [0, 0]
        self.d = {"tables": dev(self.tables), "ctx": dev(self.ctx), "starts": dev(self.starts), "seen": dev(np.array(bits, np.uint64).view(np.int64), np.int64)}

    def places(self, i, t):
        """The places that token t of sequence i sees, written from the definition."""
        c, bits = self.ctx[i], self.seen[i][t]
        at = c + bin(bits & (1 << t) - 1).count("1")
        old = range(c) if not self.window else [j for j in set(range(min(self.sinks, c))) | set(range(max(0, at - self.window + 1), c))]
        return set(old) | {c + u for u in range(self.new[i]) if bits >> u & 1}

    def call(self, L, out=None, q=None, scale=0.0, stream=None, rows=None, **over):
        d, pitch = {**self.d, **over}, self.heads * self.dim + self.pad
        return L.oa_k_tree_attention(ptr(self.q if q is None else q), pitch, ptr(self.out if out is None else out), pitch, ptr(self.cache), self.fmt, self.pages, ptr(d["tables"]), self.tables.shape[1],
                                     ptr(d["ctx"]), ptr(d["starts"]), None if self.chain else ptr(d["seen"]), len(self.ctx), self.before + self.rows + 2 if rows is None else rows, self.heads, self.n_kv,
                                     self.dim, self.window, self.sinks, scale, ptr(self.status), stream or now())

    def check(self, out=None, q=None, scale=0.0, only=None, clean=True):
        out, q = self.out if out is None else out, self.q if q is None else q
        scale, width = scale or 1.0 / math.sqrt(self.dim), self.heads * self.dim
        for i in range(len(self.ctx)) if only is None else only:
            pages = torch.tensor(self.tables[i, : self.need[i]].astype(np.int64), device="cuda")
            k, v = (self.values[j, pages].transpose(1, 2).reshape(-1, self.n_kv, self.dim) for j in (0, 1))
            for t in range(self.new[i]):
                r = int(self.starts[i]) + t
                got = out[r, :width].double().view(self.n_kv, -1, self.dim)
                see = torch.tensor(sorted(self.places(i, t)), device="cuda", dtype=torch.long)
                if not len(see):
                    assert not got.any()
                    continue
                x = q[r, :width].double().view(self.n_kv, -1, self.dim)
                p = torch.softmax(torch.einsum("khd,pkd->khp", x, k[see]) * scale, -1)
                want, size = torch.einsum("khp,pkd->khd", p, v[see]), torch.einsum("khp,pkd->khd", p, v[see].abs())
                score = torch.einsum("khd,pkd->khp", x.abs(), k[see].abs()).amax(-1, keepdim=True) * scale
                many = self.fmt != BF16 and -(-(self.before + self.rows + 2) // len(self.ctx)) * (self.heads // self.n_kv) > 8      # on the safe side of the kernels' border
                weight = 2.0 ** -8 if self.fmt == BF16 else 2.0 ** -11 + (2.0 ** -10 * (1 + 2 * score) + 2.0 ** -19 * score if many else 0.0)
                far = 0.0 if self.fmt == BF16 else len(see) * 2.0 ** -39 * v[see].abs().max()
                tol = size * (weight + 2 * (self.dim + 8) * U * score + 2.0 ** -20 + 16 * U) + far + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -133
                err = (got - want).abs()
                assert bool((err <= tol).all()), (i, t, (err / tol).max().item())
        if clean:
            mine = torch.zeros(out.shape[0], dtype=torch.bool)
            mine[self.before: self.before + self.rows] = True
            assert (out[~mine.cuda()] == 5.0).all() and (out[:, width:] == 5.0).all()


def run(L, b, **kw):
    assert b.call(L, **kw) == 0, _lib.last_error()
    torch.cuda.synchronize()


SHAPES = [(8, 2, 128), (8, 2, 64), (5, 1, 128), (6, 6, 64), (14, 2, 128), (9, 1, 64), (16, 1, 128), (32, 2, 64), (10, 2, 128)]      # heads, key/value heads, head size


@pytest.mark.parametrize("heads,n_kv,dim", SHAPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([1, 63, 64, 0], [1, 1, 1, 1]), ([130, 0, 5, 700], [5, 3, 17, 2]), ([60, 200], [64, 33])])
def test_trees(L, heads, n_kv, dim, fmt, ctx, new):
    b = Batch(heads, n_kv, dim, fmt, ctx, new, seed=heads + dim + len(ctx))
    run(L, b)
    b.check()
    assert b.status.item() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 47, 48, 56, 60, 62, 63, 64, 65, 120, 127, 128, 129, 255, 1000])
@pytest.mark.parametrize("new", [1, 8, 40])
def test_chains_that_end_anywhere(L, fmt, dim, ctx, new):
    b = Batch(4, 1, dim, fmt, [ctx, 3], [new, 2], seed=ctx, chain=True)
    run(L, b)
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(64, 0), (64, 4), (65, 1), (100, 64), (128, 65), (200, 130), (1000, 4), (2 ** 31 - 1, 7), (64, 2 ** 31 - 1)])
@pytest.mark.parametrize("chain", [True, False])
def test_windows(L, fmt, window, sinks, chain):
    b = Batch(8, 2, 64, fmt, [0, 40, 63, 64, 65, 127, 190, 500, 1000], [3, 1, 9, 64, 2, 30, 5, 4, 40], seed=window % 1000 + sinks % 100, window=window, sinks=sinks, chain=chain)
    run(L, b)
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_see_nothing(L, fmt):
    """No cached token and no bit; a window that leaves no cached token; tokens that nobody sees."""
    seen = [[0, 2, 0], [0] * 64, [1, 0, 5, 0, 0], [0]]
    b = Batch(8, 2, 128, fmt, [0, 0, 0, 0], [3, 64, 5, 1], seen=seen, seed=3, before=2)
    run(L, b)
    b.check()
    assert not b.out[2, :1024].any() and b.out[3, :1024].any() and not b.out[5:69, :1024].any()
    seen = [[(1 << t) - 1 for t in range(64)]]                                    # ancestors, and not itself: the last one's window of 64 reaches no cached token
    b = Batch(4, 2, 64, fmt, [500], [64], seen=seen, window=64, seed=4)
    run(L, b)
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_bits_of_tokens_that_are_not_there(L, fmt):
    b = Batch(4, 2, 128, fmt, [70, 3], [2, 3], seen=[[1, 3], [1, 3, 5]], seed=8)
    run(L, b)
    first = b.out.clone()
    more = b.d["seen"].clone()
    more[:2] |= -4
    more[2:5] |= -8
    run(L, b, seen=more)
    assert torch.equal(b.out, first)
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,n_kv,dim,n,top,most", [(32, 8, 128, 64, 700, 1), (32, 8, 64, 20, 2000, 7), (40, 8, 128, 11, 900, 30), (64, 8, 128, 1, 9000, 25), (28, 4, 128, 5, 3000, 64)])
def test_batches(L, fmt, heads, n_kv, dim, n, top, most):
    rng = np.random.default_rng(n)
    b = Batch(heads, n_kv, dim, fmt, rng.integers(0, top + 1, n).tolist() if n > 1 else [top], rng.integers(1, most + 1, n).tolist() if n > 1 else [most], seed=n, std=1.5, wide=5)
    run(L, b)
    b.check(only=range(0, n, 5))
    first = b.out.clone()
    for _ in range(5):                                                           # the same call gives the same bits
        run(L, b)
        assert torch.equal(b.out.view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_sequences_than_threads(L, fmt):
    rng = np.random.default_rng(1)
    n = 1500
    b = Batch(4, 1, 64, fmt, rng.integers(0, 90, n).tolist(), rng.integers(0, 3, n).tolist(), seed=9)
    run(L, b)
    b.check(only=range(0, n, 61))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [2, 20])
def test_strides_scale_and_in_place(L, fmt, new):
    b = Batch(10, 2, 128, fmt, [300, 20], [new, 1], seed=11, pad=24)
    run(L, b, scale=0.3)
    b.check(scale=0.3)
    want, q = b.out.clone(), b.q.clone()
    assert b.call(L, out=q, q=q, scale=0.3) == 0
    torch.cuda.synchronize()
    assert torch.equal(q[: b.rows, :1280], want[: b.rows, :1280]) and torch.equal(q[b.rows:], b.q[b.rows:]) and torch.equal(q[:, 1280:], b.q[:, 1280:])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 30])
def test_scores_that_grow_along_the_keys(L, fmt, new):
    """The maximum rises with every page."""
    b = Batch(4, 1, 128, fmt, [1500], [new], seed=12)
    q = b.q.clone()
    q[:] = 0.25
    k = torch.linspace(-3, 3, 1500 + new, device="cuda")
    for j in range(1500 + new):
        page, place = b.tables[0, j // PAGE], j % PAGE
        b.values[0, page, :, place] = k[j].bfloat16().double()
    if fmt == BF16:
        b.cache[0].copy_(torch.where(torch.isnan(b.cache[0]), b.cache[0], b.values[0].bfloat16()))
    else:
        one = torch.ones((), device="cuda").to(torch.float8_e4m3fn).view(torch.uint8) if fmt == E4M3 else torch.ones((), device="cuda", dtype=torch.uint8)
        b.cache[0, :, :, : PAGE * 128] = one
        b.cache[0, :, :, PAGE * 128:] = b.values[0, ..., 0].float().contiguous().view(torch.uint8)
    run(L, b, q=q)
    b.check(q=q)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("new", [1, 30])
def test_scales_of_any_size(L, fmt, new):
    """Scales from 2^-60 to 2^20 in one sequence, a scale of 0 among them."""
    def factors(shape):
        g = torch.Generator(device="cuda").manual_seed(5)
        f = torch.exp2(torch.randint(-60, 21, shape, generator=g, device="cuda").float())
        f[0] = 1.0                                                               # keys as they are: their scores decide what is looked at
        f[1, :, :, 7] = 0.0
        return f
    b = Batch(8, 2, 128, fmt, [900, 64], [new, 2], seed=13, scales=factors)
    run(L, b)
    b.check()


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e30])
def test_queries_of_any_size(L, fmt, size):
    b = Batch(8, 2, 64, fmt, [300], [9], seed=14)
    q = (b.q.float() * size).bfloat16()
    run(L, b, q=q, scale=0.125 / size)
    b.check(q=q, scale=0.125 / size)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 24])
def test_infinities_and_nan_that_are_seen(L, fmt, new):
    """A key's NaN makes its rows' results NaN, and no other sequence's; one in a place that a row does not see does nothing."""
    b = Batch(4, 2, 128, fmt, [200, 100], [new, 4], seen=[a_tree(new, np.random.default_rng(0), True), [1, 3, 5, 9]], seed=15)
    run(L, b)
    good = b.out.clone()
    page, place = int(b.tables[0, 1]), 9
    if fmt == BF16:
        b.cache[0, page, 1, place, 3] = math.nan
    else:
        b.cache[0, page, 1, PAGE * 128:].view(torch.float32)[place] = math.nan
    page, place = int(b.tables[1, 1]), (102 - 64)                                # the key of sequence 1's new token 2: seen by itself alone
    if fmt == BF16:
        b.cache[0, page, :, place] = math.nan
    else:
        b.cache[0, page, :, PAGE * 128:].view(torch.float32)[:, place] = math.nan
    run(L, b)
    at = b.starts
    assert torch.isnan(b.out[at[0]:at[1], 256:]).all() and torch.equal(b.out[at[0]:at[1], :256], good[at[0]:at[1], :256])
    assert torch.isnan(b.out[at[1] + 2]).all()
    rest = [int(at[1]) + t for t in (0, 1, 3)]
    assert torch.equal(b.out[rest], good[rest])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 24])
def test_bad_arrays_set_the_status_and_spare_the_others(L, fmt, new):
    b = Batch(8, 2, 128, fmt, [200, 100, 300], [new, new, new], seed=16, chain=True)
    for bad in (-1, b.pages, 2 ** 31 - 1, -2 ** 31):
        t = b.tables.copy()
        t[1, 0] = bad
        b.out.fill_(5.0)
        b.status.zero_()
        run(L, b, tables=dev(t))
        assert b.status.item() == 400
        b.check(only=[0, 2])
    room = b.tables.shape[1] * PAGE
    for ctx in ([200, -1, 300], [200, room + 1, 300], [200, 2 ** 31 - 1, 300], [200, -2 ** 31, 300]):
        t = b.tables.copy()
        t[t >= b.pages] = 0                                                      # what is cut to the table's room reads all of it
        b.out.fill_(5.0)
        b.status.zero_()
        run(L, b, ctx=dev(ctx), tables=dev(t))
        assert b.status.item() == 400
        b.check(only=[0, 2])
    for starts in ([0, new, new - 1, 2 * new], [0, new, 2 ** 31 - 1, 3 * new], [-1, new, 2 * new, 3 * new], [-2 ** 31, 2 ** 31 - 1, 2 * new, 3 * new]):
        b.status.zero_()
        t = b.tables.copy()
        t[t >= b.pages] = 0
        run(L, b, starts=dev(starts), tables=dev(t))
        assert b.status.item() == 400
    b.status.zero_()
    run(L, b, rows=3 * new - 1)
    assert b.status.item() == 400


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_than_64_new_tokens_are_cut(L, fmt):
    b = Batch(4, 1, 64, fmt, [80], [64], seed=17, chain=True)
    more = dev([0, 66])
    run(L, b, starts=more)
    assert b.status.item() == 400
    b.check()                                                                    # the first 64 are computed, the others left


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,n_kv,new", [(8, 2, [2, 0, 1]), (8, 2, [30, 0, 17])])
def test_a_captured_call_follows_its_arrays(L, fmt, heads, n_kv, new):
    b = Batch(heads, n_kv, 128, fmt, [333, 70, 0], new, seed=18)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    run(L, b)
    ctx, starts = torch.zeros_like(b.d["ctx"]), torch.full_like(b.d["starts"], 0)
    with torch.cuda.graph(graph, stream=side):
        assert b.call(L, ctx=ctx, starts=starts) == 0
    b.out.fill_(5.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (b.out == 5.0).all()                                                  # no sequence has a row yet
    ctx.copy_(b.d["ctx"])
    starts.copy_(b.d["starts"])
    graph.replay()
    torch.cuda.synchronize()
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 20])
def test_two_streams_at_once(L, fmt, new):
    a, b = Batch(8, 2, 128, fmt, [900] * 9, [new] * 9, seed=19), Batch(8, 2, 128, fmt, [400] * 9, [new] * 9, seed=20)
    run(L, a)
    run(L, b)
    want = a.out.clone(), b.out.clone()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for x in (a, b):
        x.out.fill_(5.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for x, st in zip((a, b), s):
            assert x.call(L, stream=C.c_void_p(st.cuda_stream)) == 0
    torch.cuda.synchronize()
    assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


@pytest.mark.parametrize("fmt", FORMATS)
def test_calls_without_a_wait_between_them(L, fmt):
    """A call's queries are the output of the one before, and its new tokens' number another: what is enqueued runs in order."""
    bs = [Batch(8, 2, 128, fmt, [500, 20], new, seed=21) for new in ([1, 1], [40, 8], [3, 2], [64, 64])]
    want = []
    for b in bs:
        run(L, b)
        want.append(b.out.clone())
        b.out.fill_(5.0)
    torch.cuda.synchronize()
    for _ in range(6):
        for b in bs:
            assert b.call(L) == 0
    torch.cuda.synchronize()
    for b, w in zip(bs, want):
        assert torch.equal(b.out, w)


def test_a_cache_beyond_32_bits(L):
    """Blocks that lie more than 4 GB into the cache, in its second plane more than 8."""
    dim, n_kv, pages = 128, 8, 70000
    for fmt in (E4M3, BF16):
        block = PAGE * (dim + 4) if fmt == E4M3 else PAGE * dim * 2
        if torch.cuda.mem_get_info()[0] < 3 * 2 * pages * n_kv * block:
            pytest.skip("not enough memory")
        cache = torch.empty((2, pages, n_kv, block), dtype=torch.uint8, device="cuda")
        b = Batch(16, n_kv, dim, fmt, [150, 40], [4, 1], seed=22)
        t = b.tables.copy()
        for i, k in enumerate(b.need):
            for p in range(k):
                t[i, p] = pages - 1 - 5 * (4 * i + p)
                cache[:, t[i, p]] = b.cache[:, b.tables[i, p]].reshape(2, n_kv, -1).view(torch.uint8)
        run(L, b)
        want = b.out.clone()
        d = dev(t)
        assert L.oa_k_tree_attention(ptr(b.q), 16 * dim, ptr(b.out), 16 * dim, ptr(cache), fmt, pages, ptr(d), t.shape[1], ptr(b.d["ctx"]), ptr(b.d["starts"]), ptr(b.d["seen"]), 2, b.rows + 2, 16, n_kv, dim,
                                     0, 0, 0.0, ptr(b.status), now()) == 0
        torch.cuda.synchronize()
        assert torch.equal(b.out, want) and b.status.item() == 0
        del cache


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_token_agrees_with_the_other_entries(L, fmt):
    """A token a sequence over a cache of bf16 is what prefix attention computes without a prefix; over 8 bits, what it computes on the cache read back is nearby."""
    b = Batch(8, 2, 128, fmt, [300, 0, 64], [1, 1, 1], seed=23, chain=True)
    run(L, b)
    b.check()
    cache = b.cache if fmt == BF16 else b.values.float().bfloat16()
    out, lens = torch.empty_like(b.q[:3]), dev([c + 1 for c in b.ctx])
    tables = dev(np.where(b.tables >= b.pages, 0, b.tables))
    assert L.oa_k_prefix_attention(ptr(b.q), 1024, ptr(out), 1024, ptr(cache.contiguous()), b.pages, None, 0, None, None, 0, ptr(tables), b.tables.shape[1], ptr(lens), 3, 8, 2, 128, 0.0, None, now()) == 0
    torch.cuda.synchronize()
    big = b.values[1].nan_to_num().abs().max().item()
    assert (out.double() - b.out[:3].double()).abs().max().item() <= big * (2.0 ** -7 + (2.0 ** -8 if fmt != BF16 else 0) + 2.0 ** -9 * (64 if fmt != BF16 else 1) ** 0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 24])
def test_queries_that_are_not_finite(L, fmt, new):
    """A NaN in a head of a row makes that head of that row NaN and nothing else."""
    b = Batch(8, 2, 128, fmt, [150, 70], [new, 2], seed=24)
    run(L, b)
    good = b.out.clone()
    q = b.q.clone()
    q[0, 3 * 128 + 5] = math.nan
    run(L, b, q=q)
    assert torch.isnan(b.out[0, 3 * 128: 4 * 128]).all()
    b.out[0, 3 * 128: 4 * 128] = good[0, 3 * 128: 4 * 128]
    assert torch.equal(b.out, good)


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_row_has_no_pitch(L, fmt):
    b = Batch(4, 1, 64, fmt, [100], [1], seed=25, chain=True)
    run(L, b)
    want = b.out.clone()
    d = b.d
    for pitch in (256, 1 << 38):
        b.out.fill_(5.0)
        assert L.oa_k_tree_attention(ptr(b.q), pitch, ptr(b.out), pitch, ptr(b.cache), fmt, b.pages, ptr(d["tables"]), b.tables.shape[1], ptr(d["ctx"]), ptr(d["starts"]), None, 1, 1, 4, 1, 64, 0, 0, 0.0, None,
                                     now()) == 0, _lib.last_error()
        torch.cuda.synchronize()
        assert torch.equal(b.out, want)


@pytest.mark.parametrize("fmt", [BF16, INT8])
@pytest.mark.parametrize("heads", [1, 16])
def test_very_many_sequences(L, fmt, heads):
    """70000 sequences of no or one new token on pages that they share."""
    n, dim = 70000, 64
    b = Batch(heads, 1, dim, fmt, [60], [1], seed=26, chain=True)
    rng = np.random.default_rng(2)
    new = (rng.random(n) < 0.7).astype(np.int32)
    starts, rows = np.concatenate([[0], np.cumsum(new)]), int(new.sum())
    tables = dev(np.full((n, 1), b.tables[0, 0]))
    ctx = dev(np.full(n, 60))
    q = b.q[:1, : heads * dim].repeat(rows, 1).contiguous()
    out = torch.full((rows + 1, heads * dim), 5.0, dtype=torch.bfloat16, device="cuda")
    s = dev(starts)
    assert L.oa_k_tree_attention(ptr(q), heads * dim, ptr(out), heads * dim, ptr(b.cache), fmt, b.pages, ptr(tables), 1, ptr(ctx), ptr(s), None, n, rows, heads, 1, dim, 0, 0, 0.0, ptr(b.status), now()) == 0
    torch.cuda.synchronize()
    assert b.status.item() == 0 and (out[rows] == 5.0).all()
    b.check(out=torch.cat([out[:1], torch.full_like(b.out[1:], 5.0)]))
    assert (out[:rows] == out[0]).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_calls_from_two_threads(L, fmt):
    import threading
    bs = [Batch(8, 2, 64, fmt, [300, 40, 700], new, seed=27) for new in ([1, 2, 1], [30, 5, 64])]
    want = []
    for b in bs:
        run(L, b)
        want.append(b.out.clone())
        b.out.fill_(5.0)
    torch.cuda.synchronize()
    streams, codes = [torch.cuda.Stream(), torch.cuda.Stream()], []

    def work(b, st):
        for _ in range(50):
            code = b.call(L, stream=C.c_void_p(st.cuda_stream))
            codes.append((code, _lib.last_error() if code else ""))
    threads = [threading.Thread(target=work, args=x) for x in zip(bs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [(0, "")] * 100, codes[0]
    for b, w in zip(bs, want):
        assert torch.equal(b.out, w)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window", [0, 70])
def test_trees_that_cross_tiles(L, fmt, window):
    """New tokens on either side of pages, tiles of keys and tiles of rows, each seeing every third one before it."""
    seen = [sum(1 << u for u in range(t + 1) if (t - u) % 3 == 0) for t in range(64)]
    ctx = [0, 1, 63, 64, 65, 100, 127, 128, 129, 191, 192, 255, 256, 320]
    b = Batch(10, 2, 128, fmt, ctx, [64] * len(ctx), seen=[seen] * len(ctx), seed=28, window=window, sinks=3 if window else 0)
    run(L, b)
    b.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("group", range(1, 17))
def test_groups_of_any_size(L, fmt, group):
    for new in ([1, 1, 0, 1], [min(64, 128 // group + 1), 17, 1, 64]):
        b = Batch(2 * group, 2, 64, fmt, [70, 200, 5, 0], new, seed=29 + group)
        run(L, b)
        b.check()


@pytest.mark.parametrize("fmt", [BF16, E4M3])
@pytest.mark.parametrize("heads,n_kv,new", [(1024, 1024, 2), (1024, 1024, 20), (2048, 128, 3)])
def test_very_many_heads(L, fmt, heads, n_kv, new):
    b = Batch(heads, n_kv, 64, fmt, [130], [new], seed=30)
    run(L, b)
    b.check()
