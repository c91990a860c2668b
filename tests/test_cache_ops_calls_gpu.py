"""Calls of the operators on a caller's paged cache as a program makes them on the B200: tables that ask for what there is not (and what is cut to what there is), captured calls, a first call that
is captured, calls from two threads on two streams.  Values against the 64-bit oracles and tolerances of test_cache_ops_gpu.py, or against an eager call's bits."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402
from test_cache_ops_gpu import PAGE, Batch, apart, assert_turned, cuda_i32, frequencies, now, ptr, randn, run, turned  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def same_bits(a, b):
    return torch.equal(a.view(torch.int16 if a.element_size() == 2 else torch.int32), b.view(torch.int16 if b.element_size() == 2 else torch.int32))


# ---- tables that ask for what there is not -----------------------------------------------------------
def full_tables(b, seed):
    """Every entry of both tables names a page of the cache, and every place holds a number: a row that is cut to its table sees only those."""
    rng = np.random.default_rng(seed)
    for table in (b.pt, b.ot):
        bad = (table < 0) | (table >= b.pages)
        table[bad] = rng.integers(0, b.pages, int(bad.sum()))
    b.cache.nan_to_num_(0.25)
    return b


# what is asked for, and the lengths and bounds that the header's cut leaves of it (None: as they were); the runs that fall are those of three prefixes
CUTS = {
    "own length": (dict(own=(1, 10 ** 6)), dict(own=(1, "width"))),
    "longest own length": (dict(own=(3, 2 ** 31 - 1)), dict(own=(3, "width"))),
    "negative length": (dict(own=(1, -5)), dict(own=(1, 0))),
    "prefix length": (dict(prefix=(0, 2 ** 31 - 1)), dict(prefix=(0, "width"))),
    "negative prefix length": (dict(prefix=(1, -1)), dict(prefix=(1, 0))),
    "runs fall": (dict(runs=[0, 4, 2, 6]), dict(runs=[0, 4, 4, 6])),
    "runs fall at once": (dict(runs=[5, 1, 0, 0]), dict(runs=[5, 5, 5, 5])),
    "runs beyond": (dict(runs=[-2, 3, 5, 90]), dict(runs=[0, 3, 5, 6])),
    "runs all beyond": (dict(runs=[9, 10, 11, 12]), dict(runs=[6, 6, 6, 6])),
}


@pytest.mark.parametrize("wide", [1, apart(6, 2), 600])
@pytest.mark.parametrize("what", list(CUTS))
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths_and_runs_are_cut_to_what_there_is(L, what, wide, dim):
    """Every row's value, the cut ones' among them, is that of the cut lengths and runs, and the status says that something was cut."""
    b = full_tables(Batch(8, 2, dim, [200, 64, 130], [0, 3, 5, 6], [30, 70, 64, 5, 0, 17], seed=12, wide=wide), 5)
    run(L, b)
    b.check()
    assert b.status.item() == 0
    asked, left = CUTS[what]

    def put(change):
        for name, value in change.items():
            if name == "runs":
                b.runs = list(value)
            else:
                lens, table = (b.own, b.ot) if name == "own" else (b.prefixes, b.pt)
                lens[value[0]] = table.shape[1] * PAGE if value[1] == "width" else value[1]

    put(asked)
    b.upload()
    b.out.fill_(5.0)
    run(L, b)
    assert b.status.item() == 400
    put(left)
    b.check()


@pytest.mark.parametrize("wide", [1, apart(4, 2), 600])
@pytest.mark.parametrize("page", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_pages_that_there_are_not_leave_the_other_rows_right(L, page, wide):
    """A bad page of one row, then of one of two prefixes: rows that do not read it have their values, and nothing behind the rows is written."""
    for which in ("own", "prefix"):
        b = full_tables(Batch(8, 2, 128, [200, 300], [0, 2, 4], [30, 70, 64, 5], seed=13, wide=wide), 6)
        bad = b.pages if page == "pages" else page
        table = b.ot if which == "own" else b.pt
        table[1, 1] = bad
        b.upload()
        run(L, b)
        assert b.status.item() == 400
        table[1, 1] = 0
        b.check(rows=[0, 2, 3] if which == "own" else [0, 1])
        assert torch.isfinite(b.out[:4]).all() and (b.out[4:] == 5.0).all()


# ---- rows ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("f32", [False, True])
def test_a_single_row_in_place_under_two_pitches(L, f32):
    dtype = torch.float32 if f32 else torch.bfloat16
    x, positions = randn(4, (1, 3, 128), dtype), cuda_i32([70001])
    freqs, _ = frequencies(L, 128)
    want, mag = turned(x, positions, freqs, 1.0, 128, 1)
    assert L.oa_k_rotary(ptr(x), 384, ptr(x), 2 ** 62, ptr(positions), 1, 3, 128, 128, 1, freqs.ctypes.data, 1.0, 0, int(f32), now()) == 0
    torch.cuda.synchronize()
    assert_turned(x, want, mag, dtype, 2.0 ** -52 * 70001)
    b = Batch(8, 2, 128, [100], [0, 1], [7], seed=3)
    run(L, b)
    pt, pl, pr, ot, ol = b.d
    q = b.q.clone()
    assert L.oa_k_prefix_attention(ptr(q), 2 ** 61, ptr(q), 1024, ptr(b.cache), b.pages, ptr(pt), b.pt.shape[1], ptr(pl), ptr(pr), 1, ptr(ot), b.ot.shape[1], ptr(ol), 1, 8, 2, 128, 0.0, None, now()) == 0
    torch.cuda.synchronize()
    assert same_bits(q, b.out[:1])


# ---- captured calls -------------------------------------------------------------------------------------
class Appends:
    """q, k and v of new tokens, rotated and written to a cache; the transposed rotation of q in fp32; copies of two pages."""

    def __init__(self, L, tokens, seed):
        self.L, self.tokens, self.heads, self.n_kv, self.dim, self.pages = L, tokens, 8, 2, 128, tokens // PAGE + 9
        self.width = (self.heads + 2 * self.n_kv) * self.dim
        self.freqs, self.amp = frequencies(L, 128, 1e6, 3, 4.0, 32.0, 1.0, 32768)
        self.qkv, self.g = randn(seed, (tokens, self.width)), randn(seed + 1, (tokens, 8 * 128), torch.float32)
        self.start = randn(seed + 2, (2, self.pages, self.n_kv, PAGE, self.dim))
        self.cache, self.q, self.dx = self.start.clone(), torch.empty(tokens, 1024, dtype=torch.bfloat16, device="cuda"), torch.empty(tokens, 1024, dtype=torch.float32, device="cuda")
        free = self.pages - 4                                                       # the last four pages are for the copies
        self.rng = np.random.default_rng(seed)
        self.positions, self.slots = cuda_i32(self.rng.integers(0, 30000, tokens)), cuda_i32(self.rng.permutation(free * PAGE)[:tokens])
        self.moves = (_lib.OaPageMove * 3)(*[_lib.OaPageMove(s, free + i, n) for i, (s, n) in enumerate([(0, 64), (0, 17), (1, 64)])])
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(self, stream=None):
        L, s, f, k0 = self.L, stream or now(), self.freqs.ctypes.data, self.qkv.data_ptr() + 2 * 1024
        rc = L.oa_k_rotary_cache(ptr(self.qkv), self.width, k0, k0 + 512, self.width, ptr(self.q), 1024, ptr(self.cache), self.pages, ptr(self.positions), ptr(self.slots), self.tokens, self.heads,
                                 self.n_kv, self.dim, 128, 1, f, self.amp, ptr(self.status), s)
        rc = rc or L.oa_k_rotary(ptr(self.g), 1024, ptr(self.dx), 1024, ptr(self.positions), self.tokens, 8, 128, 128, 0, f, self.amp, 1, 1, s)
        return rc or L.oa_k_cache_copy(ptr(self.cache), 2, self.pages, self.n_kv, self.dim, 2, self.moves, 3, s)

    def outputs(self):
        return [self.cache.clone(), self.q.clone(), self.dx.clone(), self.status.clone()]

    def reset(self):
        self.cache.copy_(self.start), self.q.zero_(), self.dx.zero_(), self.status.zero_()

    def change(self):
        """Other positions, slots and rows, where the device arrays lie."""
        free = self.pages - 4
        self.positions.copy_(cuda_i32(self.rng.integers(0, 30000, self.tokens))), self.slots.copy_(cuda_i32(self.rng.permutation(free * PAGE)[: self.tokens]))
        self.qkv.neg_(), self.g.mul_(0.5)


@pytest.mark.parametrize("tokens", [1, 6, 130, 2003])
def test_captured_calls_keep_host_arrays_and_follow_device_arrays(L, tokens):
    """A replay has the frequencies and moves that the call was captured with, whatever lies in their arrays now, and the positions, slots and rows of the replay."""
    a = Appends(L, tokens, seed=tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert a.call() == 0
    a.reset()
    freqs, moves = a.freqs.copy(), [(m.src, m.dst, m.tokens) for m in a.moves]
    for replay in range(3):
        if replay:
            a.change()
        a.freqs[:] = freqs
        for m, (src, dst, n) in zip(a.moves, moves):
            m.src, m.dst, m.tokens = src, dst, n
        a.reset()
        assert a.call() == 0
        torch.cuda.synchronize()
        want = a.outputs()
        a.freqs[:] = 1e9
        for m in a.moves:
            m.src, m.dst, m.tokens = 10 ** 6, -1, 99
        a.reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same_bits(x, y) for x, y in zip(a.outputs(), want)), replay
    assert not same_bits(a.start, a.cache) and a.status.item() == 0


FIRST = r'''
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import torch
torch.zeros(8, device="cuda").normal_()
from test_cache_ops_calls_gpu import Appends, Batch, _lib, run, same_bits
L, what = _lib.load(), sys.argv[2]
if what == "attention":
    b = Batch(8, 2, 128, [300], [0, 6], [11, 1, 64, 90, 2, 65], seed=13, wide=int(sys.argv[3]))
else:
    b = Appends(L, 130, 7)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    rc = b.call(L) if what == "attention" else b.call()
assert rc == 0, (rc, _lib.last_error())
if what == "attention":
    for _ in range(2):
        b.out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        b.check()
    first = b.out.clone()
    run(L, b)
    assert same_bits(first, b.out)
else:
    b.reset()
    graph.replay()
    torch.cuda.synchronize()
    first = b.outputs()
    b.reset()
    assert b.call() == 0
    torch.cuda.synchronize()
    assert all(same_bits(x, y) for x, y in zip(first, b.outputs()))
print("same")
'''


@pytest.mark.parametrize("what,wide", [("attention", 1), ("attention", 600), ("appends", 0)])
def test_a_process_may_capture_its_first_call(L, what, wide):
    """Nothing that the library makes at its first use (its pool of scratch memory, attributes of its kernels) ends a capture."""
    r = subprocess.run([sys.executable, "-c", FIRST, ROOT, what, str(wide)], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), (r.stdout[-500:], r.stderr[-3000:])


# ---- calls one after the other --------------------------------------------------------------------------
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n_kv,tokens", [(8, 64), (2, 3), (32, 64)])
def test_a_copy_has_what_the_calls_before_it_wrote(L, n_kv, tokens, captured):
    """Page 0 is written, copied, written again, copied, two hundred times without a wait on the host: every kernel may start before the one ahead of it has ended, and each copy holds its own step's
    keys and values."""
    steps, dim, heads = 200, 64, n_kv
    width = 3 * heads * dim
    rows, freqs = randn(9, (steps, tokens, width)), np.zeros(dim // 2)                # angles of 0: keys come out as they are
    cache = torch.zeros((2, steps + 1, n_kv, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    q, positions, slots = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device="cuda"), cuda_i32(np.arange(tokens)), cuda_i32(np.arange(tokens))
    moves = [(_lib.OaPageMove * 1)(_lib.OaPageMove(0, i + 1, tokens)) for i in range(steps)]

    def chain():
        for i in range(steps):
            at = rows[i].data_ptr()
            assert L.oa_k_rotary_cache(at, width, at + 2 * heads * dim, at + 4 * heads * dim, width, ptr(q), heads * dim, ptr(cache), steps + 1, ptr(positions), ptr(slots), tokens, heads, n_kv, dim,
                                       dim, 1, freqs.ctypes.data, 1.0, None, now()) == 0
            assert L.oa_k_cache_copy(ptr(cache), 2, steps + 1, n_kv, dim, 2, moves[i], 1, now()) == 0

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain()
    for _ in range(5):
        cache.zero_(), q.zero_()
        graph.replay() if captured else chain()
        torch.cuda.synchronize()
        kv = rows.view(steps, tokens, 3, n_kv, dim)[:, :, 1:].permute(2, 0, 3, 1, 4)        # [planes, steps, heads, tokens, channels]
        assert torch.equal(cache[:, 1:, :, :tokens], kv) and not cache[:, :, :, tokens:].any() and torch.equal(q, rows[-1, :, :heads * dim])


@pytest.mark.parametrize("wide", [1, apart(12, 2), 600])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_without_a_wait_are_those_with_one(L, wide, captured):
    """Sixty decoding steps: lengths rise on the device, a new token is rotated into its page, attention reads it, in place.  Nothing waits between them, and no step reads what a later one writes or misses
    what an earlier one wrote."""
    steps, n, heads, n_kv, dim = 60, 12, 8, 2, 128
    own = [0, 1, 30, 63, 64, 100, 3, 0, 127, 65, 10, 5]
    b = Batch(heads, n_kv, dim, [200, 300], [0, 5, 11], own, seed=21, wide=wide)
    at, b.ot = 0, np.full((n, 4), -1, np.int32)                                        # room for sixty tokens more, in pages of their own
    free = np.random.default_rng(2).permutation(200).astype(np.int32)
    cache = torch.full((2, 200, n_kv, PAGE, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    for table, lens, room in ((b.pt, b.prefixes, 0), (b.ot, own, steps)):
        for i, x in enumerate(lens):
            k = -(-(x + room) // PAGE)
            table[i, :k] = free[at:at + k]
            at += k
            for j in range(-(-x // PAGE)):
                cache[:, int(table[i, j]), :, : min(PAGE, x - j * PAGE)] = randn(i * 10 + j + room, (2, n_kv, min(PAGE, x - j * PAGE), dim))
    b.cache, b.pages, b.pad = cache, 200, 0
    b.upload()
    rows, freqs = randn(5, (steps, n, (heads + 2 * n_kv) * dim)), frequencies(L, dim)[0]
    tables, outs, start = cuda_i32(b.ot).long(), torch.empty(steps, n, heads * dim, dtype=torch.bfloat16, device="cuda"), cuda_i32(own)
    positions, slots, width = start.clone(), start.clone(), rows.shape[2]

    def steps_of(wait):
        for i in range(steps):
            positions.copy_(b.d[4])
            slots.copy_(torch.gather(tables, 1, (b.d[4] // PAGE).long()[:, None])[:, 0] * PAGE + b.d[4] % PAGE)
            k0 = rows[i].data_ptr() + 2 * heads * dim
            assert L.oa_k_rotary_cache(ptr(rows[i]), width, k0, k0 + 2 * n_kv * dim, width, ptr(outs[i]), heads * dim, ptr(cache), 200, ptr(positions), ptr(slots), n, heads, n_kv, dim, dim, 1,
                                       freqs.ctypes.data, 1.0, ptr(b.status), now()) == 0
            b.d[4].add_(1)
            if wait:
                torch.cuda.synchronize()
            assert b.call(L, q=outs[i], out=outs[i]) == 0
            if wait:
                torch.cuda.synchronize()

    def again():
        cache.copy_(before), b.d[4].copy_(start), outs.zero_()

    before = cache.clone()
    steps_of(wait=True)
    want, last = outs.clone(), cache.clone()
    assert b.status.item() == 0 and torch.isfinite(want).all() and b.d[4].tolist() == [x + steps for x in own]
    if captured:
        again()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            steps_of(wait=False)
    for _ in range(4):
        again()
        graph.replay() if captured else steps_of(wait=False)
        torch.cuda.synchronize()
        assert same_bits(outs, want) and same_bits(cache, last)
    b.own = [x + steps for x in own]
    q = torch.empty(n, heads * dim, dtype=torch.bfloat16, device="cuda")
    assert L.oa_k_rotary(ptr(rows[-1]), width, ptr(q), heads * dim, ptr(positions), n, heads, dim, dim, 1, freqs.ctypes.data, 1.0, 0, 0, now()) == 0
    b.check(out=outs[-1], q=q)


def test_two_captured_calls_at_once(L):
    """Two graphs on two streams, replayed over one another: neither has the other's scratch."""
    bs = [Batch(32, 8, 128, [900], [0, 30], [(i * 29) % 300 for i in range(30)], seed=15), Batch(8, 2, 64, [5000], [0, 50], [(i * 17) % 90 for i in range(50)], seed=16)]
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for b in bs:
        run(L, b)
        b.first = b.out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(3):
                assert b.call(L) == 0
        graphs.append(graph)
    for _ in range(20):
        for b, s, g in zip(bs, streams, graphs):
            with torch.cuda.stream(s):
                b.out.fill_(5.0)
                g.replay()
    torch.cuda.synchronize()
    for b in bs:
        assert same_bits(b.out, b.first)


@pytest.mark.parametrize("heads,n_kv,dim", [(8, 2, 128), (8, 2, 64), (5, 1, 128)])
def test_prompts_on_a_cache_that_was_cleared_once(L, heads, n_kv, dim):
    """Prompts of any length grow into pages, are rotated and written by one call and attended to by oa_k_paged_attention, whose tables name nothing (-1) behind a row's end; then pages are freed,
    handed on as they are and grown into again by shorter prompts.  The one condition is a cache that was cleared after its allocation."""
    width, pages = 8, 64
    cache = torch.zeros((2, pages, n_kv, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    rng, (freqs, amp) = np.random.default_rng(5), frequencies(L, dim)
    for lens in ([1, 63, 64, 65, 127, 128, 129, 200, 300], [300, 17, 64, 1, 100, 129, 5, 65, 191], [2, 3, 1, 66, 70, 190, 130, 64, 63]):
        n = len(lens)
        tables, have, refs = np.full((n, width), -1, np.int32), np.zeros(n, np.int32), np.zeros(pages, np.int32)
        refs[rng.permutation(pages)[:20]] = 1                                          # pages that another part of a program holds
        table = _lib.OaPageTable(tables.ctypes.data, have.ctypes.data, refs.ctypes.data, n, width, pages)
        for r, x in enumerate(lens):
            assert L.oa_host_cache_grow(table, r, x) == 0
        at = [(r, i) for r, x in enumerate(lens) for i in range(x)]
        qkv = randn(sum(lens) + dim, (len(at), (heads + 2 * n_kv) * dim))
        q, out = (torch.empty((len(at), heads * dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        k0, slots, where = qkv.data_ptr() + 2 * heads * dim, [int(tables[r, i // PAGE]) * PAGE + i % PAGE for r, i in at], cuda_i32([i for _, i in at])
        assert L.oa_k_rotary_cache(ptr(qkv), qkv.shape[1], k0, k0 + 2 * n_kv * dim, qkv.shape[1], ptr(q), heads * dim, ptr(cache), pages, ptr(where), ptr(cuda_i32(slots)), len(at), heads, n_kv, dim, dim,
                                   1, freqs.ctypes.data, amp, None, now()) == 0
        ctx = np.array(lens, np.int32)
        assert L.oa_k_paged_attention(ptr(q), ptr(out), ptr(cache), pages, tables.ctypes.data, width, ctx.ctypes.data, ctx.ctypes.data, n, heads, n_kv, dim, 0, now()) == 0
        torch.cuda.synchronize()
        first = 0
        for r, x in enumerate(lens):
            rows = torch.tensor(tables[r, : -(-x // PAGE)].astype(np.int64), device="cuda")
            k, v = (cache[p, rows].double().transpose(1, 2).reshape(-1, n_kv, dim)[:x] for p in (0, 1))
            y = q[first:first + x].double().view(x, n_kv, -1, dim)
            s = torch.einsum("tkhd,pkd->tkhp", y, k) / dim ** 0.5
            seen = (torch.arange(x, device="cuda")[None] <= torch.arange(x, device="cuda")[:, None])[:, None, None]
            p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
            want, size = torch.einsum("tkhp,pkd->tkhd", p, v), torch.einsum("tkhp,pkd->tkhd", p, v.abs())
            got = out[first:first + x].double().view(want.shape)
            # a weight rounded to bf16, scores as sums of products in fp32 that move a weight by twice that, the result's own rounding
            score = torch.einsum("tkhd,pkd->tkhp", y.abs(), k.abs()).amax(-1, keepdim=True) / dim ** 0.5
            tol = size * (2.0 ** -8 + 2 * (dim + 4) * 2.0 ** -24 * score + 2.0 ** -18) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -133
            assert bool(((got - want).abs() <= tol).all()), (lens, r, ((got - want).abs() / tol).max().item())
            first += x
        everyone = np.arange(n, dtype=np.int32)
        assert L.oa_host_cache_free(table, everyone.ctypes.data, n) == 0 and (have == 0).all() and (tables == -1).all() and refs.sum() == 20


# ---- errors ---------------------------------------------------------------------------------------------
def test_a_call_that_found_no_memory_leaves_no_error_behind(L):
    """Scratch of over a terabyte: the call says so with its code and text, nothing is launched, and the program's next CUDA call does not meet the error again."""
    buf = torch.zeros(9 << 20, dtype=torch.bfloat16, device="cuda")                     # a cache of one page, and the first of q's rows behind it
    ints, before = torch.zeros(64, dtype=torch.int32, device="cuda"), L.oa_kernel_launches()
    n, heads, n_kv, dim = 2 ** 18, 16384, 1024, 64
    q = C.c_void_p(buf.data_ptr() + 2 * n_kv * PAGE * dim * 2)                          # in place; nothing is launched that could go beyond it
    for again in range(2):
        code = L.oa_k_prefix_attention(q, heads * dim, q, heads * dim, ptr(buf), 1, ptr(ints), 10 ** 4, ptr(ints), ptr(ints), 1, ptr(ints), 8, ptr(ints), n, heads, n_kv, dim, 0.0, None, now())
        assert code == 500 and "scratch" in _lib.last_error(), (code, _lib.last_error())
        assert L.oa_kernel_launches() == before
        assert torch.ones(8, device="cuda").mul_(2).sum().item() == 16.0
    b = Batch(8, 2, 128, [100], [0, 1], [7], seed=3)
    run(L, b)
    b.check()


# ---- threads ----------------------------------------------------------------------------------------------
def test_two_threads_on_two_streams(L):
    """Each thread has a cache, tables, a stream and errors of its own; every result is the one that the calls give alone."""
    wanted = []
    for t in range(2):
        b = Batch(32, 8, 128, [900], [0, 30], [(i * 29) % 300 for i in range(30)], seed=15) if t else Batch(8, 2, 64, [5000], [0, 50], [(i * 17) % 90 for i in range(50)], seed=16)
        a = Appends(L, 700 + 600 * t, seed=t)
        run(L, b), a.reset()
        assert a.call() == 0
        torch.cuda.synchronize()
        wanted.append((b, b.out.clone(), a, a.outputs()))
    failures, start = [], threading.Barrier(2)

    def work(t):
        try:
            b, first, a, outputs = wanted[t]
            side = torch.cuda.Stream()
            stream = C.c_void_p(side.cuda_stream)
            start.wait()
            with torch.cuda.stream(side):
                for i in range(30):
                    b.out.fill_(5.0), a.reset()
                    assert b.call(L, stream=stream) == 0 and a.call(stream) == 0
                    assert L.oa_k_cache_copy(ptr(a.cache), 0 if t else 2, a.pages, 2, 128, 2 if t else 3, a.moves, 1, stream) == 400 and "cache copy" in _lib.last_error()
                    assert L.oa_k_prefix_attention(None, 0, None, 0, None, 1, None, 1, None, None, 0, None, 1, None, 1, 8, 2, 96 + t, 0.0, None, stream) == 400 and "64 or 128" in _lib.last_error()
                    if i % 10 == 9:
                        side.synchronize()
                        assert same_bits(b.out, first) and all(same_bits(x, y) for x, y in zip(a.outputs(), outputs)), (t, i)
        except BaseException as e:      # noqa: BLE001
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures
