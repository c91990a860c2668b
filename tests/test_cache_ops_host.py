"""Host side of the operators on a caller's paged cache, no GPU: rotary frequencies, the bookkeeping of pages against a plain model of it, and what the
entry points refuse before they touch a device."""
import ctypes as C
import math
import random

import numpy as np
import pytest

from opsagent_b200 import _lib

PAGE = 64


@pytest.fixture(scope="module")
def L():
    return _lib.load()


# ---- rotary frequencies ------------------------------------------------------------------------
def freqs(L, dims, base, scaling=0, factor=1.0, first=0.0, second=0.0, original=0):
    out, amp = np.full(max(1, dims // 2) + 1, np.nan), C.c_float()
    rc = L.oa_host_rotary_freqs(dims, base, scaling, factor, first, second, original, out.ctypes.data, C.byref(amp))
    assert rc == 0 and np.isnan(out[dims // 2:]).all()
    return out[: dims // 2], amp.value


@pytest.mark.parametrize("dims", [2, 6, 64, 96, 128, 256])
@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
def test_frequencies_follow_their_formulas(L, dims, scaling):
    base, factor, first, second, original = {0: (10000.0, 1.0, 0, 0, 0), 1: (10000.0, 8.0, 0, 0, 0), 2: (500000.0, 32.0, 1.0, 4.0, 8192), 3: (1e6, 4.0, 32.0, 1.0, 32768)}[scaling]
    got, amp = freqs(L, dims, base, scaling, factor, first, second, original)
    for i, f in enumerate(got):
        want = base ** (-2.0 * i / dims)
        if scaling == 1:
            want /= factor
        if scaling == 2:
            turns = original * want / (2 * math.pi)
            if turns < first:
                want /= factor
            elif turns < second:
                share = (turns - first) / (second - first)
                want = (1 - share) * want / factor + share * want
        if scaling == 3:
            where = lambda t: dims * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(where(first)), 0), min(math.ceil(where(second)), dims - 1)
            ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            want = want / factor * ramp + want * (1 - ramp)
        assert abs(f - want) <= 8 * 2.0 ** -53 * want, (i, f, want)      # a power, two products and a sum in 64 bits
    assert amp == np.float32(0.1 * math.log(factor) + 1.0 if scaling == 3 else 1.0)


@pytest.mark.parametrize("args", [(3, 1e4, 0, 1.0, 0, 0, 0), (-2, 1e4, 0, 1.0, 0, 0, 0), (258, 1e4, 0, 1.0, 0, 0, 0), (64, 0.0, 0, 1.0, 0, 0, 0), (64, math.nan, 0, 1.0, 0, 0, 0),
                                  (64, 1e4, 4, 1.0, 0, 0, 0), (64, 1e4, -1, 1.0, 0, 0, 0), (64, 1e4, 1, 0.0, 0, 0, 0), (64, 1e4, 1, math.inf, 0, 0, 0), (64, 1e4, 2, 8.0, 4.0, 1.0, 8192),
                                  (64, 1e4, 2, 8.0, 1.0, 4.0, 0), (64, 1e4, 3, 0.5, 32.0, 1.0, 4096), (64, 1.0, 3, 4.0, 32.0, 1.0, 4096), (64, 1e4, 3, 4.0, 0.0, 1.0, 4096)])
def test_frequencies_refuse(L, args):
    out, amp = np.zeros(256), C.c_float()
    assert L.oa_host_rotary_freqs(*args, out.ctypes.data, C.byref(amp)) == 400
    assert "rotary" in _lib.last_error() and not out.any()


# ---- pages --------------------------------------------------------------------------------------
class Table:
    def __init__(self, rows, width, pages):
        self.tables, self.lens, self.refs = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32)
        self.c = _lib.OaPageTable(self.tables.ctypes.data, self.lens.ctypes.data, self.refs.ctypes.data, rows, width, pages)
        self.moves, self.n = (_lib.OaPageMove * (pages + rows))(), C.c_int32(-1)

    def copy(self):
        return self.tables.copy(), self.lens.copy(), self.refs.copy()

    def same(self, was):
        return all(np.array_equal(a, b) for a, b in zip(self.copy(), was))

    def held(self, row):
        return self.tables[row, : -(-int(self.lens[row]) // PAGE)].tolist()

    def done(self):
        return [(m.src, m.dst, m.tokens) for m in self.moves[: self.n.value]]


def i32(a):
    return np.ascontiguousarray(a, np.int32)


def grow(L, t, row, n):
    return L.oa_host_cache_grow(t.c, row, n)


def free(L, t, rows):
    rows = i32(rows)
    return L.oa_host_cache_free(t.c, rows.ctypes.data, rows.size)


def fork(L, t, parent, children, cap=None):
    children = i32(children)
    return L.oa_host_cache_fork(t.c, parent, children.ctypes.data, children.size, t.moves, len(t.moves) if cap is None else cap, C.byref(t.n))


def compact(L, t, cap=None):
    return L.oa_host_cache_compact(t.c, t.moves, len(t.moves) if cap is None else cap, C.byref(t.n))


@pytest.mark.parametrize("seed", range(6))
def test_a_life_of_a_cache_against_a_plain_model(L, seed):
    """Random growing, forking, ending and compacting; the model keeps what every place holds (a name per token), moves are carried out on it."""
    rng = random.Random(seed)
    rows, width, pages = 9, 5, 22
    t = Table(rows, width, pages)
    content = [[None] * PAGE for _ in range(pages)]                       # what the cache's places hold
    text = [[] for _ in range(rows)]                                       # what each row should read
    name = 0
    for _ in range(400):
        was, what = t.copy(), rng.randrange(4)
        if what == 0:
            r, n = rng.randrange(rows), rng.choice([0, 1, 5, 63, 64, 65, 130])
            rc = grow(L, t, r, n)
            need = -(-(len(text[r]) + n) // PAGE) - -(-len(text[r]) // PAGE)
            assert rc == (400 if len(text[r]) + n > width * PAGE else 429 if need > int((was[2] == 0).sum()) else 0)
            if rc == 0:
                assert t.held(r)[len(t.held(r)) - need:] == np.flatnonzero(was[2] == 0)[:need].tolist()      # lowest-numbered
                for i in range(len(text[r]), len(text[r]) + n):
                    content[t.tables[r, i // PAGE]][i % PAGE] = name
                    text[r].append(name)
                    name += 1
        elif what == 1:
            p, kids = rng.randrange(rows), rng.sample(range(rows), rng.randint(0, 3))
            rc = fork(L, t, p, kids)
            tail = len(text[p]) % PAGE
            if p in kids or any(text[k] for k in kids):
                assert rc == 400
            elif tail and len(kids) > int((was[2] == 0).sum()):
                assert rc == 429
            else:
                assert rc == 0 and t.n.value == (len(kids) if tail else 0)
                for s, d, n in t.done():
                    assert was[2][d] == 0 and n == tail
                    content[d][:n] = content[s][:n]
                for k in kids:
                    text[k] = list(text[p])
        elif what == 2:
            some = [rng.randrange(rows) for _ in range(rng.randint(0, 3))]
            rc = free(L, t, some)
            assert rc == 0
            for r in some:
                text[r] = []
                assert (t.tables[r] == -1).all()
        else:
            rc = compact(L, t)
            assert rc == 0
            used = int((t.refs > 0).sum())
            assert (t.refs[:used] > 0).all() and not t.refs[used:].any()
            assert [m[0] for m in t.done()] == sorted(p for p in np.flatnonzero(was[2] > 0) if p >= used) and all(m[2] == PAGE for m in t.done())
            assert not {m[0] for m in t.done()} & {m[1] for m in t.done()}
            new = [list(c) for c in content]
            for s, d, _ in t.done():
                new[d] = list(content[s])
            content = new
        if rc:
            assert t.same(was)
        count = np.zeros(pages, np.int32)
        for r in range(rows):
            assert t.lens[r] == len(text[r])
            assert [content[t.tables[r, i // PAGE]][i % PAGE] for i in range(len(text[r]))] == text[r]
            np.add.at(count, t.held(r), 1)
        assert np.array_equal(count, t.refs)


def test_page_calls_refuse_and_change_nothing(L):
    t = Table(4, 3, 6)
    assert grow(L, t, 0, 70) == 0 and grow(L, t, 1, 64) == 0
    was = t.copy()
    assert grow(L, t, 4, 1) == 400 and grow(L, t, -1, 1) == 400 and grow(L, t, 0, -1) == 400 and grow(L, t, 0, 3 * PAGE) == 400 and grow(L, t, 0, 2 ** 31 - 1) == 400
    assert fork(L, t, 0, [1]) == 400 and fork(L, t, 0, [2, 2]) == 400 and fork(L, t, 0, [0]) == 400 and fork(L, t, 0, [7]) == 400 and fork(L, t, 9, [2]) == 400
    assert fork(L, t, 0, [2, 3], cap=1) == 400
    assert free(L, t, [0, 5]) == 400 and free(L, t, [-1]) == 400
    assert L.oa_host_cache_grow(None, 0, 1) == 400 and L.oa_host_cache_compact(t.c, None, 4, C.byref(t.n)) == 400 and L.oa_host_cache_compact(t.c, t.moves, 4, None) == 400
    assert t.same(was) and "compact" in _lib.last_error()


@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1, -2 ** 31, 5])          # outside the cache, and one that is free
def test_bad_pages_are_refused(L, page):
    t = Table(3, 3, 6)
    assert grow(L, t, 0, 130) == 0
    t.tables[0, 1] = page
    was = t.copy()
    assert grow(L, t, 0, 1) == 400 and fork(L, t, 0, [1]) == 400 and free(L, t, [0]) == 400 and compact(L, t) == 400
    assert t.same(was)


def test_bad_lengths_and_counts_are_refused(L):
    for n in (-1, 3 * PAGE + 1, 2 ** 31 - 1):
        t = Table(2, 3, 6)
        t.lens[0] = n
        was = t.copy()
        assert grow(L, t, 0, 1) == 400 and free(L, t, [0]) == 400 and compact(L, t) == 400 and t.same(was)
    t = Table(2, 3, 6)
    assert grow(L, t, 0, 64) == 0
    t.tables[1, 0], t.lens[1] = t.tables[0, 0], 64                          # two rows, one reference
    was = t.copy()
    assert free(L, t, [0, 1]) == 400 and t.same(was)
    t.refs[5] = -1
    was = t.copy()
    assert compact(L, t) == 400 and t.same(was)


def test_a_shared_page_that_is_not_full_is_not_grown(L):
    t = Table(2, 3, 6)
    assert grow(L, t, 0, 10) == 0
    t.tables[1, 0], t.lens[1], t.refs[0] = 0, 10, 2                         # shared by hand, without a fork
    was = t.copy()
    assert grow(L, t, 0, 1) == 400 and t.same(was)
    assert grow(L, t, 0, 0) == 0 and t.same(was)


# ---- what the GPU entry points refuse, before a device is asked for -----------------------------------
BUF = np.zeros(4096, np.int32)
P = (BUF.ctypes.data + 15) // 16 * 16


def test_rotary_refuses(L):
    f = np.ones(128)

    def call(x=P, ldx=256, out=P, ldo=256, pos=P, T=2, heads=2, dim=128, rot=64, layout=1, fr=f, amp=1.0, f32=0):
        return L.oa_k_rotary(x, ldx, out, ldo, pos, T, heads, dim, rot, layout, fr.ctypes.data if fr is not None else None, amp, 0, f32, None)

    assert call(T=0) == 0                                                    # nothing to do, nothing touched
    bad = [dict(T=-1), dict(heads=0), dict(dim=127, rot=64), dict(dim=0, rot=0), dict(rot=63), dict(rot=-2), dict(rot=130), dict(dim=512, ldx=1024, ldo=1024, rot=258), dict(layout=2),
           dict(fr=None), dict(fr=np.full(128, np.inf)), dict(amp=math.nan), dict(ldx=255), dict(ldo=255), dict(x=None), dict(out=None), dict(pos=None), dict(x=P + 1),
           dict(x=P + 2, out=P + 2, f32=1), dict(pos=P + 2), dict(out=P + 16), dict(out=P + 2 * 256 + 4), dict(ldo=264)]
    for case in bad:
        assert call(**case) == 400, case
        assert "rotary" in _lib.last_error()


def test_rotary_cache_refuses(L):
    f = np.ones(64)

    def call(q=P, ldq=256, k=P, v=P, ldkv=128, qo=P, ldqo=256, cache=P, pages=4, pos=P, slots=P, T=2, heads=2, kv=1, status=None):
        return L.oa_k_rotary_cache(q, ldq, k, v, ldkv, qo, ldqo, cache, pages, pos, slots, T, heads, kv, 128, 128, 1, f.ctypes.data, 1.0, status, None)

    assert call(T=0) == 0
    for case in [dict(kv=0), dict(pages=0), dict(ldkv=127), dict(ldq=255), dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(cache=None), dict(pos=None), dict(slots=None), dict(k=P + 1),
                 dict(slots=P + 1), dict(status=P + 2), dict(qo=P + 256), dict(T=-3)]:
        assert call(**case) == 400, case


def test_cache_copy_refuses(L):
    def call(moves, cache=P, planes=2, pages=8, kv=2, dim=64, esz=2):
        m = (_lib.OaPageMove * max(1, len(moves)))(*[_lib.OaPageMove(*x) for x in moves])
        return L.oa_k_cache_copy(cache, planes, pages, kv, dim, esz, m, len(moves), None)

    assert call([]) == 0 and call([], cache=None) == 0
    for moves in ([(0, 8, 64)], [(8, 0, 64)], [(-1, 0, 64)], [(0, -1, 64)], [(0, 1, 65)], [(0, 1, -1)], [(0, 1, 64), (2, 1, 64)], [(0, 1, 64), (1, 2, 64)], [(1, 2, 64), (0, 1, 64)], [(3, 3, 64)]):
        assert call(moves) == 400, moves
    ok = [(0, 1, 64)]
    for case in [dict(planes=0), dict(pages=0), dict(kv=0), dict(dim=0), dict(dim=4), dict(esz=1), dict(esz=8), dict(cache=None), dict(cache=P + 8), dict(dim=4096)]:
        assert call(ok, **case) == 400, case
    assert L.oa_k_cache_copy(P, 2, 8, 2, 64, 2, None, 1, None) == 400 and L.oa_k_cache_copy(P, 2, 8, 2, 64, 2, None, -1, None) == 400


def test_prefix_attention_refuses(L):
    def call(q=P, ldq=1024, out=P, ldo=1024, cache=P, pages=8, pt=P, mp=2, pl=P, pr=P, n=1, ot=P, mo=2, ol=P, seqs=3, heads=8, kv=2, dim=128, scale=0.0, status=None):
        return L.oa_k_prefix_attention(q, ldq, out, ldo, cache, pages, pt, mp, pl, pr, n, ot, mo, ol, seqs, heads, kv, dim, scale, status, None)

    assert call(seqs=0) == 0
    for case in [dict(dim=96), dict(dim=32), dict(heads=7), dict(heads=0), dict(kv=0), dict(heads=34, ldq=8192, ldo=8192), dict(seqs=-1), dict(seqs=(1 << 20) + 1), dict(mo=0), dict(mp=0), dict(n=33),
                 dict(n=-1), dict(pages=0), dict(pages=1 << 24), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(ldq=1023), dict(ldq=1028), dict(ldo=1000), dict(ldo=1028), dict(q=None),
                 dict(out=None), dict(cache=None), dict(pt=None), dict(pl=None), dict(pr=None), dict(ot=None), dict(ol=None), dict(q=P + 2), dict(out=P + 8), dict(cache=P + 8), dict(pt=P + 2),
                 dict(status=P + 1), dict(out=P + 16)]:
        assert call(**case) == 400, case
        assert "prefix attention" in _lib.last_error()


def test_rows_that_overlap_are_refused(L):
    """Addresses alone: nothing behind them is touched before a device is found."""
    f, far = np.ones(64), 1 << 40

    def rotary(q=far, ldq=512, k=far + 512, v=far + 768, ldkv=512, qo=far, ldqo=512, cache=2 * far, T=5):
        _rc = L.oa_k_rotary_cache(q, ldq, k, v, ldkv, qo, ldqo, cache, 4, P, P, T, 2, 1, 128, 128, 1, f.ctypes.data, 1.0, None, None)
        return _rc, _lib.last_error()

    assert "overlap" not in rotary()[1]                                       # rows of q, k and v next to each other, q turned in place
    assert "overlap" not in rotary(T=1, qo=far + 1024)[1] and "overlap" not in rotary(qo=far + 10240, ldqo=256)[1]
    for case in [dict(qo=far + 512), dict(qo=far + 256), dict(k=far + 510), dict(v=far + 256), dict(qo=far + 1024 + 896), dict(qo=far + 3 * 1024 - 128), dict(qo=far - 16), dict(qo=far + 768, ldqo=256),
                 dict(cache=far), dict(cache=far - 4 * 2 * 64 * 128 * 2 + 16), dict(qo=2 * far + 64), dict(k=2 * far + 65536, ldkv=128)]:
        code, text = rotary(**case)
        assert code == 400 and "overlap" in text, case

    def attention(out, cache=2 * far):
        _rc = L.oa_k_prefix_attention(far, 1024, out, 1024, cache, 8, P, 2, P, P, 1, P, 2, P, 3, 8, 2, 128, 0.0, None, None)
        return _rc, _lib.last_error()

    assert "overlap" not in attention(far)[1] and "overlap" not in attention(far + 6144)[1] and "overlap" not in attention(2 * far - 6144)[1]
    for out in (far + 16, far + 6128, 2 * far - 6128, 2 * far, 2 * far + 8 * 2 * 2 * 64 * 128 * 2 - 16):
        code, text = attention(out)
        assert code == 400 and "overlap" in text, out


def test_host_memory_is_not_run_on(L):
    """Arguments in order, memory that is not a device's: an error, with or without a GPU, and no launch."""
    f = np.ones(64)
    before = L.oa_kernel_launches()
    assert L.oa_k_rotary(P, 256, P, 256, P, 2, 2, 128, 128, 1, f.ctypes.data, 1.0, 0, 0, None) in (400, 500)
    assert L.oa_k_cache_copy(P, 2, 8, 2, 64, 2, (_lib.OaPageMove * 1)(_lib.OaPageMove(0, 1, 3)), 1, None) in (400, 500)
    assert L.oa_k_prefix_attention(P, 1024, P, 1024, P, 8, P, 2, P, P, 1, P, 2, P, 3, 8, 2, 128, 0.0, None, None) in (400, 500)
    assert L.oa_kernel_launches() == before
