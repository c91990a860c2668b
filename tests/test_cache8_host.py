"""What the operators on caches of 8 bits and on several new tokens refuse before they touch a device, no GPU."""
import math

import numpy as np
import pytest

from opsagent_b200 import _lib

P, Q = 1 << 20, 3 << 20                                                                      # an address that is never followed


@pytest.fixture(scope="module")
def L():
    return _lib.load()


ROWS = [dict(dim=8), dict(dim=72), dict(dim=0), dict(dim=272), dict(kv=0), dict(kv=4097), dict(pages=0), dict(pages=-1), dict(fmt=0), dict(fmt=3), dict(T=-1), dict(ld=127), dict(k=None), dict(v=None),
        dict(cache=None), dict(slots=None), dict(k=P + 1), dict(v=P + 4097), dict(cache=2 * P + 8), dict(slots=P + 2), dict(status=P + 3), dict(ld=1 << 38), dict(k=2 * P), dict(v=2 * P + 100), dict(k=2 * P - 512),
        dict(slots=P + 8), dict(slots=P + 4096 - 16), dict(slots=P + 4096 + 256), dict(slots=2 * P - 16), dict(slots=2 * P + 8), dict(status=P), dict(status=P + 4096 + 1276), dict(status=2 * P + 4), dict(status=Q), dict(status=Q + 16)]


@pytest.mark.parametrize("case", ROWS)
@pytest.mark.parametrize("read", [False, True])
def test_rows_refuse(L, case, read):
    a = dict(k=P, v=P + 4096, ld=128, cache=2 * P, pages=4, slots=Q, T=5, kv=2, dim=64, fmt=1, status=None)
    a.update(case)
    if read:
        rc = L.oa_k_cache8_read(a["cache"], a["pages"], a["slots"], a["T"], a["kv"], a["dim"], a["fmt"], a["k"], a["v"], a["ld"], a["status"], None)
    else:
        rc = L.oa_k_cache8_write(a["k"], a["v"], a["ld"], a["cache"], a["pages"], a["slots"], a["T"], a["kv"], a["dim"], a["fmt"], a["status"], None)
    assert rc == 400 and "8-bit cache" in _lib.last_error(), case


def test_rows_that_are_read_do_not_overlap(L):
    def read(k, v, ld, T=5):
        rc = L.oa_k_cache8_read(1 << 40, 4, Q, T, 2, 64, 1, k, v, ld, None, None)
        return rc == 400 and "overlap" in _lib.last_error()
    assert read(P, P, 128) and read(P, P + 64, 256) and read(P, P + 256, 200) and read(P, P + 1024, 128)
    assert not read(P, P + 256, 256) and not read(P, P + 5 * 256, 128) and not read(P, P + 256, 128, T=1)


def test_no_rows_and_no_moves(L):
    assert L.oa_k_cache8_write(None, None, 128, None, 4, None, 0, 2, 64, 1, None, None) == 0 and L.oa_k_cache8_read(None, 4, None, 0, 2, 64, 2, None, None, 128, None, None) == 0
    assert L.oa_k_cache8_copy(None, 2, 8, 2, 64, None, 0, None) == 0


def test_copy_refuses(L):
    def call(moves, cache=P, planes=2, pages=8, kv=2, dim=64):
        m = (_lib.OaPageMove * max(1, len(moves)))(*[_lib.OaPageMove(*x) for x in moves])
        return L.oa_k_cache8_copy(cache, planes, pages, kv, dim, m, len(moves), None)
    for moves in ([(0, 8, 64)], [(8, 0, 64)], [(-1, 0, 64)], [(0, -1, 64)], [(0, 1, 65)], [(0, 1, -1)], [(0, 1, 64), (2, 1, 64)], [(0, 1, 64), (1, 2, 64)], [(1, 2, 64), (0, 1, 64)], [(3, 3, 64)]):
        assert call(moves) == 400 and "cache copy" in _lib.last_error(), moves
    for case in [dict(planes=0), dict(pages=0), dict(kv=0), dict(kv=4097), dict(dim=0), dict(dim=8), dict(dim=264), dict(cache=None), dict(cache=P + 8)]:
        assert call([(0, 1, 64)], **case) == 400 and "8-bit cache" in _lib.last_error(), case
    assert L.oa_k_cache8_copy(P, 2, 8, 2, 64, None, 1, None) == 400 and L.oa_k_cache8_copy(P, 2, 8, 2, 64, None, -1, None) == 400


def attention(L, q=P, ldq=1024, out=P, ldo=1024, cache=1 << 40, fmt=1, pages=8, tables=Q, width=4, ctx=Q + 4096, starts=Q + 8192, seen=Q + 12288, seqs=3, rows=9, heads=8, kv=2, dim=128, window=0, sinks=0, scale=0.0, status=None):
    return L.oa_k_tree_attention(q, ldq, out, ldo, cache, fmt, pages, tables, width, ctx, starts, seen, seqs, rows, heads, kv, dim, window, sinks, scale, status, None)


@pytest.mark.parametrize("case", [
    dict(dim=96), dict(dim=32), dict(dim=256), dict(fmt=3), dict(fmt=-1), dict(heads=7), dict(heads=0), dict(kv=0), dict(kv=1025, heads=1025, ldq=1 << 18, ldo=1 << 18), dict(heads=34, ldq=8192, ldo=8192), dict(seqs=-1),
    dict(seqs=(1 << 20) + 1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(width=0), dict(width=(1 << 24) + 1), dict(pages=0), dict(pages=1 << 24), dict(fmt=0, pages=1 << 24), dict(window=63), dict(window=1),
    dict(window=-64), dict(sinks=-1, window=64), dict(sinks=1), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(ldq=1023), dict(ldq=1028), dict(ldo=1000), dict(ldo=1028), dict(q=None), dict(out=None),
    dict(cache=None), dict(tables=None), dict(ctx=None), dict(starts=None), dict(q=P + 2), dict(out=P + 8), dict(cache=(1 << 40) + 8), dict(tables=P + 2), dict(ctx=P + 1), dict(starts=P + 2), dict(seen=P + 4),
    dict(status=P + 1), dict(out=P + 16), dict(out=P + 9 * 2048 - 16), dict(ldq=1 << 37), dict(ldo=1 << 37, out=1 << 30), dict(out=(1 << 40) - 2048), dict(out=(1 << 40) + 8 * 2 * 2 * 64 * 132 - 16),
    dict(out=Q + 32), dict(out=Q + 4096), dict(out=Q + 4096 - 9 * 2048 + 16), dict(out=Q + 8192), dict(out=Q + 12288), dict(out=Q + 12288 + 64), dict(status=P + 9 * 2048 - 4), dict(out=Q + 65536, status=Q + 65536),
    dict(status=Q), dict(status=Q + 44), dict(status=Q + 4096 + 8), dict(status=Q + 8192 + 12), dict(status=Q + 12288 + 68), dict(status=(1 << 40) + 64), dict(q=Q + 65536, status=Q + 65536 + 9 * 2048 - 4)])
def test_attention_refuses(L, case):
    assert attention(L, **case) == 400, case
    assert "tree attention" in _lib.last_error()


def test_attention_beside_its_arrays(L):
    for case in [dict(status=Q + 48), dict(status=Q + 4096 + 12), dict(status=Q + 8192 + 16), dict(status=Q + 12288 + 72), dict(status=P + 9 * 2048), dict(status=P - 4), dict(out=Q + 12288 + 80, seen=Q + 12288), dict(seen=None, out=Q + 12288),
                 dict(status=(1 << 40) - 4), dict(status=(1 << 40) + 8 * 2 * 2 * 64 * 132)]:
        assert "tree attention" not in (attention(L, **case), _lib.last_error())[1], case


def test_attention_of_nothing(L):
    assert attention(L, seqs=0) == 0 and attention(L, rows=0) == 0
    beside = "overlap" not in (attention(L, out=P + 9 * 2048), _lib.last_error())[1]
    assert beside and "overlap" not in (attention(L, out=(1 << 40) + 8 * 2 * 2 * 64 * 132), _lib.last_error())[1] and "overlap" not in (attention(L, out=(1 << 40) - 9 * 2048), _lib.last_error())[1]


def test_host_memory_is_not_run_on(L):
    before = L.oa_kernel_launches()
    x = np.zeros(1 << 20, np.uint8)
    p = (x.ctypes.data + 1023) // 1024 * 1024
    moves = (_lib.OaPageMove * 1)(_lib.OaPageMove(0, 1, 3))
    assert L.oa_k_cache8_write(p, p + 4096, 128, p + 65536, 2, p + 8192, 2, 2, 64, 1, None, None) in (400, 500)
    assert L.oa_k_cache8_read(p + 65536, 2, p + 8192, 2, 2, 64, 1, p, p + 4096, 128, None, None) in (400, 500)
    assert L.oa_k_cache8_copy(p, 2, 2, 2, 64, moves, 1, None) in (400, 500)
    assert L.oa_k_tree_attention(p, 128, p + 4096, 128, p + 65536, 1, 2, p + 8192, 1, p + 8192, p + 8192, None, 1, 1, 2, 2, 64, 0, 0, 0.0, None, None) in (400, 500)
    assert L.oa_kernel_launches() == before


def test_copies_in_caches_that_no_memory_holds(L):
    """What a launch cannot count is refused as other arguments are, and not as a fault of the device."""
    one = (_lib.OaPageMove * 1)(_lib.OaPageMove(0, 1, 64))
    for planes, pages, kv, dim in [(2 ** 31 - 1, 8, 4096, 256), (2 ** 31 - 1, 2 ** 31 - 1, 1, 16), (2 ** 22, 64, 8, 128), (64, 2 ** 30, 4096, 64)]:
        assert L.oa_k_cache8_copy(P, planes, pages, kv, dim, one, 1, None) == 400 and "memory" in _lib.last_error(), (planes, pages)
        assert L.oa_k_cache_copy(P, planes, pages, kv, dim, 2, one, 1, None) == 400 and "memory" in _lib.last_error(), (planes, pages)
    for planes, pages, kv, dim in [(2, 2, 1, 16), (128, 2 ** 15, 8, 128)]:
        assert "memory reaches" not in (L.oa_k_cache8_copy(P, planes, pages, kv, dim, one, 1, None), _lib.last_error())[1]
        assert "memory reaches" not in (L.oa_k_cache_copy(P, planes, pages, kv, dim, 2, one, 1, None), _lib.last_error())[1]
