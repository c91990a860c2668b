"""Caches of 8 bits at sizes whose offsets pass 32 bits: blocks of a cache, rows far apart, copies between them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402
from test_cache8_gpu import E4M3, INT8, dev, now, parts, ptr, quantised, randn  # noqa: E402


@pytest.fixture(scope="module")
def L():
    return _lib.load()


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_a_cache_beyond_32_bits(L, fmt):
    """5.4 GB: tokens of the last pages written, read back, and copied to the first one's neighbour and the other way round."""
    pages, n_kv, dim = 40000, 8, 128
    cache = torch.zeros((2, pages, n_kv, 64 * (dim + 4)), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 2 ** 32
    slots = np.array([0, 5, (pages - 1) * 64 + 63, (pages - 2) * 64, 20000 * 64 + 7], np.int32)
    kv = randn(1, (len(slots), 2, n_kv, dim))
    s, ld = dev(slots), 2 * n_kv * dim
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = kv[:, 0], kv[:, 1]
    assert L.oa_k_cache8_write(ptr(k), ptr(v), ld, ptr(cache), pages, ptr(s), len(slots), n_kv, dim, fmt, ptr(status), now()) == 0, _lib.last_error()
    out = torch.empty_like(kv)
    assert L.oa_k_cache8_read(ptr(cache), pages, ptr(s), len(slots), n_kv, dim, fmt, ptr(out[:, 0]), ptr(out[:, 1]), ld, ptr(status), now()) == 0, _lib.last_error()
    y, scale = (torch.from_numpy(x).cuda() for x in quantised(kv, fmt))           # [token, plane, head, ..]
    bits, scales = parts(cache, dim)
    for i, slot in enumerate(slots.tolist()):
        assert torch.equal(bits[:, slot // 64, :, slot % 64], y[i]) and torch.equal(scales[:, slot // 64, :, slot % 64], scale[i]), slot
    assert torch.equal(out, ((y.view(torch.float8_e4m3fn) if fmt == E4M3 else y.view(torch.int8)).float() * scale[..., None]).bfloat16())
    moves = (_lib.OaPageMove * 2)(_lib.OaPageMove(pages - 1, 1, 64), _lib.OaPageMove(0, pages - 3, 6))
    assert L.oa_k_cache8_copy(ptr(cache), 2, pages, n_kv, dim, moves, 2, now()) == 0, _lib.last_error()
    torch.cuda.synchronize()
    assert torch.equal(cache[:, 1], cache[:, pages - 1]) and cache[:, 1].any() and status.item() == 0
    assert torch.equal(bits[:, pages - 3, :, :6], bits[:, 0, :, :6]) and torch.equal(scales[:, pages - 3, :, :6], scales[:, 0, :, :6]) and not bits[:, pages - 3, :, 6:].any()


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_rows_that_are_gigabytes_apart(L, fmt):
    """Three rows with a pitch of 2^30 elements and eight more: the last one starts 4.3 GB behind the first."""
    n_kv, dim, ld = 2, 64, 2 ** 30 + 8
    memory = torch.empty(2 * ld + 2 * n_kv * dim, dtype=torch.bfloat16, device="cuda")
    rows = [memory[i * ld: i * ld + 2 * n_kv * dim] for i in range(3)]
    want = randn(2, (3, 2 * n_kv * dim))
    for r, w in zip(rows, want):
        r.copy_(w)
    small, large = (torch.zeros((2, 3, n_kv, 64 * (dim + 4)), dtype=torch.uint8, device="cuda") for _ in range(2))
    s = dev([70, 3, 191])
    wide = 2 * n_kv * dim
    v = n_kv * dim * 2                                                           # values lie behind the keys of their row
    assert L.oa_k_cache8_write(want.data_ptr(), want.data_ptr() + v, wide, ptr(small), 3, ptr(s), 3, n_kv, dim, fmt, None, now()) == 0, _lib.last_error()
    assert L.oa_k_cache8_write(memory.data_ptr(), memory.data_ptr() + v, ld, ptr(large), 3, ptr(s), 3, n_kv, dim, fmt, None, now()) == 0, _lib.last_error()
    torch.cuda.synchronize()
    assert torch.equal(small, large) and small.any()
    for r in rows:
        r.zero_()
    back = torch.empty_like(want)
    assert L.oa_k_cache8_read(ptr(small), 3, ptr(s), 3, n_kv, dim, fmt, back.data_ptr(), back.data_ptr() + v, wide, None, now()) == 0, _lib.last_error()
    assert L.oa_k_cache8_read(ptr(small), 3, ptr(s), 3, n_kv, dim, fmt, memory.data_ptr(), memory.data_ptr() + v, ld, None, now()) == 0, _lib.last_error()
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(rows), back) and back.any()
