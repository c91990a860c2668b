"""Caches of 8 bits on the B200, through the C ABI: rows quantised as they are written, read back, pages copied, and a run of them with rotary positions, page tables and attention.

Writing and copying are defined to the bit.  Reading is one product in fp32 and one rounding to bf16, which torch does with the same bits."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402

PAGE = 64
E4M3, INT8 = 1, 2


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def ptr(t, offset=0):
    return C.c_void_p(t.data_ptr() + offset) if t is not None else None


def now():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def dev(a):
    return torch.from_numpy(np.array(a, np.int32)).cuda()


def randn(seed, shape, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()


def e4m3_of(x):
    """Bits of the nearest e4m3 value, ties to even: all 127 magnitudes are compared, in 64 bits."""
    codes = np.arange(127)
    mags = np.where(codes >> 3 > 0, (1 + (codes & 7) / 8) * 2.0 ** ((codes >> 3) - 7), (codes & 7) / 8 * 2.0 ** -6)
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    hi = np.minimum(np.searchsorted(mags, a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = mags[hi] - a, a - mags[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), mags


def quantised(x, fmt):
    """x [..., dim] bf16 -> (bytes, scales): IEEE divisions in fp32, by numpy."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(-1)
    with np.errstate(all="ignore"):
        scale = (top / np.float32(448 if fmt == E4M3 else 127)).astype(np.float32)
        y = (x / scale[..., None]).astype(np.float32)
    dead = ~(scale > 0) | ~np.isfinite(top)
    y = np.where(dead[..., None], np.float32(0), y)
    b = e4m3_of(y)[0] if fmt == E4M3 else np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    return b, np.where(np.isfinite(top), scale, np.float32(np.nan))


def test_the_oracle_knows_e4m3():
    codes, mags = e4m3_of([0.0, 1.0, 448.0, 500.0, 2.0 ** -9, 2.0 ** -10, 1.0625, 1.1875, -0.5])
    assert codes.tolist() == [0, 0x38, 0x7e, 0x7e, 1, 0, 0x38, 0x3a, 0xb0]
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert (mags == want).all()


def parts(cache, dim):
    return cache[..., : PAGE * dim].unflatten(-1, (PAGE, dim)), cache[..., PAGE * dim:].view(torch.float32)


def slots_of(tokens, pages, seed):
    return np.random.default_rng(seed).permutation(pages * PAGE)[:tokens].astype(np.int32)


CASES = [  # tokens, key/value heads, head size, row padding, offset of the first element
    (1, 1, 16, 0, 0), (1, 8, 64, 0, 0), (5, 3, 80, 0, 0), (7, 2, 128, 8, 0), (33, 8, 64, 3, 0), (70, 1, 256, 0, 0), (6, 4, 192, 0, 1), (300, 8, 128, 0, 0), (129, 5, 48, 16, 3), (1000, 2, 112, 0, 0)]


@pytest.mark.parametrize("tokens,n_kv,dim,pad,off", CASES)
@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_write_and_read(L, tokens, n_kv, dim, pad, off, fmt):
    pages, pitch = -(-tokens // PAGE) + 2, 2 * n_kv * dim + pad
    memory = randn(tokens + dim, (tokens * pitch + off + 64,))
    rows = memory[off: off + tokens * pitch].view(tokens, pitch)
    rows[:, ::7] *= 30.0
    k, v = (rows[:, i * n_kv * dim: (i + 1) * n_kv * dim].unflatten(1, (n_kv, dim)) for i in (0, 1))
    if tokens > 4:
        k[1] = 0.0
        k[2, 0, 1], v[3, 0, 0] = math.inf, math.nan
        v[4] *= 2.0 ** -125
    slots = slots_of(tokens, pages, tokens)
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    cache = torch.randint(0, 256, (2, pages, n_kv, PAGE * (dim + 4)), dtype=torch.uint8, device="cuda")
    want, status, s = cache.clone(), torch.zeros(1, dtype=torch.int32, device="cuda"), dev(slots)
    assert L.oa_k_cache8_write(ptr(rows), ptr(rows, 2 * n_kv * dim), pitch, ptr(cache), pages, ptr(s), tokens, n_kv, dim, fmt, ptr(status), now()) == 0, _lib.last_error()
    torch.cuda.synchronize()
    live = slots >= 0
    at = torch.tensor(slots[live].astype(np.int64), device="cuda")
    for plane, x in enumerate((k, v)):
        y, scale = quantised(x[torch.tensor(live, device="cuda")], fmt)
        values, scales = parts(want[plane], dim)
        values[at // PAGE, :, at % PAGE] = torch.from_numpy(y).cuda()
        scales[at // PAGE, :, at % PAGE] = torch.from_numpy(scale).cuda()
    (a, sa), (b, sb) = parts(cache, dim), parts(want, dim)
    assert torch.equal(a, b) and torch.equal(torch.isnan(sa), torch.isnan(sb)) and torch.equal(sa.nan_to_num(), sb.nan_to_num()) and status.item() == 0
    out = torch.full((tokens * pitch + off + 64,), 5.0, dtype=torch.bfloat16, device="cuda")
    got = out[off: off + tokens * pitch].view(tokens, pitch)
    assert L.oa_k_cache8_read(ptr(cache), pages, ptr(s), tokens, n_kv, dim, fmt, ptr(got), ptr(got, 2 * n_kv * dim), pitch, ptr(status), now()) == 0, _lib.last_error()
    torch.cuda.synchronize()
    for plane in (0, 1):
        values, scales = parts(cache[plane], dim)
        y = values[at // PAGE, :, at % PAGE].view(torch.float8_e4m3fn if fmt == E4M3 else torch.int8).float() * scales[at // PAGE, :, at % PAGE][..., None]
        mine = got[:, plane * n_kv * dim: (plane + 1) * n_kv * dim].unflatten(1, (n_kv, dim))
        alive = torch.tensor(live, device="cuda")
        assert torch.equal(torch.isnan(mine[alive]), torch.isnan(y)) and torch.equal(mine[alive].nan_to_num(), y.bfloat16().nan_to_num())
        assert (mine[~alive] == 5.0).all()
        x = (k, v)[plane][alive].double()
        fine = torch.isfinite(x).all(-1, keepdim=True) & (x.abs().amax(-1, keepdim=True) > 2.0 ** -100)
        top = x.abs().amax(-1, keepdim=True)
        # a value is off by half of its step (2^-4 of it, or half of 2^-9 of the scale; half of a scale for int8), by the roundings of scale and quotient, and by that of the result
        step = torch.maximum(x.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10) if fmt == E4M3 else top / 127 / 2
        assert bool((((mine[alive].double() - x).abs() <= step * (1 + 2.0 ** -20) + x.abs() * (2.0 ** -8 * 1.07 + 2.0 ** -22) + step * 2.0 ** -8) | ~fine).all())
    assert (got[:, 2 * n_kv * dim:] == 5.0).all() and (out[:off] == 5.0).all() and (out[off + tokens * pitch:] == 5.0).all()


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_every_value_is_written_to_the_nearest(L, fmt):
    """All magnitudes of bf16 between 2^-14 and 1 under a largest one of 1, and the ties among them."""
    bits = torch.arange(0x3880, 0x3f81, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).cuda()
    n = -(-len(bits) // 126)
    x = torch.ones((n, 128), dtype=torch.bfloat16, device="cuda")
    for i in range(n):
        part = bits[i * 126: (i + 1) * 126]
        x[i, 1: 1 + len(part)] = part * (-1) ** i
    x[:, 127] = torch.where(torch.arange(n, device="cuda") % 2 == 0, -0.0, 0.0)      # zeros keep their sign
    cache, s = torch.zeros((2, -(-n // PAGE), 1, PAGE * 132), dtype=torch.uint8, device="cuda"), dev(np.arange(n))
    assert L.oa_k_cache8_write(ptr(x), ptr(x), 128, ptr(cache), cache.shape[1], ptr(s), n, 1, 128, fmt, None, now()) == 0
    torch.cuda.synchronize()
    y, scale = quantised(x, fmt)
    values, scales = parts(cache, 128)
    for plane in (0, 1):
        assert torch.equal(values[plane, :, 0].reshape(-1, 128)[:n].cpu(), torch.from_numpy(y)) and torch.equal(scales[plane, :, 0].reshape(-1)[:n].cpu(), torch.from_numpy(scale))


def test_slots_beyond_the_cache_set_the_status(L):
    x, status = randn(1, (4, 2, 2, 64)), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = torch.zeros((2, 3, 2, PAGE * 68), dtype=torch.uint8, device="cuda")
    for bad in (3 * PAGE, 2 ** 31 - 1):
        cache.zero_()
        status.zero_()
        s = dev([5, bad, -2 ** 31, 70])
        assert L.oa_k_cache8_write(ptr(x), ptr(x, 256), 256, ptr(cache), 3, ptr(s), 4, 2, 64, INT8, ptr(status), now()) == 0
        out = torch.full_like(x, 5.0)
        assert L.oa_k_cache8_read(ptr(cache), 3, ptr(s), 4, 2, 64, INT8, ptr(out), ptr(out, 256), 256, ptr(status), now()) == 0
        torch.cuda.synchronize()
        assert status.item() == 400 and (out[1:3] == 5.0).all() and int((parts(cache, 64)[1] != 0).sum()) == 8
    back = dev([70, 5, 5, 70])                                                    # the same place twice
    assert L.oa_k_cache8_read(ptr(cache), 3, ptr(back), 4, 2, 64, INT8, ptr(out), ptr(out, 256), 256, None, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[3]) and torch.equal(out[1], out[2]) and not torch.equal(out[0], out[1])


@pytest.mark.parametrize("planes,n_kv,dim,n", [(2, 1, 16, 1), (6, 8, 64, 4), (4, 8, 128, 30), (2, 3, 80, 70), (2, 2, 256, 5), (2, 1, 64, 3000)])
@pytest.mark.parametrize("tokens", [64, 1, 2, 3, 20, 63])
@pytest.mark.parametrize("shared", [False, True])
def test_copy(L, planes, n_kv, dim, n, tokens, shared):
    sources = 1 if shared else n
    pages = n + sources + 2
    order = np.random.default_rng(n).permutation(pages)
    cache = torch.randint(0, 256, (planes, pages, n_kv, PAGE * (dim + 4)), dtype=torch.uint8, device="cuda")
    want = cache.clone()
    moves = (_lib.OaPageMove * n)()
    for i in range(n):
        k = tokens if i % 3 != 2 else max(0, tokens - 1)
        moves[i] = _lib.OaPageMove(int(order[i % sources]), int(order[sources + i]), k)
    for (a, b) in zip(parts(want, dim), parts(cache, dim)):
        for some in (0, 1):                                                      # those of every third move are one place fewer
            pick = [m for i, m in enumerate(moves) if (i % 3 == 2) == bool(some)]
            if pick and pick[0].tokens:
                a[:, [m.dst for m in pick], :, : pick[0].tokens] = b[:, [m.src for m in pick], :, : pick[0].tokens]
    assert L.oa_k_cache8_copy(ptr(cache), planes, pages, n_kv, dim, moves, n, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128])
def test_conversations_on_a_cache_of_8_bits(L, fmt, dim):
    """As they are used together: a prompt rotated and written, forked, drafts written behind each branch and attended to, the accepted ones kept, pages compacted, read back."""
    heads, n_kv, pages, width, layers = 8, 2, 24, 4, 1
    cache = torch.randint(0, 256, (2 * layers, pages, n_kv, PAGE * (dim + 4)), dtype=torch.uint8, device="cuda")
    tables, lens, refs = np.full((4, width), -1, np.int32), np.zeros(4, np.int32), np.zeros(pages, np.int32)
    table = _lib.OaPageTable(tables.ctypes.data, lens.ctypes.data, refs.ctypes.data, 4, width, pages)
    freqs, amp = np.zeros(dim // 2), C.c_float()
    assert L.oa_host_rotary_freqs(dim, 10000.0, 0, 1.0, 0.0, 0.0, 0, freqs.ctypes.data, C.byref(amp)) == 0
    wide = (heads + 2 * n_kv) * dim
    text = [[] for _ in range(4)]                                                # what each row's places hold: rotated keys, values

    def append(row, count, seed):
        qkv = randn(seed, (count, wide))
        at = int(lens[row])
        assert L.oa_host_cache_grow(table, row, count) == 0
        pos = np.arange(at, at + count)
        slots = dev(tables[row][pos // PAGE] * PAGE + pos % PAGE)
        positions = dev(pos)
        assert L.oa_k_rotary(ptr(qkv), wide, ptr(qkv), wide, ptr(positions), count, heads + n_kv, dim, dim, 1, freqs.ctypes.data, 1.0, 0, 0, now()) == 0      # queries and keys, in place
        assert L.oa_k_cache8_write(ptr(qkv, 2 * heads * dim), ptr(qkv, 2 * (heads + n_kv) * dim), wide, ptr(cache), pages, ptr(slots), count, n_kv, dim, fmt, None, now()) == 0
        torch.cuda.synchronize()
        y, s = quantised(qkv[:, heads * dim:].reshape(count, 2, n_kv, dim), fmt)
        y = torch.from_numpy(y).view(torch.float8_e4m3fn if fmt == E4M3 else torch.int8).double() * torch.from_numpy(s).double()[..., None]
        text[row] += list(y.cuda())
        return qkv

    def attend(rows, qkvs, ctx, new):
        q = torch.cat([x[:, : heads * dim] for x in qkvs]).contiguous()
        starts = dev(np.concatenate([[0], np.cumsum(new)]))
        t, c = dev(np.where(tables[rows] < 0, 0, tables[rows])), dev(ctx)
        out = torch.empty_like(q)
        assert L.oa_k_tree_attention(ptr(q), heads * dim, ptr(out), heads * dim, ptr(cache), fmt, pages, ptr(t), width, ptr(c), ptr(starts), None, len(rows), q.shape[0], heads, n_kv, dim, 0, 0, 0.0, None, now()) == 0
        torch.cuda.synchronize()
        r = 0
        for row, n0, n in zip(rows, ctx, new):
            for u in range(n):
                kv = torch.stack(text[row][: n0 + u + 1])                        # [place, plane, head, channel]
                x = q[r].double().view(n_kv, -1, dim)
                p = torch.softmax(torch.einsum("khd,pkd->khp", x, kv[:, 0]) / math.sqrt(dim), -1)
                want, size = torch.einsum("khp,pkd->khd", p, kv[:, 1]), torch.einsum("khp,pkd->khd", p, kv[:, 1].abs())
                score = torch.einsum("khd,pkd->khp", x.abs(), kv[:, 0].abs()).amax(-1, keepdim=True) / math.sqrt(dim)
                # fp16: weights, scales, and keys and values times these, 2^-11 each (a score's error twice, in a weight and in their sum)
                tol = size * (3 * 2.0 ** -11 + 2 * 2.0 ** -10 * score + 2 * (dim + 8) * 2.0 ** -24 * score + 2.0 ** -19) + want.abs() * 2.0 ** -8 * 1.01 + 2.0 ** -30
                assert bool(((out[r].double().view(n_kv, -1, dim) - want).abs() <= tol).all())
                r += 1

    attend([0], [append(0, 100, 1)[36:]], [36], [64])                            # a prompt's last 64 tokens
    children = np.array([1, 2, 3], np.int32)
    moves, n = (_lib.OaPageMove * pages)(), C.c_int32()
    assert L.oa_host_cache_fork(table, 0, children.ctypes.data, 3, moves, pages, n) == 0 and n.value == 3
    assert L.oa_k_cache8_copy(ptr(cache), 2 * layers, pages, n_kv, dim, moves, n.value, now()) == 0
    for c in children:
        text[c] = list(text[0])
    drafts = [append(r, k, 10 + r) for r, k in ((1, 5), (2, 30), (3, 1))]
    attend([1, 2, 3], drafts, [100, 100, 100], [5, 30, 1])
    lens[1], text[1] = 102, text[1][:102]                                        # two drafts of five are kept: the next tokens go over the others
    attend([1, 2, 3], [append(r, 2, 20 + r) for r in (1, 2, 3)], [102, 130, 101], [2, 2, 2])
    ended = np.array([0, 2], np.int32)
    assert L.oa_host_cache_free(table, ended.ctypes.data, 2) == 0 and L.oa_host_cache_compact(table, moves, pages, n) == 0
    assert L.oa_k_cache8_copy(ptr(cache), 2 * layers, pages, n_kv, dim, moves, n.value, now()) == 0
    attend([1, 3], [append(r, 3, 30 + r) for r in (1, 3)], [104, 103], [3, 3])
    pos = np.arange(int(lens[1]))
    slots = dev(tables[1][pos // PAGE] * PAGE + pos % PAGE)
    out = torch.empty((len(pos), 2, n_kv, dim), dtype=torch.bfloat16, device="cuda")
    assert L.oa_k_cache8_read(ptr(cache), pages, ptr(slots), len(pos), n_kv, dim, fmt, ptr(out), ptr(out, 2 * n_kv * dim), 2 * n_kv * dim, None, now()) == 0
    torch.cuda.synchronize()
    want = torch.stack(text[1])
    assert len(text[1]) == len(pos) and bool(((out.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01).all())


def test_captured_writes_reads_and_copies(L):
    x, cache, s = randn(3, (70, 2, 2, 64)), torch.zeros((2, 5, 2, PAGE * 68), dtype=torch.uint8, device="cuda"), dev(np.arange(70) + 20)
    out = torch.zeros_like(x)
    moves = (_lib.OaPageMove * 2)(_lib.OaPageMove(0, 3, 64), _lib.OaPageMove(1, 4, 26))
    back = dev(np.concatenate([np.arange(44) + 20 + 192, np.arange(26) + 256]))
    L.oa_k_cache8_copy(ptr(cache), 2, 5, 2, 64, moves, 2, now())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        assert L.oa_k_cache8_write(ptr(x), ptr(x, 256), 256, ptr(cache), 5, ptr(s), 70, 2, 64, E4M3, None, now()) == 0
        assert L.oa_k_cache8_copy(ptr(cache), 2, 5, 2, 64, moves, 2, now()) == 0
        assert L.oa_k_cache8_read(ptr(cache), 5, ptr(back), 70, 2, 64, E4M3, ptr(out), ptr(out, 256), 256, None, now()) == 0
    for seed in (4, 5):
        x.copy_(randn(seed, x.shape))
        graph.replay()
        torch.cuda.synchronize()
        y, scale = quantised(x, E4M3)
        want = (torch.from_numpy(y).view(torch.float8_e4m3fn).float() * torch.from_numpy(scale)[..., None]).bfloat16()
        assert torch.equal(out.cpu(), want)
