"""The operators on a caller's paged cache on the B200, through the C ABI, against plain implementations in 64 bits: rotary positions (alone and with the
write to the cache), copies of pages, decode attention over shared prefixes, and a run of them together.

Tolerances come from arithmetic.  A rounding to bf16 is off by at most 2^-8 of the value, to fp32 by 2^-24.  `u` below is 2^-24.
 rotary: cos and sin are off by at most 8 u + the angle's error (its rounding to fp32 and sincospif's two ulps, the amplitude's product), the two products and the
   sum add 3 u of |a| + |b|: 12 u amplitude (|a| + |b|), and then the output's own rounding.  The angle's own error is 2^-52 of the angle (two roundings in 64 bits).
 attention: a probability is rounded to bf16 for the second product (2^-8 of p |v| summed up, over l), scores are sums of D products in fp32 ((D + 4) u of the sum of
   |q k|, scaled), which moves p by twice that at most (its own, and l's), 2^x by 2^-21; joining parts rounds a dozen times in fp32; the output rounds once."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from opsagent_b200 import _lib  # noqa: E402

PAGE, U = 64, 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def now():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def cuda_i32(a):
    return torch.tensor(np.ascontiguousarray(a, np.int32), device="cuda")


def randn(seed, shape, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def frequencies(L, dims, base=10000.0, scaling=0, factor=1.0, first=0.0, second=0.0, original=0):
    f, amp = np.zeros(max(1, dims // 2)), C.c_float()
    assert L.oa_host_rotary_freqs(dims, base, scaling, factor, first, second, original, f.ctypes.data, C.byref(amp)) == 0
    return f, amp.value


# ---- rotary ------------------------------------------------------------------------------------
def turned(x, positions, freqs, amplitude, dims, layout, transpose=False):
    """-> (values, |a| + |b| of each channel's pair, amplitude included) in 64 bits."""
    half = dims // 2
    y, mag = x.double().clone(), x.double().abs()
    angle = positions.double()[:, None] * torch.from_numpy(freqs[:half]).cuda()
    c, s = (angle.cos() * amplitude)[:, None], (angle.sin() * amplitude)[:, None]
    s = -s if transpose else s
    i = torch.arange(half, device="cuda")
    ia, ib = (i, i + half) if layout == 1 else (2 * i, 2 * i + 1)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(amplitude)
    return y, mag


def assert_turned(got, want, mag, dtype, angle_error=0.0):
    err = (got.double() - want).abs()
    tol = (12 * U + angle_error) * mag + HALF_STEP[dtype] * (want.abs() + 12 * U * mag) + 2.0 ** -133
    assert bool((err <= tol).all()), (err - tol).max().item()


ROTARY = [  # tokens, heads, head size, rotated, layout, fp32, row padding, transposed
    (1, 1, 2, 2, 1, False, 0, False), (1, 32, 128, 128, 1, False, 0, False), (5, 3, 64, 64, 0, False, 0, False), (7, 5, 128, 96, 1, False, 8, True), (33, 4, 128, 64, 0, False, 0, True),
    (3, 2, 128, 0, 1, False, 0, False), (4, 3, 80, 20, 1, False, 0, False), (6, 3, 80, 20, 0, False, 2, False), (9, 2, 256, 256, 1, False, 0, False), (2, 2, 66, 66, 0, False, 6, False),
    (300, 8, 64, 32, 1, False, 24, False), (150, 40, 128, 128, 0, False, 0, False), (17, 3, 128, 128, 1, True, 0, True), (5, 7, 64, 40, 0, True, 4, False), (4, 2, 96, 2, 1, True, 1, False),
    (513, 2, 64, 64, 0, True, 0, False)]


@pytest.mark.parametrize("tokens,heads,dim,rot,layout,f32,pad,transpose", ROTARY)
@pytest.mark.parametrize("in_place", [False, True])
def test_rotary(L, tokens, heads, dim, rot, layout, f32, pad, transpose, in_place):
    dtype, width = torch.float32 if f32 else torch.bfloat16, heads * dim
    freqs, _ = frequencies(L, rot)
    amp = 1.0 if rot != 96 else 1.25
    rows = randn(tokens + dim, (tokens + 1, width + pad), dtype)               # a row behind the last, and columns behind each row's end
    positions = cuda_i32(np.arange(tokens) * 37 + 11)
    out = rows.clone() if in_place else torch.full_like(rows, 7.0)
    src = out if in_place else rows
    want, mag = turned(rows[:tokens, :width].reshape(tokens, heads, dim), positions, freqs, amp, rot, layout, transpose)
    assert L.oa_k_rotary(ptr(src), width + pad, ptr(out), width + pad, ptr(positions), tokens, heads, dim, rot, layout, freqs.ctypes.data, amp, int(transpose), int(f32), now()) == 0
    torch.cuda.synchronize()
    got = out[:tokens, :width].reshape(tokens, heads, dim)
    assert_turned(got, want, mag, dtype, 2.0 ** -52 * 37 * tokens)
    assert torch.equal(got[..., rot:], rows[:tokens, :width].reshape(tokens, heads, dim)[..., rot:])
    rest = rows if in_place else torch.full_like(rows, 7.0)
    assert torch.equal(out[tokens:], rest[tokens:]) and torch.equal(out[:, width:], rest[:, width:])


def test_rotary_unaligned_rows(L):
    """A pointer two bytes off a 16-byte boundary takes the element path, with the same bits."""
    x = randn(3, (6, 256))
    odd = torch.empty(6 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 256)
    odd.copy_(x)
    freqs, _ = frequencies(L, 128)
    positions, outs = cuda_i32([0, 1, 5, 100, 8191, 100000]), []
    for src in (x, odd):
        for layout in (0, 1):
            out = torch.empty_like(x)
            assert L.oa_k_rotary(ptr(src), 256, ptr(out), 256, ptr(positions), 6, 2, 128, 128, layout, freqs.ctypes.data, 1.0, 0, 0, now()) == 0
            outs.append(out)
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and not torch.equal(outs[0], outs[1])


def test_rotary_far_positions(L):
    """Positions of up to 31 bits, against angles in 80 bits."""
    at = np.array([0, 1, -1, 131071, 10 ** 6 + 1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], np.int64)
    freqs, _ = frequencies(L, 64, base=500000.0)
    x = randn(9, (len(at), 1, 64), torch.float32)
    out = torch.empty_like(x)
    assert L.oa_k_rotary(ptr(x), 64, ptr(out), 64, ptr(cuda_i32(at)), len(at), 1, 64, 64, 1, freqs.ctypes.data, 1.0, 0, 1, now()) == 0
    angle = at.astype(np.longdouble)[:, None] * freqs.astype(np.longdouble)
    c, s = np.cos(angle)[:, None].astype(np.float64), np.sin(angle)[:, None].astype(np.float64)
    a, b = np.split(x.cpu().double().numpy(), 2, -1)
    want = torch.from_numpy(np.concatenate([a * c - b * s, a * s + b * c], -1)).cuda()
    mag = torch.from_numpy(np.concatenate([abs(a) + abs(b)] * 2, -1)).cuda()
    # 2^-52 of an angle of at most 2^31 (the kernel's two roundings), and 80-bit angles that are 2^-33 off
    assert_turned(out, want, mag, torch.float32, 2.0 ** -21 + 2.0 ** -33)


def test_rotary_gradient_against_differences(L):
    """<g, y(x + h e) - y(x - h e)> / 2h is what the transposed call gives (the map is linear: h = 1 has no error of its own)."""
    t, heads, dim, rot = 3, 2, 16, 12
    for layout in (0, 1):
        freqs, _ = frequencies(L, rot)
        positions, x, g = cuda_i32([3, 900, 70000]), randn(1, (t, heads * dim), torch.float32), randn(2, (t, heads * dim), torch.float32)
        call = lambda src, out, tr: L.oa_k_rotary(ptr(src), heads * dim, ptr(out), heads * dim, ptr(positions), t, heads, dim, rot, layout, freqs.ctypes.data, 1.1, tr, 1, now())  # noqa: E731
        grad = torch.empty_like(x)
        assert call(g, grad, 1) == 0
        for k in range(t * heads * dim):
            up, down = x.clone(), x.clone()
            up.view(-1)[k] += 1.0
            down.view(-1)[k] -= 1.0
            a, b = torch.empty_like(x), torch.empty_like(x)
            assert call(up, a, 0) == 0 and call(down, b, 0) == 0
            want = (g.double() * (a.double() - b.double())).sum() / 2
            # two results and two sums x +- 1 in fp32 (16 u of values up to 8, times 1.1 sqrt 2), against two terms of g
            assert abs(grad.view(-1)[k].item() - want.item()) <= 32 * U * 8 * 1.6 * 2 * g.abs().max().item()


def test_rotary_keeps_special_values(L):
    x = torch.zeros(1, 64, device="cuda")
    x[0, 5], x[0, 37 + 3], x[0, 20] = math.inf, math.nan, -0.0
    freqs, _ = frequencies(L, 64)
    out = torch.empty_like(x)
    assert L.oa_k_rotary(ptr(x), 64, ptr(out), 64, ptr(cuda_i32([1])), 1, 1, 64, 64, 1, freqs.ctypes.data, 1.0, 0, 1, now()) == 0
    bad = [5, 37, 8, 40]
    assert not torch.isfinite(out[0, bad]).any() and torch.isfinite(out).sum() == 60


@pytest.mark.parametrize("tokens,heads,n_kv,dim,rot,layout", [(1, 32, 8, 64, 64, 1), (130, 8, 2, 128, 128, 1), (70, 10, 2, 128, 64, 0), (5, 3, 3, 48, 22, 1), (200, 4, 1, 64, 16, 0)])
def test_rotary_cache(L, tokens, heads, n_kv, dim, rot, layout):
    pages, width = -(-tokens // PAGE) + 3, (heads + 2 * n_kv) * dim
    qkv, cache = randn(tokens, (tokens, width)), randn(1, (2, pages, n_kv, PAGE, dim))
    freqs, amp = frequencies(L, rot, 1e6, 3, 4.0, 32.0, 1.0, 32768)
    rng = np.random.default_rng(tokens)
    slots = rng.permutation(pages * PAGE)[:tokens].astype(np.int32)
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]                          # a padding row
    if tokens > 4:
        slots[1], slots[3] = pages * PAGE, 2 ** 31 - 1                          # beyond the cache
    positions, status = cuda_i32(rng.integers(0, 100000, tokens)), torch.zeros(1, dtype=torch.int32, device="cuda")
    before, q_out = cache.clone(), torch.full((tokens + 1, heads * dim), 3.0, dtype=torch.bfloat16, device="cuda")
    k0 = qkv.data_ptr() + 2 * heads * dim
    assert L.oa_k_rotary_cache(ptr(qkv), width, k0, k0 + 2 * n_kv * dim, width, ptr(q_out), heads * dim, ptr(cache), pages, ptr(positions), ptr(cuda_i32(slots)), tokens, heads, n_kv, dim, rot,
                               layout, freqs.ctypes.data, amp, ptr(status), now()) == 0
    torch.cuda.synchronize()
    x = qkv.view(tokens, -1, dim)
    error = 2.0 ** -52 * 100000
    want, mag = turned(x, positions, freqs, amp, rot, layout)
    assert_turned(q_out[:tokens].view(tokens, heads, dim), want[:, :heads], mag[:, :heads], torch.bfloat16, error)
    assert (q_out[tokens] == 3.0).all()
    untouched = torch.ones(pages * PAGE, dtype=torch.bool)
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < pages * PAGE:
            continue
        untouched[s] = False
        assert_turned(cache[0, s // PAGE, :, s % PAGE], want[t, heads:heads + n_kv], mag[t, heads:heads + n_kv], torch.bfloat16, error)
        assert torch.equal(cache[1, s // PAGE, :, s % PAGE], x[t, heads + n_kv:])
    rows = lambda c: c.transpose(2, 3).reshape(2, pages * PAGE, -1)[:, untouched.cuda()]  # noqa: E731
    assert torch.equal(rows(cache), rows(before))
    assert status.item() == (400 if tokens > 4 else 0)


@pytest.mark.parametrize("heads,dim,rot,layout,f32,pad", [(2, 64, 64, 1, False, 0), (3, 128, 96, 0, False, 8), (2, 66, 30, 1, False, 6), (1, 600, 256, 0, False, 0), (2, 520, 256, 1, True, 1), (1, 2048, 64, 1, False, 0),
                                                           (17, 64, 32, 0, True, 0)])
def test_rotary_of_more_rows_than_run_at_once(L, heads, dim, rot, layout, f32, pad):
    """Every CTA takes several rows; heads of more pieces than a CTA has threads, too."""
    tokens, dtype, width = 2003, torch.float32 if f32 else torch.bfloat16, heads * dim
    freqs, _ = frequencies(L, rot)
    x, positions = randn(dim, (tokens, width + pad), dtype), cuda_i32((np.arange(tokens) * 7919) % 4099)
    out = torch.empty_like(x)
    assert L.oa_k_rotary(ptr(x), width + pad, ptr(out), width + pad, ptr(positions), tokens, heads, dim, rot, layout, freqs.ctypes.data, 1.0, 0, int(f32), now()) == 0
    torch.cuda.synchronize()
    rows = x[:, :width].reshape(tokens, heads, dim)
    got = out[:, :width].reshape(tokens, heads, dim)
    want, mag = turned(rows, positions, freqs, 1.0, rot, layout)
    assert_turned(got, want, mag, dtype, 2.0 ** -52 * 4099)
    assert torch.equal(got[..., rot:], rows[..., rot:])


@pytest.mark.parametrize("layout", [0, 1])
def test_rotary_cache_in_place_on_fused_rows(L, layout):
    """q, k and v next to each other in a row, q turned in place: what the two calls apart give, and k and v stay."""
    tokens, heads, n_kv, dim, pages = 1500, 4, 2, 64, 30
    width = (heads + 2 * n_kv) * dim
    freqs, _ = frequencies(L, dim)
    qkv, cache = randn(1, (tokens, width)), randn(2, (2, pages, n_kv, PAGE, dim))
    slots, positions = np.random.default_rng(3).permutation(pages * PAGE)[:tokens], cuda_i32(np.arange(tokens) % 777)
    want_q, want_k = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device="cuda"), torch.empty(tokens, n_kv * dim, dtype=torch.bfloat16, device="cuda")
    k0 = qkv.data_ptr() + 2 * heads * dim
    assert L.oa_k_rotary(ptr(qkv), width, ptr(want_q), heads * dim, ptr(positions), tokens, heads, dim, dim, layout, freqs.ctypes.data, 1.0, 0, 0, now()) == 0
    assert L.oa_k_rotary(k0, width, ptr(want_k), n_kv * dim, ptr(positions), tokens, n_kv, dim, dim, layout, freqs.ctypes.data, 1.0, 0, 0, now()) == 0
    before = qkv.clone()
    assert L.oa_k_rotary_cache(ptr(qkv), width, k0, k0 + 2 * n_kv * dim, width, ptr(qkv), width, ptr(cache), pages, ptr(positions), ptr(cuda_i32(slots)), tokens, heads, n_kv, dim, dim, layout,
                               freqs.ctypes.data, 1.0, None, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(qkv[:, :heads * dim], want_q) and torch.equal(qkv[:, heads * dim:], before[:, heads * dim:])
    s = torch.tensor(slots, device="cuda")
    assert torch.equal(cache[0, s // PAGE, :, s % PAGE].reshape(tokens, -1), want_k)
    assert torch.equal(cache[1, s // PAGE, :, s % PAGE].reshape(tokens, -1), before[:, (heads + n_kv) * dim:])


# ---- copies of pages -----------------------------------------------------------------------------
@pytest.mark.parametrize("planes,pages,n_kv,dim,dtype,n,tokens", [
    (2, 9, 1, 8, torch.bfloat16, 3, (64,)), (4, 40, 8, 128, torch.bfloat16, 17, (64,)), (6, 30, 8, 64, torch.bfloat16, 13, (1, 63, 20, 0)), (2, 30, 3, 80, torch.bfloat16, 12, (5, 64)),
    (3, 21, 2, 36, torch.float32, 9, (33, 64)), (2, 6000, 1, 8, torch.bfloat16, 2900, (64, 7)), (2, 140, 1, 512, torch.bfloat16, 65, (64,))])
def test_cache_copy(L, planes, pages, n_kv, dim, dtype, n, tokens):
    cache = randn(pages, (planes, pages, n_kv, PAGE, dim), dtype)
    order = np.random.default_rng(n).permutation(pages)
    src, dst = order[:n], order[n:2 * n]
    src = src[np.arange(n) // 2 * 2 % n]                                         # every other source has two targets
    want, moves = cache.clone(), (_lib.OaPageMove * n)()
    for i in range(n):
        k = tokens[i % len(tokens)]
        moves[i] = _lib.OaPageMove(int(src[i]), int(dst[i]), k)
        want[:, dst[i], :, :k] = cache[:, src[i], :, :k]
    assert L.oa_k_cache_copy(ptr(cache), planes, pages, n_kv, dim, cache.element_size(), moves, n, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("runs", [(70,), (20, 13, 1, 30, 6), (2,) * 35])
def test_cache_copy_of_pages_that_go_to_many(L, runs):
    """Enough work that a CTA writes what it has read to several pages; sources change and lengths differ within its share."""
    planes, n_kv, dim = 16, 8, 128
    n, pages = sum(runs), sum(runs) + len(runs)
    order, cache = np.random.default_rng(len(runs)).permutation(pages), randn(len(runs), (planes, pages, n_kv, PAGE, dim))
    want, moves, at = cache.clone(), (_lib.OaPageMove * n)(), 0
    for r, count in enumerate(runs):
        for i in range(count):
            k, dst = (64, 49, 64, 0, 1)[(at + i) % 5] if r % 2 else 49, int(order[len(runs) + at + i])
            moves[at + i] = _lib.OaPageMove(int(order[r]), dst, k)
            want[:, dst, :, :k] = cache[:, order[r], :, :k]
        at += count
    assert L.oa_k_cache_copy(ptr(cache), planes, pages, n_kv, dim, 2, moves, n, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache.view(torch.int16), want.view(torch.int16))


def test_cache_copy_of_no_places(L):
    cache = randn(1, (2, 4, 1, PAGE, 8))
    want, moves = cache.clone(), (_lib.OaPageMove * 2)(_lib.OaPageMove(0, 1, 0), _lib.OaPageMove(0, 2, 0))
    assert L.oa_k_cache_copy(ptr(cache), 2, 4, 1, 8, 2, moves, 2, now()) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


# ---- decode attention over shared prefixes -------------------------------------------------------
def apart(n, n_kv):
    """A table of prefixes so wide that prefixes are work of their own."""
    return (1200 if n <= 8 else 600) // (n * n_kv) + 1


class Batch:
    """Pages anywhere in a cache whose unused places hold NaN."""

    def __init__(self, heads, n_kv, dim, prefixes, runs, own, seed=0, spare=3, pad=0, scale_q=1.0, wide=1):
        self.heads, self.n_kv, self.dim, self.prefixes, self.runs, self.own = heads, n_kv, dim, list(prefixes), list(runs), list(own)
        n, rng = len(self.own), np.random.default_rng(seed)
        need = [-(-x // PAGE) for x in self.prefixes + self.own]
        self.pages = sum(need) + spare
        order, at = rng.permutation(self.pages), 0
        width = [max([wide] + need[: len(prefixes)]), max(need[len(prefixes):] + [1]) + 1]
        self.pt, self.ot = np.full((max(1, len(prefixes)), width[0]), -7, np.int32), np.full((max(1, n), width[1]), 10 ** 9, np.int32)
        for i, k in enumerate(need):
            (self.pt[i] if i < len(prefixes) else self.ot[i - len(prefixes)])[:k] = order[at:at + k]
            at += k
        self.cache = randn(seed + 1, (2, self.pages, n_kv, PAGE, dim))
        used = torch.zeros(self.pages, PAGE, dtype=torch.bool)
        for i, x in enumerate(self.prefixes + self.own):
            row = self.pt[i] if i < len(prefixes) else self.ot[i - len(prefixes)]
            for p in range(0, x, PAGE):
                used[row[p // PAGE], : min(PAGE, x - p)] = True
        self.cache.masked_fill_(~used.cuda()[None, :, None, :, None], math.nan)
        self.pad = pad
        self.q = randn(seed + 2, (n, heads * dim + pad), std=scale_q)
        self.out = torch.full((n + 2, heads * dim + pad), 5.0, dtype=torch.bfloat16, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.upload()

    def upload(self):
        self.d = [cuda_i32(x) for x in (self.pt, self.prefixes or [0], self.runs or [0], self.ot, self.own)]

    def call(self, L, out=None, scale=0.0, stream=None, q=None):
        pt, pl, pr, ot, ol = self.d
        pitch = self.heads * self.dim + self.pad
        return L.oa_k_prefix_attention(ptr(self.q if q is None else q), pitch, ptr(self.out if out is None else out), pitch, ptr(self.cache), self.pages, ptr(pt), self.pt.shape[1], ptr(pl), ptr(pr),
                                       len(self.prefixes), ptr(ot), self.ot.shape[1], ptr(ol), len(self.own), self.heads, self.n_kv, self.dim, scale, ptr(self.status), stream or now())

    def keys(self, plane, row, n):
        pages = row[: -(-n // PAGE)].astype(np.int64)
        assert ((0 <= pages) & (pages < self.pages)).all()                        # judged here: an index out of bounds on the device ends the process's use of it
        pages = torch.tensor(pages, device="cuda")
        return self.cache[plane, pages].double().transpose(1, 2).reshape(-1, self.n_kv, self.dim)[:n]

    def check(self, out=None, scale=0.0, rows=None, q=None):
        out, q = self.out if out is None else out, self.q if q is None else q
        n, scale = len(self.own), scale or 1.0 / math.sqrt(self.dim)
        for i in range(n) if rows is None else rows:
            g = next((g for g in range(len(self.prefixes)) if self.runs[g] <= i < self.runs[g + 1]), None)
            kv = [torch.cat([self.keys(p, self.pt[g], self.prefixes[g]) if g is not None else self.cache.new_zeros((0, self.n_kv, self.dim)).double(), self.keys(p, self.ot[i], self.own[i])])
                  for p in (0, 1)]
            got = out[i, : self.heads * self.dim].double().view(self.n_kv, -1, self.dim)
            if kv[0].shape[0] == 0:
                assert not got.any()
                continue
            x = q[i, : self.heads * self.dim].double().view(self.n_kv, -1, self.dim)
            p = torch.softmax(torch.einsum("khd,pkd->khp", x, kv[0]) * scale, -1)
            want, size = torch.einsum("khp,pkd->khd", p, kv[1]), torch.einsum("khp,pkd->khd", p, kv[1].abs())
            score = torch.einsum("khd,pkd->khp", x.abs(), kv[0].abs()).amax(-1, keepdim=True) * scale
            tol = size * (2.0 ** -8 + 2 * (self.dim + 4) * U * score + 2.0 ** -20 + 16 * U) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -133
            err = (got - want).abs()
            assert bool((err <= tol).all()), (i, (err / tol).max().item())
        if rows is None and out is self.out:
            assert (out[n:] == 5.0).all() and (out[:, self.heads * self.dim:] == 5.0).all()


def run(L, b, **kw):
    assert b.call(L, **kw) == 0
    torch.cuda.synchronize()


SHAPES = [  # heads, key/value heads, head size
    (8, 2, 128), (8, 2, 64), (5, 1, 128), (6, 6, 64), (4, 2, 128), (14, 2, 128), (9, 1, 64), (32, 2, 128), (16, 1, 64), (24, 2, 128)]


@pytest.mark.parametrize("heads,n_kv,dim", SHAPES)
@pytest.mark.parametrize("prefix,own", [(1, [1]), (64, [0, 1]), (130, [5, 64, 65, 0, 200]), (500, [3] * 40)])
@pytest.mark.parametrize("wide", [False, True])
def test_prefix_attention(L, heads, n_kv, dim, prefix, own, wide):
    b = Batch(heads, n_kv, dim, [prefix], [0, len(own)], own, seed=heads + prefix, wide=apart(len(own), n_kv) if wide else 1)
    run(L, b)
    b.check()
    assert b.status.item() == 0


@pytest.mark.parametrize("prefix", [63, 65, 127, 128, 129, 192, 255, 256, 257, 1000])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("wide", [1, apart(3, 1), 4000])
def test_prefixes_that_end_anywhere(L, prefix, dim, wide):
    b = Batch(4, 1, dim, [prefix], [0, 3], [0, 17, 16], seed=prefix, wide=wide)
    run(L, b)
    b.check()


@pytest.mark.parametrize("own", [1, 15, 16, 17, 31, 33, 47, 48, 49, 63, 64, 65, 127, 129, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_own_parts_that_end_anywhere(L, own, dim):
    b = Batch(8, 2, dim, [70], [0, 2], [own, 1], seed=own)
    run(L, b)
    b.check()


@pytest.mark.parametrize("wide", [1, apart(11, 2), 2000])
def test_rows_without_a_prefix_and_rows_that_see_nothing(L, wide):
    b = Batch(8, 2, 128, [100, 0, 300], [1, 3, 5, 9], [0, 0, 7, 0, 9, 0, 80, 0, 0, 0, 4], seed=5, wide=wide)      # rows 0, 9 and 10 have no prefix, 3 and 4 an empty one
    run(L, b)
    b.check()
    assert not b.out[[0, 3, 9], :1024].any() and b.out[10, :1024].any()


def test_no_prefix_at_all(L):
    b = Batch(8, 2, 64, [], [], [0, 1, 300, 64, 900], seed=6)
    run(L, b)
    b.check()


@pytest.mark.parametrize("wide", [1, apart(75, 1), 3000])
def test_many_prefixes(L, wide):
    lens = [(i * 37) % 211 for i in range(32)]
    runs = [0] + [min(70, 2 * i + (i % 3)) for i in range(1, 33)]
    b = Batch(8, 1, 64, lens, runs, [(i * 13) % 90 for i in range(75)], seed=7, wide=wide)
    run(L, b)
    b.check()


@pytest.mark.parametrize("heads,n_kv,dim,n,prefix,top", [(32, 8, 128, 128, 1536, 300), (32, 8, 64, 40, 4000, 60), (40, 8, 128, 67, 777, 200), (64, 8, 128, 20, 9000, 700), (28, 4, 128, 9, 64, 3000)])
def test_batches(L, heads, n_kv, dim, n, prefix, top):
    own = np.random.default_rng(n).integers(0, top + 1, n).tolist()
    b = Batch(heads, n_kv, dim, [prefix], [0, n], own, seed=n, scale_q=2.0)
    run(L, b)
    b.check(rows=range(0, n, 7))
    first = b.out.clone()
    for _ in range(5):                                                           # the same call gives the same bits
        run(L, b)
        assert torch.equal(b.out.view(torch.int16), first.view(torch.int16))


# tables with room for prefixes far longer than these: rows are taken two tiles at a time, whose second one may have no rows
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,n_kv,prefixes,runs,wide", [
    (32, 2, [1000], [0, 17], 400), (5, 1, [64, 0, 129, 700], [0, 9, 9, 36, 63], 900), (12, 12, [300, 257], [1, 130, 140], 120), (16, 4, [1, 2000, 63], [0, 33, 97, 104], 200), (48, 3, [640], [2, 11], 400)])
def test_tables_with_room_for_long_prefixes(L, heads, n_kv, prefixes, runs, wide, dim):
    b = Batch(heads, n_kv, dim, prefixes, runs, [(i * 31) % 140 for i in range(runs[-1] + 1)], seed=heads, wide=wide)
    run(L, b)
    b.check()
    first = b.out.clone()
    run(L, b)
    assert torch.equal(first, b.out) and b.status.item() == 0


# more rows than one tile has, with such a table
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 1000, 5000])
@pytest.mark.parametrize("heads,n_kv,rows", [(8, 2, 40), (5, 1, 77)])
def test_rows_of_several_tiles(L, heads, n_kv, rows, prefix):
    b = Batch(heads, n_kv, 128, [prefix], [0, rows], [(i * 31) % 140 for i in range(rows)], seed=prefix + heads, wide=2000, scale_q=1.5)
    run(L, b)
    b.check()
    first = b.out.clone()
    run(L, b)
    assert torch.equal(first, b.out) and b.status.item() == 0


def test_rows_of_several_tiles_on_many_prefixes(L):
    """Runs of one row, of one tile, of a tile and a row, of three tiles; prefixes of one place and of many; pieces of one tile and of several for a CTA."""
    rows, lens = [1, 32, 33, 96, 2, 64, 130], [700, 1, 3000, 65, 129, 0, 257]
    runs = np.concatenate([[3], 3 + np.cumsum(rows)]).tolist()
    b = Batch(16, 4, 128, lens, runs, [(i * 13) % 90 for i in range(runs[-1] + 2)], seed=23, wide=1000)
    run(L, b)
    b.check()
    assert b.status.item() == 0


def test_rows_of_several_tiles_keep_what_masks_and_maxima_ask_for(L):
    """Scores that rise along the keys, then tables with a page that there is not."""
    b = Batch(8, 2, 128, [700], [0, 50], [5] * 50, seed=24, wide=2000)
    ramp = torch.arange(700, device="cuda", dtype=torch.float32) / 40
    direction = torch.nn.functional.normalize(randn(3, (128,), torch.float32), dim=0)
    for i, page in enumerate(b.pt[0, :11]):
        n = min(PAGE, 700 - i * PAGE)
        b.cache[0, page, :, :n] = (ramp[i * PAGE:i * PAGE + n, None] * direction * 8).bfloat16()
    b.q[:] = (direction * 8).bfloat16().repeat(8)
    run(L, b)
    b.check()
    b.cache.nan_to_num_(0.0)
    b.pt[0, 3] = b.pages
    b.upload()
    run(L, b)
    assert b.status.item() == 400 and torch.isfinite(b.out).all() and (b.out[50:] == 5.0).all()


def test_one_long_sequence(L):
    b = Batch(8, 2, 128, [40], [0, 1], [20011], seed=8)
    run(L, b)
    b.check()


@pytest.mark.parametrize("wide", [1, apart(6, 2), 2000])
def test_scores_that_grow_along_the_keys(L, wide):
    """Every tile raises the maximum by far more than the reference may lag behind."""
    b = Batch(8, 2, 128, [700], [0, 6], [200] * 6, seed=9, wide=wide)
    ramp = torch.arange(700, device="cuda", dtype=torch.float32) / 40
    direction = torch.nn.functional.normalize(randn(3, (128,), torch.float32), dim=0)
    for i, page in enumerate(b.pt[0, :11]):
        n = min(PAGE, 700 - i * PAGE)
        b.cache[0, page, :, :n] = (ramp[i * PAGE:i * PAGE + n, None] * direction * 8).bfloat16()
    b.q[:] = (direction * 8).bfloat16().repeat(8)
    run(L, b)
    b.check()


def test_strides_scale_and_in_place(L):
    b = Batch(8, 2, 128, [200], [0, 9], [30, 0, 64, 1, 100, 5, 7, 9, 11], seed=10, pad=24)
    run(L, b, scale=0.3)
    b.check(scale=0.3)
    q = b.q.clone()
    run(L, b, out=b.q, scale=0.3)
    assert torch.equal(b.q[:, :1024], b.out[:9, :1024]) and torch.equal(b.q[:, 1024:], q[:, 1024:])


@pytest.mark.parametrize("wide", [1, apart(3, 2), 2000])
def test_infinities_and_nan_that_are_seen(L, wide):
    """-inf scores leave a key out, a NaN or +inf key makes its rows NaN, as the plain softmax does; other heads stay."""
    b = Batch(4, 2, 64, [150], [0, 3], [70, 3, 0], seed=11, wide=wide)
    b.q[:, 0], b.q[:, 64] = 1.0, 1.0
    b.q[:, 128 + 1] = 1.0
    b.cache[0, b.pt[0, 0], 0, 3, 0] = -math.inf                                   # head 0 of the cache: a score of -inf (or inf where q is negative: q is 1 there)
    b.cache[0, b.ot[1, 0], 1, 1, 1] = math.nan                                    # row 1's own key, head 1 of the cache
    b.q[:, 0] = b.q[:, 64] = 1.0
    run(L, b)
    out = b.out[:3, :256].view(3, 2, 2, 64)
    assert torch.isfinite(out[:, 0]).all() and torch.isnan(out[1, 1]).all() and torch.isfinite(out[[0, 2], 1]).all()
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[3] = False
    k, v = (torch.cat([b.keys(p, b.pt[0], 150)[keep], b.keys(p, b.ot[0], 70)])[:, 0] for p in (0, 1))
    x = b.q[0, :128].double().view(2, 64)
    p = torch.softmax(x @ k.T / 8, -1)
    tol = (p @ v.abs()) * (2.0 ** -8 + 2.0 ** -13) + (p @ v).abs() * 2.0 ** -7
    assert bool(((out[0, 0].double() - p @ v).abs() <= tol).all())
    b.cache[0, b.pt[0, :3], 0, :, 0] = -math.inf                                  # no score of the prefix left: the own part decides, and row 2 is NaN like a softmax of -inf alone
    run(L, b)
    out = b.out[:3, :256].view(3, 2, 2, 64)
    k, v = (b.keys(p, b.ot[0], 70)[:, 0] for p in (0, 1))
    p = torch.softmax(x @ k.T / 8, -1)
    tol = (p @ v.abs()) * (2.0 ** -8 + 2.0 ** -13) + (p @ v).abs() * 2.0 ** -7
    assert bool(((out[0, 0].double() - p @ v).abs() <= tol).all()) and torch.isnan(out[2, 0]).all()


@pytest.mark.parametrize("wide", [1, apart(4, 2), 2000])
def test_bad_tables_set_the_status_and_spare_the_others(L, wide):
    own = [30, 70, 64, 5]
    good = Batch(8, 2, 128, [200], [0, 4], own, seed=12, wide=wide)
    run(L, good)
    assert good.status.item() == 0
    for what in ("own page", "own page below", "own length", "negative length", "prefix page", "prefix length", "runs fall", "runs beyond"):
        b = Batch(8, 2, 128, [200], [0, 4], own, seed=12, wide=wide)
        b.cache.nan_to_num_(0.0)
        rows = [0, 2, 3]
        if what == "own page":
            b.ot[1, 0] = b.pages
        if what == "own page below":
            b.ot[1, 1] = -1
        if what == "own length":
            b.own[1] = 10 ** 6
        if what == "negative length":
            b.own[1] = -5
        if what == "prefix page":
            b.pt[0, 1], rows = 2 ** 30, []
        if what == "prefix length":
            b.prefixes[0], rows = 2 ** 31 - 1, []
        if what == "runs fall":
            b.runs, rows = [3, 1], []
        if what == "runs beyond":
            b.runs = [-2, 9]
            rows = [0, 1, 2, 3]                                                   # cut to what there is
        b.upload()
        run(L, b)
        assert b.status.item() == 400, what
        for i in rows:
            assert torch.equal(b.out[i], good.out[i]) or what in ("own length", "negative length"), what
        assert (b.out[4:] == 5.0).all()


@pytest.mark.parametrize("wide", [1, apart(6, 2), 2000])
def test_a_captured_call_follows_its_tables(L, wide):
    """Two graphs and eager calls in between; lengths change between replays (a row ends, another grows, the prefix grows)."""
    b, c = Batch(8, 2, 128, [300], [0, 6], [11, 1, 64, 90, 2, 65], seed=13, wide=wide), Batch(8, 2, 64, [90, 64], [0, 2, 5], [100, 3, 0, 0, 700], seed=14)
    run(L, b), run(L, c)
    graphs = []
    side = torch.cuda.Stream()
    for x in (b, c):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            assert x.call(L) == 0
        graphs.append(g)
    for prefix, own in [(300, [10, 0, 64, 90, 1, 33]), (299, [11, 1, 64, 0, 2, 5]), (128, [0, 0, 0, 1, 0, 65])]:
        b.prefixes, b.own = [prefix], own
        b.d[1].copy_(cuda_i32(b.prefixes)), b.d[4].copy_(cuda_i32(own))
        cache = b.cache.clone()
        b.cache.nan_to_num_(0.5)                                                  # what was behind an end may be seen now
        b.out.fill_(5.0), c.out.fill_(5.0)
        graphs[0].replay(), graphs[1].replay(), graphs[0].replay()
        assert c.call(L) == 0
        torch.cuda.synchronize()
        b.check(), c.check()
        b.cache.copy_(cache)


def test_two_streams_at_once(L):
    """Calls on two streams share nothing."""
    bs = [Batch(32, 8, 128, [900], [0, 30], [(i * 29) % 300 for i in range(30)], seed=15), Batch(8, 2, 64, [5000], [0, 50], [(i * 17) % 90 for i in range(50)], seed=16)]
    for b in bs:
        run(L, b)
        b.first = b.out.clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for b, s in zip(bs, streams):
            with torch.cuda.stream(s):
                b.out.fill_(5.0)
                assert b.call(L, stream=C.c_void_p(s.cuda_stream)) == 0
    torch.cuda.synchronize()
    for b in bs:
        assert torch.equal(b.out.view(torch.int16), b.first.view(torch.int16))


def test_a_cache_beyond_32_bits(L):
    """Pages whose bytes lie beyond 2^32 (and elements beyond 2^31) from the cache's start: copies, rotary writes and attention."""
    n_kv, dim, pages, heads = 8, 128, 40000, 32
    plane = n_kv * PAGE * dim
    assert 2 * pages * plane * 2 > 2 ** 33
    cache = torch.empty((2, pages, n_kv, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    far = [pages - 1, pages - 2, 39000, 12]
    cache[:, far] = randn(1, (2, 4, n_kv, PAGE, dim))
    moves = (_lib.OaPageMove * 2)(_lib.OaPageMove(pages - 1, 38000, 64), _lib.OaPageMove(12, 39999 - 2, 30))
    assert L.oa_k_cache_copy(ptr(cache), 2, pages, n_kv, dim, 2, moves, 2, now()) == 0
    assert torch.equal(cache[:, 38000], cache[:, pages - 1]) and torch.equal(cache[:, 39997, :, :30], cache[:, 12, :, :30])
    b = Batch(heads, n_kv, dim, [100], [0, 2], [50, 100], seed=17)
    b.cache, b.pages = cache, pages
    b.pt[0, :2], b.ot[0, 0], b.ot[1, :2] = [pages - 1, 39000], 38000, [pages - 2, 12]
    b.upload()
    qkv = randn(2, (2, (heads + 2 * n_kv) * dim))
    freqs, _ = frequencies(L, dim)
    slots, at = [38000 * PAGE + 49, 12 * PAGE + 35], qkv.data_ptr() + 2 * heads * dim
    assert L.oa_k_rotary_cache(ptr(qkv), qkv.shape[1], at, at + 2 * n_kv * dim, qkv.shape[1], ptr(b.q), heads * dim, ptr(cache), pages, ptr(cuda_i32([149, 199])), ptr(cuda_i32(slots)), 2, heads, n_kv,
                               dim, dim, 1, freqs.ctypes.data, 1.0, None, now()) == 0
    assert torch.equal(cache[1, 12, :, 35], qkv[1, (heads + n_kv) * dim:].view(n_kv, dim))
    run(L, b)
    b.check()


# ---- together -------------------------------------------------------------------------------------
def test_conversations_from_one_prompt(L):
    """A prompt's pages are forked for five conversations, each gets new tokens over four steps (rotated, written, attended), two end, the rest is compacted and goes
    on: every step's attention is the one over each conversation's whole history in 64 bits, and that of oa_k_paged_attention."""
    heads, n_kv, dim, rows, width, pages, prompt = 8, 2, 128, 6, 8, 40, 150
    rng = np.random.default_rng(3)
    tables, lens, refs = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32)
    table = _lib.OaPageTable(tables.ctypes.data, lens.ctypes.data, refs.ctypes.data, rows, width, pages)
    moves, n = (_lib.OaPageMove * pages)(), C.c_int32()
    cache = torch.full((2, pages, n_kv, PAGE, dim), math.nan, dtype=torch.bfloat16, device="cuda")
    freqs, amp = frequencies(L, dim, 500000.0, 2, 32.0, 1.0, 4.0, 8192)
    refs[[0, 3, 4]] = 1                                                            # pages that another part of a program holds
    history = {r: [] for r in range(rows)}                                          # each row's keys and values as they were given, positions from 0

    def append(which, count):
        start = {r: int(lens[r]) for r in which}
        for r in which:
            assert L.oa_host_cache_grow(table, r, count) == 0
        at = [(r, i) for r in which for i in range(start[r], start[r] + count)]
        qkv = randn(int(rng.integers(1 << 30)), (len(at), (heads + 2 * n_kv) * dim))
        slots = [int(tables[r, i // PAGE]) * PAGE + i % PAGE for r, i in at]
        q = torch.empty((len(at), heads * dim), dtype=torch.bfloat16, device="cuda")
        k0 = qkv.data_ptr() + 2 * heads * dim
        assert L.oa_k_rotary_cache(ptr(qkv), qkv.shape[1], k0, k0 + 2 * n_kv * dim, qkv.shape[1], ptr(q), heads * dim, ptr(cache), pages, ptr(cuda_i32([i for _, i in at])), ptr(cuda_i32(slots)),
                                   len(at), heads, n_kv, dim, dim, 1, freqs.ctypes.data, amp, None, now()) == 0
        for j, (r, _) in enumerate(at):
            history[r].append(qkv[j].view(-1, dim)[heads:])
        return q

    def attend(which, q):
        shared = prompt // PAGE                                                    # the prompt's full pages lie in every row's table
        own = [int(lens[r]) - shared * PAGE for r in which]
        out = torch.empty_like(q)
        t = cuda_i32(tables[which])
        prefix = t[:1, :shared].contiguous()
        own_tables = t[:, shared:].contiguous()
        assert L.oa_k_prefix_attention(ptr(q), heads * dim, ptr(out), heads * dim, ptr(cache), pages, ptr(prefix), shared, ptr(cuda_i32([shared * PAGE])), ptr(cuda_i32([0, len(which)])), 1,
                                       ptr(own_tables), own_tables.shape[1], ptr(cuda_i32(own)), len(which), heads, n_kv, dim, 0.0, None, now()) == 0
        whole, host, ctx = torch.empty_like(q), np.maximum(tables[which], 0), lens[which].copy()
        clean = torch.nan_to_num(cache, 0.0)                                       # that entry asks for finite places behind an end
        assert L.oa_k_paged_attention(ptr(q), ptr(whole), ptr(clean), pages, host.ctypes.data, width, ctx.ctypes.data, None, len(which), heads, n_kv, dim, 0, now()) == 0
        torch.cuda.synchronize()
        for j, r in enumerate(which):
            x = torch.stack(history[r])
            k, _ = turned(x[:, :n_kv], torch.arange(len(x), device="cuda"), freqs, amp, dim, 1)
            k, v, y = k.bfloat16().double(), x[:, n_kv:].double(), q[j].double().view(n_kv, -1, dim)
            p = torch.softmax(torch.einsum("khd,pkd->khp", y, k) / math.sqrt(dim), -1)
            want, size = torch.einsum("khp,pkd->khd", p, v), torch.einsum("khp,pkd->khd", p, v.abs())
            # keys that lie within 2^-19 of a rounding step may be a whole step of bf16 off: 2^-7 of |q k| on few keys, bounded here on all
            score = torch.einsum("khd,pkd->khp", y.abs(), k.abs()) / math.sqrt(dim) * 2.0 ** -7 * 2.0 ** -9
            tol = (size * (2.0 ** -8 + 2 * score.amax(-1, keepdim=True) + 2.0 ** -12) + want.abs() * 2.0 ** -7).view(-1)
            assert bool(((out[j].double() - want.view(-1)).abs() <= tol).all()) and bool(((whole[j].double() - want.view(-1)).abs() <= tol).all())

    append([0], prompt)
    children = np.array([1, 2, 3, 4, 5], np.int32)
    assert L.oa_host_cache_fork(table, 0, children.ctypes.data, 5, moves, pages, C.byref(n)) == 0 and n.value == 5
    assert L.oa_k_cache_copy(ptr(cache), 2, pages, n_kv, dim, 2, moves, n.value, now()) == 0
    for r in range(1, 6):
        history[r] = list(history[0])
    append([2], 77)
    for _ in range(4):
        attend([1, 2, 3, 4, 5], append([1, 2, 3, 4, 5], 1))
    ended = np.array([0, 3], np.int32)
    assert L.oa_host_cache_free(table, ended.ctypes.data, 2) == 0
    refs[[0, 3, 4]] = 0
    assert L.oa_host_cache_compact(table, moves, pages, C.byref(n)) == 0 and n.value > 0
    assert L.oa_k_cache_copy(ptr(cache), 2, pages, n_kv, dim, 2, moves, n.value, now()) == 0
    cache[:, int((refs > 0).sum()):] = math.nan
    for _ in range(3):
        attend([1, 2, 4, 5], append([1, 2, 4, 5], 1))
