"""The operators on a caller's paged cache at the limits of what their entry points accept, no GPU: the arithmetic that deals out units of work, rows whose lengths
come near 31 bits, and arguments at the edge of a refusal."""
import ctypes as C
import glob
import os
import random
import re
import subprocess

import numpy as np
import pytest

from opsagent_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAGE = 64


@pytest.fixture(scope="module")
def L():
    return _lib.load()


# ---- units of work -----------------------------------------------------------------------------
SRC_UNITS = r'''
#include <cstdio>
#include "opsagent_b200/csrc/work_units.hpp"
int main() {                                             // lines of (grid, total, unit) -> busy CTAs, the unit's CTA, that CTA's first unit and the next one's
    long long grid, total, unit;
    while (std::scanf("%lld %lld %lld", &grid, &total, &unit) == 3) {
        const long long busy = oa::busy_ctas(grid, total); const int cta = oa::cta_of(unit, busy, total);
        std::printf("%lld %d %lld %lld\n", busy, cta, (long long)oa::first_unit(cta, busy, total), (long long)oa::first_unit(cta + 1, busy, total));
    }
    return 0;
}
'''


def test_units_are_dealt_out_exactly_beyond_32_bits(tmp_path):
    """Whole-number arithmetic of any length says whose a unit is, from one unit up to the most that prefix attention accepts (2^20 sequences of 2^10 heads and 2^24 pages a table):
    a dividend below 2^32 over a divisor beyond it is 0, not what is left of the divisor."""
    src, exe, rng = tmp_path / "units.cpp", tmp_path / "units", random.Random(1)
    src.write_text(SRC_UNITS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{ROOT}", str(src), "-o", str(exe)], check=True)
    most = 2 ** 20 * 2 ** 10 * (1 + 2 * 2 ** 24)
    totals = [1, 2, 147, 148, 149, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 1, 2 ** 34 + 1024, 2 ** 40 + 3, most] + [int(2 ** rng.uniform(0, 55)) for _ in range(200)]
    asked = []
    for total in totals:
        for grid in (1, 7, 132, 148):
            busy, page_units = min(grid, total), min(total, 2 ** 24 + 1)
            edges = {total * c // busy + d for c in (0, 1, busy // 2, busy - 1, busy) for d in (-1, 0, 1)} | {page_units - 1, page_units, rng.randrange(total)}
            asked += [(grid, total, u) for u in sorted(edges) if 0 <= u < total]
    r = subprocess.run([str(exe)], input="\n".join("%d %d %d" % x for x in asked), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-500:]
    got = [tuple(map(int, line.split())) for line in r.stdout.splitlines()]
    assert len(got) == len(asked)
    for (grid, total, unit), g in zip(asked, got):
        busy = min(grid, total)
        cta = next(c for c in range(busy) if total * c // busy <= unit < total * (c + 1) // busy)
        assert g == (busy, cta, total * cta // busy, total * (cta + 1) // busy), (grid, total, unit, g)


# ---- pages -------------------------------------------------------------------------------------
def test_a_row_that_would_pass_31_bits_is_not_grown(L):
    """A table with room for more tokens than a length can count: the last ones that fit are given, one more is refused and changes nothing."""
    width, full = 2 ** 25 + 8, 2 ** 31 - PAGE                             # a row of one page named over and over
    tables, lens, refs = np.zeros((1, width), np.int32), np.array([full], np.int32), np.array([2 ** 30, 0], np.int32)
    tables[0, full // PAGE:] = -1
    t = _lib.OaPageTable(tables.ctypes.data, lens.ctypes.data, refs.ctypes.data, 1, width, 2)
    for more in (PAGE, 200, 2 ** 31 - 1):
        assert L.oa_host_cache_grow(t, 0, more) == 400
        assert "page table" in _lib.last_error() and lens.tolist() == [full] and refs.tolist() == [2 ** 30, 0] and (tables[0, full // PAGE:] == -1).all()
    assert L.oa_host_cache_grow(t, 0, PAGE - 1) == 0
    assert lens.tolist() == [2 ** 31 - 1] and refs.tolist() == [2 ** 30, 1] and tables[0, full // PAGE] == 1 and (tables[0, full // PAGE + 1:] == -1).all()
    assert L.oa_host_cache_grow(t, 0, 1) == 400 and L.oa_host_cache_grow(t, 0, 0) == 0 and lens.tolist() == [2 ** 31 - 1]


# ---- order of a kernel's first steps ---------------------------------------------------------------
def _kernels(source):
    """Bodies of the __global__ functions of a CUDA source, without comments."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", source, flags=re.S)
    for part in text.split("__global__")[1:]:
        at = depth = part.index("{")
        depth = 0
        for i in range(at, len(part)):
            depth += {"{": 1, "}": -1}.get(part[i], 0)
            if depth == 0:
                yield part[:at], part[at:i + 1]
                break


def test_tensor_memory_is_held_before_the_next_kernel_may_start():
    """A kernel that lets its successor start while one of its own CTAs still waits for tensor memory could wait for columns that the successor, which waits for it, has taken.  The signal comes
    behind the allocation: behind a barrier of the whole CTA, or from the warp that allocates and no other."""
    seen = 0
    for path in sorted(glob.glob(os.path.join(ROOT, "opsagent_b200", "csrc", "*.cu"))):
        for head, body in _kernels(open(path).read()):
            alloc = re.search(r"tmem_alloc<|tcgen05\.alloc", body)
            if not alloc:
                continue
            seen += 1
            first = body.find("griddep_launch()")
            assert first > alloc.start(), (path, head.strip()[-200:])
            behind_barrier = "__syncthreads()" in body[alloc.start():first]
            same_warp = body[:alloc.start()].endswith("if (warp == 1) ") and body[:first].endswith("if (warp == 1) ")
            assert behind_barrier or same_warp, (path, head.strip()[-200:])
    assert seen >= 8


def test_copies_do_not_read_by_the_read_only_path():
    """A page may have been written by the kernel ahead, which has not ended when the copy's CTAs start: loads that ask for memory nobody writes while their kernel lives are not for it."""
    for name in ("cache_copy.cu", "common.cuh"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "opsagent_b200", "csrc", name)).read())
        assert not re.search(r"ld\.global\.nc|__ldg\(", text), name


# ---- pitches and rows ------------------------------------------------------------------------------
BUF, FREQS = np.zeros(4096, np.int32), np.ones(128)
P, FAR = (BUF.ctypes.data + 15) // 16 * 16, 1 << 40                       # addresses alone: nothing behind them is touched before a device is found


def rotary(L, x=P, ldx=256, out=P, ldo=256, T=2, f32=0):
    return L.oa_k_rotary(x, ldx, out, ldo, P, T, 2, 128, 64, 1, FREQS.ctypes.data, 1.0, 0, f32, None), _lib.last_error()


def rotary_cache(L, q=FAR, ldq=512, k=FAR + 512, v=FAR + 768, ldkv=512, out=FAR, ldo=512, T=5):
    return L.oa_k_rotary_cache(q, ldq, k, v, ldkv, out, ldo, 2 * FAR, 4, P, P, T, 2, 1, 128, 128, 1, FREQS.ctypes.data, 1.0, None, None), _lib.last_error()


def attention(L, q=FAR, ldq=1024, out=FAR, ldo=1024, n=3, scale=0.0):
    return L.oa_k_prefix_attention(q, ldq, out, ldo, 2 * FAR, 8, P, 2, P, P, 1, P, 2, P, n, 8, 2, 128, scale, None, None), _lib.last_error()


PITCHES = [2 ** 39, 2 ** 45, 2 ** 61, 2 ** 62, 2 ** 63 - 8]


@pytest.mark.parametrize("pitch", PITCHES)
def test_pitches_that_no_memory_has_are_refused(L, pitch):
    """Two rows so far apart that their addresses leave 64 bits, or that no device holds both: refused, and the process goes on."""
    for f32 in (0, 1):
        assert rotary(L, ldx=pitch, ldo=pitch, f32=f32)[0] == 400 and "apart" in _lib.last_error()
        for case in [dict(ldx=pitch, out=P + 2 ** 20), dict(ldo=pitch, out=P + 2 ** 20), dict(ldx=pitch // 64, ldo=pitch // 64, T=100), dict(ldx=pitch, ldo=pitch, out=P + 16)]:
            assert rotary(L, **case, f32=f32)[0] == 400 and "rotary" in _lib.last_error(), case
    for case in [dict(ldq=pitch), dict(ldkv=pitch), dict(ldo=pitch, out=3 * FAR), dict(ldq=pitch, ldo=pitch), dict(ldq=pitch, ldo=pitch, ldkv=pitch)]:
        assert rotary_cache(L, **case)[0] == 400 and "apart" in _lib.last_error(), case
    for case in [dict(ldq=pitch), dict(ldo=pitch, out=3 * FAR), dict(ldq=pitch, ldo=pitch)]:
        assert attention(L, **case)[0] == 400 and "apart" in _lib.last_error(), case


@pytest.mark.parametrize("pitch", PITCHES)
def test_a_single_row_may_have_any_pitch(L, pitch):
    """Nothing lies a pitch away from a single row.  Only overlaps are judged here: without a device the call ends behind that."""
    for f32 in (0, 1):
        assert rotary(L, ldx=pitch, ldo=pitch, T=1, f32=f32)[0] != 400 or "device" in _lib.last_error()
        code, text = rotary(L, ldx=pitch, out=P + 16, ldo=pitch, T=1, f32=f32)
        assert code == 400 and "overlap" in text
        assert "overlap" not in rotary(L, ldx=pitch, out=P + 1024, ldo=pitch, T=1, f32=f32)[1]
    assert "overlap" not in rotary_cache(L, ldq=pitch, ldkv=pitch, ldo=pitch, T=1)[1] and "apart" not in rotary_cache(L, ldq=pitch, ldkv=pitch, ldo=pitch, T=1)[1]
    assert "overlap" not in attention(L, ldq=pitch, ldo=pitch, n=1)[1] and "apart" not in attention(L, ldq=pitch, ldo=pitch, n=1)[1]


def test_a_single_row_is_turned_in_place_under_any_two_pitches(L):
    """out is x itself, whatever the pitches of the one row are; two rows under two pitches are not the same rows."""
    assert "overlap" not in rotary(L, ldo=264, T=1)[1] and "overlap" not in rotary(L, ldx=1024, T=1, f32=1)[1]
    assert "overlap" not in rotary_cache(L, ldo=256, T=1)[1] and "overlap" not in attention(L, ldo=2048, n=1)[1]
    for code, text in (rotary(L, ldo=264), rotary_cache(L, ldo=256, T=2), attention(L, ldo=2048, n=2), rotary(L, out=P + 16, ldo=264, T=1)):
        assert code == 400 and "overlap" in text


def test_a_scale_beyond_fp32_in_powers_of_two_is_refused(L):
    """Scores are taken times scale log2(e) in fp32: where that is infinite, a score of 0 would become NaN."""
    largest = np.nextafter(np.float32(np.finfo(np.float32).max / 1.4426950408889634), np.float32(0))
    assert attention(L, scale=float(largest))[0] != 400 or "device" in _lib.last_error()
    for scale in (2.4e38, float(np.finfo(np.float32).max)):
        code, text = attention(L, scale=scale)
        assert code == 400 and "scale" in text
