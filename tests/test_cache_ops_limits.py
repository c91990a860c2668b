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
