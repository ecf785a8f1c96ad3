"""csrc/paged_rule.h, what the kernels over a paged cache take from numbers in device memory, on the CPU: divisions, rows of
sequences, what a query sees and the tiles that cover it, for any values of those numbers."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from helpers import ROOT

DRIVER = """
#include "paged_rule.h"
using namespace mi;
extern "C" int quotient(int n, int d) { return divide(n, make_divider(d)); }
extern "C" void span(int s, int e, int len, int rows, int* out) { const Span x = span_of(s, e, len, rows); out[0] = x.first; out[1] = x.n; out[2] = x.pos; }
extern "C" int cap_of(int pages, int size) { return capacity(pages, size); }
extern "C" int seen(int p, int j, int w, int s) { return sees(p, j, w, s); }
extern "C" int every(int j0, int size, int lo, int hi, int cap, int w, int s) { return all_seen(j0, size, lo, hi, cap, w, s); }
extern "C" void tiles(int lo, int hi, int cap, int w, int s, int size, int* out) {
    const Tiles t = tiles_of(lo, hi, cap, w, s, size);
    out[0] = t.count; out[1] = t.end; out[2] = t.count ? tile_at(t, t.count - 1) : -1;
    for (int i = 0; i < t.count && i < 60; ++i) out[3 + i] = tile_at(t, i);
}
"""
BIG = 2 ** 31 - 1


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("rule")
    src, so = d / "paged.cpp", str(d / "paged.so")
    src.write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "adreno-llms_amd", "csrc"), "-o", so, str(src)])
    return ctypes.CDLL(so)


def test_divide(rule):
    rng = random.Random(1)
    ds = list(range(1, 300)) + [2 ** k + e for k in range(8, 31) for e in (-1, 0, 1)] + [BIG] + [rng.randint(1, BIG) for _ in range(300)]
    for d in ds:
        ns = [0, 1, d - 1, d, d + 1, BIG, BIG - 1, BIG // d * d, BIG // d * d - 1] + [rng.randint(0, BIG) for _ in range(20)]
        for n in ns:
            if 0 <= n <= BIG:
                assert rule.quotient(n, d) == n // d, (n, d)


def test_rows_of_a_sequence(rule):
    out = (ctypes.c_int * 3)()
    for s in (-BIG, -1, 0, 3, 10, BIG):
        for e in (-BIG, -1, 0, 3, 7, 10, 11, BIG):
            for length in (-BIG, -1, 0, 2, 100, BIG):
                rule.span(s, e, length, 10, out)
                first, n, pos = out
                assert 0 <= first <= 10 and 0 <= n <= 10 - first and pos == max(length, 0) - n
                if 0 <= s <= e <= 10:
                    assert (first, n) == (s, e - s)
    assert rule.cap_of(3, 16) == 48 and rule.cap_of(BIG, BIG) == BIG


def _sees(p, j, w, s):
    return j <= p and (w <= 0 or j > p - w or j < s)


def test_tiles_cover_what_is_seen(rule):
    rng, out = random.Random(2), (ctypes.c_int * 64)()
    for _ in range(4000):
        size = rng.choice([16, 32, 64])
        lo = rng.randint(-20, 400)
        hi = lo + rng.choice([0, 1, 5, 15, 70])
        cap, w = rng.choice([0, 1, 40, 300, 10000]), rng.choice([-3, 0, 1, 2, 17, 64, 100, 399, 5000])
        s = rng.choice([0, 1, 4, 37, 64, 1000])
        rule.tiles(lo, hi, cap, w, s, size, out)
        count, end, last = out[0], out[1], out[2]
        got = [out[3 + i] for i in range(count)]
        assert count <= 60 and got == sorted(set(got))
        seen = {j for p in range(max(lo, 0), hi + 1) for j in range(min(p + 1, cap)) if _sees(p, j, w, s)}
        assert {j // size for j in seen} <= set(got), (lo, hi, cap, w, s, size)
        # none for nothing, but for what lies between the window of the first and the last query, and the table's end
        assert all(0 <= t * size < max(end, 1) for t in got)
        if seen:
            assert end >= max(seen) + 1 and end <= cap and last == got[-1]
        for t in got:
            j0 = t * size
            every = all(j in seen and all(_sees(p, j, w, s) for p in range(lo, hi + 1)) for j in range(j0, j0 + size)) if lo >= 0 else False
            said = rule.every(j0, size, lo, hi, cap, w, s)       # (a tile that is seen in part as first positions may not count)
            assert said == every or (not said and 0 < s < j0 + size), (j0, size, lo, hi, cap, w, s)
        for p in (lo, hi):
            for j in range(0, 60, 7):
                if p >= 0:
                    assert rule.seen(p, j, w, s) == _sees(p, j, w, s)


def test_numbers_of_any_size(rule):
    out = (ctypes.c_int * 64)()
    for lo in (-BIG, -1, 0, 5, BIG - 1, BIG):
        for hi in (lo, BIG):
            for cap in (0, 1, BIG):
                for w in (-BIG, 0, 1, 5, BIG):
                    for s in (0, 1, BIG):
                        rule.tiles(lo, hi, cap, w, s, 32, out)
                        assert out[0] >= 0 and (out[0] == 0 or 0 <= out[2] <= (cap - 1) // 32)
                        for j0 in (0, BIG - 31):
                            if hi >= 0:
                                rule.every(j0, 32, lo, hi, cap, w, s)
                                rule.seen(hi, j0, w, s)
