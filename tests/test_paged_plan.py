"""csrc/paged_plan.h, which kernels serve a call of mi_attention and how keys are shared out to blocks, on the CPU: every sequence's
rows are some launch's, the blocks suffice for any lengths, and no launch has many that nothing can come to."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from helpers import ROOT

DRIVER = """
#include "paged_plan.h"
using namespace mi;
static const Room kAll{32u << 20, 16384};
// of a call: for each launch wavefronts, slices, target, least, from, to, blocks per key/value head (blocks too many for an int: -1), threads
extern "C" int launches(const int* v, int room, int cus, int* out) {
    const AttentionSize a{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]};
    const PagedLaunches r = attention_launches(a, room ? kAll : Room{}, cus);
    for (int i = 0; i < r.n; ++i) {
        const PagedLaunch& l = r.of[i];
        const int64_t each = l.blocks % a.n_kv_heads ? -2 : l.blocks / a.n_kv_heads;
        const int x[8] = {l.wavefronts, l.slices, l.plan.target, l.plan.least, l.plan.from, l.plan.to, each > 0x7fffffff ? -1 : static_cast<int>(each), l.threads};
        for (int k = 0; k < 8; ++k) out[8 * i + k] = x[k];
    }
    return r.n;
}
extern "C" int down(int start, int end) { return goes_down(start, end); }
extern "C" int span_n(int start, int end, int rows) { return span_of(start, end, 0, rows).n; }
// items of a launch over the sequences (rows n, positions len each), and the greatest number of parts of a set
extern "C" void items(const int* v, const int* l, const int* n, const int* len, long long* out) {
    Plan plan;
    plan.target = l[2], plan.least = l[3], plan.from = l[4], plan.to = l[5], plan.nrep = v[4] / v[5];
    const int rows = l[0] ? 32 * l[0] : kRows, keys = l[0] ? kChunkKeys : kKeys;
    float all = 0;
    int first = 0;
    for (int pass = 0; pass < 2; ++pass) {
        const int share = share_of(all, plan);
        out[0] = out[1] = out[2] = 0;
        first = 0;
        for (int b = 0; b < v[0]; first += n[b++]) {
            const Cost c = cost_of(plan, span_of(first, first + n[b], len[b], v[1]), v[3], v[7], v[8], rows, keys);
            all += pass ? 0 : static_cast<float>(c.sets) * static_cast<float>(c.tiles);
            const long long chunks = c.sets ? (c.tiles - 1) / share + 1 : 0;
            out[0] += c.sets * chunks;
            out[1] += c.sets;
            out[2] = chunks > out[2] ? chunks : out[2];
        }
    }
}
"""
NAMES = "n_seqs n_tokens max_tokens cap n_heads n_kv_heads head_dim window sinks".split()


class Launch:
    def __init__(self, raw):
        self.raw = list(raw)
        self.wavefronts, self.slices, self.target, self.least, self.first, self.last, self.each, self.threads = raw
        self.rows = 32 * self.wavefronts or 16


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("plan")
    src, so = d / "plan.cpp", str(d / "plan.so")
    src.write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "adreno-llms_amd", "csrc"), "-o", so, str(src)])
    lib = ctypes.CDLL(so)

    def launches(room=True, cus=256, **size):
        v, out = (ctypes.c_int * 9)(*[size.get(n, 0) for n in NAMES]), (ctypes.c_int * 16)()
        return [Launch(out[8 * i:8 * i + 8]) for i in range(lib.launches(v, int(room), cus, out))]

    def items(launch, new, lengths, **size):
        """(items, sets, most parts of a set) per key/value head"""
        v, out = (ctypes.c_int * 9)(*[size.get(n, 0) for n in NAMES]), (ctypes.c_longlong * 3)()
        lib.items(v, (ctypes.c_int * 8)(*launch.raw), (ctypes.c_int * len(new))(*new), (ctypes.c_int * len(new))(*lengths), out)
        return list(out)

    rule = lambda: None                                                            # noqa: E731
    rule.launches, rule.items, rule.down, rule.span_n = launches, items, lib.down, lib.span_n
    return rule


def _size(new, lengths, heads=32, kv=8, D=128, pad=0, **more):
    return dict(dict(n_seqs=len(new), n_tokens=sum(new) + pad, max_tokens=max(new), cap=-(-max(lengths) // 64) * 64, n_heads=heads, n_kv_heads=kv,
                     head_dim=D), **more)


def test_blocks_suffice_and_every_row_has_a_launch(rule):
    rng = random.Random(3)
    seen = set()
    for _ in range(3000):
        seqs = rng.choice([1, 2, 5, 17, 64, 65, 200])
        form = rng.choice(["step", "few", "chunk", "mixed", "mixed"])
        top = dict(step=1, few=9, chunk=700, mixed=700)[form]
        new = [rng.choice([0, 1, 1, 1]) if form == "mixed" and b % 4 else rng.randint(0 if form == "mixed" else 1, top) for b in range(seqs)]
        if not sum(new):
            continue
        lengths = [n + rng.choice([0, 5, 900, 6000]) for n in new]
        heads, kv, D = rng.choice([(14, 2, 64), (9, 3, 64), (12, 12, 64), (32, 8, 128), (8, 1, 128), (40, 1, 64)])
        window = rng.choice([0, 0, 100, 1000])
        size = _size(new, lengths, heads, kv, D, pad=rng.choice([0, 0, 33, 4000]), window=window, sinks=rng.choice([0, 4]))
        if rng.random() < 0.2:
            size["max_tokens"] = rng.choice([0, 1, 7, 5000])                       # a wrong hint
        all_launches = rule.launches(room=rng.random() < 0.8, **size)
        nrep = heads // kv
        for n in new:
            if n:
                assert sum(x.first <= n * nrep <= x.last for x in all_launches) == 1, (size, n)
        for x in all_launches:
            n, sets, parts = rule.items(x, new, lengths, **size)
            assert sets <= n <= x.each and x.threads == 64 * (x.wavefronts * x.slices or 4), (size, x.raw, n)
            assert parts <= 1 or (x.target > 0 and x.each * kv <= 16384 // max(x.wavefronts, 1)), (size, x.raw)
            if parts:
                seen.add((D, x.wavefronts, x.slices, parts > 1))
    assert {(D, w, s, p) for D, w, s in [(64, 0, 1), (64, 2, 4), (64, 4, 1), (128, 0, 1), (128, 4, 2), (128, 4, 1)] for p in (0, 1)} == seen


def test_a_launch_counts_its_own_sequences(rule):
    """A launch of sequences of a few rows, or of many, is not sized by the rows of the others."""
    # decode rows of long conversations beside one chunk of a prompt: the few rows' keys are split
    new, lengths = [1] * 16 + [2032], [32768] * 16 + [2032]
    many, few = rule.launches(**_size(new, lengths))
    assert many.wavefronts and not few.wavefronts and few.target == 3 * 256 // 8 and few.each - few.target <= 17 * 2
    assert rule.items(few, new, lengths, **_size(new, lengths))[2] > 4
    # one chunk among 63 single tokens: room for parts and slices of it
    new, lengths = [1] * 63 + [256], [3000] * 63 + [3000]
    many, few = rule.launches(**_size(new, lengths))
    assert (many.wavefronts, many.slices) == (4, 2) and many.target >= 128 // 8 and few.target == 3 * 256 // 8
    # and a batch of which nothing can be long enough for the kernel for many rows, whatever the hint says
    one, = rule.launches(**dict(_size([1] * 3, [100000] * 3), max_tokens=4096, cap=2 ** 24))
    assert one.wavefronts == 0 and one.last >= 12


def test_rows_that_no_two_sequences_share(rule):
    """Wherever q_start does not go down, whatever else it holds, the sequences' rows are no more than the batch's; one that goes down
    has more, so it has to be told apart."""
    rng = random.Random(4)
    big, ups, more = 2 ** 31 - 1, 0, 0
    for _ in range(20000):
        rows = rng.choice([1, 7, 100])
        start = [rng.choice([-big, -1, 0, 0, 3, 5, 7, 50, 100, 101, big]) for _ in range(rng.randint(2, 6))]
        if rng.random() < 0.5:
            start.sort()
        down = any(rule.down(s, e) for s, e in zip(start, start[1:]))
        all_rows = sum(rule.span_n(s, e, rows) for s, e in zip(start, start[1:]))
        ups += not down
        more += all_rows > rows
        assert down or all_rows <= rows
    assert ups > 5000 and more > 500
    # the blocks of such a call would not be all there: 6 sequences of the same 5 rows, counted as 5 rows
    size = dict(_size([5] * 6, [3000] * 6, heads=14, kv=2, D=64), n_tokens=5, max_tokens=1)
    one, = rule.launches(**size)
    n, sets, parts = rule.items(one, [5] * 6, [3000] * 6, **dict(size, n_tokens=30))
    assert parts > 1 and sets > one.each - one.target and any(rule.down(s, e) for s, e in zip([0, 5, 0], [5, 0, 5]))


def test_cases_come_to_the_kernels_that_they_are_for(rule):
    """On 256 compute units, those of the device that they are written for."""
    from helpers import mil                                                        # noqa: F401
    from test_paged_kernels_gpu import FEW, MANY, UNDER_WINDOW, WIDE, WINDOW_CACHE

    def of(case, page, columns=0, **more):
        pages = max(-(-max(case["lengths"]) // page), columns // page)
        size = _size(case["new"], case["lengths"], case["heads"], case["kv_heads"], case["D"], pad=case.get("pad", 0), cap=pages * page, **more)
        return rule.launches(**size)

    for (D, slices), (case, columns) in MANY.items():
        for page in (16, 100, 48, 5):
            many, few = of(case, page, columns)
            assert (many.wavefronts, many.slices, few.wavefronts) == (2 if slices == 4 else 4, slices, 0), (D, slices, page)
    for case in FEW.values():
        assert [x.wavefronts for x in of(case, 16)] == [0]
    for slices, pad, window, sinks in UNDER_WINDOW:
        many = of(dict(WINDOW_CACHE, pad=pad), 16, window=window, sinks=sinks)[0]
        assert many.wavefronts and many.slices == slices, (pad, window, sinks)
    assert WIDE == 2 ** 20
