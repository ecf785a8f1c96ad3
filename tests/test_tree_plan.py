"""csrc/paged_plan.h, which kernel serves a call of mi_attention_tree and how keys are shared out to its blocks, on the CPU: the blocks
suffice for any trees and lengths, also with the least share that fits; and csrc/beam_rule.h, how logits are cut up."""
import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

from helpers import ROOT

DRIVER = """
#include "beam_rule.h"
#include "paged_plan.h"
using namespace mi;
static const Room kAll{32u << 20, 16384};
static PagedLaunch launch_of(const int* v, int room, int cus) {
    return tree_launch(AttentionSize{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9] == 0}, room ? kAll : Room{}, cus);
}
// wavefronts, slices, sets, target, blocks per key/value head, threads
extern "C" void launch(const int* v, int room, int cus, int* out) {
    const PagedLaunch l = launch_of(v, room, cus);
    const int x[6] = {l.wavefronts, l.slices, l.sets, l.plan.target, static_cast<int>(l.blocks % v[5] ? -1 : l.blocks / v[5]), l.threads};
    for (int k = 0; k < 6; ++k) out[k] = x[k];
}
// share, items, sets, most parts of a set: by the first share, then by the least that fits
extern "C" void items(const int* v, int room, int cus, const int* n, const int* len, int* out) {
    const PagedLaunch l = launch_of(v, room, cus);
    const int rows = l.wavefronts ? 32 * l.wavefronts : kRows * l.sets, keys = l.wavefronts ? kChunkKeys : kKeys;
    auto of = [&](auto f) {
        for (int b = 0, first = 0; b < v[0]; first += n[b++]) f(cost_of(l.plan, span_of(first, first + n[b], len[b], v[1]), v[3], v[7], v[8], rows, keys));
    };
    float all = 0;
    of([&](Cost c) { all += static_cast<float>(c.sets) * static_cast<float>(c.tiles); });
    int share = share_of(all, l.plan);
    for (int pass = 0; pass < 2; ++pass, out += 4) {
        out[0] = share, out[1] = out[2] = out[3] = 0;
        of([&](Cost c) {
            out[1] += items_of(c, share), out[2] += c.sets;
            const int parts = c.sets ? (c.tiles - 1) / share + 1 : 0;
            out[3] = parts > out[3] ? parts : out[3];
        });
        if (l.plan.target > 0) share = even_share(share, static_cast<int>(l.blocks / v[5]), [&](int s) {
            int sum = 0;
            of([&](Cost c) { sum += items_of(c, s); });
            return sum;
        });
    }
}
// share, items: by share_of, then by round_share (sequences' sets and tiles; sums in fp32 as on the device, the quotients by a reciprocal that is `off` too great)
extern "C" void rounds(int n, const int* sets, const int* tiles, int target, int resident, int least, int blocks, float off, int* out) {
    Plan plan;
    plan.target = target, plan.least = least;
    float all = 0;
    int every = 0, most = 0;
    for (int b = 0; b < n; ++b) all += static_cast<float>(sets[b]) * static_cast<float>(tiles[b]), every += sets[b], most = tiles[b] > most ? tiles[b] : most;
    const auto items = [&](int share) {
        float sum = 0;
        for (int b = 0; b < n; ++b) {
            const float x = share > tree_worth(tiles[b]) ? share : tree_worth(tiles[b]);
            sum += static_cast<float>(sets[b]) * (static_cast<float>(static_cast<int>((static_cast<float>(tiles[b]) - 0.5f) * (1.0f / x * off))) + 1.0f);
        }
        return static_cast<int>(sum);
    };
    int share = share_of(all, plan);
    for (int pass = 0; pass < 2; ++pass, out += 2) {
        out[0] = share, out[1] = 0;
        for (int b = 0; b < n; ++b) out[1] += items_of({sets[b], tiles[b]}, share > tree_worth(tiles[b]) ? share : tree_worth(tiles[b]));
        share = round_share(share, all, every, most, plan, resident, blocks, items);
    }
}
extern "C" void apart(unsigned in, unsigned sets, unsigned pairs, unsigned* out) {
    const SetOfPair x = eight_apart(in, sets, pairs);
    out[0] = x.set, out[1] = x.pair;
}
extern "C" unsigned up(unsigned h) { return ascending(h); }
extern "C" unsigned back(unsigned a) { return half_bits(a); }
extern "C" int token(int tile, int lane, int e) { return token_of(tile, lane, e); }
extern "C" int tiles(int vocab) { return tiles_of_row(vocab); }
extern "C" long long fit(long long bytes, int beams, int vocab) { return groups_that_fit(bytes, beams, vocab); }
"""
NAMES = "n_seqs n_tokens max_tokens cap n_heads n_kv_heads head_dim window sinks codes".split()


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("tree_plan")
    src, so = d / "plan.cpp", str(d / "plan.so")
    src.write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "adreno-llms_amd", "csrc"), "-o", so, str(src)])
    lib = ctypes.CDLL(so)
    lib.fit.restype, lib.fit.argtypes = ctypes.c_longlong, [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]

    def size(s):
        return (ctypes.c_int * 10)(*[s.get(n, 0) for n in NAMES])

    def launch(s, room=True, cus=256):
        out = (ctypes.c_int * 6)()
        lib.launch(size(s), int(room), cus, out)
        return dict(zip("wavefronts slices sets target each threads".split(), out))

    def items(s, new, lengths, room=True, cus=256):
        out = (ctypes.c_int * 8)()
        lib.items(size(s), int(room), cus, (ctypes.c_int * len(new))(*new), (ctypes.c_int * len(new))(*lengths), out)
        return list(out[:4]), list(out[4:])

    lib.launch_of, lib.items_of = launch, items
    return lib


def size_of(new, lengths, heads, kv, D, pad=0, page=64, columns=0, **more):
    pages = max(-(-max(lengths) // page), columns // page, 1)
    return dict(dict(n_seqs=len(new), n_tokens=sum(new) + pad, max_tokens=max(new), cap=pages * page, n_heads=heads, n_kv_heads=kv, head_dim=D), **more)


def test_blocks_suffice(rule):
    rng = random.Random(5)
    seen = set()
    for _ in range(3000):
        seqs = rng.choice([1, 2, 5, 17, 64, 65, 200])
        new = [rng.randint(0, rng.choice([2, 24, 64, 130])) for _ in range(seqs)]
        if not sum(new):
            continue
        lengths = [n + rng.choice([0, 5, 900, 6000, 30000]) for n in new]
        heads, kv, D = rng.choice([(14, 2, 64), (9, 3, 64), (12, 12, 64), (32, 8, 128), (8, 1, 128), (40, 1, 64), (16, 8, 128)])
        s = size_of(new, lengths, heads, kv, D, pad=rng.choice([0, 0, 33, 4000]), window=rng.choice([0, 0, 100, 1000]), sinks=rng.choice([0, 4]))
        if rng.random() < 0.2:
            s["max_tokens"] = rng.choice([0, 1, 7, 5000])                          # a wrong hint
        s["codes"] = rng.choice([0, 1])
        room = rng.random() < 0.8
        l = rule.launch_of(s, room)
        assert l["threads"] == 64 * (l["wavefronts"] or 4) and l["slices"] == 1
        for share, n, sets, parts in rule.items_of(s, new, lengths, room):
            assert sets <= n <= l["each"], (s, l, n)
            assert parts <= 1 or (l["target"] > 0 and l["each"] * kv <= 16384 // max(l["wavefronts"], 1)), (s, l)
        (first, _, _, _), (even, _, _, _) = rule.items_of(s, new, lengths, room)
        assert first // 2 < even <= first or first == 1
        seen.add((D, l["wavefronts"], l["sets"], parts > 1))
    assert seen >= {(D, w, s, p) for D in (64, 128) for w, s in ((0, 1), (0, 2), (4, 1)) for p in (True, False)}, seen


def test_cases_come_to_the_kernels_that_they_are_for(rule):
    """On 256 compute units, those of the device that they are written for."""
    from test_tree_attention_gpu import CASES, COLUMNS, WIDER

    for codes in (0, 1):                                                           # fp16; int8 or Q4
        seen = set()
        for case in CASES:
            for columns in COLUMNS + [WIDER] * (case is CASES[8]):
                l = rule.launch_of(size_of(case["new"], case["lengths"], case["heads"], case["kv_heads"], case["D"], case.get("pad", 0), case["page"], columns,
                                           codes=codes))
                seen.add((case["D"], case["page"] % 16 == 0, l["wavefronts"], l["sets"]))
        assert seen == {(D, whole, w, s) for D in (64, 128) for whole in (True, False) for w, s in ((0, 1), (0, 2), (4, 1))}, (codes, seen)


def test_halves_ascend(rule):
    """Over all fp16 numbers: the order of their values, both zeros alike, infinities outermost; and back."""
    h = np.arange(65536, dtype=np.uint16)
    value = h.view(np.float16)
    number = np.isfinite(value) | np.isinf(value)
    up = np.array([rule.up(int(x)) for x in h])
    order = np.argsort(value[number].astype(np.float64), kind="stable")
    v, u = value[number].astype(np.float64)[order], up[number][order]
    assert ((np.diff(v) > 0) == (np.diff(u) > 0)).all() and ((np.diff(v) == 0) == (np.diff(u) == 0)).all()
    back = np.array([rule.back(int(x)) for x in up], np.uint32).astype(np.uint16).view(np.float16)
    assert (back[number] == value[number]).all()
    least = min(rule.up(int(x)) for x in h[np.isfinite(value)])
    assert least == 0x400 and rule.up(0xfc00) == 0x3ff


def test_tiles_hold_every_token_once(rule):
    tokens = [rule.token(tile, lane, e) for tile in range(3) for lane in range(64) for e in range(64)]
    assert sorted(tokens) == list(range(3 * 4096))
    assert [rule.tiles(v) for v in (1, 4096, 4097, 1 << 21)] == [1, 1, 2, 512]
    for beams, vocab in ((1, 1), (5, 200), (8, 151936), (64, 1 << 21)):
        n, room = rule.fit(16 << 20, beams, vocab), 136 * beams * rule.tiles(vocab)
        assert n * room <= 16 << 20 < (n + 1) * room and n >= 1


def test_sets_of_a_pair_are_eight_blocks_apart(rule):
    out = (ctypes.c_uint * 2)()
    for sets in (1, 2, 3, 7, 16):
        for pairs in (1, 2, 7, 8, 9, 15, 16, 40, 61):
            where = {}
            for i in range(sets * pairs):
                rule.apart(i, sets, pairs, out)
                where[out[0], out[1]] = i
            assert sorted(where) == [(s, p) for s in range(sets) for p in range(pairs)]
            for p in range(pairs):
                step = 8 if p < pairs // 8 * 8 else pairs % 8
                assert [where[s, p] - where[0, p] for s in range(sets)] == [s * step for s in range(sets)]


def test_rounds_fit_the_launch(rule):
    """A share by rounds of blocks never makes more items than the launch has blocks, and with one round or two where it says so."""
    rng = random.Random(9)
    better = 0
    for _ in range(4000):
        n, resident, kv = rng.choice([1, 2, 7, 32, 64]), rng.choice([1, 2]), rng.choice([1, 2, 3, 5, 8, 12])
        sets = [rng.choice([0, 1, 2, 4, rng.randint(1, 30)]) for _ in range(n)]
        tiles = [rng.choice([1, rng.randint(1, 40), rng.randint(1, 600), rng.randint(1, 30000)]) for _ in range(n)]
        target = rng.choice([resident * 256 // kv, rng.randint(1, 300)])
        least, blocks = rng.choice([1, 16]), target + sum(sets) + rng.choice([0, 0, 50])
        out = (ctypes.c_int * 4)()
        off = rng.choice([1.0, 1.0 + 2.0 ** -22, 1.0 - 2.0 ** -22])
        rule.rounds(n, (ctypes.c_int * n)(*sets), (ctypes.c_int * n)(*tiles), target, resident, least, blocks, ctypes.c_float(off), out)
        assert 1 <= out[2] and out[3] <= blocks and out[3] >= sum(sets), (sets, tiles, target, resident, list(out))
        better += out[2] != out[0]
    assert better > 1000
