"""mi_attention_tree against a plain evaluation in 64 bits (tree_lib.TreeCache.expect).  Everything that no row may see is NaN in
these caches; a chain of drafts is what mi_attention makes of the same rows."""
import ctypes

import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache, quantise, values
from tree_lib import TreeCache, ancestors

pytestmark = pytest.mark.gpu
KINDS = [mil.KV_F16, mil.KV_INT8, mil.KV_Q4]


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


COLUMNS = [0, 2 ** 14, 2 ** 20]
WIDER = 2 ** 16


@pytest.fixture(autouse=True, params=COLUMNS, ids=["tight", "middle", "wide"])
def columns(request, monkeypatch):
    """Small batches run on the kernel for few rows, 16 to a wavefront; under a page table for so many positions 32 to a wavefront, and
    under one for a million on the kernel for many rows."""
    monkeypatch.setattr(Cache, "columns", request.param)
    return request.param


CASES = [
    dict(heads=14, kv_heads=2, D=64, page=16, lengths=[40], new=[16]),
    dict(heads=14, kv_heads=2, D=64, page=16, lengths=[16], new=[16]),                       # nothing but drafts
    dict(heads=9, kv_heads=3, D=64, page=64, lengths=[1, 5, 64, 65, 0, 300], new=[1, 4, 33, 31, 0, 32], pad=3),
    dict(heads=8, kv_heads=8, D=128, page=1, lengths=[130, 17], new=[40, 17]),
    dict(heads=32, kv_heads=8, D=128, page=48, lengths=[700, 97, 48, 49], new=[64, 37, 1, 24]),
    dict(heads=15, kv_heads=5, D=64, page=100, lengths=[1500, 199, 101], new=[100, 99, 3], gap=3),
    dict(heads=8, kv_heads=1, D=128, page=32, lengths=[460, 333], new=[130, 129]),
    dict(heads=4, kv_heads=1, D=64, page=2048, lengths=[5000], new=[65], spare=0),
    dict(heads=16, kv_heads=2, D=128, page=100, lengths=[300, 77], new=[30, 20]),
    dict(heads=14, kv_heads=2, D=64, page=36, lengths=[90, 20], new=[12, 20]),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("kind", KINDS)
def test_against_64_bits(queue, kind, case):
    c = TreeCache(kind, seed=1, **case).upload()
    c.check(c.attend(queue))
    c.check(c.attend(queue, ld_out=c.heads * c.D + 5), what="rows apart")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", [CASES[6], CASES[8]])
def test_wider_tables(queue, kind, case, monkeypatch):
    """Codes of width 128 come to 32 rows to a wavefront under tables for more positions than fp16."""
    monkeypatch.setattr(Cache, "columns", WIDER)
    c = TreeCache(kind, seed=6, **case).upload()
    c.check(c.attend(queue))
    c.check(c.attend(queue, window=50, sinks=2), 50, 2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 37), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("case", [CASES[0], CASES[2], CASES[4], CASES[5]])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_Q4])
def test_windows(queue, kind, case, window, sinks):
    c = TreeCache(kind, seed=2, **case).upload()
    c.check(c.attend(queue, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("case", [CASES[2], CASES[5], CASES[6]])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_INT8])
def test_any_bits(queue, kind, case):
    """Masks that are no trees: later rows, not the row's own, none at all (with nothing before: zeros)."""
    rng = np.random.default_rng(3)
    masks = [rng.random((n, n)) < 0.3 for n in case["new"]]
    for m in masks:
        m[::5] = False
    c = TreeCache(kind, seed=3, masks=masks, **case).upload()
    c.check(c.attend(queue))


def test_rows_that_see_nothing(queue):
    n = 40
    masks = [np.zeros((n, n), bool)]
    masks[0][3, 7] = True
    c = TreeCache(mil.KV_F16, 14, 2, 64, 16, [n], [n], masks=masks).upload()
    got = c.attend(queue)
    c.check(got)
    assert (got[[r for r in range(n) if r != 3]] == 0).all()


@pytest.mark.parametrize("words", [1, 2, 3, 7])
def test_words(queue, words):
    """Rows past the words are seen by none; words past the rows count for nothing."""
    c = TreeCache(mil.KV_F16, 14, 2, 64, 16, [300, 80], [70, 33], words=words, seed=4).upload()
    c.check(c.attend(queue))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", [CASES[0], CASES[4], CASES[6]])
def test_a_chain_is_a_text(queue, kind, case):
    """Bits of a lower triangle: what mi_attention has to give."""
    masks = [np.tril(np.ones((n, n), bool)) for n in case["new"]]
    c = TreeCache(kind, seed=5, masks=masks, **case).upload()
    plain = Cache.__new__(Cache)
    plain.__dict__ = c.__dict__
    plain.check(c.attend(queue))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_INT8])
def test_infinities_and_nans_of_drafts_that_are_not_seen(queue, kind, bad):
    """Every odd draft's keys and values are NaN or infinite; the even ones do not see them."""
    n, m = 48, 200
    masks = [np.tril(np.ones((n, n), bool))]
    masks[0][::2, 1::2] = False
    c = TreeCache(kind, 14, 2, 64, 16, [m], [n], masks=masks, seed=6)
    c.k[0][m - n + 1::2] = bad
    c.v[0][m - n + 1::2] = bad
    c.fill()
    got = c.upload().attend(queue)
    masks[0][1::2] = False                                # (the odd ones are not looked at)
    c.check(got, rows=slice(0, n, 2))


def test_repeated_and_captured(queue):
    """The same bits again, and from a graph that follows lengths and bits on the device."""
    c = TreeCache(mil.KV_INT8, 14, 2, 64, 64, [900, 3000, 64], [24, 17, 9], seed=7).upload()
    first = c.attend(queue)
    assert (c.attend(queue).view(np.uint16) == first.view(np.uint16)).all()
    width = c.heads * c.D
    out = mil.Buffer.from_host(np.zeros((c.rows, width), np.uint16))
    seen = mil.Buffer.from_host(np.ascontiguousarray(c.seen))
    call = mil.AttentionCall(c.cache, c.batch, c.heads, c.dev_qkv, out, ld_q=c.ld)
    mask = mil.TreeMask(seen, c.words)
    assert mil.lib().mi_graph_begin(queue.handle)
    assert mil.attention_tree(queue, call, mask)
    graph = mil.lib().mi_graph_end(queue.handle)
    assert graph
    for turn in range(3):
        assert mil.lib().mi_graph_launch(graph, queue.handle)
        queue.finish()
        got = out.read(np.float16, (c.rows, c.heads, c.D))
        c.check(got, what=turn)
        rng = np.random.default_rng(turn)
        c.masks = [ancestors([-1] + [int(rng.integers(0, i)) for i in range(1, n)]) for n in c.new]
        bits = np.zeros((c.rows, 32 * c.words), bool)
        for b, m in enumerate(c.masks):
            bits[c.start[b]:c.start[b] + len(m), :len(m)] = m
        c.seen = np.packbits(bits.reshape(c.rows, c.words, 32), axis=2, bitorder="little").view(np.uint32)[..., 0]
        seen.write(np.ascontiguousarray(c.seen))
        queue.finish()
    mil.lib().mi_graph_destroy(graph)


def test_long(queue):
    """Parts of a sequence that meet in the workspace, the drafts in the last of them."""
    c = TreeCache(mil.KV_F16, 14, 2, 64, 16, [9000, 70], [30, 1], seed=8).upload()
    c.check(c.attend(queue))


def test_a_stream_without_a_workspace(queue):
    hip = ctypes.CDLL("libamdhip64.so")
    foreign = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(foreign)) == 0
    c = TreeCache(mil.KV_Q4, 14, 2, 64, 16, [3000, 70], [30, 40], seed=9).upload()
    out = mil.Buffer.from_host(np.zeros((c.rows, c.heads * c.D), np.uint16))
    seen = mil.Buffer.from_host(np.ascontiguousarray(c.seen))
    call = mil.AttentionCall(c.cache, c.batch, c.heads, c.dev_qkv, out, ld_q=c.ld)
    assert mil.attention_tree(foreign, call, mil.TreeMask(seen, c.words))
    assert hip.hipStreamSynchronize(foreign) == 0
    c.check(out.read(np.float16, (c.rows, c.heads, c.D)))
    assert hip.hipStreamDestroy(foreign) == 0


class Odd(TreeCache):
    """Sequences whose lengths or pages on the device are not those that the cache was made with."""

    def bend(self, lengths=None, table=None):
        if lengths is not None:
            self.bent = list(lengths)
            self.dev_len.write(np.array(lengths, np.int32))
        if table is not None:
            self.bent_table = table
            self.dev_table.write(table)
        return self

    def visible(self, b, window, sinks):
        n, m = self.new[b], self.lengths[b]
        end, base = self.bent[b], self.bent[b] - n
        seen = np.zeros((n, m), bool)
        for p in range(min(m, max(end, 0))):
            page = self.bent_table[b, p // self.page]
            if not 0 <= page < self.n_pages:
                continue
            if p < base:
                place = np.clip(self.position[self.start[b]:self.start[b] + n], base, end - 1)
                seen[:, p] = (p > place - window) | (p < sinks) if window > 0 else True
            else:
                seen[:, p] = self.masks[b][:, p - base]
        return seen


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_Q4])
def test_lengths_and_pages_that_do_not_fit(queue, kind, window):
    """Fewer positions than drafts (the first ones have no place), none, less than none; pages that are not in the pool."""
    c = Odd(kind, 14, 2, 64, 16, [60, 40, 33, 50, 90], [16, 20, 20, 9, 30], seed=11).upload()
    table = c.table.copy()
    table[0, 1], table[4, 2], table[4, 5] = -1, c.n_pages, 2 ** 31 - 1
    c.bend([60, 13, 0, -5, 90], table)
    got = c.attend(queue, window=window, sinks=3)
    c.check(got, window, 3)
    assert (got[36:65] == 0).all()


def test_many_sequences_and_wrong_hints(queue):
    """More than the 64 that are planned at a time, of all sizes; max_tokens says how many there are at most, or does not."""
    rng = np.random.default_rng(12)
    new = [int(x) for x in rng.integers(0, 9, 150)]
    new[77] = 60
    c = TreeCache(mil.KV_F16, 9, 3, 64, 16, [n + int(rng.integers(0, 60)) for n in new], new, seed=12, pad=5).upload()
    want = c.expect()
    for hint in (60, 0, 1, 7, 5000):
        c.batch.max_tokens = hint
        got = c.attend(queue)[:sum(new)].astype(np.float64)
        assert (np.abs(got - want[0]) <= want[1]).all(), hint


def test_streams_at_once(queue):
    """Two streams, each with a workspace of its own, and parts that meet in it."""
    queues = [queue, mil.Queue()]
    caches = [TreeCache(mil.KV_F16, 14, 2, 64, 16, [3000 + 77 * i], [40], seed=13 + i).upload() for i in range(2)]
    calls = []
    for c in caches:
        out = mil.Buffer.from_host(np.zeros((c.rows, c.heads * c.D), np.uint16))
        mask = mil.TreeMask(mil.Buffer.from_host(np.ascontiguousarray(c.seen)), c.words)
        calls.append((mil.AttentionCall(c.cache, c.batch, c.heads, c.dev_qkv, out, ld_q=c.ld), mask, out))
    for _ in range(20):
        for q, (call, mask, _out) in zip(queues, calls):
            assert mil.attention_tree(q, call, mask)
    for q, c, (_call, _mask, out) in zip(queues, caches, calls):
        q.finish()
        c.check(out.read(np.float16, (c.rows, c.heads, c.D)))


@pytest.mark.parametrize("scale", [1e-30, 300.0, 65504.0])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_INT8])
def test_scales(queue, kind, scale):
    """Weights all alike, and scores of thousands and millions, whose products are rounded before the base is taken off."""
    c = TreeCache(kind, 14, 2, 64, 16, [200, 90], [40, 7], seed=14).upload()
    got = c.attend(queue, scale=scale)
    assert np.isfinite(got[:47]).all()
    if scale < 1:
        c.check(got, scale=scale)
    else:                                                 # the greatest score has (nearly) all the weight
        for b, (n, m) in enumerate(zip(c.new, c.lengths)):
            k, v = (values(kind, *quantise(kind, x[b])).astype(np.float64) for x in (c.k, c.v))
            seen = c.visible(b, 0, 0)
            for r in range(n):
                for h in range(c.heads):
                    s = k[:, h // 7] @ c.qkv[c.start[b] + r, h * 64:(h + 1) * 64].astype(np.float64) * scale
                    s[~seen[r]] = -np.inf
                    order = np.argsort(-s)
                    # a second score may take weight where it is within fp32's error of the sum (64 2^-24 of it) and 20 of the first
                    if s[order[0]] - s[order[1]] > 20 + 2.0 ** -17 * np.abs(s[order[0]]):
                        want = v[order[0], h // 7]
                        assert (np.abs(got[c.start[b] + r, h] - want) <= 2.0 ** -9 * np.abs(want) + 2.0 ** -16).all()


@pytest.mark.parametrize("heads,kv_heads", [(12, 6), (28, 7), (10, 5), (12, 12), (6, 3), (16, 8)])
@pytest.mark.parametrize("lengths,new", [([2100], [50]), ([900, 33, 0, 1500], [40, 33, 0, 17]), ([70] * 70, [12] * 70)])
def test_sets_of_rows_that_share_their_keys(queue, heads, kv_heads, lengths, new):
    """Several sets of rows in several parts for numbers of key/value heads that do not go into eight, and in a batch of one; twice, as
    the parts of a set meet in memory that the first call leaves ready for the next."""
    c = TreeCache(mil.KV_F16, heads, kv_heads, 64, 16, lengths, new, seed=12).upload()
    got = c.attend(queue)
    c.check(got)
    assert np.array_equal(got.view(np.uint16), c.attend(queue).view(np.uint16))
    c.check(c.attend(queue, window=600, sinks=3), 600, 3)


@pytest.mark.parametrize("heads,kv_heads,lengths,new", [
    (14, 2, [3000, 900, 2000], [30, 24, 9]), (32, 8, [2500] * 4, [32] * 4), (16, 4, [1700] * 5, [12] * 5), (8, 1, [4000, 1, 3900], [16, 1, 16]),
    (12, 12, [2200, 700], [40, 3]), (14, 2, [1500] * 66, [4] * 66),
])
def test_rounds_of_blocks(queue, heads, kv_heads, lengths, new):
    """Width 128, where blocks take a compute unit for themselves and shares of keys follow from the rounds that they make."""
    c = TreeCache(mil.KV_INT8, heads, kv_heads, 128, 64, lengths, new, seed=13).upload()
    got = c.attend(queue)
    c.check(got)
    assert np.array_equal(got.view(np.uint16), c.attend(queue).view(np.uint16))
