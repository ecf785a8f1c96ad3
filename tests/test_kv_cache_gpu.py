"""mi_kv_write and mi_kv_read: codes, scales and values bit for bit as the definition in 64 bits gives them, and nothing else
touched."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache, quantise, values

pytestmark = pytest.mark.gpu
KINDS = [mil.KV_F16, mil.KV_INT8, mil.KV_Q4]


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def _write(c, queue):
    at = c.dev_qkv.ptr + 2 * c.heads * c.D
    assert mil.kv_write(queue, c.cache, c.batch, at, at + 2 * c.kv * c.D, c.ld, c.ld)
    queue.finish()


def _read(c, queue, ld=0, before=0x1234, batch=None, rows=None):
    width, rows = c.kv * c.D, rows or c.rows
    outs = [mil.Buffer.from_host(np.full((rows, ld or width), before, np.uint16)) for _ in "kv"]
    assert mil.kv_read(queue, c.cache, batch or c.batch, *outs, ld, ld)
    queue.finish()
    return [o.read(np.uint16, (rows, ld or width)) for o in outs]


def _blank(c):
    """The pools without the batch's rows."""
    keep = [(k.copy(), v.copy()) for k, v in zip(c.k, c.v)]
    lengths = c.lengths
    c.lengths = [m - n for m, n in zip(c.lengths, c.new)]
    c.k, c.v = [k[:m] for (k, _), m in zip(keep, c.lengths)], [v[:m] for (_, v), m in zip(keep, c.lengths)]
    c.fill()
    before = c.pool, c.scale
    c.lengths, c.k, c.v = lengths, [k for k, _ in keep], [v for _, v in keep]
    c.fill()
    return before


CASES = [
    dict(heads=14, kv_heads=2, D=64, page=16, lengths=[24], new=[1]),
    dict(heads=9, kv_heads=3, D=64, page=48, lengths=[1, 49, 200, 0, 96], new=[1, 2, 200, 0, 48], pad=5),
    dict(heads=8, kv_heads=8, D=128, page=1, lengths=[7, 3], new=[7, 1]),
    dict(heads=8, kv_heads=1, D=128, page=100, lengths=[333], new=[333], pad=1),
    dict(heads=15, kv_heads=5, D=64, page=256, lengths=list(range(1, 90)), new=[1] * 89, gap=1),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("kind", KINDS)
def test_write_and_read(queue, kind, case):
    c = Cache(kind, seed=3, **case)
    want, want_scale = c.pool, c.scale
    c.pool, c.scale = _blank(c)
    c.upload()
    c.pool, c.scale = want, want_scale
    _write(c, queue)
    pool, scale = c.read_pools()
    for name in "kv":
        assert np.array_equal(pool[name], want[name])
        assert scale[name] is None or np.array_equal(scale[name], want_scale[name])
    width = c.kv * c.D
    for ld in (0, width + 3):
        for got, rows in zip(_read(c, queue, ld), (c.k, c.v)):
            n = sum(c.new)
            new = [values(kind, *quantise(kind, r[m - n_:])) for r, m, n_ in zip(rows, c.lengths, c.new)]
            assert np.array_equal(got[:n, :width], np.concatenate(new).reshape(n, width).view(np.uint16))
            assert (got[n:] == 0x1234).all() and (got[:, width:] == 0x1234).all()


@pytest.mark.parametrize("kind", KINDS)
def test_every_position_reads_back(queue, kind):
    c = Cache(kind, 4, 2, 64, 32, [70, 0, 33, 128], [1, 0, 1, 1], seed=5).upload()
    start = np.concatenate([[0], np.cumsum(c.lengths)]).astype(np.int32)
    rows, dev = int(start[-1]), mil.Buffer.from_host(start)
    batch = mil.KVBatch(4, rows, 128, c.max_pages, dev, c.dev_len, c.dev_table)
    for got, each in zip(_read(c, queue, batch=batch, rows=rows), (c.k, c.v)):
        want = np.concatenate([values(kind, *quantise(kind, r)) for r in each]).reshape(rows, -1)
        assert np.array_equal(got, want.view(np.uint16))


@pytest.mark.parametrize("kind", [mil.KV_INT8, mil.KV_Q4])
def test_what_a_scale_can_be(queue, kind):
    """Every finite fp16 number as a row's greatest, the others at every fraction of it; zeros, the smallest and greatest
    numbers, infinities and NaN (which stay in their row or 32 elements)."""
    tops = np.arange(0x7c00, dtype=np.uint16).view(np.float16)
    n = len(tops)
    c = Cache(kind, 1, 1, 64, 512, [n], [n], seed=9, spare=0)      # (62 whole pages)
    rng = np.random.default_rng(2)
    rows = (rng.uniform(-1, 1, (n, 64)) * tops[:, None].astype(np.float64)).astype(np.float16)
    rows[:, 5], rows[:, 40] = tops, -tops
    half = tops.astype(np.float64)[:, None] / (127 if kind == mil.KV_INT8 else 7) * (np.arange(8)[None] + 0.5)
    rows[:, 8:16] = np.where(np.abs(half) <= np.abs(tops[:, None]), half, 0).astype(np.float16)      # ties
    for r, (at, x) in enumerate([(0, np.inf), (63, -np.inf), (31, np.nan), (32, np.nan)]):
        rows[1000 * r, at] = x
    c.k, c.v = [rows.reshape(n, 1, 64)], [rows[::-1].reshape(n, 1, 64).copy()]
    c.qkv[:, 64:128], c.qkv[:, 128:192] = rows, rows[::-1]
    c.fill()
    want, want_scale = c.pool, c.scale
    c.upload()
    _write(c, queue)
    pool, scale = c.read_pools()
    for name in "kv":
        finite = (want_scale[name] & 0x7fff) <= 0x7c00
        assert np.array_equal(pool[name], want[name])
        assert np.array_equal(scale[name][finite], want_scale[name][finite])
        assert ((scale[name][~finite] & 0x7fff) > 0x7c00).all() and 0 < (~finite).sum() <= 4
    for got, each in zip(_read(c, queue), (c.k, c.v)):
        back = values(kind, *quantise(kind, each[0])).reshape(n, 64)
        got = got.view(np.float16)
        assert np.array_equal(np.isnan(got), np.isnan(back)) and np.isfinite(got[~np.isnan(got)]).all()
        ok = ~np.isnan(back)
        assert np.array_equal(got[ok].view(np.uint16), back[ok].view(np.uint16))


@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_a_place(queue, kind):
    """Positions past the table or before 0, and pages that are not in the pool: skipped by the write, zeros for the read."""
    c = Cache(kind, 2, 2, 64, 16, [40, 30, 20, 5], [40, 3, 2, 5], seed=6)
    c.table[0, 1], c.table[1, 1], c.table[3, 0] = -7, c.n_pages, 2 ** 31 - 1
    places = c.table.copy()
    c.upload()
    c.dev_len.write(np.array([40, 30, c.max_pages * 16 + 1, 5], np.int32))
    at = c.dev_qkv.ptr + 2 * c.heads * c.D
    assert mil.kv_write(queue, c.cache, c.batch, at, at + 2 * c.kv * c.D, c.ld, c.ld)
    queue.finish()
    pool, _ = c.read_pools()
    # rows of sequences 0 (positions 16 .. 31), 1 (27 .. 29) and 3 have no page; sequence 2's are at 47 (no page: -1) and 48
    for name in "kv":
        assert np.array_equal(pool[name], c.pool[name])
    lost = np.zeros(c.rows, bool)
    lost[16:32] = lost[40:43] = lost[43:45] = lost[45:50] = True
    assert places[2, 2] == -1
    for got in _read(c, queue):
        assert (got[lost] == 0).all() and (got[~lost] != 0).any(axis=1).all()


def test_in_a_recorded_graph(queue):
    """The lengths are read by the kernels: a recorded write and read follows them."""
    c = Cache(mil.KV_INT8, 2, 2, 64, 16, [64, 64], [1, 1], seed=8)
    want = {n: c.pool[n].copy() for n in "kv"}
    c.upload()
    for n in "kv":
        c.dev[n].write(np.full_like(c.pool[n], 3))
    outs = [mil.Buffer(c.rows * 2 * 64 * 2) for _ in "kv"]
    at = c.dev_qkv.ptr + 2 * c.heads * c.D

    def both():
        assert mil.kv_write(queue, c.cache, c.batch, at, at + 2 * c.kv * c.D, c.ld, c.ld)
        assert mil.kv_read(queue, c.cache, c.batch, *outs)

    both()
    queue.finish()
    with mil.Graph(queue) as graph:
        both()
    for p in (0, 15, 16, 63):
        c.dev_len.write(np.array([p + 1, 64 - p], np.int32))
        rows = c.qkv.copy()
        w = c.heads * c.D
        for b, pos in enumerate((p, 63 - p)):
            rows[b, w:w + 128], rows[b, w + 128:w + 256] = c.k[b][pos].reshape(-1), c.v[b][pos].reshape(-1)
        c.dev_qkv.write(rows)
        graph.launch()
        queue.finish()
        for out, each in zip(outs, (c.k, c.v)):
            got = out.read(np.uint16, (2, 128))
            new = np.stack([each[0][p].reshape(-1), each[1][63 - p].reshape(-1)]).reshape(2, 2, 64)
            assert np.array_equal(got, values(c.kind, *quantise(c.kind, new)).view(np.uint16).reshape(2, 128))
    pool, _ = c.read_pools()
    for b, pos in ((0, 15), (1, 0)):
        page, slot = c.table[b][pos // 16], pos % 16
        assert np.array_equal(pool["k"][page, :, slot], want["k"][page, :, slot])
