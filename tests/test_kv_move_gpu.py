"""mi_kv_keep and mi_kv_reorder against copies on the host, byte for byte, of every pool, scale and table whole."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache

pytestmark = pytest.mark.gpu
KINDS = [mil.KV_F16, mil.KV_INT8, mil.KV_Q4]


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def layers(kind, n, heads, D, page, lengths, new, seed, **more):
    """n caches with the same page table and other values."""
    made = [Cache(kind, heads, heads, D, page, lengths, new, seed=seed, **more)]
    for i in range(1, n):
        c = Cache(kind, heads, heads, D, page, lengths, new, seed=seed + i, **more)
        c.table = made[0].table
        c.fill()
        made.append(c)
    return [c.upload() for c in made]


def same(got, want):
    for g, w in zip(got, want):
        for name in "kv":
            assert (g[name] is None and w[name] is None) or (g[name] == w[name]).all()


KEEP = [
    dict(heads=2, D=64, page=16, lengths=[40, 17, 3, 90], new=[16, 16, 3, 70]),
    dict(heads=8, D=128, page=5, lengths=[64, 200], new=[64, 130]),
    dict(heads=5, D=64, page=48, lengths=[100, 0, 49], new=[10, 0, 49], pad=7),
    dict(heads=1, D=64, page=1, lengths=[33], new=[33]),
    dict(heads=20, D=128, page=100, lengths=[250, 101], new=[40, 2]),
]


@pytest.mark.parametrize("case", KEEP)
@pytest.mark.parametrize("kind", KINDS)
def test_keep(queue, kind, case):
    rng = np.random.default_rng(1)
    caches = layers(kind, 3, seed=1, **case)
    c = caches[0]
    for paths in ("some", "all", "none", "last", "close"):
        keep, kept = np.full(max(c.rows, 1), -77, np.int32), np.zeros(len(c.new), np.int32)
        for b, n in enumerate(c.new):
            path = {"some": np.sort(rng.choice(n, rng.integers(0, n + 1), replace=False)) if n else [], "all": np.arange(n), "none": [],
                    "last": np.arange(n)[-1:], "close": np.arange(1, n)}[paths]
            keep[c.start[b]:c.start[b] + len(path)], kept[b] = path, len(path)
        pools = [x.read_pools() for x in caches]
        for both in pools:
            for what in both:
                for name in "kv":
                    if what[name] is None:
                        continue
                    for b, n in enumerate(c.new):
                        at = np.arange(c.lengths[b] - n, c.lengths[b])
                        src = at[keep[c.start[b]:c.start[b] + kept[b]]]
                        dst = at[:kept[b]]
                        rows = what[name][c.table[b][src // c.page], :, src % c.page].copy()
                        what[name][c.table[b][dst // c.page], :, dst % c.page] = rows
        held = [mil.Buffer.from_host(x) for x in (keep, kept, np.zeros(len(kept), np.int32))]
        assert mil.kv_keep(queue, mil.KVCaches([x.cache for x in caches]), c.batch, *held)
        queue.finish()
        for x, want in zip(caches, pools):
            same(x.read_pools(), want)
        assert (held[2].read(np.int32, kept.shape) == np.array(c.lengths) - c.new + kept).all()


def test_keep_many_layers(queue):
    """More caches than a launch takes; lengths may be left alone."""
    caches = layers(mil.KV_INT8, 70, 2, 64, 16, [40], [20], seed=3)
    before = [x.read_pools() for x in caches]
    held = [mil.Buffer.from_host(np.array(x, np.int32)) for x in ([3, 5, 19] + [0] * 17, [3])]
    assert mil.kv_keep(queue, mil.KVCaches([x.cache for x in caches]), caches[0].batch, *held)
    queue.finish()
    c = caches[0]
    for x, both in zip(caches, before):
        for what in both:
            for name in "kv":
                for i, j in ((0, 3), (1, 5), (2, 19)):
                    what[name][c.table[0][(20 + i) // 16], :, (20 + i) % 16] = what[name][c.table[0][(20 + j) // 16], :, (20 + j) % 16]
        same(x.read_pools(), both)


def test_keep_numbers_out_of_range(queue):
    """Such numbers move nothing, and counts are taken as 0 to n."""
    c = Cache(mil.KV_F16, 2, 2, 64, 16, [40, 40, 40], [8, 8, 8], seed=4).upload()
    want = c.read_pools()
    keep = np.array([-1, 8, 2 ** 31 - 1, 5, 0, 0, 0, 0] + [3] * 8 + [-2 ** 31, 1, 2, 3, 4, 5, 6, 1000], np.int32)
    kept = np.array([4, -3, 1000], np.int32)
    for name in "kv":
        pool = want[0][name]
        pool[c.table[0][35 // 16], :, 35 % 16] = pool[c.table[0][37 // 16], :, 37 % 16]
    held = [mil.Buffer.from_host(x) for x in (keep, kept, np.zeros(3, np.int32))]
    assert mil.kv_keep(queue, mil.KVCaches([c.cache]), c.batch, *held)
    queue.finish()
    same(c.read_pools(), want)
    assert held[2].read(np.int32, (3,)).tolist() == [36, 32, 40]


def test_keep_places_outside_the_cache(queue):
    """Rows in pages that are not in the pool, past the table, or before position 0 move nowhere and nothing moves onto them."""
    c = Cache(mil.KV_INT8, 2, 2, 64, 16, [48, 32], [32, 32], seed=5).upload()
    table = c.table.copy()
    table[0, 2] = 1000
    c.dev_table.write(table)
    c.dev_len.write(np.array([48, 20], np.int32))          # the second has more rows than positions
    want = c.read_pools()
    keep = np.concatenate([np.arange(1, 33), np.arange(1, 33)]).astype(np.int32)
    for what in want:
        for name in "kv":
            pool = what[name]
            if pool is None:
                continue
            for i in range(15):                            # 16 + i <- 17 + i, below position 32
                pool[table[0, 1], :, i] = pool[table[0, 1], :, i + 1]
            for p in range(19):                            # the second begins at -12: positions 0 .. 18
                pool[table[1, p // 16], :, p % 16] = pool[table[1, (p + 1) // 16], :, (p + 1) % 16]
    held = [mil.Buffer.from_host(x) for x in (keep, np.array([31, 31], np.int32))]
    assert mil.kv_keep(queue, mil.KVCaches([c.cache]), c.batch, *held)
    queue.finish()
    same(c.read_pools(), want)


REORDER = [
    dict(heads=2, D=64, page=16, lengths=[40, 40, 40, 17, 17], new=[0] * 5),
    dict(heads=8, D=128, page=100, lengths=[250, 250, 250, 99, 100, 101], new=[0] * 6),
    dict(heads=5, D=64, page=1, lengths=[7, 0, 3], new=[0] * 3),
    dict(heads=3, D=128, page=48, lengths=[0, 48, 49, 47], new=[0] * 4),
    dict(heads=1, D=64, page=3000, lengths=[2999, 1], new=[0] * 2),
]


@pytest.mark.parametrize("case", REORDER)
@pytest.mark.parametrize("kind", KINDS)
def test_reorder(queue, kind, case):
    n = len(case["lengths"])
    caches = layers(kind, 3, seed=2, spare=n + 2, **case)
    c = caches[0]
    free = [p for p in range(c.n_pages) if p not in set(c.table.ravel().tolist())]
    for turn in range(3):
        rng = np.random.default_rng(turn)
        source = [np.arange(n), rng.integers(0, n, n), rng.integers(0, n, n)][turn]
        if turn == 2:
            source[0] = -1
            source[-1] = n
        fresh = np.array(free[:n], np.int32)
        lengths = np.array(c.lengths, np.int32)
        new_len, table = np.zeros(n, np.int32), np.full_like(c.table, -1)
        pools = [x.read_pools() for x in caches]
        for b, f in enumerate(source):
            if not 0 <= f < n:
                continue
            m = new_len[b] = lengths[f]
            used, full, tail = -(-m // c.page), m // c.page, m % c.page
            table[b, :used] = c.table[f, :used]
            if tail and f != b:
                table[b, full] = fresh[b]
                for both in pools:
                    for what in both:
                        for name in "kv":
                            if what[name] is not None:
                                what[name][fresh[b], :, :tail] = what[name][c.table[f, full], :, :tail]
        held = [mil.Buffer.from_host(np.ascontiguousarray(x, np.int32)) for x in
                (lengths, c.table, source, fresh, np.full(n, -9), np.full_like(c.table, -9))]
        assert mil.kv_reorder(queue, mil.KVCaches([x.cache for x in caches]), mil.ReorderCall(n, c.max_pages, *held))
        queue.finish()
        for x, want in zip(caches, pools):
            same(x.read_pools(), want)
        assert (held[4].read(np.int32, (n,)) == new_len).all() and (held[5].read(np.int32, table.shape) == table).all()


def test_reorder_many_layers_and_bad_pages(queue):
    """More caches than a launch takes; lengths past the table, below 0, and pages that are not there copy nothing."""
    caches = layers(mil.KV_Q4, 40, 2, 64, 16, [40, 40, 40, 40], [0] * 4, seed=6, spare=6)
    c = caches[0]
    free = [p for p in range(c.n_pages) if p not in set(c.table.ravel().tolist())]
    table = c.table.copy()
    table[2, 2] = c.n_pages
    lengths = np.array([40, 200, 40, -3], np.int32)
    source, fresh = np.array([1, 0, 3, 2], np.int32), np.array([free[0], c.n_pages + 3, free[2], free[3]], np.int32)
    held = [mil.Buffer.from_host(x) for x in (lengths, table, source, fresh, np.full(4, -9, np.int32), np.full_like(table, -9))]
    before = [x.read_pools() for x in caches]
    assert mil.kv_reorder(queue, mil.KVCaches([x.cache for x in caches]), mil.ReorderCall(4, c.max_pages, *held))
    queue.finish()
    for x, want in zip(caches, before):
        same(x.read_pools(), want)
    got = held[5].read(np.int32, table.shape)
    assert held[4].read(np.int32, (4,)).tolist() == [200, 40, -3, 40]
    assert got[0].tolist() == table[1].tolist() and got[1].tolist() == [*table[0][:2], fresh[1]] and (got[2] == -1).all()
    assert got[3].tolist() == [*table[2][:2], free[3]]
    table[0, 0] = table[0, 0]
    # and all of them where they are there
    source, lengths = np.array([0, 0, 0, 0], np.int32), np.array([40] * 4, np.int32)
    held = [mil.Buffer.from_host(np.array(x, np.int32)) for x in (lengths, c.table, source, free[:4], [-9] * 4, np.full_like(table, -9))]
    assert mil.kv_reorder(queue, mil.KVCaches([x.cache for x in caches]), mil.ReorderCall(4, c.max_pages, *held))
    queue.finish()
    for x, both in zip(caches, before):
        for what in both:
            for name in "kv":
                for b in (1, 2, 3):
                    what[name][free[b], :, :8] = what[name][c.table[0, 2], :, :8]
        same(x.read_pools(), both)


def test_pools_beyond_4_gib(queue):
    """Pages at offsets that 32 bits do not hold: drafts attended, kept, and their sequence copied, out there."""
    from tree_lib import TreeCache

    page, kv, D, n_pages = 64, 8, 128, 36000
    small = TreeCache(mil.KV_F16, 16, kv, D, page, [300, 70], [20, 30], seed=24)
    size = kv * page * D * 2
    assert n_pages * size > 2 ** 32
    far = np.full_like(small.table, -1)
    used = [(b, i) for b in range(2) for i in range(small.max_pages) if small.table[b, i] >= 0]
    places = [n_pages - 1, 16384, 16383, 1, 35001, 32769, 20000][:len(used)]
    pools = [mil.Buffer(n_pages * size) for _ in "kv"]
    for (b, i), to in zip(used, places):
        far[b, i] = to
        for pool, name in zip(pools, "kv"):
            host = np.ascontiguousarray(small.pool[name][small.table[b, i]])
            assert mil.lib().mi_memcpy_h2d(pool.ptr + to * size, host.ctypes.data, size, None)
    small.upload()
    small.dev_table.write(far)
    small.cache = mil.KVCache(mil.KV_F16, n_pages, page, kv, D, *pools)
    small.check(small.attend(queue))

    def rows(b, table, p):
        """Keys and values at position p."""
        got = []
        for pool in pools:
            host = np.empty((kv, page, D), np.uint16)
            assert mil.lib().mi_memcpy_d2h(host.ctypes.data, pool.ptr + int(table[b, p // page]) * size, size, None)
            got.append(host[:, p % page])
        return np.array(got)

    caches = mil.KVCaches([small.cache])
    keep = np.full(50, -1, np.int32)
    keep[:3], keep[20:22] = [1, 5, 19], [0, 29]
    held = [mil.Buffer.from_host(x) for x in (keep, np.array([3, 2], np.int32))]
    assert mil.kv_keep(queue, caches, small.batch, *held)
    queue.finish()
    for b, before, path in ((0, 280, [1, 5, 19]), (1, 40, [0, 29])):
        for i, j in enumerate(path):
            want = np.array([small.k[b][before + j], small.v[b][before + j]]).view(np.uint16)
            assert (rows(b, far, before + i) == want).all()
    lengths, source, fresh = np.array([283, 42], np.int32), np.array([1, 0], np.int32), np.array([35999 - 7, 33333], np.int32)
    held = [mil.Buffer.from_host(x) for x in (lengths, far, source, fresh, np.zeros(2, np.int32), np.zeros_like(far))]
    assert mil.kv_reorder(queue, caches, mil.ReorderCall(2, small.max_pages, *held))
    queue.finish()
    table = held[5].read(np.int32, far.shape)
    assert table[0, 0] == fresh[0] and table[1].tolist() == [*far[0, :4], fresh[1]]
    for b, f, p in ((0, 1, 0), (0, 1, 41), (1, 0, 256), (1, 0, 282)):
        assert (rows(b, table, p) == rows(f, far, p)).all()


def test_captured(queue):
    """Graphs that follow paths, lengths and sources in device memory."""
    c = Cache(mil.KV_INT8, 4, 4, 64, 16, [40, 33, 50], [20, 9, 30], seed=7, spare=6).upload()
    free = [p for p in range(c.n_pages) if p not in set(c.table.ravel().tolist())][:3]
    n = len(c.lengths)
    buf = lambda x: mil.Buffer.from_host(np.array(x, np.int32))  # noqa: E731
    keep, kept, new_len = buf([0] * c.rows), buf([0] * n), buf([0] * n)
    source, fresh, after, table = buf(list(range(n))), buf(free), buf([0] * n), buf(c.table)
    caches = mil.KVCaches([c.cache])
    call = mil.ReorderCall(n, c.max_pages, new_len, c.dev_table, source, fresh, after, table)
    assert mil.lib().mi_graph_begin(queue.handle)
    assert mil.kv_keep(queue, caches, c.batch, keep, kept, new_len) and mil.kv_reorder(queue, caches, call)
    graph = mil.lib().mi_graph_end(queue.handle)
    assert graph
    for turn in range(3):
        rng = np.random.default_rng(turn)
        paths = [np.sort(rng.choice(m, rng.integers(1, m), replace=False)) for m in c.new]
        flat = np.full(c.rows, -1, np.int32)
        for s, p in zip(c.start, paths):
            flat[s:s + len(p)] = p
        frm = rng.integers(0, n, n)
        keep.write(flat)
        kept.write(np.array([len(p) for p in paths], np.int32))
        source.write(frm.astype(np.int32))
        pools = c.read_pools()
        lengths = [m - k + len(p) for m, k, p in zip(c.lengths, c.new, paths)]
        for what in pools:
            for name in "kv":
                pool = what[name]
                for b, p in enumerate(paths):
                    at = c.lengths[b] - c.new[b]
                    moved = pool[c.table[b][(at + p) // 16], :, (at + p) % 16].copy()
                    to = at + np.arange(len(p))
                    pool[c.table[b][to // 16], :, to % 16] = moved
                for b, f in enumerate(frm):
                    if f != b and lengths[f] % 16:
                        pool[free[b], :, :lengths[f] % 16] = pool[c.table[f][lengths[f] // 16], :, :lengths[f] % 16]
        assert mil.lib().mi_graph_launch(graph, queue.handle)
        queue.finish()
        same(c.read_pools(), pools)
        assert after.read(np.int32, (n,)).tolist() == [lengths[f] for f in frm]
    mil.lib().mi_graph_destroy(graph)
