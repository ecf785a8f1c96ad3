"""mi_attention against a plain evaluation in 64 bits of the values that the cache holds, with tolerances that count the
roundings (paged_lib.Cache.expect).  Everything that no row may see is NaN in these caches."""
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


STEPS = [
    dict(heads=14, kv_heads=2, D=64, page=16, lengths=[24], new=[1]),
    dict(heads=9, kv_heads=3, D=64, page=64, lengths=[1, 2, 31, 32, 33, 63, 64, 65, 500, 0], new=[1] * 9 + [0], pad=2),
    dict(heads=8, kv_heads=8, D=128, page=1, lengths=[130, 17], new=[1, 1]),
    dict(heads=32, kv_heads=8, D=128, page=48, lengths=[700, 47, 48, 49], new=[1, 1, 1, 1]),
    dict(heads=15, kv_heads=5, D=64, page=100, lengths=[1500, 99, 101], new=[1, 1, 1], gap=3),
    dict(heads=40, kv_heads=1, D=128, page=32, lengths=[260], new=[1]),
    dict(heads=16, kv_heads=8, D=64, page=8, lengths=list(range(1, 140, 2)), new=[1] * 70),
    dict(heads=4, kv_heads=1, D=64, page=2048, lengths=[5000], new=[1], spare=0),
]
CHUNKS = [
    dict(heads=14, kv_heads=2, D=64, page=16, lengths=[300], new=[300]),
    dict(heads=9, kv_heads=3, D=64, page=48, lengths=[257, 130], new=[129, 130]),
    dict(heads=8, kv_heads=2, D=128, page=64, lengths=[200, 1], new=[77, 1], pad=7),
    dict(heads=12, kv_heads=12, D=64, page=100, lengths=[333], new=[65]),
    dict(heads=8, kv_heads=1, D=128, page=5, lengths=[90, 40], new=[33, 40]),
    dict(heads=32, kv_heads=8, D=128, page=16, lengths=[600, 0, 900, 30, 64], new=[1, 0, 70, 30, 1], pad=19, gap=1),
    dict(heads=15, kv_heads=5, D=64, page=32, lengths=[1100], new=[2]),
]


@pytest.mark.parametrize("case", STEPS + CHUNKS)
@pytest.mark.parametrize("kind", KINDS)
def test_against_64_bits(queue, kind, case):
    c = Cache(kind, seed=1, **case).upload()
    c.check(c.attend(queue))
    c.check(c.attend(queue, ld_out=c.heads * c.D + 5), what="rows apart")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 37), (64, 64), (250, 1), (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("case", [STEPS[1], STEPS[4], CHUNKS[0], CHUNKS[2], CHUNKS[5]])
@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_Q4])
def test_windows(queue, kind, case, window, sinks):
    c = Cache(kind, seed=2, **case).upload()
    c.check(c.attend(queue, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("kind", KINDS)
def test_scales(queue, kind):
    for scale in (1.0, 2.0 ** -10, 3.7, 1e-30):
        c = Cache(kind, 14, 2, 64, 16, [200, 90], [60, 1], seed=4).upload()
        c.check(c.attend(queue, scale=scale), scale=scale, what=scale)


@pytest.mark.parametrize("form", [dict(lengths=[150, 64], new=[150, 20]), dict(lengths=[700], new=[1])])
@pytest.mark.parametrize("kind", KINDS)
def test_what_a_masked_position_holds_does_not_matter(queue, kind, form):
    """NaN and infinities in a chunk's later rows, which earlier rows of the same tile must not take up, and in
    positions behind the window."""
    c = Cache(kind, 14, 2, 64, 16, seed=7, **form)
    m, n = c.lengths[0], c.new[0]
    for name, bad in ((c.k, np.nan), (c.v, np.inf), (c.v, np.nan)):
        name[0][m - 5, :, 11] = bad
    c.fill()
    c.upload()
    got = c.attend(queue)
    # the rows that do not see it: as ever.  (Not bit for bit what they are without it: a row that shares a tile with such a place may
    # be summed in another order; the tolerance holds for any.)
    unseen = np.r_[0:max(n - 5, 0), n:sum(c.new)]
    c.check(got, rows=unseen)
    assert np.isnan(got[n - 1]).any()
    # with a window of 3 the last two rows do not see the position any more
    got = c.attend(queue, window=3)
    c.check(got, window=3, rows=np.r_[0:max(n - 5, 0), max(n - 2, 0):n])
    if n > 2:
        assert np.isnan(got[n - 3]).any() and np.isnan(got[n - 5]).any()


def test_infinite_values_that_are_seen(queue):
    c = Cache(mil.KV_F16, 14, 2, 64, 16, [40], [40], seed=7)
    c.v[0][20, 1, 3], c.v[0][25, 1, 3] = np.inf, -np.inf
    c.fill()
    got = c.upload().attend(queue)[:, 7:, 3]
    assert np.isfinite(got[:20]).all() and (got[20:25] == np.inf).all() and np.isnan(got[25:]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_are_not_in_the_pool(queue, kind):
    """Positions in such pages are not seen; a sequence that has nothing else gives zeros."""
    c = Cache(kind, 14, 2, 64, 16, [100, 40, 16], [1, 20, 1], seed=11)
    whole = c.table.copy()
    c.table[0, 2], c.table[2, 0] = c.n_pages, -3
    c.upload()
    got = c.attend(queue)
    assert (got[21].view(np.uint16) == 0).all()
    other = Cache(kind, 14, 2, 64, 16, [84, 40, 16], [1, 20, 1], seed=11)           # the same without positions 32 .. 47
    for x, y in ((other.k, c.k), (other.v, c.v)):
        x[0], x[1] = np.delete(y[0], range(32, 48), 0), y[1]
    other.qkv[:] = c.qkv
    want, tol = other.expect()
    assert (np.abs(got[:21].astype(np.float64) - want[:21]) <= tol[:21]).all()
    assert (whole[0, :7] >= 0).all()


def test_rows_before_the_first_position(queue):
    """More rows than positions: the rows before position 0 see nothing."""
    c = Cache(mil.KV_F16, 14, 2, 64, 16, [40], [40], seed=12).upload()
    c.dev_len.write(np.array([25], np.int32))
    got = c.attend(queue)
    assert (got[:15].view(np.uint16) == 0).all() and np.isfinite(got).all() and (got[15] != 0).any()


def test_the_same_bits_again(queue):
    c = Cache(mil.KV_INT8, 14, 2, 64, 16, [3000, 700, 90, 1], [1, 1, 1, 1], seed=13).upload()
    first = c.attend(queue)
    for _ in range(5):
        assert np.array_equal(c.attend(queue).view(np.uint16), first.view(np.uint16))


def test_streams_without_a_workspace_and_the_null_stream(queue):
    c = Cache(mil.KV_F16, 14, 2, 64, 16, [3000, 5], [1, 1], seed=14).upload()
    c.check(c.attend(mil.Queue(default=True)), what="null stream")
    import ctypes
    hip = ctypes.CDLL("libamdhip64.so")
    handle = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0

    class Foreign(mil.Queue):
        def __init__(self, h):
            self.handle = h

        def __del__(self):
            pass

    c.check(c.attend(Foreign(handle.value)), what="a stream from elsewhere")
    assert hip.hipStreamDestroy(handle) == 0


def test_two_streams_at_once(queue):
    other = mil.Queue()
    a = Cache(mil.KV_F16, 14, 2, 64, 16, [4000, 800], [1, 1], seed=15).upload()
    b = Cache(mil.KV_INT8, 14, 2, 64, 16, [2000, 3000], [1, 1], seed=16).upload()
    outs = [mil.Buffer(c.rows * c.heads * c.D * 2) for c in (a, b)]
    calls = [mil.AttentionCall(c.cache, c.batch, c.heads, c.dev_qkv, o, ld_q=c.ld) for c, o in zip((a, b), outs)]
    for _ in range(20):
        assert mil.attention(queue, calls[0]) and mil.attention(other, calls[1])
    queue.finish(), other.finish()
    for c, o in zip((a, b), outs):
        c.check(o.read(np.float16, (c.rows, c.heads, c.D)))


@pytest.mark.parametrize("kind", KINDS)
def test_steps_of_a_recorded_graph(queue, kind):
    """Write and attention recorded once and replayed for 40 tokens of three sequences: the lengths on the device say
    where each token goes and what it sees."""
    c = Cache(kind, 14, 2, 64, 16, [70, 100, 41], [1, 1, 1], seed=17)
    first = [30, 60, 1]
    c.upload()
    fresh = Cache(kind, 14, 2, 64, 16, [70, 100, 41], [1, 1, 1], seed=17)
    for n in "kv":                                              # what is to come is not there yet
        for b, f in enumerate(first):
            p = np.arange(f, c.lengths[b])
            fresh.pool[n][fresh.table[b][p // 16], :, p % 16] = 0x7e
        c.dev[n].write(fresh.pool[n])
    width, at = c.heads * c.D, c.dev_qkv.ptr + 2 * c.heads * c.D
    out = mil.Buffer(3 * width * 2)
    call = mil.AttentionCall(c.cache, c.batch, c.heads, c.dev_qkv, out, ld_q=c.ld)

    def step():
        assert mil.kv_write(queue, c.cache, c.batch, at, at + 2 * c.kv * c.D, c.ld, c.ld)
        assert mil.attention(queue, call)

    rng, graph = np.random.default_rng(1), None
    for t in range(40):
        now = [f + t for f in first]
        rows = np.full((3, c.ld), np.nan, np.float16)
        rows[:, :width] = rng.standard_normal((3, width)).astype(np.float16)
        for b, p in enumerate(now):
            rows[b, width:width + 128], rows[b, width + 128:width + 256] = c.k[b][p].reshape(-1), c.v[b][p].reshape(-1)
        c.dev_qkv.write(rows)
        c.dev_len.write(np.array([p + 1 for p in now], np.int32))
        if t == 0:
            step()
        else:
            if graph is None:
                with mil.Graph(queue) as graph:
                    step()
            graph.launch()
        queue.finish()
        if t % 13 == 0 or t == 39:
            part = Cache(kind, 14, 2, 64, 16, [p + 1 for p in now], [1, 1, 1])
            part.k, part.v = [k[:p + 1] for k, p in zip(c.k, now)], [v[:p + 1] for v, p in zip(c.v, now)]
            part.qkv[:] = rows
            part.check(out.read(np.float16, (3, c.heads, c.D)), what=t)
