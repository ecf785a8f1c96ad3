"""Every kernel of mi_attention by itself (which one a call comes to is paged_plan.h's; test_paged_plan.py looks that these cases come
to the ones they are for), and what masked places hold under a window in the one for many rows."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache

pytestmark = pytest.mark.gpu
KINDS = [mil.KV_F16, mil.KV_INT8, mil.KV_Q4]
WIDE = 2 ** 20                                         # positions of a page table that takes chunks to the kernel for many rows

# (width, slices): the cache, positions of the page table.  Rows of padding make the batch one of many blocks: no slices.
MANY = {
    (64, 4): (dict(heads=8, kv_heads=4, D=64, lengths=[700, 90, 400], new=[150, 90, 1]), WIDE),
    (64, 1): (dict(heads=8, kv_heads=4, D=64, lengths=[700, 90, 400], new=[150, 90, 1], pad=2000), 0),
    (128, 2): (dict(heads=16, kv_heads=8, D=128, lengths=[500, 90, 400], new=[100, 90, 1]), WIDE),
    (128, 1): (dict(heads=16, kv_heads=8, D=128, lengths=[500, 90, 400], new=[100, 90, 1], pad=3200), 0),
}
FEW = {D: dict(heads=8, kv_heads=4, D=D, lengths=[700, 33, 400], new=[1, 9, 1]) for D in (64, 128)}
# Under a window: two sequences of which many rows share tiles; (slices, rows of padding, window, sinks)
UNDER_WINDOW = [(1, 3500, 16, 4), (1, 3500, 3, 0), (1, 3500, 64, 64), (1, 3500, 1, 1), (1, 3500, 100, 37), (4, 1450, 200, 5), (4, 1450, 200, 0),
                (4, 1450, 215, 130)]
WINDOW_CACHE = dict(heads=8, kv_heads=4, D=64, page=16, lengths=[500, 300], new=[250, 200])


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


@pytest.mark.parametrize("page", [16, 100, 48, 5])     # (one after the other in one process: each has an LDS limit to be raised)
@pytest.mark.parametrize("D,slices", sorted(MANY))
@pytest.mark.parametrize("kind", KINDS)
def test_many_rows(monkeypatch, queue, kind, D, slices, page):
    case, columns = MANY[D, slices]
    monkeypatch.setattr(Cache, "columns", columns)
    c = Cache(kind, page=page, seed=61, **case).upload()
    c.check(c.attend(queue))


@pytest.mark.parametrize("page", [16, 100])
@pytest.mark.parametrize("D", sorted(FEW))
@pytest.mark.parametrize("kind", KINDS)
def test_few_rows(queue, kind, D, page):
    c = Cache(kind, page=page, seed=62, **FEW[D]).upload()
    c.check(c.attend(queue))


@pytest.mark.parametrize("slices,pad,window,sinks", UNDER_WINDOW)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", KINDS)
def test_what_a_window_leaves_behind_does_not_matter(queue, kind, bad, slices, pad, window, sinks):
    """Infinities and NaN among the values: at the causal edge and behind the window (key/value heads 0 and 1), right behind the sinks (2),
    and in a sink, where there is one (3: every row sees it).  Rows that see none are as ever, the others have it."""
    c = Cache(kind, seed=63, pad=pad, **WINDOW_CACHE)
    places = {0: [494], 1: [255, 490], 2: [sinks], 3: [0]}
    for head, at in places.items():
        c.v[0][at, head, 9] = bad
    c.k[0][260, 0, 5] = np.nan                              # and a key
    places[0] = [494, 260]
    c.fill()
    got = c.upload().attend(queue, window=window, sinks=sinks)
    want, tol = c.expect(window, sinks)
    p = np.arange(250, 500)
    for head, at in places.items():
        sees = np.zeros((250, len(at)), bool)
        for i, j in enumerate(at):
            sees[:, i] = (j <= p) & ((j > p - window) | (j < sinks))
        clean, own = ~sees.any(1), slice(2 * head, 2 * head + 2)
        off = np.abs(got[:250, own].astype(np.float64) - want[:250, own]) <= tol[:250, own]
        assert off[clean].all(), (head, np.nonzero(~off & clean[:, None, None])[0][:5])
        seen = sees[:, [j != 260 for j in at]].any(1)
        assert not np.isfinite(got[:250, own, 9][seen]).any()
        if head == 0:
            assert np.isnan(got[:250, own][sees[:, 1]]).all()
        assert head == 3 or clean.sum() >= 15, "the test has to have rows to look at"
    rest = slice(250, 450)
    assert (np.abs(got[rest].astype(np.float64) - want[rest]) <= tol[rest]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 70])
def test_small_weights_count(queue, kind, n):
    """9000 positions at 2^-22 of the greatest weight, 0.2 % of its sum, with values a hundred times as large: a sixth of the output,
    many times what it may be off by."""
    c = Cache(kind, 14, 2, 64, 32, [9000], [n], seed=64)
    c.qkv[:, :14 * 64] = 1.0                                # q k: scores 15.2 and 0
    c.k[0][:] = 0
    c.k[0][17] = 1.9
    c.v[0][:] = np.abs(c.v[0]) * 100
    c.v[0][17] = 1.0
    c.fill()
    got = c.upload().attend(queue)
    c.check(got)
    want, tol = c.expect()
    assert (want - 1.0 > 10 * tol).mean() > 0.99 and (tol > 0).all()


@pytest.mark.parametrize("form", ["few", "many"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", [mil.KV_INT8, mil.KV_Q4])
def test_scales_at_multiples_of_8_bytes(monkeypatch, queue, kind, D, form):
    case, columns = (FEW[D], 0) if form == "few" else MANY[D, 4 if D == 64 else 2]
    monkeypatch.setattr(Cache, "columns", columns)
    c = Cache(kind, page=16, seed=65, **case).upload()
    held = []
    for name in "kv":
        scales = c.scale[name].reshape(-1)
        held.append(mil.Buffer.from_host(np.concatenate([np.full(4, 0x7e00, np.uint16), scales])))
        assert held[-1].ptr % 16 == 0
    c.cache = mil.KVCache(kind, c.n_pages, 16, c.kv, D, c.dev["k"], c.dev["v"], *(b.ptr + 8 for b in held))
    c.check(c.attend(queue))
    at = c.dev_qkv.ptr + 2 * c.heads * D
    assert mil.kv_write(queue, c.cache, c.batch, at, at + 2 * c.kv * D, c.ld, c.ld)
    queue.finish()
    for name, b in zip("kv", held):
        assert np.array_equal(b.read(np.uint16, (4 + c.scale[name].size,))[4:], c.scale[name].reshape(-1))
