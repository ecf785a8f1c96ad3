"""mi_attention at the last positions that an int counts, 2^31 - 2 and before: offsets within tiles must not pass them."""
import numpy as np
import pytest

from helpers import mil

pytestmark = pytest.mark.gpu
LAST = 2 ** 31 - 1                                     # positions


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


@pytest.mark.parametrize("page", [2 ** 16, 100003])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (300, 3), (64, 0), (1, 1)])
@pytest.mark.parametrize("n,rows", [(1, 1), (90, 90), (90, 2 ** 16)])
def test_a_window_at_the_end(queue, n, rows, window, sinks, page):
    """A sequence of 2^31 - 1 positions of which all but the last page (and the first, for sinks) are nowhere.  (Many rows of padding
    take it to the kernel for many rows.)"""
    D, heads, rng = 64, 2, np.random.default_rng(41)
    max_pages = -(-LAST // page)
    table = np.full(max_pages, -1, np.int32)
    pages = sorted({0, (LAST - 700) // page, (LAST - 1) // page})
    table[pages] = np.arange(len(pages))
    near = np.arange(LAST - 700, LAST)
    pos = np.concatenate([np.arange(sinks), near])
    k, v = (rng.standard_normal((len(pos), D)).astype(np.float16) for _ in "kv")
    pool = {x: np.full((len(pages), 1, page, D), np.nan, np.float16) for x in "kv"}
    for name, each in (("k", k), ("v", v)):
        pool[name][table[pos // page], 0, pos % page] = each
    q = np.full((rows, heads, D), np.nan, np.float16)
    q[:n] = rng.standard_normal((n, heads, D))
    bufs = {x: mil.Buffer.from_host(pool[x]) for x in "kv"}
    cache = mil.KVCache(mil.KV_F16, len(pages), page, 1, D, bufs["k"], bufs["v"])
    batch = mil.KVBatch(1, rows, n, max_pages, mil.Buffer.from_host(np.array([0, n], np.int32)),
                        mil.Buffer.from_host(np.array([LAST], np.int32)), mil.Buffer.from_host(table))
    out = mil.Buffer.from_host(np.full((rows, heads, D), 0x1234, np.uint16))
    call = mil.AttentionCall(cache, batch, heads, mil.Buffer.from_host(q), out, window=window, sinks=sinks)
    assert mil.attention(queue, call)
    queue.finish()
    got = out.read(np.uint16, (rows, heads, D))
    assert (got[n:] == 0x1234).all()
    got = got[:n].view(np.float16).astype(np.float64)
    p = np.arange(LAST - n, LAST)[:, None]
    seen = (pos[None] <= p) & ((pos[None] > p - window) | (pos[None] < sinks))
    assert seen.any(1).all()
    for h in range(heads):
        score = np.where(seen, q[:n, h].astype(np.float64) @ k.astype(np.float64).T / 8, -np.inf)
        w = np.exp(score - score.max(1, keepdims=True))
        total = w.sum(1, keepdims=True)
        want, mean = w @ v.astype(np.float64) / total, w @ np.abs(v.astype(np.float64)) / total
        # the output's rounding, the weights' over and under the line, and a score's fp32 sum of 64 products (below 2^6 in size)
        tol = 2.0 ** -11 * np.abs(want) + (2 * 2.0 ** -11 + 2 * 64 * 2.0 ** -18) * mean + 2.0 ** -25
        assert (np.abs(got[:, h] - want) <= tol).all(), (h, np.abs(got[:, h] - want).max())
