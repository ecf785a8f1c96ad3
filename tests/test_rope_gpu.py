"""mi_rope against the formula in more than 64 bits.

What an output may be off by: half a step of fp16 for its rounding (2^-11 of it, 2^-25 below the normal numbers), and (|x| + |y|) times
the error of cosine and sine: an angle's turns are off by three roundings of 2^-53 of their number, and 2^-26 when the rest is
rounded to fp32, 2 pi times that in the angle, 2^-22 for cosine and sine themselves (two units in their last place) and 2^-23 for two
roundings of the sum."""
import ctypes

import numpy as np
import pytest

from helpers import mil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def expect(x, heads, D, rot, inv_freq, position, axis, interleaved):
    """Rows [n, heads * D] -> (turned rows, tolerance)."""
    x = x.reshape(len(x), heads, D).astype(np.float64)
    out, tol = x.copy(), np.zeros_like(x)
    for i in range(rot // 2):
        angle = position[axis[i]].astype(np.longdouble) * np.longdouble(inv_freq[i])
        c, s = np.cos(angle).astype(np.float64)[:, None], np.sin(angle).astype(np.float64)[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        turns = np.abs(angle.astype(np.float64))[:, None] / (2 * np.pi)
        off = (np.abs(x[..., a]) + np.abs(x[..., b])) * (2 * np.pi * (3 * 2.0 ** -53 * turns + 2.0 ** -26) + 2.0 ** -22 + 2.0 ** -23)
        tol[..., a] = tol[..., b] = off
    tol[..., :rot] += 2.0 ** -11 * np.abs(out[..., :rot]) + 2.0 ** -25
    return out.reshape(len(x), -1), tol.reshape(len(x), -1)


def check(got, want, tol):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), [int(z[0]) for z in np.nonzero(bad)], got[bad][:4], want[bad][:4], tol[bad][:4])


def run(queue, n, heads, kv, D, rot, sections=None, interleaved=False, first=0, gap=0, shift=0, in_place=False, seed=0, theta=1e6):
    """Rows q | k | v side by side, `gap` more elements from row to row, `shift` elements into their allocation."""
    rng = np.random.default_rng(seed)
    ld = (heads + 2 * kv) * D + gap
    flat = rng.standard_normal(n * ld + shift).astype(np.float16)
    x = flat[shift:].reshape(n, ld)
    sections = sections or [rot // 2]
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    position = (first + rng.integers(0, 4096, (len(sections), n))).astype(np.int32)
    inv_freq = (theta ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32)
    held = [mil.Buffer.from_host(z) for z in (flat, inv_freq if rot else np.zeros(1, np.float32), position)]
    wide, narrow = heads * D, kv * D
    q = held[0].ptr + 2 * shift
    k = q + 2 * wide
    outs = [mil.Buffer.from_host(np.full(n * (w + 3) + 1, 0x1234, np.uint16)) for w in (wide, narrow)]
    to = dict(q_out=q, k_out=k, ld_q_out=ld, ld_k_out=ld) if in_place else \
        dict(q_out=outs[0].ptr + 2 * (gap % 2), k_out=outs[1], ld_q_out=wide + 3 * (gap > 0), ld_k_out=narrow + 3 * (gap > 0))
    call = mil.RopeCall(n, heads, kv, D, rot, held[1], held[2], q=q, k=k, ld_q=ld, ld_k=ld, axis=axis if len(sections) > 1 else None,
                        interleaved=interleaved, **to)
    assert mil.rope(queue, call)
    queue.finish()
    after = held[0].read(np.float16, flat.shape)
    if in_place:
        rows = after[shift:].reshape(n, ld)
        got_q, got_k = rows[:, :wide], rows[:, wide:wide + narrow]
        assert (rows[:, wide + narrow:].view(np.uint16) == x[:, wide + narrow:].view(np.uint16)).all() and \
            (after[:shift].view(np.uint16) == flat[:shift].view(np.uint16)).all()
    else:
        assert (after.view(np.uint16) == flat.view(np.uint16)).all()
        got = []
        for buf, w, s in ((outs[0], wide, gap % 2), (outs[1], narrow, 0)):
            all_of = buf.read(np.uint16, (n * (w + 3) + 1,))
            step = w + 3 * (gap > 0)
            used = np.zeros(len(all_of), bool)
            at = s + np.arange(n)[:, None] * step + np.arange(w)[None]
            used[at] = True
            assert (all_of[~used] == 0x1234).all(), "written beside the rows"
            got.append(all_of[at].view(np.float16))
        got_q, got_k = got
    for rows, lo, h in ((got_q, 0, heads), (got_k, wide, kv)):
        if h:
            check(rows, *expect(x[:, lo:lo + h * D], h, D, rot, inv_freq, position, axis, interleaved))


SHAPES = [(14, 2, 64, 64), (9, 3, 64, 32), (32, 8, 128, 128), (15, 5, 64, 64), (1, 0, 128, 64), (0, 7, 64, 64), (6, 2, 96, 96), (4, 1, 80, 48),
          (3, 2, 256, 256), (5, 1, 250, 36), (2, 1, 2, 2), (3, 1, 64, 0), (64, 8, 128, 128), (1, 1, 16, 16), (7, 1, 48, 16)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,D,rot", SHAPES)
def test_against_the_formula(queue, heads, kv, D, rot, interleaved, in_place):
    for n, gap, shift in ((1, 0, 0), (5, 0, 0), (67, 8, 8), (6, 1, 0), (5, 16, 3)):
        run(queue, n, heads, kv, D, rot, interleaved=interleaved, in_place=in_place, gap=gap, shift=shift, seed=n)


@pytest.mark.parametrize("sections", [[16, 24, 24], [32, 32], [1, 62, 1], [10, 20, 30, 4], [64, 0, 0, 0]])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(queue, sections, interleaved):
    run(queue, 300, 8, 2, 128, 128, sections=sections, interleaved=interleaved, seed=1)


@pytest.mark.parametrize("first", [0, 131072, 4000000, 2 ** 31 - 5000, -5000, -2 ** 31])
def test_far_positions(queue, first):
    run(queue, 40, 4, 2, 64, 64, first=first, seed=2)


def test_many_rows(queue):
    run(queue, 3001, 14, 2, 64, 64, seed=3)
    run(queue, 1030, 40, 8, 128, 128, sections=[16, 24, 24], seed=4, interleaved=True)


def test_turned_back(queue):
    """Negative positions turn back: each rounding on the way is half a step of at most |x| + |y|."""
    n, D, heads = 50, 64, 3
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, heads * D)).astype(np.float16)
    position = rng.integers(0, 100000, (1, n)).astype(np.int32)
    inv = (1e4 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    there, here = mil.Buffer.from_host(position), mil.Buffer.from_host(-position)
    freq, rows = mil.Buffer.from_host(inv), mil.Buffer.from_host(x)
    for p in (there, here):
        assert mil.rope(queue, mil.RopeCall(n, heads, 0, D, D, freq, p, q=rows, q_out=rows))
    queue.finish()
    size = np.abs(x.astype(np.float64)).reshape(n, heads, 2, D // 2).sum(2, keepdims=True).repeat(2, 2).reshape(n, -1)
    assert (np.abs(rows.read(np.float16, x.shape).astype(np.float64) - x) <= size * (3 * 2.0 ** -11 + 2.0 ** -18) + 2.0 ** -23).all()


def test_infinities_and_nans_go_by_the_formula(queue):
    x = np.ones((4, 64), np.float16)
    x[0, 3], x[1, 40], x[2, 5] = np.inf, np.nan, 65504
    inv = np.full(32, 0.7, np.float32)
    held = [mil.Buffer.from_host(z) for z in (x, inv, np.array([1, 1, 1, 0], np.int32))]
    assert mil.rope(queue, mil.RopeCall(4, 1, 0, 64, 64, held[1], held[2], q=held[0], q_out=held[0]))
    queue.finish()
    got = held[0].read(np.float16, x.shape).astype(np.float64)
    assert np.isinf(got[0, [3, 35]]).all() and np.isnan(got[1, [8, 40]]).all()
    assert np.isfinite(np.delete(got[0], [3, 35])).all() and np.isfinite(np.delete(got[1], [8, 40])).all() and (got[3] == 1).all()


def test_captured(queue):
    """A graph follows the positions in device memory, and gives the bits of the call."""
    n, rng = 33, np.random.default_rng(6)
    x = rng.standard_normal((n, 16 * 64)).astype(np.float16)
    held = [mil.Buffer.from_host(z) for z in (x, (1e4 ** (-np.arange(32) / 32)).astype(np.float32), np.zeros((1, n), np.int32))]
    outs = [mil.Buffer.from_host(np.zeros_like(x)) for _ in range(2)]
    calls = [mil.RopeCall(n, 16, 0, 64, 64, held[1], held[2], q=held[0], q_out=o) for o in outs]
    assert mil.lib().mi_graph_begin(queue.handle)
    assert mil.rope(queue, calls[0])
    graph = mil.lib().mi_graph_end(queue.handle)
    for turn in range(3):
        held[2].write(rng.integers(0, 10 ** 6, (1, n)).astype(np.int32))
        assert mil.lib().mi_graph_launch(graph, queue.handle) and mil.rope(queue, calls[1])
        queue.finish()
        got = [o.read(np.uint16, x.shape) for o in outs]
        assert (got[0] == got[1]).all() and got[0].any()
    mil.lib().mi_graph_destroy(graph)
