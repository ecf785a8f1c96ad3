"""mi_rope at angles of billions of turns, seen through outputs that are small: where cos a and sin a are nearly alike, 1 cos a - 1 sin a is
below fp16's normal numbers, whose steps of 2^-24 leave nothing of the angle's error out.

What such an output (x = y = 1, |cos a - sin a| < 2^-14) may be off by: the angle's error times |sin a + cos a| = sqrt 2, the angle being off by
2 pi 2^-26 from its rounding to fp32, in turns below a half (the 64-bit part before it: 2^-53 of a turn); two units in the last place, 2^-23,
for cosine and for sine, both below 1; and half a step, 2^-25, for the output.  (1 s is s, and c - s of two numbers so near to each other is exact.)"""
import numpy as np
import pytest

from helpers import mil

pytestmark = pytest.mark.gpu
TOLERANCE = np.sqrt(2) * 2 * np.pi * 2.0 ** -26 + 2 * 2.0 ** -23 + 2.0 ** -25


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def small_ones(inv_freq, sign):
    """Positions near 2^31 whose angles leave cos a - sin a small, and those differences (80-bit numbers hold the angle as it is)."""
    position = sign * (2 ** 31 - 1 - np.arange(2 ** 21, dtype=np.int64))
    angle = position.astype(np.longdouble) * np.longdouble(np.float32(inv_freq))
    left = np.cos(angle) - np.sin(angle)
    some = np.abs(left) < 2.0 ** -14
    return position[some].astype(np.int32), left[some].astype(np.float64)


@pytest.mark.skipif(np.finfo(np.longdouble).nmant < 63, reason="needs 64 bits of an angle")
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("inv_freq", [1.0, 0.7, 65.0, 1e4])
@pytest.mark.parametrize("D", [16, 18])
def test_far_angles(queue, inv_freq, sign, D):
    position, want = small_ones(inv_freq, sign)
    n, pairs = len(position), D // 2
    assert n >= 20
    held = [mil.Buffer.from_host(x) for x in (np.ones((n, D), np.float16), np.full(pairs, inv_freq, np.float32), position)]
    out = mil.Buffer.from_host(np.zeros((n, D), np.float16))
    assert mil.rope(queue, mil.RopeCall(n, 1, 0, D, D, held[1], held[2], q=held[0], q_out=out))
    queue.finish()
    got = out.read(np.float16, (n, D))[:, :pairs].astype(np.float64)
    assert (np.abs(got - want[:, None]) <= TOLERANCE).all(), (np.abs(got - want[:, None]).max(), TOLERANCE)
