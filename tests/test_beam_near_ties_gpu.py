"""mi_beam_select where beams (nearly) tie: rows alike in everything are equal whatever their alignment; rows whose sums are nearer to each other
than the logarithm's error (2^-20, of fp32's exponentials) come in either order, and all else is as it has to be."""
import ctypes

import numpy as np
import pytest

from helpers import mil
from test_beam_select_gpu import check, expect, make, queue, select  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams,vocab,n_out,extra", [(4, 30000, 12, 0), (4, 30000, 12, 3), (9, 5001, 40, 1), (20, 4100, 33, 5), (64, 700, 64, 1), (2, 151936, 4, 7)])
def test_rows_that_are_alike(queue, beams, vocab, n_out, extra):  # noqa: F811
    """ld makes every row begin at another alignment; the lowest rows come first, token by token."""
    rng = np.random.default_rng(beams)
    row, score = make(rng, 1, vocab)
    logits, scores = np.repeat(row, beams, 0), np.repeat(score, beams)
    hip = ctypes.CDLL("libamdhip64.so")
    foreign = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(foreign)) == 0
    for q in (queue, foreign):
        check(select(q, logits, scores, 1, beams, vocab, n_out, ld=vocab + extra), expect(logits, scores, 1, beams, n_out))
    assert hip.hipStreamDestroy(foreign) == 0


@pytest.mark.parametrize("beams,vocab,n_out", [(2, 30000, 16), (5, 9000, 20), (16, 5000, 32), (24, 5000, 64), (3, 300, 30)])
def test_rows_of_the_same_logits_in_another_order(queue, beams, vocab, n_out):  # noqa: F811
    rng = np.random.default_rng(vocab)
    row, score = make(rng, 1, vocab)
    logits = np.stack([row[0][rng.permutation(vocab)] for _ in range(beams)])
    scores = np.repeat(score, beams)
    got, want = select(queue, logits, scores, 1, beams, vocab, n_out), expect(logits, scores, 1, beams, n_out)
    x = row[0].astype(np.float64)
    off = 2.0 ** -24 * np.abs(want[0]) + 2.0 ** -20
    assert (np.abs(got[0] - want[0]) <= off).all()
    value, token, source = got[0][0], got[1][0], got[2][0]
    assert len(set(zip(token.tolist(), source.tolist()))) == n_out
    true = float(score[0]) + logits[source, token].astype(np.float64) - (x.max() + np.log(np.exp(x - x.max()).sum()))
    assert (np.abs(value - true) <= off[0]).all() and (np.diff(value) <= 0).all()
    for r in range(beams):                                # within a row the order is that of its logits, then its tokens, and none is left out
        mine = token[source == r]
        order = np.argsort(-logits[r].astype(np.float64), kind="stable")[:len(mine)]
        assert (mine == order).all()
