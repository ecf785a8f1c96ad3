"""mi_beam_select against the definition in 64 bits: tokens and rows whole numbers that have to be equal, scores to their rounding
(2^-24 of them) and 2^-20 for the logarithm of the sum, whose exponentials are fp32's (each off by 2^-21 at most where it counts)."""
import ctypes

import numpy as np
import pytest

from helpers import mil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def expect(logits, score, groups, beams, n_out):
    tokens, rows, scores = (np.full((groups, n_out), -1, np.int32), np.full((groups, n_out), -1, np.int32),
                            np.full((groups, n_out), -np.inf))
    for g in range(groups):
        best = []
        for r in range(g * beams, (g + 1) * beams):
            x = logits[r].astype(np.float64)
            top = x.max()
            if not np.isfinite(score[r]) or not np.isfinite(top) or np.isnan(x).any():
                continue
            value = float(score[r]) + x - (top + np.log(np.exp(x - top).sum()))
            some = np.argsort(-x, kind="stable")[:n_out]
            best += [(-value[t], r, int(t)) for t in some if np.isfinite(x[t])]
        best.sort()
        for i, (v, r, t) in enumerate(best[:n_out]):
            scores[g, i], rows[g, i], tokens[g, i] = -v, r, t
    return scores, tokens, rows


def select(queue, logits, score, groups, beams, vocab, n_out, ld=0, shift=0):
    ld = ld or vocab
    flat = np.full(shift + groups * beams * ld, np.float16(np.nan))
    rows = flat[shift:].reshape(groups * beams, ld)
    rows[:, :vocab] = logits
    held = [mil.Buffer.from_host(flat), mil.Buffer.from_host(score)]
    outs = [mil.Buffer.from_host(np.full(groups * n_out + 2, 0x12345678, np.int32)) for _ in range(3)]
    assert mil.beam_select(queue, mil.BeamCall(groups, beams, vocab, n_out, held[0].ptr + 2 * shift, held[1], *outs, ld=ld))
    if isinstance(queue, mil.Queue):
        queue.finish()
    else:
        mil.lib().mi_stream_sync(queue)
    got = [o.read(np.int32, (groups * n_out + 2,)) for o in outs]
    assert all((x[-2:] == 0x12345678).all() for x in got), "written behind the outputs"
    got = [x[:-2].reshape(groups, n_out) for x in got]
    return got[0].view(np.float32), got[1], got[2]


def check(got, want):
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all(), (got[1:], want[1:])
    some = np.isfinite(want[0])
    assert (np.isfinite(got[0]) == some).all() and (got[0][~some] == -np.inf).all()
    assert (np.abs(got[0][some] - want[0][some]) <= 2.0 ** -24 * np.abs(want[0][some]) + 2.0 ** -20).all()


def make(rng, rows, vocab, sigma=2.5):
    return (rng.standard_normal((rows, vocab)) * sigma).astype(np.float16), (rng.standard_normal(rows) - 20).astype(np.float32)


@pytest.mark.parametrize("groups,beams,vocab,n_out", [
    (1, 1, 1, 1), (1, 1, 1, 4), (1, 4, 151936, 8), (3, 5, 49152, 10), (2, 8, 65536, 16), (7, 3, 4097, 6), (1, 64, 4096, 64), (2, 9, 12345, 64),
    (5, 2, 63, 4), (40, 4, 500, 8), (1, 2, 300001, 3), (2, 1, 8191, 1), (3, 17, 100, 34)])
def test_against_64_bits(queue, groups, beams, vocab, n_out):
    rng = np.random.default_rng(vocab)
    logits, score = make(rng, groups * beams, vocab)
    check(select(queue, logits, score, groups, beams, vocab, n_out), expect(logits, score, groups, beams, n_out))


@pytest.mark.parametrize("shift,extra", [(1, 0), (0, 1), (3, 8), (4, 3), (8, 16)])
def test_rows_apart_and_unaligned(queue, shift, extra):
    rng = np.random.default_rng(5)
    logits, score = make(rng, 6, 9001)
    check(select(queue, logits, score, 2, 3, 9001, 6, ld=9001 + extra, shift=shift), expect(logits, score, 2, 3, 6))


@pytest.mark.parametrize("vocab", [40, 4096, 5000, 151936])
def test_ties_go_to_the_lowest(queue, vocab):
    """All logits alike; a few values over many tokens; both zeros; beams that are alike."""
    rng = np.random.default_rng(6)
    score = np.full(6, -3.0, np.float32)
    score[3:] = [-2.0, -3.0, -2.0]
    for kind in range(5):
        logits = np.zeros((6, vocab), np.float16)
        if kind == 1:
            logits[:] = rng.integers(0, 3, logits.shape)
        if kind == 2:
            logits[:] = np.where(rng.random(logits.shape) < 0.5, np.float16(-0.0), np.float16(0.0))
            logits[:, 7] = -1
        if kind == 3:
            logits[:] = rng.integers(0, 3, vocab)[None]
        if kind == 4:
            logits[:] = np.linspace(4, -4, vocab)[None]
        check(select(queue, logits, score, 2, 3, vocab, 20), expect(logits, score, 2, 3, 20))


def test_forbidden_tokens_and_beams_that_are_not_there(queue):
    rng = np.random.default_rng(7)
    vocab, beams = 10000, 5
    logits, score = make(rng, 4 * beams, vocab)
    logits[:, rng.permutation(vocab)[:vocab // 2]] = -np.inf
    logits[0, :] = -np.inf                                # a row of nothing
    logits[1, 5:] = -np.inf                               # five tokens
    logits[5:10] = -np.inf                                # group 1: two tokens in all
    logits[6, [77, 9999]] = [1, 2]
    score[10:14] = -np.inf                                # group 2: a first step, one beam
    logits[15, 44], logits[16, 45] = np.nan, np.inf       # group 3: rows that are broken, scores that are
    score[17], score[18] = np.nan, np.inf
    got, want = select(queue, logits, score, 4, beams, vocab, 10), expect(logits, score, 4, beams, 10)
    check(got, want)
    assert (got[1][1, 2:] == -1).all() and set(got[2][2]) == {14} and set(got[2][3]) == {19}


def test_all_of_a_group_gone(queue):
    logits, score = np.full((2, 700), -np.inf, np.float16), np.zeros(2, np.float32)
    got = select(queue, logits, score, 1, 2, 700, 5)
    assert (got[0] == -np.inf).all() and (got[1] == -1).all() and (got[2] == -1).all()


def test_extreme_logits(queue):
    rng = np.random.default_rng(8)
    vocab = 20000
    logits = rng.choice(np.array([65504, -65504, 60000, 2.0 ** -24, -2.0 ** -24, 0], np.float16), (6, vocab))
    logits[3] = -65504
    logits[4] = rng.standard_normal(vocab) * 1e-5
    score = np.array([0, -1, 1, 7, 100, 3], np.float32)
    check(select(queue, logits, score, 2, 3, vocab, 12), expect(logits, score, 2, 3, 12))


def test_more_groups_than_the_workspace_holds(queue):
    """16 MB hold the tiles of about 30000 rows of 4 tiles: the rest goes in another pair of launches."""
    rng = np.random.default_rng(9)
    vocab, groups, beams = 200, 25000, 5                  # 125000 tiles of 136 bytes
    logits, score = make(rng, groups * beams, vocab)
    got = select(queue, logits, score, groups, beams, vocab, 3)
    some = np.concatenate([np.arange(5), np.arange(groups // 2, groups // 2 + 5), np.arange(24660, 24680), np.arange(groups - 5, groups)])
    rows = (some[:, None] * beams + np.arange(beams)).ravel()
    want = expect(logits[rows], score[rows], len(some), beams, 3)
    check([x[some] for x in got[:2]] + [got[2][some] - (some * beams - np.arange(len(some)) * beams)[:, None]], want)


def test_other_streams(queue):
    """The null stream, and one that has no workspace, whose single launch gives the same bits."""
    hip = ctypes.CDLL("libamdhip64.so")
    foreign = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(foreign)) == 0
    for groups, beams, vocab, n_out in ((1, 4, 151936, 8), (3, 5, 4097, 64), (2, 64, 300, 64), (1, 2, 2 ** 21, 5)):
        rng = np.random.default_rng(vocab)
        logits, score = make(rng, groups * beams, vocab)
        own = select(queue, logits, score, groups, beams, vocab, n_out)
        check(own, expect(logits, score, groups, beams, n_out))
        for other in (mil.Queue(default=True), foreign):
            got = select(other, logits, score, groups, beams, vocab, n_out)
            assert all((x.view(np.int32) == y.view(np.int32)).all() for x, y in zip(got, own))
    assert hip.hipStreamDestroy(foreign) == 0


def test_captured(queue):
    """A graph on the stream, replayed with the stream's other users of the workspace in between."""
    rng = np.random.default_rng(10)
    groups, beams, vocab, n_out = 2, 4, 20000, 8
    logits, score = make(rng, groups * beams, vocab)
    held = [mil.Buffer.from_host(logits), mil.Buffer.from_host(score)]
    outs = [mil.Buffer.from_host(np.zeros((groups, n_out), np.int32)) for _ in range(3)]
    call = mil.BeamCall(groups, beams, vocab, n_out, *held, *outs)
    assert mil.lib().mi_graph_begin(queue.handle)
    assert mil.beam_select(queue, call)
    graph = mil.lib().mi_graph_end(queue.handle)
    for turn in range(3):
        logits, score = make(rng, groups * beams, vocab)
        held[0].write(logits)
        held[1].write(score)
        other = make(rng, 6, 5000)
        check(select(queue, *other, 2, 3, 5000, 6), expect(*other, 2, 3, 6))
        assert mil.lib().mi_graph_launch(graph, queue.handle)
        queue.finish()
        got = [o.read(t, (groups, n_out)) for o, t in zip(outs, (np.float32, np.int32, np.int32))]
        check(got, expect(logits, score, groups, beams, n_out))
    mil.lib().mi_graph_destroy(graph)


def test_streams_at_once(queue):
    """Two streams, each with a workspace of its own."""
    rng = np.random.default_rng(11)
    queues, held, calls, outs = [queue, mil.Queue()], [], [], []
    for i in range(2):
        logits, score = make(rng, 8, 30000)
        held.append((logits, score, mil.Buffer.from_host(logits), mil.Buffer.from_host(score)))
        outs.append([mil.Buffer.from_host(np.zeros((2, 8), np.int32)) for _ in range(3)])
        calls.append(mil.BeamCall(2, 4, 30000, 8, *held[i][2:], *outs[i]))
    for _ in range(30):
        for q, call in zip(queues, calls):
            assert mil.beam_select(q, call)
    for q, (logits, score, _, _), out in zip(queues, held, outs):
        q.finish()
        check([o.read(t, (2, 8)) for o, t in zip(out, (np.float32, np.int32, np.int32))], expect(logits, score, 2, 4, 8))


@pytest.mark.parametrize("beams", [1, 2, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("n_out", [1, 2, 16, 24, 25, 63, 64])
def test_every_number_of_beams_and_outputs(queue, beams, n_out):
    """Scores nearly alike, so that all rows offer; among them rows that tie in everything, and logits of few values."""
    rng = np.random.default_rng(beams * 100 + n_out)
    for levels in (0, 5, 400):
        logits, score = make(rng, 2 * beams, 5000)
        if levels:
            logits = (np.rint(logits.astype(np.float32) * levels / 8) * 8 / levels).astype(np.float16)
        score[:] = np.where(rng.random(2 * beams) < 0.5, -20, score / 100 - 20)
        logits[beams:][::3] = logits[beams]
        score[beams:][::3] = score[beams]
        check(select(queue, logits, score, 2, beams, 5000, n_out), expect(logits, score, 2, beams, n_out))


@pytest.mark.parametrize("score", [1e6, -3e7, 2.0 ** 28])
def test_scores_far_from_zero(queue, score):
    """The order is that of the 64-bit sums, which fp32's steps at the scores do not show."""
    rng = np.random.default_rng(12)
    logits, _ = make(rng, 4, 3000)
    scores = np.full(4, score, np.float32)
    got, want = select(queue, logits, scores, 1, 4, 3000, 12), expect(logits, scores, 1, 4, 12)
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all() and (got[0] == want[0].astype(np.float32)).all()
