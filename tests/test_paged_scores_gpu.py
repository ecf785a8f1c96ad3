"""mi_attention where the products of queries and keys are large: a row's weights come from the differences of its scores, however
far from 0 these are.  Scores here are sums that fp32 holds exactly, so what the rows have to give is known."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache

pytestmark = pytest.mark.gpu
KINDS = [mil.KV_F16, mil.KV_INT8, mil.KV_Q4]
# (rows of new tokens, positions, pages as wide as): the kernel for few rows, alone and in parts, and the one for many, in one
# piece and in parts
FORMS = [(1, 40, 0), (1, 3000, 0), (70, 200, 2 ** 20), (70, 3000, 2 ** 20)]


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


def _cache(monkeypatch, kind, D, form, q, k):
    """Queries all `q`, keys all `k` (a number that every kind holds: a scale's 127 or 7 times a power of two)."""
    n, m, columns = form
    monkeypatch.setattr(Cache, "columns", columns)
    c = Cache(kind, 4, 2, D, 16, [m], [n], seed=31)
    c.qkv[:, :4 * D] = q
    c.k[0][:] = k
    return c


def _check(c, got, want, mean):
    """want: [rows, kv heads, D] in 64 bits.  Equal weights are equal exactly, so an output is off by its own rounding, 2^-11 of it, and
    by fp32 sums of m terms and the quotient, (m + 2) 2^-24 of the mean of |v|; 2^-25 where fp16 has its smallest steps."""
    got = got.astype(np.float64).reshape(len(got), 2, 2, c.D)
    tol = 2.0 ** -11 * np.abs(want) + (c.lengths[0] + 2) * 2.0 ** -24 * mean + 2.0 ** -25
    bad = ~(np.abs(got - want[:, :, None]) <= tol[:, :, None])
    assert not bad.any(), (int(bad.sum()), got[bad][:4], np.broadcast_to(want[:, :, None], got.shape)[bad][:4])


def _values(c):
    from paged_lib import quantise, values
    return values(c.kind, *quantise(c.kind, c.v[0])).astype(np.float64)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D,q,scale", [(64, 24576.0, 0.123), (128, 24576.0, 0.0884), (64, 3.0, 65504.0), (64, 96.0, 11.7), (128, 24.0, 1.37)])
@pytest.mark.parametrize("kind", KINDS)
def test_equal_scores_far_from_0(monkeypatch, queue, kind, D, q, scale, sign, form):
    """All keys alike: the mean of the values.  Scores of up to 10^10 either way, around 2^18 to 2^34 steps of the exponent."""
    k = 7 * 2.0 ** 11 if q > 1000 else 7 * 2.0 ** 6
    c = _cache(monkeypatch, kind, D, form, sign * q, k)
    c.fill()
    n, m, _ = form
    v = _values(c)
    want, mean = (np.cumsum(x, 0)[m - n:] / np.arange(m - n + 1, m + 1)[:, None, None] for x in (v, np.abs(v)))
    _check(c, c.upload().attend(queue, scale=scale), want, mean)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("at", [0, 17, -3])
@pytest.mark.parametrize("kind", KINDS)
def test_one_key_above_all_others_far_from_0(monkeypatch, queue, kind, at, form):
    """A key whose score is a seventh above the others' in the 10^9s: rows that see it give its value, those before it a mean."""
    c = _cache(monkeypatch, kind, 64, form, 24576.0, 6 * 2.0 ** 11)
    n, m, _ = form
    at = at % m
    c.k[0][:, :, 0] = 7 * 2.0 ** 11                       # (each row's greatest, so that 6 is a code as well)
    c.k[0][at] = 7 * 2.0 ** 11
    c.fill()
    v = _values(c)
    want, mean = (np.cumsum(x, 0)[m - n:] / np.arange(m - n + 1, m + 1)[:, None, None] for x in (v, np.abs(v)))
    for r in range(n):
        if m - n + r >= at:
            want[r], mean[r] = v[at], np.abs(v[at])
    if kind == mil.KV_INT8:                              # (6 of 7 is 108.9 codes of 127: the rows are still alike)
        assert (c.pool["k"][c.table[0, 0]][:, 1] == 109).any()
    _check(c, c.upload().attend(queue, scale=0.123), want, mean)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("odd", [1.0, np.inf, np.nan])
def test_scores_of_minus_infinity_alone_give_zeros(monkeypatch, queue, odd, form):
    """Whatever the values are."""
    c = _cache(monkeypatch, mil.KV_F16, 64, form, 1.0, 0.0)
    c.k[0][:, :, 5] = -np.inf
    c.v[0][::3, :, 7] = odd
    c.fill()
    assert (c.upload().attend(queue).view(np.uint16) & 0x7fff == 0).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", KINDS)
def test_heads_of_either_kind_side_by_side(monkeypatch, queue, kind, form):
    """One head of a group with scores in the 10^8s, the other with ordinary ones: rows of one matrix, each as by itself."""
    n, m, columns = form
    monkeypatch.setattr(Cache, "columns", columns)
    c = Cache(kind, 4, 2, 64, 16, [m], [n], seed=33)
    for head in (0, 2):
        c.qkv[:, head * 64:head * 64 + 64] = 0
        c.qkv[:, head * 64] = 3 * 2.0 ** 13
    for b in c.k:
        b[:, :, 0] = 7 * 2.0 ** 9                         # (its products with the far heads' queries: 21 2^22)
        b[:, :, 1:] = np.clip(b[:, :, 1:], -3, 3)
    for head in (1, 3):
        c.qkv[:, head * 64] = 0
    if kind != mil.KV_F16:                               # (a scale for so large an element leaves the others 0: ordinary scores are)
        c.k[0][:, :, 1:] = 0
    c.fill()
    got = c.upload().attend(queue, scale=7.3)
    v = _values(c)
    want, mean = (np.cumsum(x, 0)[m - n:] / np.arange(m - n + 1, m + 1)[:, None, None] for x in (v, np.abs(v)))
    far = got[:, [0, 2]].astype(np.float64)
    tol = 2.0 ** -11 * np.abs(want) + (m + 2) * 2.0 ** -24 * mean + 2.0 ** -25
    assert (np.abs(far - want) <= tol).all()
    want, tol = c.expect(scale=7.3)
    assert (np.abs(got[:n].astype(np.float64) - want) <= tol)[:, [1, 3]].all()
