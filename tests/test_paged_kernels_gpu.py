"""Every kernel of mi_attention by itself (which one a call comes to is paged_plan.h's; test_paged_plan.py looks that these cases come
to the ones they are for)."""
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
