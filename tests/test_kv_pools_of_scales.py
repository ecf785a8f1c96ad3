"""What mi_kv_keep and mi_kv_reorder refuse of the scales of quantised caches: a pool of scales that is there twice would have its rows moved twice,
by blocks of one launch that nothing orders, and a row could be left with another one's scale.  (No GPU: an accepted call would go on to mi_init and
fail there.)"""
import pytest

from helpers import mil
from test_several_refusals import keep, no_gpu, reorder


def caches(kind, *scales):
    """Caches with pools of their own and these pools of scales, keys' and values'."""
    return [dict(kind=kind, k=65536 * (2 * i + 1), v=65536 * (2 * i + 2), k_scale=k, v_scale=v) for i, (k, v) in enumerate(scales)]


@pytest.mark.parametrize("kind", [mil.KV_INT8, mil.KV_Q4])
@pytest.mark.parametrize("scales,which", [
    ([(256, 256)], 0), ([(256, 512), (1024, 1024)], 1), ([(256, 512), (256, 1024)], 1), ([(256, 512), (1024, 512)], 1), ([(256, 512), (512, 1024)], 1),
    ([(256, 512), (1024, 256)], 1), ([(256, 512), (1024, 2048), (4096, 8192), (16384, 1024)], 3),
])
def test_scales_that_are_there_twice(capfd, kind, scales, which):
    made = caches(kind, *scales)
    assert not keep(made) and not reorder(made)
    err = capfd.readouterr().err
    assert err.count(f"scales of cache {which} are there twice") == 2 and err.count("ERROR: mi_kv_keep: ") == err.count("ERROR: mi_kv_reorder: ") == 1, err


@no_gpu
def test_scales_of_their_own_and_those_that_are_not_used(capfd):
    """fp16 caches' are not looked at."""
    for kind in (mil.KV_INT8, mil.KV_Q4):
        assert not keep(caches(kind, (256, 512), (1024, 2048))) and not reorder(caches(kind, (256, 512), (1024, 2048)))
    assert not keep(caches(mil.KV_F16, (256, 256), (256, None))) and not reorder(caches(mil.KV_F16, (None, None), (None, None)))
    assert "twice" not in capfd.readouterr().err
