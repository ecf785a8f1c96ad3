"""A call of mi_attention that is refused has done nothing, also where only the second of its launches cannot be made."""
import numpy as np
import pytest

from helpers import mil

pytestmark = pytest.mark.gpu


def test_refused_before_anything_is_enqueued(capfd):
    """2100 sequences of 34100 rows, 4096 heads of their own: the launch for sequences of many rows would fit, the one for
    those of few has more blocks than a grid counts.  (All rows but the 64 of the first sequence are padding.)"""
    assert mil.lib().mi_init(0) == 1
    queue, heads, D, page, seqs, rows, real = mil.Queue(), 4096, 64, 64, 2100, 34100, 64
    width = heads * D
    pools = [mil.Buffer.from_host(np.zeros((heads, page, D), np.float16)) for _ in "kv"]
    cache = mil.KVCache(mil.KV_F16, 1, page, heads, D, *pools)
    start = np.full(seqs + 1, real, np.int32)
    start[0] = 0
    length, table = np.zeros(seqs, np.int32), np.zeros((seqs, 1), np.int32)
    length[0] = real
    held = [mil.Buffer.from_host(x) for x in (start, length, table)]
    q, out = (mil.Buffer.from_host(np.full((real, width), x, np.uint16)) for x in (0, 0x1234))

    def call(n):
        return mil.attention(queue, mil.AttentionCall(cache, mil.KVBatch(seqs, n, real, 1, *held), heads, q, out))

    assert not call(rows)
    queue.finish()
    assert "more than a launch counts" in capfd.readouterr().err
    assert (out.read(np.uint16, (real, width)) == 0x1234).all()
    assert call(real)                                      # and fewer are taken
    queue.finish()
    assert (out.read(np.uint16, (real, width)) == 0).all()
