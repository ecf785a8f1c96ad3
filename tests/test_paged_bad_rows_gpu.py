"""mi_attention after a call whose q_start goes down, so that sequences share rows: whatever that call computes, the stream's later
ones are as ever."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("columns,new", [(0, 1), (2 ** 20, 60)], ids=["few", "many"])
@pytest.mark.parametrize("at", [0, 63, 70])
def test_a_q_start_that_goes_down(monkeypatch, columns, new, at):
    assert mil.lib().mi_init(0) == 1
    queue = mil.Queue()
    monkeypatch.setattr(Cache, "columns", columns)
    seqs = at + 8
    good = Cache(mil.KV_F16, 14, 2, 64, 16, [1500] * 4, [new] * 4, seed=51).upload()
    bad = Cache(mil.KV_F16, 14, 2, 64, 16, [1] * at + [1500] * 8, [0] * at + [new] * 8, seed=52).upload()
    start = np.zeros(seqs + 1, np.int32)
    start[at:] = np.where(np.arange(seqs + 1 - at) % 2, new, 0)                # 0, new, 0, new, ..
    bad.dev_start.write(start)
    bad.batch = mil.KVBatch(seqs, new, new, bad.max_pages, bad.dev_start, bad.dev_len, bad.dev_table)
    out = mil.Buffer.from_host(np.full((bad.rows, 14 * 64), 0x1234, np.uint16))
    for _ in range(3):
        assert mil.attention(queue, mil.AttentionCall(bad.cache, bad.batch, 14, bad.dev_qkv, out, ld_q=bad.ld))
        queue.finish()
        assert (out.read(np.uint16, (bad.rows, 14 * 64))[new:] == 0x1234).all()
        good.check(good.attend(queue))
        # a product whose slices of K meet by the same counters
    N, K = 64, 4864
    w, x = mil.synth_normal_f16(1, 0.02, (N, K)), mil.synth_normal_f16(2, 1.0, (40, K))
    held = [mil.Buffer.from_host(a) for a in (w, x)] + [mil.Buffer(40 * N * 2)]
    assert mil.pytorch_linear(queue, 40, N, K, held[1], held[0], held[2])
    queue.finish()
    want = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.abs(held[2].read(np.float16, (40, N)).astype(np.float64) - want).max() < 1e-2
