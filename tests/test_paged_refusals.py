"""What mi_kv_write, mi_kv_read and mi_attention refuse, said before any device is looked for; and that nothing to do is
nothing to refuse.  (No GPU: an accepted call would go on to mi_init and fail there.)"""
import ctypes
import os

import pytest

from helpers import mil

GOOD = dict(kind=0, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, k=4096, v=8192, k_scale=None, v_scale=None)
BATCH = dict(n_seqs=1, n_tokens=3, max_tokens=3, max_pages=2, q_start=256, kv_len=512, pages=1024)
CALL = dict(n_heads=4, q=4096, out=8192)


def _all(cache=None, batch=None, call=None, rows=None):
    c, b = mil.KVCache(**dict(GOOD, **(cache or {}))), mil.KVBatch(**dict(BATCH, **(batch or {})))
    rows = dict(dict(k=4096, v=8192, ld_k=128, ld_v=128), **(rows or {}))
    args = [ctypes.addressof(c), ctypes.addressof(b), rows["k"], rows["ld_k"], rows["v"], rows["ld_v"]]
    a = mil.AttentionCall(c, b, **dict(CALL, **(call or {})))
    return [mil.lib().mi_kv_write(None, *args), mil.lib().mi_kv_read(None, *args), mil.lib().mi_attention(None, ctypes.addressof(a))]


@pytest.mark.parametrize("bad,word", [
    (dict(cache=dict(kind=1)), "bad cache"), (dict(cache=dict(head_dim=96)), "bad cache"), (dict(cache=dict(page_size=0)), "bad cache"),
    (dict(cache=dict(n_pages=0)), "bad cache"), (dict(cache=dict(n_kv_heads=0)), "bad cache"),
    (dict(cache=dict(k=None)), "aligned"), (dict(cache=dict(v=8200)), "aligned"),
    (dict(cache=dict(kind=8)), "aligned"), (dict(cache=dict(kind=4, k_scale=256, v_scale=258)), "aligned"),
    (dict(cache=dict(page_size=1 << 24, n_kv_heads=2, head_dim=64)), "2 GiB"),
    (dict(batch=dict(n_seqs=-1)), "bad batch"), (dict(batch=dict(n_tokens=-1)), "bad batch"), (dict(batch=dict(max_pages=0)), "bad batch"),
    (dict(batch=dict(q_start=None)), "bad batch"), (dict(batch=dict(kv_len=None)), "bad batch"), (dict(batch=dict(pages=514)), "bad batch"),
])
def test_of_all_three(capfd, bad, word):
    assert _all(**bad) == [0, 0, 0]
    err = capfd.readouterr().err
    assert err.count("ERROR: ") == 3 and err.count(word) == 3, err
    assert all(name in err for name in ("mi_kv_write", "mi_kv_read", "mi_attention"))


@pytest.mark.parametrize("rows", [dict(k=None), dict(v=None), dict(ld_k=127), dict(ld_v=0), dict(ld_v=-128), dict(k=4097)])
def test_of_rows(capfd, rows):
    assert _all(batch=dict(n_tokens=0))[:2] == [1, 1]
    capfd.readouterr()
    assert _all(batch=dict(n_tokens=0), rows=rows)[:2] == [0, 0]
    assert capfd.readouterr().err.count("bad rows") == 2


@pytest.mark.parametrize("call", [
    dict(n_heads=0), dict(n_heads=3), dict(n_heads=-2), dict(q=None), dict(out=None), dict(q=4097), dict(out=8193), dict(ld_q=255),
    dict(ld_out=255), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e6),
    dict(sinks=-1)])
def test_of_a_call(capfd, call):
    assert _all(batch=dict(n_tokens=0), call=call)[2] == 0
    assert "mi_attention: bad argument" in capfd.readouterr().err


def test_null_and_too_many(capfd):
    assert mil.lib().mi_attention(None, None) == 0
    assert mil.lib().mi_kv_write(None, None, None, None, 0, None, 0) == 0
    assert mil.lib().mi_kv_read(None, None, None, None, 0, None, 0) == 0
    c = mil.KVCache(**dict(GOOD, n_kv_heads=1 << 12, page_size=1))
    b = mil.KVBatch(**dict(BATCH, n_tokens=1 << 30))
    ld = (1 << 12) * 64
    args = [ctypes.addressof(c), ctypes.addressof(b), 4096, ld, 8192, ld]
    assert mil.lib().mi_kv_write(None, *args) == 0 and mil.lib().mi_kv_read(None, *args) == 0
    a = mil.AttentionCall(c, b, 1 << 12, 4096, 8192)
    assert mil.lib().mi_attention(None, ctypes.addressof(a)) == 0
    err = capfd.readouterr().err
    assert err.count("null") == 3 and err.count("more than a launch counts") == 3


def test_nothing_to_do():
    assert _all(batch=dict(n_tokens=0)) == [1, 1, 1]
    assert _all(batch=dict(n_seqs=0, q_start=None, kv_len=None, pages=None)) == [1, 1, 1]


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="would run")
def test_a_good_call_goes_on_to_the_device(capfd):
    assert _all() == [0, 0, 0]
    assert "bad" not in capfd.readouterr().err
