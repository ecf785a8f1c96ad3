"""mi_kv_write and mi_kv_read count the elements of a row in ints, 512 at a time: rows that would take them past an int are refused,
before any device is looked for."""
import ctypes
import os

import pytest

from helpers import mil


def _both(kv_heads, rows):
    c = mil.KVCache(mil.KV_Q4, 1, 1, kv_heads, 64, 4096, 8192, 4096, 8192)            # (32 bytes of each head: the page is below 2 GiB)
    b = mil.KVBatch(1, rows, 1, 1, 256, 512, 1024)
    ld = kv_heads * 64
    args = [ctypes.addressof(c), ctypes.addressof(b), 4096, ld, 8192, ld]
    return [mil.lib().mi_kv_write(None, *args), mil.lib().mi_kv_read(None, *args)]


@pytest.mark.parametrize("kv_heads", [2 ** 25 - 1, 2 ** 25 - 7])
def test_rows_of_nearly_2_31_elements_are_refused(capfd, kv_heads):
    assert _both(kv_heads, 0) == [0, 0] and _both(kv_heads, 1) == [0, 0]
    assert capfd.readouterr().err.count("more than a launch counts") == 4


def test_rows_below_are_taken(capfd):
    assert _both(2 ** 25 - 9, 0) == [1, 1]
    assert not capfd.readouterr().err


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="would run")
def test_and_go_on_to_the_device(capfd):
    assert _both(2 ** 25 - 9, 1) == [0, 0]
    assert "more than" not in capfd.readouterr().err
