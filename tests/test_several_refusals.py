"""What mi_rope, mi_attention_tree, mi_kv_keep, mi_kv_reorder and mi_beam_select refuse, said before any device is looked for; and
that nothing to do is nothing to refuse.  (No GPU: an accepted call would go on to mi_init and fail there.)"""
import ctypes
import os

import pytest

from helpers import mil

CACHE = dict(kind=0, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, k=4096, v=8192, k_scale=None, v_scale=None)
BATCH = dict(n_seqs=1, n_tokens=3, max_tokens=3, max_pages=2, q_start=256, kv_len=512, pages=1024)
no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="would run")


def at(x):
    return ctypes.addressof(x)


def rope(**more):
    given = dict(dict(n_tokens=3, n_heads=4, n_kv_heads=2, head_dim=64, rot_dim=64, inv_freq=256, position=512, q=4096, q_out=8192, k=12288,
                      k_out=16384), **more)
    n_axes = given.pop("n_axes", None)
    call = mil.RopeCall(**given)
    if n_axes is not None:
        call.n_axes = n_axes
    return mil.rope(None, call)


@pytest.mark.parametrize("bad,word", [
    (dict(n_tokens=-1), "n_tokens=-1"), (dict(n_heads=-1), "n_heads=-1"), (dict(n_kv_heads=-2), "n_kv_heads=-2"),
    (dict(head_dim=0, rot_dim=0), "head_dim=0"), (dict(head_dim=63, rot_dim=62), "head_dim=63"), (dict(head_dim=258), "head_dim=258"),
    (dict(rot_dim=66), "rot_dim=66"), (dict(rot_dim=-2), "rot_dim=-2"), (dict(rot_dim=33), "rot_dim=33"),
    (dict(n_axes=0), "n_axes=0"), (dict(n_axes=5), "n_axes=5"), (dict(axis=[0] * 31 + [2], n_axes=2), "axis[31]=2 of 2"),
    (dict(q=None), "bad rows (q"), (dict(q=4097), "bad rows (q"), (dict(q_out=None), "bad rows (q"), (dict(q_out=8193), "bad rows (q"),
    (dict(ld_q=255), "bad rows (q"), (dict(ld_q_out=255), "bad rows (q"), (dict(q_out=4096, ld_q=512), "bad rows (q"),
    (dict(k=None), "bad rows (k"), (dict(k_out=None), "bad rows (k"), (dict(ld_k=127), "bad rows (k"), (dict(ld_k_out=-128), "bad rows (k"),
    (dict(inv_freq=None), "inv_freq"), (dict(inv_freq=258), "inv_freq"), (dict(position=None), "position"), (dict(position=513), "position"),
    (dict(n_heads=1 << 24, ld_q=1 << 30, ld_q_out=1 << 30), "more than a launch counts"), (dict(n_tokens=1 << 30), "more than a launch counts"),
])
def test_rope(capfd, bad, word):
    assert not rope(**bad)
    err = capfd.readouterr().err
    assert err.count("ERROR: mi_rope: ") == 1 and word in err, err


def test_rope_null_and_nothing(capfd):
    assert mil.lib().mi_rope(None, None) == 0 and "null" in capfd.readouterr().err
    assert rope(n_tokens=0) and rope(n_heads=0, n_kv_heads=0, q=None, q_out=None, k=None, k_out=None)
    with pytest.raises(ValueError):
        rope(axis=[0] * 31)


def tree(cache=None, batch=None, call=None, mask=None):
    c, b = mil.KVCache(**dict(CACHE, **(cache or {}))), mil.KVBatch(**dict(BATCH, **(batch or {})))
    a = mil.AttentionCall(c, b, **dict(dict(n_heads=4, q=4096, out=8192), **(call or {})))
    return mil.attention_tree(None, a, mil.TreeMask(**dict(dict(seen=256, words=1, position=512), **(mask or {}))))


@pytest.mark.parametrize("bad,word", [
    (dict(cache=dict(kind=1)), "bad cache"), (dict(cache=dict(k=8)), "aligned"), (dict(batch=dict(n_seqs=-1)), "bad batch"),
    (dict(call=dict(n_heads=3)), "bad argument"), (dict(call=dict(scale=0.0)), "bad argument"), (dict(call=dict(sinks=-1)), "bad argument"),
    (dict(call=dict(ld_q=255)), "bad argument"), (dict(mask=dict(words=0)), "words=0"), (dict(mask=dict(words=65537)), "words=65537"),
    (dict(mask=dict(seen=None)), "seen"), (dict(mask=dict(seen=258)), "seen"), (dict(mask=dict(position=None), call=dict(window=5)), "window=5"),
    (dict(mask=dict(position=514)), "position"),
])
def test_tree(capfd, bad, word):
    assert not tree(**bad)
    err = capfd.readouterr().err
    assert err.count("ERROR: mi_attention_tree: ") == 1 and word in err, err


def test_tree_null_and_nothing(capfd):
    assert mil.lib().mi_attention_tree(None, None, 8) == 0
    c, b = mil.KVCache(**CACHE), mil.KVBatch(**BATCH)
    assert mil.lib().mi_attention_tree(None, at(mil.AttentionCall(c, b, 4, 4096, 8192)), None) == 0
    assert capfd.readouterr().err.count("null") == 2
    assert tree(batch=dict(n_tokens=0)) and tree(batch=dict(n_seqs=0, q_start=None, kv_len=None, pages=None))


def keep(caches=({},), batch=None, **more):
    made = [mil.KVCache(**dict(CACHE, **c)) for c in caches]
    given = dict(dict(keep=256, kept=2048, new_len=4096), **more)
    return mil.kv_keep(None, mil.KVCaches(made), mil.KVBatch(**dict(BATCH, **(batch or {}))), **given)


@pytest.mark.parametrize("bad,word", [
    (dict(caches=()), "no caches"), (dict(caches=({}, dict(kind=9))), "bad cache"), (dict(caches=({}, dict(k=None))), "aligned"),
    (dict(caches=({}, dict(n_pages=5))), "cache 1 differs"), (dict(caches=({}, {}, dict(page_size=32))), "cache 2 differs"),
    (dict(caches=({}, dict(head_dim=128))), "cache 1 differs"), (dict(caches=({}, dict(n_kv_heads=1))), "cache 1 differs"),
    (dict(caches=({}, dict(kind=8, k_scale=256, v_scale=512))), "cache 1 differs"), (dict(batch=dict(max_pages=0)), "bad batch"),
    (dict(batch=dict(kv_len=None)), "bad batch"), (dict(keep=None), "bad argument"), (dict(keep=258), "bad argument"),
    (dict(kept=None), "bad argument"), (dict(kept=2049), "bad argument"), (dict(new_len=2), "bad argument"), (dict(new_len=2048), "bad argument"),
    (dict(new_len=512), "bad argument"), (dict(batch=dict(n_seqs=1 << 30)), "more than a launch counts"),
])
def test_keep(capfd, bad, word):
    assert not keep(**bad)
    err = capfd.readouterr().err
    assert err.count("ERROR: mi_kv_keep: ") == 1 and word in err, err


def reorder(caches=({},), **more):
    made = [mil.KVCache(**dict(CACHE, **c)) for c in caches]
    given = dict(dict(n_seqs=2, max_pages=3, kv_len=256, pages=512, source=1024, fresh=2048, new_len=4096, new_pages=8192), **more)
    return mil.kv_reorder(None, mil.KVCaches(made), mil.ReorderCall(**given))


@pytest.mark.parametrize("bad,word", [
    (dict(caches=()), "no caches"), (dict(caches=({}, dict(v=8))), "aligned"), (dict(caches=({}, dict(n_pages=5))), "cache 1 differs"),
    (dict(n_seqs=-1), "bad batch"), (dict(max_pages=0), "bad batch"), (dict(kv_len=None), "bad batch"), (dict(pages=513), "bad batch"),
    (dict(source=None), "bad argument"), (dict(fresh=2050), "bad argument"), (dict(new_len=None), "bad argument"),
    (dict(new_pages=None), "bad argument"), (dict(new_len=256), "bad argument"), (dict(new_pages=512), "bad argument"),
    (dict(new_pages=4096), "bad argument"), (dict(new_len=2048), "bad argument"), (dict(n_seqs=1 << 30), "more than a launch counts"),
])
def test_reorder(capfd, bad, word):
    assert not reorder(**bad)
    err = capfd.readouterr().err
    assert err.count("ERROR: mi_kv_reorder: ") == 1 and word in err, err


def test_moves_null_and_nothing(capfd):
    caches = mil.KVCaches([mil.KVCache(**CACHE)])
    assert mil.lib().mi_kv_keep(None, None, 1, at(mil.KVBatch(**BATCH)), 256, 2048, None) == 0
    assert mil.lib().mi_kv_keep(None, caches._at, 1, None, 256, 2048, None) == 0
    assert mil.lib().mi_kv_reorder(None, caches._at, 1, None) == 0 and mil.lib().mi_kv_reorder(None, None, 1, at(mil.ReorderCall(0, 1, *[256] * 6))) == 0
    assert capfd.readouterr().err.count("ERROR") == 4
    assert keep(batch=dict(n_seqs=0), keep=None, kept=None, new_len=None)
    assert reorder(n_seqs=0, kv_len=None, pages=None, source=None, fresh=None, new_len=None, new_pages=None)


def beam(**more):
    given = dict(dict(n_groups=1, beams=2, vocab=100, n_out=4, logits=4096, score=256, out_score=512, out_token=1024, out_row=2048), **more)
    return mil.beam_select(None, mil.BeamCall(**given))


@pytest.mark.parametrize("bad,word", [
    (dict(n_groups=-1), "n_groups=-1"), (dict(beams=0), "beams=0"), (dict(beams=65), "beams=65"), (dict(n_out=0), "n_out=0"),
    (dict(n_out=65), "n_out=65"), (dict(vocab=0, ld=5), "vocab=0"), (dict(vocab=(1 << 21) + 1), "vocab=2097153"), (dict(ld=99), "ld=99"),
    (dict(logits=None), "logits="), (dict(logits=4097), "logits="), (dict(score=None), "score="), (dict(score=258), "score="),
    (dict(out_score=None), "out_score="), (dict(out_token=1026), "out_token="), (dict(out_row=None), "out_row="),
    (dict(n_groups=1 << 30), "more than a launch counts"),
])
def test_beam(capfd, bad, word):
    assert not beam(**bad)
    err = capfd.readouterr().err
    assert err.count("ERROR: mi_beam_select: ") == 1 and word in err, err


def test_beam_null_and_nothing(capfd):
    assert mil.lib().mi_beam_select(None, None) == 0 and "null" in capfd.readouterr().err
    assert beam(n_groups=0, logits=None)


@no_gpu
def test_good_calls_go_on_to_the_device(capfd):
    assert not any((rope(), tree(), keep(), reorder(), beam()))
    assert "bad" not in capfd.readouterr().err


@pytest.mark.parametrize("pools,which", [
    ([(4096, 8192), (16384, 32768), (4096, 65536)], 2), ([(4096, 8192), (8192, 16384)], 1), ([(4096, 4096)], 0),
    ([(4096, 8192), (16384, 8192)], 1), ([(4096, 8192), (16384, 32768), (65536, 16384)], 2),
])
def test_a_pool_that_is_there_twice(capfd, pools, which):
    """Its rows would be moved twice, by two wavefronts at once."""
    caches = [dict(k=k, v=v) for k, v in pools]
    assert not keep(caches) and not reorder(caches)
    err = capfd.readouterr().err
    assert err.count(f"a pool of cache {which} is there twice") == 2, err


def test_lengths_do_not_replace_what_is_read(capfd):
    assert not keep(new_len=256, keep=256) and not keep(new_len=BATCH["pages"]) and not keep(new_len=BATCH["q_start"])
    assert capfd.readouterr().err.count("bad argument") == 3
