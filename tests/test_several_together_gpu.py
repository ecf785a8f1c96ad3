"""The calls of several continuations as a host makes them, one layer and its cache in pages:

trees of drafts: rotary positions of the drafts' queries and keys, rows into the cache, attention over the tree, the accepted path kept,
and the next token after it, whose attention has to be that of a sequence that was written in its own order all along;
beams: continuations chosen from logits, beams that go on as copies of others, and the next token of each, whose attention has to be
that of a cache of its own."""
import numpy as np
import pytest

from helpers import mil
from paged_lib import quantise, values
from test_beam_select_gpu import expect as best_of
from test_rope_gpu import expect as turned
from tree_lib import ancestors, tree

pytestmark = pytest.mark.gpu
HEADS, KV, D, PAGE, PAGES = 14, 2, 64, 16, 40
INV = (1e4 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)


@pytest.fixture(scope="module")
def queue():
    assert mil.lib().mi_init(0) == 1
    return mil.Queue()


class Host:
    """What a host keeps: pools, page tables and lengths in device memory."""

    def __init__(self, queue, kind, seqs):
        self.queue, self.kind, self.seqs = queue, kind, seqs
        row = {mil.KV_F16: 2 * D, mil.KV_INT8: D, mil.KV_Q4: D // 2}[kind]
        scales = {mil.KV_F16: 0, mil.KV_INT8: 1, mil.KV_Q4: D // 32}[kind]
        self.pools = [mil.Buffer.from_host(np.full(PAGES * KV * PAGE * row, 255, np.uint8)) for _ in "kv"]
        self.scales = [mil.Buffer.from_host(np.full(PAGES * KV * PAGE * max(scales, 1), 0x7e00, np.uint16)) for _ in "kv"]
        self.cache = mil.KVCache(kind, PAGES, PAGE, KV, D, *self.pools, *(self.scales if scales else (None, None)))
        order = np.random.default_rng(1).permutation(PAGES)
        self.columns = PAGES // seqs // 2
        self.table = mil.Buffer.from_host(order[:seqs * self.columns].reshape(seqs, -1).astype(np.int32))
        self.fresh = order[seqs * self.columns:].astype(np.int32)
        self.lengths = mil.Buffer.from_host(np.zeros(seqs, np.int32))

    def batch(self, new, lengths):
        self.lengths.write(np.array(lengths, np.int32))
        self.start = mil.Buffer.from_host(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        return mil.KVBatch(self.seqs, sum(new), max(new), self.columns, self.start, self.lengths, self.table)

    def rotate(self, qkv, position):
        """Rows q | k | v on the device with q and k turned in place, as fp16 rows on the host too."""
        n, ld = qkv.shape
        dev, pos, inv = mil.Buffer.from_host(qkv), mil.Buffer.from_host(np.array(position, np.int32)), mil.Buffer.from_host(INV)
        k = dev.ptr + 2 * HEADS * D
        assert mil.rope(self.queue, mil.RopeCall(n, HEADS, KV, D, D, inv, pos, q=dev, q_out=dev, k=k, k_out=k, ld_q=ld, ld_k=ld, ld_q_out=ld,
                                                 ld_k_out=ld))
        self.queue.finish()
        got = dev.read(np.float16, qkv.shape)
        want, tol = turned(qkv[:, :(HEADS + KV) * D], HEADS + KV, D, D, INV, np.array([position]), [0] * (D // 2), False)
        assert (np.abs(got[:, :(HEADS + KV) * D].astype(np.float64) - want) <= tol).all() and (got[:, (HEADS + KV) * D:] == qkv[:, (HEADS + KV) * D:]).all()
        return dev, got

    def write(self, batch, dev, ld):
        assert mil.kv_write(self.queue, self.cache, batch, dev.ptr + 2 * HEADS * D, dev.ptr + 2 * (HEADS + KV) * D, ld, ld)

    def attend(self, batch, dev, ld, mask=None):
        out = mil.Buffer.from_host(np.zeros((batch.n_tokens, HEADS * D), np.float16))
        call = mil.AttentionCall(self.cache, batch, HEADS, dev, out, ld_q=ld)
        assert mil.attention_tree(self.queue, call, mask) if mask else mil.attention(self.queue, call)
        self.queue.finish()
        return out.read(np.float16, (batch.n_tokens, HEADS, D))


def new_rows(rng, n):
    return rng.standard_normal((n, (HEADS + 2 * KV) * D)).astype(np.float16)


def attention_of(kind, q, rows):
    """One query [HEADS * D] over cached rows (turned q | k | v): (output, how far it may be off: the roundings that paged_lib counts)."""
    k, v = (values(kind, *quantise(kind, rows[:, a * D:(a + KV) * D].reshape(-1, KV, D))).astype(np.float64) for a in (HEADS, HEADS + KV))
    out, tol = np.empty((HEADS, D)), np.empty((HEADS, D))
    for h in range(HEADS):
        x, kh, vh = q[h * D:(h + 1) * D].astype(np.float64), k[:, h // (HEADS // KV)], v[:, h // (HEADS // KV)]
        s = kh @ x * D ** -0.5
        w = np.exp(s - s.max())
        out[h], mean = w @ vh / w.sum(), w @ np.abs(vh) / w.sum()
        off = 2.0 ** -21 + D * 2.0 ** -24 * (np.abs(kh) @ np.abs(x)).max() * D ** -0.5
        tol[h] = 2.0 ** -11 * np.abs(out[h]) + (2 * 2.0 ** -11 + 2 * off) * mean + len(rows) * 2.0 ** -31 * np.abs(vh).max() + 2.0 ** -25
    return out, tol


def near(got, want, tol):
    assert (np.abs(got.astype(np.float64) - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_INT8, mil.KV_Q4])
def test_trees_of_drafts(queue, kind):
    rng = np.random.default_rng(2)
    host, before = Host(queue, kind, 3), [37, 5, 64]
    texts = [None] * 3                                    # of each sequence its rows, turned, in the order of the text
    batch = host.batch(before, before)
    dev, got = host.rotate(new_rows(rng, sum(before)), np.concatenate([np.arange(n) for n in before]))
    host.write(batch, dev, got.shape[1])
    for b, (lo, n) in enumerate(zip(np.cumsum([0] + before), before)):
        texts[b] = got[lo:lo + n]
    for turn in range(4):
        new = [int(rng.integers(3, 20)) for _ in range(3)]
        parents = [tree(rng, n) for n in new]
        seen = [ancestors(p) for p in parents]
        bits = np.zeros((sum(new), 32), bool)
        start = np.concatenate([[0], np.cumsum(new)])
        for s, m in zip(start, seen):
            bits[s:s + len(m), :len(m)] = m
        mask = mil.TreeMask(mil.Buffer.from_host(np.packbits(bits, axis=1, bitorder="little").view(np.uint32)), 1)
        position = np.concatenate([len(t) + m.sum(1) - 1 for t, m in zip(texts, seen)])
        batch = host.batch(new, [len(t) + n for t, n in zip(texts, new)])
        dev, got = host.rotate(new_rows(rng, sum(new)), position)
        host.write(batch, dev, got.shape[1])
        out = host.attend(batch, dev, got.shape[1], mask)
        keep, kept, paths = np.full(sum(new), -1, np.int32), np.zeros(3, np.int32), []
        for b in range(3):
            for i in range(new[b]):
                rows = np.concatenate([texts[b], got[start[b]:start[b + 1]][seen[b][i]]])
                near(out[start[b] + i], *attention_of(kind, got[start[b] + i, :HEADS * D], rows))
            path = np.nonzero(seen[b][rng.integers(0, new[b])])[0]
            paths.append(path)
            keep[start[b]:start[b] + len(path)], kept[b] = path, len(path)
        held = [mil.Buffer.from_host(x) for x in (keep, kept, np.zeros(3, np.int32))]
        assert mil.kv_keep(queue, mil.KVCaches([host.cache]), batch, *held)
        queue.finish()
        for b in range(3):
            texts[b] = np.concatenate([texts[b], got[start[b]:start[b + 1]][paths[b]]])
        assert held[2].read(np.int32, (3,)).tolist() == [len(t) for t in texts]
        # the next token after the path: an ordinary step
        batch = host.batch([1] * 3, [len(t) + 1 for t in texts])
        dev, got = host.rotate(new_rows(rng, 3), [len(t) for t in texts])
        host.write(batch, dev, got.shape[1])
        out = host.attend(batch, dev, got.shape[1])
        for b in range(3):
            texts[b] = np.concatenate([texts[b], got[b:b + 1]])
            near(out[b], *attention_of(kind, got[b, :HEADS * D], texts[b]))


@pytest.mark.parametrize("kind", [mil.KV_F16, mil.KV_INT8])
def test_beams(queue, kind):
    rng = np.random.default_rng(3)
    beams, vocab = 4, 5000
    host = Host(queue, kind, beams)
    table = host.table.read(np.int32, (beams, host.columns))
    spare = list(host.fresh)
    # a prompt that all beams share but for its last page's rows
    n = 21
    dev, got = host.rotate(np.tile(new_rows(rng, n), (beams, 1)), np.tile(np.arange(n), beams))
    host.write(host.batch([n] * beams, [n] * beams), dev, got.shape[1])
    texts = [got[:n] for _ in range(beams)]
    score = np.array([0.0] + [-np.inf] * (beams - 1), np.float32)
    for turn in range(14):
        logits = (rng.standard_normal((beams, vocab)) * 2).astype(np.float16)
        held = [mil.Buffer.from_host(x) for x in (logits, score)]
        outs = [mil.Buffer.from_host(np.zeros((1, beams), np.int32)) for _ in range(3)]
        assert mil.beam_select(queue, mil.BeamCall(1, beams, vocab, beams, *held, *outs))
        fresh = [spare.pop(0) for _ in range(beams)]
        lens = mil.Buffer.from_host(np.array([len(t) for t in texts], np.int32))
        new_len, new_table = mil.Buffer.from_host(np.zeros(beams, np.int32)), mil.Buffer.from_host(np.full((beams, host.columns), -9, np.int32))
        # (the rows that were chosen go from call to call on the device)
        assert mil.kv_reorder(queue, mil.KVCaches([host.cache]), mil.ReorderCall(
            beams, host.columns, lens, host.table, outs[2], mil.Buffer.from_host(np.array(fresh, np.int32)), new_len, new_table))
        queue.finish()
        want = best_of(logits, score, 1, beams, beams)
        token, source = outs[1].read(np.int32, (beams,)), outs[2].read(np.int32, (beams,))
        assert (token == want[1][0]).all() and (source == want[2][0]).all()
        score = outs[0].read(np.float32, (beams,))
        texts = [texts[s] for s in source]
        assert new_len.read(np.int32, (beams,)).tolist() == [len(t) for t in texts]
        table = new_table.read(np.int32, (beams, host.columns))
        used = -(-len(texts[0]) // PAGE)
        spare += sorted(set(range(PAGES)) - set(table[:, :used].ravel().tolist()) - set(spare))
        if len(texts[0]) % PAGE == 0:                     # a page for the next rows
            table[:, used] = [spare.pop(0) for _ in range(beams)]
        host.table.write(table)
        batch = host.batch([1] * beams, [len(t) + 1 for t in texts])
        dev, got = host.rotate(new_rows(rng, beams), [len(t) for t in texts])
        host.write(batch, dev, got.shape[1])
        out = host.attend(batch, dev, got.shape[1])
        for b in range(beams):
            texts[b] = np.concatenate([texts[b], got[b:b + 1]])
            near(out[b], *attention_of(kind, got[b, :HEADS * D], texts[b]))
