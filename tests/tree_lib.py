"""Drafted tokens over a paged cache for the tests: trees, their masks, and what mi_attention_tree has to give, in 64 bits."""
import numpy as np

from helpers import mil
from paged_lib import Cache, quantise, values


def tree(rng, n, roots=1):
    """Parents of a random tree in drafting order; the first `roots` tokens have none."""
    return [-1 if i < roots else int(rng.integers(0, i)) for i in range(n)]


def ancestors(parents):
    """bool [n, n]: row i sees its ancestors and itself."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


class TreeCache(Cache):
    """`masks`: of every sequence bool [n, n], which of its new rows a row sees; by default random trees of ancestors.  `depths`: how far a
    row's place in the text lies behind the earlier positions."""

    def __init__(self, *args, masks=None, words=None, **more):
        super().__init__(*args, **more)
        rng = np.random.default_rng(more.get("seed", 0) + 77)
        self.masks = masks if masks is not None else [ancestors(tree(rng, n, roots=1 + (n > 5 and b % 2))) for b, n in enumerate(self.new)]
        self.depths = [np.maximum(m.sum(1) - 1, 0) for m in self.masks]
        self.words = words or max(1, -(-max(self.new + [1]) // 32))
        bits = np.zeros((self.rows, 32 * self.words), bool)
        self.position = np.full(self.rows, -5, np.int32)
        for b, (n, m) in enumerate(zip(self.new, self.masks)):
            w, s = min(n, bits.shape[1]), self.start[b]
            bits[s:s + n, :w] = m[:, :w]
            bits[s:s + n, n:] = True                      # (rows that the sequence does not have)
            self.position[s:s + n] = self.lengths[b] - n + self.depths[b]
        self.seen = np.packbits(bits.reshape(self.rows, self.words, 32), axis=2, bitorder="little").view(np.uint32)[..., 0]

    def attend(self, queue, window=0, sinks=0, scale=None, ld_out=0, before=0x1234):
        width = self.heads * self.D
        ld = ld_out or width
        out = mil.Buffer.from_host(np.full((self.rows, ld), before, np.uint16))
        held = mil.Buffer.from_host(np.ascontiguousarray(self.seen)), mil.Buffer.from_host(self.position)
        call = mil.AttentionCall(self.cache, self.batch, self.heads, self.dev_qkv, out, ld_q=self.ld, ld_out=ld, scale=scale, window=window,
                                 sinks=sinks)
        assert mil.attention_tree(queue, call, mil.TreeMask(held[0], self.words, held[1] if window > 0 else None))
        queue.finish()
        got = out.read(np.uint16, (self.rows, ld))
        assert (got[:, width:] == before).all(), "written beside the rows"
        assert (got[sum(self.new):] == before).all(), "padding rows written"
        return got[:, :width].copy().view(np.float16).reshape(self.rows, self.heads, self.D)

    def visible(self, b, window, sinks):
        n, m = self.new[b], self.lengths[b]
        seen = np.zeros((n, m), bool)
        j = np.arange(m - n)[None]
        place = np.clip(self.position[self.start[b]:self.start[b] + n], m - n, m - 1)[:, None]
        seen[:, :m - n] = (j > place - window) | (j < sinks) if window > 0 else True
        drafts = self.masks[b].copy()
        drafts[:, 32 * self.words:] = False
        seen[:, m - n:] = drafts
        return seen

    def expect(self, window=0, sinks=0, scale=None):
        """(rows, how far an output may be off): the roundings that Cache.expect counts."""
        scale = self.D ** -0.5 if scale is None else scale
        want, tol = np.zeros((sum(self.new), self.heads, self.D)), np.zeros((sum(self.new), self.heads, self.D))
        group = self.heads // self.kv
        for b, (n, m) in enumerate(zip(self.new, self.lengths)):
            if not n:
                continue
            k, v = (values(self.kind, *quantise(self.kind, x[b])).astype(np.float64) for x in (self.k, self.v))
            s, seen = self.start[b], self.visible(b, window, sinks)
            for h in range(self.heads):
                q = self.qkv[s:s + n, h * self.D:(h + 1) * self.D].astype(np.float64)
                for r in range(n):
                    at = np.nonzero(seen[r])[0]
                    if not len(at):
                        continue
                    kh, vh = k[at, h // group], v[at, h // group]
                    with np.errstate(invalid="ignore"):
                        score, size = kh @ q[r] * scale, np.abs(kh) @ np.abs(q[r]) * scale
                    w = np.exp(score - score.max())
                    out, mean = w @ vh / w.sum(), w @ np.abs(vh) / w.sum()
                    off = 2.0 ** -21 + self.D * 2.0 ** -24 * size.max()
                    want[s + r, h] = out
                    tol[s + r, h] = 2.0 ** -11 * np.abs(out) + (2 * 2.0 ** -11 + 2 * off) * mean + m * 2.0 ** -31 * np.abs(vh).max() + 2.0 ** -25
        return want, tol
