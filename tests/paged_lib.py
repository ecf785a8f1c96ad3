"""A paged cache and its sequences for the tests, and what write, read and attention have to give, in 64 bits."""
import numpy as np

from helpers import mil

NAN = 0x7e00                                          # an fp16 NaN


def quantise(kind, x):
    """fp16 rows [..., D] -> (stored codes, fp16 scales), by the definition in 64 bits."""
    if kind == mil.KV_F16:
        return x, None
    size, top, most = (x.shape[-1], 127, 515.5) if kind == mil.KV_INT8 else (32, 7, 9352.0)
    f = x.astype(np.float64).reshape(*x.shape[:-1], x.shape[-1] // size, size)
    finite = np.isfinite(f).all(-1, keepdims=True)
    f = np.where(finite, f, 0.0)
    scale = np.minimum(np.abs(f).max(-1, keepdims=True) / top, most).astype(np.float16)
    wide = scale.astype(np.float64)
    code = np.clip(np.rint(np.divide(f, wide, out=np.zeros_like(f), where=wide > 0)), -127 if top == 127 else -8, top)
    code = code.reshape(x.shape).astype(np.int32)
    scale = np.where(finite, scale, np.float16(np.nan))[..., 0]
    if kind == mil.KV_INT8:
        return code.astype(np.int8), scale[..., 0]
    u = (code + 8).astype(np.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4), scale


def values(kind, code, scale):
    """What stored rows stand for, fp16."""
    if kind == mil.KV_F16:
        return code
    if kind == mil.KV_Q4:
        wide = np.empty((*code.shape[:-1], code.shape[-1] * 2), np.float64)
        wide[..., 0::2], wide[..., 1::2] = (code & 15).astype(np.float64) - 8, (code >> 4).astype(np.float64) - 8
        each = np.repeat(scale.astype(np.float64), 32, -1)
    else:
        wide, each = code.astype(np.float64), scale.astype(np.float64)[..., None]
    with np.errstate(invalid="ignore"):
        return (wide * each).astype(np.float16)


class Cache:
    """Sequences of `lengths` positions whose last `new` are the batch's rows, in pages handed out in a random order.  What no
    sequence has written is NaN all over: pages of nobody, the rest of last pages, scales."""

    columns = 0                                       # of the page table, in positions: at least that many (the tail is not used)

    def __init__(self, kind, heads, kv_heads, D, page, lengths, new, seed=0, pad=0, spare=3, max_pages=None, sigma=1.0, gap=0):
        rng = np.random.default_rng(seed)
        self.kind, self.heads, self.kv, self.D, self.page = kind, heads, kv_heads, D, page
        self.lengths, self.new = list(lengths), list(new)
        self.k = [(rng.standard_normal((n, kv_heads, D)) * sigma).astype(np.float16) for n in lengths]
        self.v = [(rng.standard_normal((n, kv_heads, D)) * sigma).astype(np.float16) for n in lengths]
        used = [-(-n // page) for n in lengths]
        self.n_pages = sum(used) + spare
        self.max_pages = max_pages or max(max(used), 1, self.columns // page)
        order, at = rng.permutation(self.n_pages), 0
        self.table = np.full((len(lengths), self.max_pages), -1, np.int32)
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.rows = sum(new) + pad
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.ld = (heads + 2 * kv_heads) * D + gap                   # rows of q | k | v side by side
        self.qkv = np.full((self.rows, self.ld), np.nan, np.float16)
        self.qkv[:, :heads * D] = (rng.standard_normal((self.rows, heads * D)) * sigma).astype(np.float16)
        for b in range(len(lengths)):
            if self.new[b]:
                n, m, s = self.new[b], self.lengths[b], self.start[b]
                w = kv_heads * D
                self.qkv[s:s + n, heads * D:heads * D + w] = self.k[b][m - n:].reshape(n, w)
                self.qkv[s:s + n, heads * D + w:heads * D + 2 * w] = self.v[b][m - n:].reshape(n, w)
        self.fill()

    def fill(self):
        """The pools on the host, from self.k and self.v."""
        shape = (self.n_pages, self.kv, self.page)
        row = {mil.KV_F16: (np.uint16, self.D, NAN), mil.KV_INT8: (np.int8, self.D, -1), mil.KV_Q4: (np.uint8, self.D // 2, 255)}
        dtype, width, fill = row[self.kind]
        scales = {mil.KV_F16: None, mil.KV_INT8: shape, mil.KV_Q4: (*shape, self.D // 32)}[self.kind]
        self.pool = {n: np.full((*shape, width), fill, dtype) for n in "kv"}
        self.scale = {n: None if scales is None else np.full(scales, NAN, np.uint16) for n in "kv"}
        for b, m in enumerate(self.lengths):
            for name, rows in (("k", self.k[b]), ("v", self.v[b])):
                code, scale = quantise(self.kind, rows)
                p = np.arange(m)
                pages, slots = self.table[b][p // self.page], p % self.page
                self.pool[name][pages, :, slots] = code.view(np.uint16) if self.kind == mil.KV_F16 else code
                if scale is not None:
                    self.scale[name][pages, :, slots] = scale.view(np.uint16)

    # ---- on the device

    def upload(self):
        buf = mil.Buffer.from_host
        self.dev = {n: buf(self.pool[n]) for n in "kv"}
        self.dev_scale = {n: None if self.scale[n] is None else buf(self.scale[n]) for n in "kv"}
        self.cache = mil.KVCache(self.kind, self.n_pages, self.page, self.kv, self.D, self.dev["k"], self.dev["v"],
                                 self.dev_scale["k"], self.dev_scale["v"])
        self.dev_len = buf(np.array(self.lengths, np.int32))
        self.dev_table, self.dev_start = buf(self.table), buf(self.start)
        self.batch = mil.KVBatch(len(self.lengths), self.rows, max(self.new + [0]), self.max_pages, self.dev_start, self.dev_len,
                                 self.dev_table)
        self.dev_qkv = buf(self.qkv)
        return self

    def read_pools(self):
        return ({n: self.dev[n].read(self.pool[n].dtype, self.pool[n].shape) for n in "kv"},
                {n: None if self.scale[n] is None else self.dev_scale[n].read(np.uint16, self.scale[n].shape) for n in "kv"})

    def attend(self, queue, window=0, sinks=0, scale=None, ld_out=0, before=0x1234):
        """mi_attention's rows, [rows, heads, D]; `before`: what the output holds ahead of the call."""
        width = self.heads * self.D
        ld = ld_out or width
        out = mil.Buffer.from_host(np.full((self.rows, ld), before, np.uint16))
        call = mil.AttentionCall(self.cache, self.batch, self.heads, self.dev_qkv, out, ld_q=self.ld, ld_out=ld, scale=scale,
                                 window=window, sinks=sinks)
        assert mil.attention(queue, call)
        queue.finish()
        got = out.read(np.uint16, (self.rows, ld))
        assert (got[:, width:] == before).all(), "written beside the rows"
        assert (got[sum(self.new):] == before).all(), "padding rows written"
        return got[:, :width].copy().view(np.float16).reshape(self.rows, self.heads, self.D)

    # ---- the definition

    def expect(self, window=0, sinks=0, scale=None):
        """(rows, how far an output may be off), both [rows of sequences, heads, D] in 64 bits.

        What an output is off by, at most: half a step of fp16 (2^-11 of it) for its own rounding, 2^-11 of the weighted mean of |v|
        twice for the rounding of the weights, over and under the line, n weights that are too small for fp16 (below 2^-14
        when the greatest is 2^7 or more: 2^-25 each, relative to it 2^-32), and the scores' fp32 sums: a score that is off by e changes its
        weight by a factor 1 + e, and e <= D 2^-24 scale sum |q k| (<= 2^-12 for D = 128 and N(0, 1) values; taken as
        computed) + 2^-21 for the exponential."""
        scale = self.D ** -0.5 if scale is None else scale
        want, tol = np.zeros((sum(self.new), self.heads, self.D)), np.zeros((sum(self.new), self.heads, self.D))
        group = self.heads // self.kv
        for b, (n, m) in enumerate(zip(self.new, self.lengths)):
            if not n:
                continue
            k, v = (values(self.kind, *quantise(self.kind, x[b])).astype(np.float64) for x in (self.k, self.v))
            s = self.start[b]
            p, j = np.arange(m - n, m)[:, None], np.arange(m)[None]
            seen = j <= p
            if window > 0:
                seen &= (j > p - window) | (j < sinks)
            for h in range(self.heads):
                q = self.qkv[s:s + n, h * self.D:(h + 1) * self.D].astype(np.float64)
                kh, vh = k[:, h // group], v[:, h // group]
                with np.errstate(invalid="ignore"):
                    score = np.where(seen, q @ kh.T * scale, -np.inf)
                    size = np.where(seen, np.abs(q) @ np.abs(kh).T * scale, 0.0)
                top = score.max(1, keepdims=True)
                none = ~seen.any(1)
                w = np.exp(score - np.where(none[:, None], 0.0, top))
                total = np.where(none, 1.0, w.sum(1))[:, None]
                # (what no row sees must not count, whatever it holds)
                safe = np.where(seen.any(0)[:, None], vh, 0.0)
                if np.isfinite(safe).all():
                    out, mean = w @ safe / total, w @ np.abs(safe) / total
                else:
                    out, mean = np.empty((n, self.D)), np.empty((n, self.D))
                    for r in range(n):
                        out[r] = w[r, seen[r]] @ vh[seen[r]] / total[r]
                        mean[r] = w[r, seen[r]] @ np.abs(vh[seen[r]]) / total[r]
                off = 2.0 ** -21 + self.D * 2.0 ** -24 * np.nan_to_num(size, nan=0.0, posinf=0.0).max(1, keepdims=True)
                most = np.nan_to_num(np.abs(safe), nan=0.0, posinf=0.0).max(initial=0.0)
                want[s:s + n, h] = out
                tol[s:s + n, h] = 2.0 ** -11 * np.abs(out) + (2 * 2.0 ** -11 + 2 * off) * mean + m * 2.0 ** -31 * most + 2.0 ** -25
        return want, tol

    def check(self, got, window=0, sinks=0, scale=None, what="", rows=slice(None)):
        want, tol = (x[rows] for x in self.expect(window, sinks, scale))
        got = got[:sum(self.new)][rows].astype(np.float64)
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (what, int(bad.sum()), [int(x[0]) for x in np.nonzero(bad)], got[bad][:4], want[bad][:4], tol[bad][:4])
