"""What the paged key/value cache and the attention over it are measured by: calls that a program makes which serves
many conversations at once, over the range of caches, head layouts and lengths of such programs.

`listed()` names twelve cases, `draw(rng)` makes another one of the same ranges, `prepare(case, seed)` what the program
has in hand before the call (a pool of pages in use, the page tables, new rows), `run(state)` is one pass, `exact` the
result in 64 bits, `work` what a pass cannot do without.  With `own` false, `run` is the plain form.

Kinds of case:

  write      new rows of keys and values go into their pages, and are quantised on the way.  Returned: the pool (fp16), or
             the new rows read back out of it (int8, Q4), as the values that the codes stand for.
  read       the last rows of every sequence out of their pages, as contiguous fp16 rows: what a host does that hands a
             conversation on, or runs another attention over it.
  attention  the queries of every sequence's new tokens against its cache, the new tokens' own rows included: one new
             token each is a decode step, more are a chunk of a prompt.  `window` > 0: a query sees that many positions
             up to its own, and the first `sinks` ones.

The cache holds, per token and key/value head, `width` values: fp16; int8 codes with an fp16 scale (amax / 127); or 4-bit
codes with an fp16 scale for each 32 (amax / 7), two to a byte, the even element in the low half, stored plus 8.  A value is
the fp16 number nearest to code * scale.  Pools are [pages, kv_heads, page, row], scales [pages, kv_heads, page(, width / 32)].
"""
import importlib
import math
import random

import torch

own = False

ALONE = dict(seqs=1, spread=0, window=0, sinks=0)


def _case(kind, cache, heads, kv_heads, width, page, new, length, **more):
    return dict(dict(ALONE, kind=kind, cache=cache, heads=heads, kv_heads=kv_heads, width=width, page=page, new=new,
                     length=length), **more)


def listed():
    return [
        # the second dozen of tokens of a conversation that is alone on the card: latency is all of it
        dict(_case("attention", "f16", 14, 2, 64, 16, 1, 24), name="step_f16_one"),
        # a decode step of a batch of conversations of a 0.5B model, up to 4096 positions, of all lengths
        dict(_case("attention", "int8", 14, 2, 64, 64, 1, 4096, seqs=32, spread=1), name="step_int8_32"),
        # eight long documents being answered, wide heads: the most bytes
        dict(_case("attention", "f16", 32, 8, 128, 128, 1, 32768, seqs=8, spread=2), name="step_f16_long"),
        # an odd number of conversations of a 360M model in pages that end inside every tile
        dict(_case("attention", "q4", 15, 5, 64, 48, 1, 2500, seqs=61, spread=3), name="step_q4_odd"),
        # a long prompt at once
        dict(_case("attention", "f16", 14, 2, 64, 16, 2048, 2048), name="prompt_f16_2048"),
        # a next turn: a few hundred tokens behind what the conversation has in its cache
        dict(_case("attention", "int8", 14, 2, 64, 32, 300, 1200), name="turn_int8_300_at_900"),
        # chunks of some prompts and a single token of the other conversations in one batch, padded to a round size
        dict(_case("attention", "f16", 32, 8, 128, 16, 500, 3701, seqs=17, spread=4, mixed=True), name="mixed_f16_17"),
        # a decode step of a model with a window, far behind the window's length
        dict(_case("attention", "int8", 16, 8, 128, 64, 1, 8000, seqs=16, spread=5, window=1024, sinks=4),
             name="window_step_int8"),
        # a prompt of such a model, several windows long: the most operations
        dict(_case("attention", "f16", 32, 8, 128, 64, 4096, 4096, window=1000, sinks=5), name="window_prompt_f16_4096"),
        # a decode step's rows of sixteen conversations: latency
        dict(_case("write", "f16", 14, 2, 64, 16, 1, 900, seqs=16, spread=6), name="write_f16_step"),
        # a prompt's rows, quantised as they are written, and read back for an attention that wants them in fp16
        dict(_case("write", "int8", 32, 8, 128, 64, 2048, 2048), name="write_int8_2048"),
        # whole conversations handed on
        dict(_case("read", "q4", 32, 8, 128, 32, 8000, 8000, seqs=6, spread=7), name="read_q4_6"),
    ]


HEADS = ((14, 2, 64), (9, 3, 64), (15, 5, 64), (16, 8, 64), (12, 12, 64), (32, 8, 128), (16, 8, 128), (8, 1, 128))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "write", "read"])
    heads, kv_heads, width = rng.choice(HEADS)
    cache, page = rng.choice(["f16", "int8", "q4"]), rng.choice([16, 16, 32, 48, 64, 100, 128, 256])
    form = rng.choice(["step", "step", "chunk", "mixed"])
    seqs = _log_int(rng, 1, 64) if form == "step" else 1 if form == "chunk" else rng.randint(2, 17)
    length = _log_int(rng, 20, (16000 if form == "step" and seqs <= 16 else 4000) // (2 if kind == "read" else 1))
    new = 1 if form == "step" else rng.randint(2, min(length, 2048 if form == "chunk" else 500))
    case = _case(kind, cache, heads, kv_heads, width, page, length if kind == "read" else new, length, seqs=seqs,
                 spread=rng.randint(10, 1000))
    if form == "mixed":
        case["mixed"] = True
    if kind == "attention" and rng.random() < 0.35:
        case["window"], case["sinks"] = _log_int(rng, 16, 2000), rng.choice([0, 1, 4, 37])
    return case


def _lengths(case):
    """New tokens and positions (these included) of every sequence: the first as long as the case says, the others of all
    lengths from an eighth of it.  In a mixed batch three of four sequences have a single new token, and one is empty."""
    rng, new, length = random.Random(case["spread"]), [case["new"]], [case["length"]]
    for b in range(1, case["seqs"]):
        length.append(max(1, _log_int(rng, max(1, case["length"] // 8), case["length"])))
        n = case["new"] if not case.get("mixed") else rng.randint(1, case["new"]) if b % 4 == 0 else 1
        new.append(min(length[-1], n))
        if case.get("mixed") and b == 2:
            new[-1], length[-1] = 0, 0
    return new, length


def _rows(case):
    """Rows of the batch: in a mixed one the rows behind the last sequence fill it up to a multiple of 64."""
    n = sum(_lengths(case)[0])
    return (n + 63) // 64 * 64 if case.get("mixed") else n


# ---- the cache's number formats, in torch ------------------------------------------------------------------

def _blocks(case):
    """(values that share a scale, largest code) of a quantised cache."""
    return (case["width"], 127) if case["cache"] == "int8" else (32, 7)


def _encode(case, x):
    """fp16 rows [..., width] -> (codes as they are stored, scales)."""
    if case["cache"] == "f16":
        return x, None
    block, top = _blocks(case)
    f = x.float().unflatten(-1, (-1, block))
    scale = (f.abs().amax(-1, keepdim=True) / top).half()
    code = torch.where(scale > 0, torch.round(f / scale.float()), 0.0).clamp_(-127 if top == 127 else -8, top)
    code = code.flatten(-2)
    scale = scale.squeeze(-1)
    if case["cache"] == "int8":
        return code.to(torch.int8), scale.squeeze(-1)
    code = (code + 8).to(torch.uint8).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), scale


def _decode(case, code, scale):
    """The values that stored rows stand for, fp16."""
    if case["cache"] == "f16":
        return code
    if case["cache"] == "q4":
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2).to(torch.int16) - 8
        scale = scale.repeat_interleave(32, -1)
    else:
        scale = scale.unsqueeze(-1)
    return (code.float() * scale.float()).half()


# ---- what a program holds before the call ------------------------------------------------------------------

_queue = None


def _mil():
    return importlib.import_module("adreno-llms_amd")


def queue():
    """The program's one stream."""
    global _queue
    if _queue is None:
        mil = _mil()
        assert mil.lib().mi_init(0) == 1
        _queue = mil.Queue()
    return _queue


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    new, length = _lengths(case)
    seqs, heads, kv, width, page = case["seqs"], case["heads"], case["kv_heads"], case["width"], case["page"]
    used = [-(-n // page) for n in length]
    most = max(used)
    n_pages = sum(used) + 3
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").half()  # noqa: E731
    # the pool in use, every page of it: what other conversations left behind lies next to these
    state = dict(case=case, n_pages=n_pages)
    for name in ("k", "v"):
        code, scale = _encode(case, normal(n_pages, kv, page, width))
        state[name + "_pool"], state[name + "_scale"] = code.contiguous(), scale
    # pages in the order in which they were handed out over time; what a sequence does not have is -1
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    have = torch.arange(most, device="cuda")[None] < torch.tensor(used, device="cuda")[:, None]
    table = torch.full((seqs, most), -1, dtype=torch.int32, device="cuda")
    table[have] = order[:sum(used)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    rows = _rows(case)
    state.update(table=table, start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                 length=torch.tensor(length, dtype=torch.int32, device="cuda"))
    # queries, keys and values of the new tokens side by side, as one product with the stacked weights leaves them
    state["qkv"] = normal(rows, (heads + 2 * kv) * width)
    if case["kind"] == "attention":
        state["out"] = torch.zeros(rows, heads * width, dtype=torch.float16, device="cuda")
    else:
        state["k_out"], state["v_out"] = (torch.zeros(rows, kv * width, dtype=torch.float16, device="cuda") for _ in "kv")
    if own:      # the descriptors of the cache, the batch and the call: pointers and sizes
        mil, at = _mil(), lambda t: None if t is None else t.data_ptr()  # noqa: E731
        kind = {"f16": mil.KV_F16, "int8": mil.KV_INT8, "q4": mil.KV_Q4}[case["cache"]]
        cache = mil.KVCache(kind, n_pages, page, kv, width, at(state["k_pool"]), at(state["v_pool"]),
                            at(state["k_scale"]), at(state["v_scale"]))
        batch = mil.KVBatch(seqs, rows, max(new), most, at(state["start"]), at(state["length"]), at(table))
        state.update(cache=cache, batch=batch)
        if case["kind"] == "attention":
            state["call"] = mil.AttentionCall(cache, batch, heads, at(state["qkv"]), at(state["out"]),
                                              ld_q=state["qkv"].shape[1], scale=1.0 / math.sqrt(width),
                                              window=case["window"], sinks=case["sinks"])
        queue()
    torch.cuda.synchronize()
    return state


# ---- one pass --------------------------------------------------------------------------------------

def _places(state):
    """Of every row that belongs to a sequence: (row, page, row in the page)."""
    start, length, page = state["start"].long(), state["length"].long(), state["case"]["page"]
    row = torch.arange(state["qkv"].shape[0], device="cuda")
    b = torch.searchsorted(start, row, right=True) - 1
    inside = row < start[-1]
    row, b = row[inside], b[inside]
    at = length[b] - start[b + 1] + row
    return row, state["table"].long()[b, at // page], at % page


def _plain_read(state):
    """The new rows out of their pages, behind one another."""
    case = state["case"]
    row, pages, slot = _places(state)
    got = []
    for name in ("k", "v"):
        scale = state[name + "_scale"]
        out = torch.zeros_like(state[name + "_out"])
        out[row] = _decode(case, state[name + "_pool"][pages, :, slot],
                           None if scale is None else scale[pages, :, slot]).flatten(1)
        got.append(out)
    return got


def _plain_write(state):
    case = state["case"]
    q_width, kv_width = case["heads"] * case["width"], case["kv_heads"] * case["width"]
    row, pages, slot = _places(state)
    for name, at in (("k", q_width), ("v", q_width + kv_width)):
        new = state["qkv"][row, at:at + kv_width].unflatten(1, (case["kv_heads"], case["width"]))
        code, scale = _encode(case, new)
        state[name + "_pool"][pages, :, slot] = code
        if scale is not None:
            state[name + "_scale"][pages, :, slot] = scale


def _plain_attention(state):
    case, table, start, length = state["case"], state["table"].long(), state["start"].long(), state["length"].long()
    heads, kv, width, page = case["heads"], case["kv_heads"], case["width"], case["page"]
    rows, seqs = state["qkv"].shape[0], case["seqs"]
    # every sequence's keys and values as [sequence, kv head, position, width]
    pages = table.clamp(min=0)
    k, v = (_decode(case, state[n + "_pool"][pages], None if state[n + "_scale"] is None else state[n + "_scale"][pages])
            .float().transpose(1, 2).flatten(2, 3) for n in ("k", "v"))
    # queries as [sequence, kv head, (query head of it, new token), width], the shorter sequences padded
    most = case["new"]
    token = start[:-1, None] + torch.arange(most, device="cuda")
    there = torch.arange(most, device="cuda") < (start[1:] - start[:-1])[:, None]
    q = state["qkv"][:, :heads * width][token.clamp(max=rows - 1)].float()
    q = q.view(seqs, most, kv, heads // kv, width).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(width)).unflatten(2, (heads // kv, most))
    key = torch.arange(k.shape[2], device="cuda")
    mine = (length - start[1:])[:, None] + token                      # the new tokens' own positions
    seen = key <= mine[:, :, None]
    if case["window"]:
        seen &= (key > mine[:, :, None] - case["window"]) | (key < case["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.exp_()
    total = score.sum(-1)
    out = torch.matmul(score.flatten(2, 3), v).unflatten(2, (heads // kv, most))
    out /= total.clamp(min=1e-30)[..., None]
    out = out.permute(0, 3, 1, 2, 4).flatten(2)
    result = torch.zeros_like(state["out"])
    result[token[there]] = out[there].half()
    return result


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        mil = _mil()
        if kind == "attention":
            assert mil.attention(_queue, state["call"])
            return state["out"]
        if kind == "write":
            at = state["qkv"].data_ptr() + 2 * case["heads"] * case["width"]
            ld = state["qkv"].shape[1]
            assert mil.kv_write(_queue, state["cache"], state["batch"], at, at + 2 * case["kv_heads"] * case["width"], ld, ld)
            if case["cache"] == "f16":
                return state["k_pool"], state["v_pool"]
        assert mil.kv_read(_queue, state["cache"], state["batch"], state["k_out"].data_ptr(), state["v_out"].data_ptr())
        return state["k_out"], state["v_out"]
    if kind == "attention":
        return _plain_attention(state)
    if kind == "write":
        _plain_write(state)
        if case["cache"] == "f16":
            return state["k_pool"], state["v_pool"]
    return tuple(_plain_read(state))


# ---- what a pass cannot do without -----------------------------------------------------------------

def _row_bytes(case):
    """Bytes of one token's keys (or values) in the cache, all heads."""
    return case["kv_heads"] * {"f16": 2 * case["width"], "int8": case["width"] + 2,
                               "q4": case["width"] // 2 + 2 * (case["width"] // 32)}[case["cache"]]


def _seen(case, position):
    """Positions that a query at `position` sees."""
    if not case["window"]:
        return position + 1
    first = max(0, position - case["window"] + 1)
    return position + 1 - first + min(first, case["sinks"])


def work(case):
    new, length = _lengths(case)
    kv_width = case["kv_heads"] * case["width"]
    if case["kind"] != "attention":
        passes = 2 if case["kind"] == "write" and case["cache"] != "f16" else 1   # written, and read back
        return dict(bytes=passes * sum(new) * 2 * (2 * kv_width + _row_bytes(case)), flops=0)
    pairs = sum(_seen(case, p) for n, m in zip(new, length) for p in range(m - n, m))
    # rows of the cache that any of a sequence's queries sees
    rows = sum(min(m, _seen(case, m - n) + n - 1 if case["window"] else m) for n, m in zip(new, length) if n)
    return dict(bytes=rows * 2 * _row_bytes(case) + sum(new) * case["heads"] * case["width"] * 4,
                flops=4 * pairs * case["heads"] * case["width"])


# ---- the definition in 64 bits -----------------------------------------------------------------------

def _values(state, name, pages):
    """The cached values of whole pages [n, kv_heads, page, width] in 64 bits, each the nearest fp16 number to code * scale."""
    stored, cache = state[name + "_pool"][pages], state["case"]["cache"]
    if cache == "f16":
        return stored.double()
    scale = state[name + "_scale"][pages].double()
    if cache == "int8":
        return (stored.double() * scale[..., None]).half().double()
    low, high = (stored % 16).double() - 8, torch.div(stored, 16, rounding_mode="floor").double() - 8
    both = torch.empty(*stored.shape[:-1], 2 * stored.shape[-1], dtype=torch.float64, device="cuda")
    both[..., 0::2], both[..., 1::2] = low, high
    each = torch.arange(both.shape[-1], device="cuda") // 32
    return (both * scale[..., each]).half().double()


def _rounded(case, x):
    """What rows [..., width] become by being written and read."""
    size, top = (case["width"], 127) if case["cache"] == "int8" else (32, 7)
    parts = x.double().reshape(*x.shape[:-1], x.shape[-1] // size, size)
    scale = (parts.abs().max(-1).values / top).half().double()
    code = (parts / scale.clamp(min=2.0 ** -24)[..., None]).round().clamp(-127 if top == 127 else -8, top)
    return (code * scale[..., None]).half().double().reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    new, length = _lengths(case)
    heads, kv, width, page = case["heads"], case["kv_heads"], case["width"], case["page"]
    table, first = state["table"].tolist(), 0
    if case["kind"] == "write":
        got = []
        for name, shift in (("k", heads), ("v", heads + kv)):
            rows = state["qkv"].view(-1, heads + 2 * kv, width)[:, shift:shift + kv]
            if case["cache"] == "f16":
                whole, first = state[name + "_pool"].double(), 0
                for b in range(case["seqs"]):
                    for i in range(new[b]):
                        p = length[b] - new[b] + i
                        whole[table[b][p // page], :, p % page] = rows[first + i].double()
                    first += new[b]
                got.append(whole)
            else:
                back = torch.zeros(rows.shape[0], kv * width, dtype=torch.float64, device="cuda")
                back[:sum(new)] = _rounded(case, rows[:sum(new)]).reshape(sum(new), -1)
                got.append(back)
        return tuple(got)
    if case["kind"] == "read":
        outs = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (state["k_out"], state["v_out"])]
    else:
        outs = [torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")]
    for b in range(case["seqs"]):
        n, m = new[b], length[b]
        if not n:
            continue
        pages = torch.tensor(table[b][:-(-m // page)], device="cuda")
        k, v = (_values(state, name, pages).permute(1, 0, 2, 3).reshape(kv, -1, width)[:, :m] for name in "kv")
        if case["kind"] == "read":
            for out, t in zip(outs, (k, v)):
                out[first:first + n] = t[:, m - n:].permute(1, 0, 2).reshape(n, -1)
        else:
            q = state["qkv"][first:first + n, :heads * width].double().view(n, heads, width)
            p = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
            for h in range(heads):
                g = h // (heads // kv)
                s = (q[:, h] @ k[g].T / math.sqrt(width)).masked_fill(hidden, -math.inf)
                outs[0][first:first + n, h * width:(h + 1) * width] = torch.softmax(s, 1) @ v[g]
        first += n
    return tuple(outs) if case["kind"] == "read" else outs[0]
