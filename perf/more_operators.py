"""What serving several continuations of a sequence over one paged cache is measured by: rotary positions of new rows,
attention of a tree of drafted tokens, the accepted path kept in the cache, beam search's selection, and beams that go on
as copies of others.

`listed()` names twelve cases, `draw(rng)` makes another one of the same ranges, `prepare(case, seed)` what the program
has in hand before the call, `run(state)` is one pass, `exact` the result in 64 bits, `work` what a pass cannot do
without.  With `own` false, `run` is the plain form.

Kinds of case:

  rope     queries and keys of new rows, side by side as one product with the stacked weights leaves them, turned by their
           rows' positions.  `sections`: how many pairs of a head go by each axis of the position (time, height, width), or
           one entry for all of them.  `split` true: elements i and i + rot / 2 are a pair, false: 2 i and 2 i + 1.
  tree     the queries of drafted tokens that form a tree against the cache and against their ancestors (and themselves)
           among the drafts, whose keys and values lie behind the sequence's others.  `window` > 0: of the earlier positions
           a query sees those less than `window` before its own, and the first `sinks` ones.
  keep     of every sequence's drafts the accepted path moves to the positions behind the sequence, in all layers.
  select   of every group's beams, the best continuations: n_out of beams x vocab by score + log softmax(logits), the best
           first, ties to the lowest beam and token.
  reorder  every beam goes on as a copy of one of its group: whole pages shared, the rows of the last page copied into a page
           of its own, in all layers.
"""
import importlib
import math
import random

import torch

own = False


def _case(kind, **more):
    return dict({"rope": dict(tokens=1, heads=14, kv_heads=2, width=64, rot=64, sections="32", split=True, first=0),
                 "tree": dict(cache="f16", heads=14, kv_heads=2, width=64, page=64, seqs=1, nodes=16, length=1000, spread=0,
                              window=0, sinks=0),
                 "keep": dict(layers=24, kv_heads=2, width=64, page=16, seqs=16, nodes=24, length=200, spread=0),
                 "select": dict(groups=1, beams=4, vocab=151936, n_out=8),
                 "reorder": dict(layers=24, kv_heads=2, width=64, page=16, groups=4, beams=4, length=200, spread=0)}[kind],
                kind=kind, **more)


def listed():
    return [
        # one layer's rows of a decode step of sixteen conversations, far along: latency is all of it
        dict(_case("rope", tokens=16, first=1000000), name="rope_step_16"),
        # a prompt of text and pictures, wide heads, three axes: the most bytes of one layer's rows
        dict(_case("rope", tokens=4096, heads=32, kv_heads=8, width=128, rot=128, sections="16,24,24"), name="rope_pictures_4096"),
        # a conversation that is alone on the card, sixteen drafts ahead
        dict(_case("tree", nodes=16, length=900, page=16), name="tree_f16_one"),
        # a batch of conversations of a 0.5B model in int8, up to 4096 positions, two dozen drafts each
        dict(_case("tree", cache="int8", seqs=32, nodes=24, length=4096, spread=1), name="tree_int8_32"),
        # eight long documents, wide heads, sixty-four drafts each: the most bytes and operations
        dict(_case("tree", heads=32, kv_heads=8, width=128, page=128, seqs=8, nodes=64, length=16384, spread=2), name="tree_f16_long"),
        # an odd number of conversations of a 360M model in Q4, pages that end inside a tile, trees of all sizes, a window
        dict(_case("tree", cache="q4", heads=15, kv_heads=5, page=48, seqs=13, nodes=100, length=2500, spread=3, window=1024, sinks=4),
             name="tree_q4_window"),
        # what sixteen conversations accepted of their drafts, all layers of a 0.5B model: latency
        dict(_case("keep", spread=4), name="keep_16"),
        # many conversations and wide heads, long paths, half of the layers at a time: the most rows
        dict(_case("keep", layers=16, kv_heads=8, width=128, page=32, seqs=48, nodes=64, spread=5), name="keep_48_wide"),
        # four beams of one sequence
        dict(_case("select"), name="select_4"),
        # thirty-two groups of eight beams: the most logits
        dict(_case("select", groups=32, beams=8, n_out=16), name="select_32x8"),
        # four groups of four beams, small pages: latency
        dict(_case("reorder", spread=6), name="reorder_4x4"),
        # eight groups of six beams, wide heads, an odd page, half of the layers at a time: the most rows
        dict(_case("reorder", layers=16, kv_heads=8, width=128, page=100, groups=8, beams=6, length=300, spread=7),
             name="reorder_8x6_wide"),
    ]


HEADS = ((14, 2, 64), (9, 3, 64), (15, 5, 64), (16, 8, 64), (12, 12, 64), (32, 8, 128), (16, 8, 128), (8, 1, 128))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "tree", "tree", "tree", "keep", "select", "select", "reorder"])
    heads, kv_heads, width = rng.choice(HEADS)
    spread = rng.randint(10, 100000)
    if kind == "rope":
        rot = rng.choice([width, width, width // 2])
        half = rot // 2
        sections = rng.choice([str(half), f"{half // 4},{half // 8 * 3},{half // 8 * 3}", f"{half // 2},{half // 2}"])
        return _case(kind, tokens=_log_int(rng, 1, 4096), heads=heads, kv_heads=kv_heads, width=width, rot=rot, sections=sections,
                     split=rng.random() < 0.7, first=_log_int(rng, 1, 4000000))
    if kind == "tree":
        seqs = _log_int(rng, 1, 32)
        case = _case(kind, cache=rng.choice(["f16", "int8", "q4"]), heads=heads, kv_heads=kv_heads, width=width,
                     page=rng.choice([16, 16, 32, 48, 64, 100, 128]), seqs=seqs, nodes=_log_int(rng, 2, 128 if seqs <= 8 else 64),
                     length=_log_int(rng, 1, 16000 if seqs <= 8 else 4000), spread=spread)
        if rng.random() < 0.3:
            case["window"], case["sinks"] = _log_int(rng, 16, 2000), rng.choice([0, 1, 4, 37])
        return case
    page = rng.choice([16, 32, 48, 64, 100])
    if kind == "keep":
        return _case(kind, layers=_log_int(rng, 1, 16), kv_heads=kv_heads, width=width, page=page, seqs=_log_int(rng, 1, 48),
                     nodes=rng.randint(2, 64), length=rng.randint(1, 300), spread=spread)
    if kind == "select":
        beams = rng.randint(1, 10)
        return _case(kind, groups=_log_int(rng, 1, 24), beams=beams, vocab=rng.choice([151936, 65536, 49152, _log_int(rng, 64, 150000)]),
                     n_out=rng.choice([beams, 2 * beams]))
    return _case(kind, layers=_log_int(rng, 1, 16), kv_heads=kv_heads, width=width, page=page, groups=_log_int(rng, 1, 8),
                 beams=rng.randint(2, 6), length=rng.randint(1, 300), spread=spread)


# ---- the host's side of a batch ----------------------------------------------------------------------

def _tree_sizes(case):
    """Drafts and earlier positions of every sequence: the first as many as the case says, the others of all sizes."""
    rng, nodes, before = random.Random(case["spread"]), [case["nodes"]], [case["length"]]
    for _ in range(1, case["seqs"]):
        nodes.append(rng.randint(max(1, case["nodes"] // 4), case["nodes"]))
        before.append(_log_int(rng, max(1, case["length"] // 8), case["length"]))
    return nodes, before


def _tree_parents(rng, n):
    """A tree in the order in which its tokens were drafted, the first being the root."""
    return [-1] + [rng.randint(max(0, (i - 1) // 3 - 2), max(0, (i - 1) // 2)) for i in range(1, n)]


def _tree_rows(case):
    """Of every row: its parent's number among the sequence's drafts (-1: a root), and its depth."""
    rng, parents, depths = random.Random(case["spread"] + 1), [], []
    for n in _tree_sizes(case)[0]:
        p, d = _tree_parents(rng, n), []
        for i in range(n):
            d.append(0 if p[i] < 0 else d[p[i]] + 1)
        parents.append(p)
        depths.append(d)
    return parents, depths


def _paths(case):
    """Of every sequence the drafts that are accepted, from the root down: a few that lie where they belong already, the
    others behind all the places that the path will have."""
    rng, paths = random.Random(case["spread"] + 2), []
    for n in _tree_sizes(case)[0]:
        most = rng.randint(1, max(1, n // 4))
        stay = rng.randint(1, min(3, most))
        rest = sorted(rng.sample(range(most, n), min(most - stay, n - most)))
        paths.append(list(range(stay)) + rest)
    return paths


def _beam_sizes(case):
    """Positions of every beam (those of a group are of one length), and the beam that each goes on as a copy of."""
    rng, length, source = random.Random(case["spread"]), [], []
    for g in range(case["groups"]):
        n = case["length"] if g == 0 else rng.randint(max(1, case["length"] // 2), case["length"])
        length += [n] * case["beams"]
        source += [g * case["beams"] + rng.randrange(case["beams"]) for _ in range(case["beams"])]
    return length, source


def _page_tables(case, lengths, gen):
    """(pages in the pool, table, further pages): pages in the order in which they were handed out over time."""
    used = [-(-n // case["page"]) for n in lengths]
    most, total = max(used), sum(used)
    n_pages = total + len(lengths) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    have = torch.arange(most, device="cuda")[None] < torch.tensor(used, device="cuda")[:, None]
    table = torch.full((len(lengths), most), -1, dtype=torch.int32, device="cuda")
    table[have] = order[:total]
    return n_pages, table, order[total:total + len(lengths)].contiguous()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(n):
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    return start


# ---- the cache's number formats, in torch ------------------------------------------------------------------

def _encode(case, x):
    """fp16 rows [..., width] -> (codes as they are stored, scales)."""
    if case["cache"] == "f16":
        return x, None
    size, top = (case["width"], 127) if case["cache"] == "int8" else (32, 7)
    f = x.float().unflatten(-1, (-1, size))
    scale = (f.abs().amax(-1, keepdim=True) / top).half()
    code = torch.where(scale > 0, torch.round(f / scale.float()), 0.0).clamp_(-127 if top == 127 else -8, top).flatten(-2)
    scale = scale.squeeze(-1)
    if case["cache"] == "int8":
        return code.to(torch.int8), scale.squeeze(-1).contiguous()
    code = (code + 8).to(torch.uint8).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), scale.contiguous()


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


def _at(t):
    return None if t is None else t.data_ptr()


def _positions(case):
    """Positions [axes, tokens]: text counts on along all axes; every third stretch of 256 rows is a picture 16 wide, whose
    rows have one time, and the line and column that they lie in."""
    axes = len(case["sections"].split(","))
    at = torch.arange(case["tokens"], device="cuda")
    if axes == 1:
        return (at + case["first"]).to(torch.int32)[None].contiguous()
    stretch, inside = at // 256, at % 256
    picture = stretch % 3 == 2
    start = stretch * 256 + case["first"]
    place = [torch.where(picture, start, start + inside), torch.where(picture, start + inside // 16, start + inside),
             torch.where(picture, start + inside % 16, start + inside)]
    return torch.stack(place[-axes:]).to(torch.int32).contiguous()


def _axis_of_pair(case):
    return [a for a, n in enumerate(case["sections"].split(",")) for _ in range(int(n))]


def _prepare_rope(case, gen):
    heads, kv, width, rot = case["heads"], case["kv_heads"], case["width"], case["rot"]
    state = dict(qkv=torch.randn(case["tokens"], (heads + 2 * kv) * width, generator=gen, device="cuda").half(),
                 position=_positions(case),
                 inv_freq=1e6 ** (torch.arange(rot // 2, device="cuda", dtype=torch.float32) * (-2.0 / rot)),
                 q=torch.zeros(case["tokens"], heads * width, dtype=torch.float16, device="cuda"),
                 k=torch.zeros(case["tokens"], kv * width, dtype=torch.float16, device="cuda"))
    state["axis"] = torch.tensor(_axis_of_pair(case), device="cuda")
    if own:
        ld = state["qkv"].shape[1]
        state["call"] = _mil().RopeCall(case["tokens"], heads, kv, width, rot, _at(state["inv_freq"]), _at(state["position"]),
                                        q=_at(state["qkv"]), q_out=_at(state["q"]), k=_at(state["qkv"]) + 2 * heads * width,
                                        k_out=_at(state["k"]), ld_q=ld, ld_k=ld, axis=_axis_of_pair(case),
                                        interleaved=not case["split"])
    return state


def _prepare_tree(case, gen):
    nodes, before = _tree_sizes(case)
    parents, depths = _tree_rows(case)
    heads, kv, width, page, seqs = case["heads"], case["kv_heads"], case["width"], case["page"], case["seqs"]
    n_pages, table, _ = _page_tables(case, [n + m for n, m in zip(nodes, before)], gen)
    rows, words = sum(nodes), (max(nodes) + 31) // 32
    state = dict(n_pages=n_pages, table=table, start=_ints(_starts(nodes)), length=_ints([n + m for n, m in zip(nodes, before)]))
    for name in ("k", "v"):
        code, scale = _encode(case, torch.randn(n_pages, kv, page, width, generator=gen, device="cuda").half())
        state[name + "_pool"], state[name + "_scale"] = code.contiguous(), scale
    state["q"] = torch.randn(rows, heads * width, generator=gen, device="cuda").half()
    state["out"] = torch.zeros_like(state["q"])
    bits, position = [], []
    for p, d, m in zip(parents, depths, before):
        seen = []
        for i, up in enumerate(p):
            seen.append((seen[up] if up >= 0 else 0) | 1 << i)
        bits += [[x >> (32 * w) & 0xffffffff for w in range(words)] for x in seen]
        position += [m + x for x in d]
    state["seen"] = torch.tensor(bits, dtype=torch.int64, device="cuda").to(torch.int32)
    state["position"] = _ints(position)
    if own:
        mil = _mil()
        kind = {"f16": mil.KV_F16, "int8": mil.KV_INT8, "q4": mil.KV_Q4}[case["cache"]]
        cache = mil.KVCache(kind, n_pages, page, kv, width, _at(state["k_pool"]), _at(state["v_pool"]), _at(state["k_scale"]),
                            _at(state["v_scale"]))
        batch = mil.KVBatch(seqs, rows, max(nodes), table.shape[1], _at(state["start"]), _at(state["length"]), _at(table))
        state["call"] = mil.AttentionCall(cache, batch, heads, _at(state["q"]), _at(state["out"]), window=case["window"],
                                          sinks=case["sinks"])
        state["tree"] = mil.TreeMask(_at(state["seen"]), words, _at(state["position"]))
    return state


def _layers(case, n_pages, gen):
    """The pools of all layers, keys and values, fp16: what lies in the pages does not matter to a copy."""
    return [torch.randn(n_pages, case["kv_heads"], case["page"], case["width"], generator=gen, device="cuda").half()
            for _ in range(2 * case["layers"])]


def _caches(case, n_pages, pools):
    mil = _mil()
    return mil.KVCaches([mil.KVCache(mil.KV_F16, n_pages, case["page"], case["kv_heads"], case["width"], _at(pools[2 * i]), _at(pools[2 * i + 1]))
                         for i in range(case["layers"])])


def _prepare_keep(case, gen):
    nodes, before = _tree_sizes(case)
    paths = _paths(case)
    n_pages, table, _ = _page_tables(case, [n + m for n, m in zip(nodes, before)], gen)
    start = _starts(nodes)
    keep = torch.full((start[-1],), -1, dtype=torch.int32)
    for s, p in zip(start, paths):
        keep[s:s + len(p)] = torch.tensor(p, dtype=torch.int32)
    state = dict(pools=_layers(case, n_pages, gen), table=table, start=_ints(start), keep=keep.cuda(),
                 length=_ints([n + m for n, m in zip(nodes, before)]), kept=_ints([len(p) for p in paths]),
                 new_length=torch.zeros(case["seqs"], dtype=torch.int32, device="cuda"))
    if own:
        state["caches"] = _caches(case, n_pages, state["pools"])
        state["batch"] = _mil().KVBatch(case["seqs"], start[-1], max(nodes), table.shape[1], _at(state["start"]), _at(state["length"]),
                                        _at(table))
    return state


def _prepare_select(case, gen):
    rows, vocab = case["groups"] * case["beams"], case["vocab"]
    logits = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5).half()
    # some tokens that a grammar or a list of words forbids, and sums of log probabilities of some dozen tokens so far
    logits[:, torch.randint(vocab, (max(1, vocab // 50),), generator=gen, device="cuda")] = -math.inf
    score = -20.0 + torch.randn(rows, generator=gen, device="cuda")
    shape = (case["groups"], case["n_out"])
    state = dict(logits=logits, score=score, out_score=torch.zeros(shape, device="cuda"),
                 out_token=torch.zeros(shape, dtype=torch.int32, device="cuda"), out_row=torch.zeros(shape, dtype=torch.int32, device="cuda"))
    if own:
        state["call"] = _mil().BeamCall(case["groups"], case["beams"], vocab, case["n_out"], _at(logits), _at(score),
                                        _at(state["out_score"]), _at(state["out_token"]), _at(state["out_row"]))
    return state


def _prepare_reorder(case, gen):
    length, source = _beam_sizes(case)
    n_pages, table, fresh = _page_tables(case, length, gen)
    state = dict(pools=_layers(case, n_pages, gen), table=table, fresh=fresh, length=_ints(length), source=_ints(source),
                 new_table=torch.zeros_like(table), new_length=torch.zeros(len(length), dtype=torch.int32, device="cuda"))
    if own:
        state["caches"] = _caches(case, n_pages, state["pools"])
        state["call"] = _mil().ReorderCall(len(length), table.shape[1], _at(state["length"]), _at(table), _at(state["source"]),
                                           _at(fresh), _at(state["new_length"]), _at(state["new_table"]))
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = globals()["_prepare_" + case["kind"]](case, gen)
    state["case"] = case
    if own:
        queue()
    torch.cuda.synchronize()
    return state


# ---- one pass --------------------------------------------------------------------------------------

def _plain_rope(state):
    case = state["case"]
    heads, kv, width, rot = case["heads"], case["kv_heads"], case["width"], case["rot"]
    angle = state["position"].double()[state["axis"]].T * state["inv_freq"].double()      # [tokens, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = state["qkv"][:, :(heads + kv) * width].view(case["tokens"], heads + kv, width).float()
    if case["split"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    turned = (a * cos - b * sin, b * cos + a * sin)
    both = torch.cat(turned, -1) if case["split"] else torch.stack(turned, -1).flatten(-2)
    out = torch.cat((both, x[..., rot:]), -1).half().flatten(1)
    return out[:, :heads * width].contiguous(), out[:, heads * width:].contiguous()


def _plain_tree(state):
    case, table, start, length = state["case"], state["table"].long(), state["start"].long(), state["length"].long()
    heads, kv, width, seqs, most = case["heads"], case["kv_heads"], case["width"], case["seqs"], case["nodes"]
    rows = state["q"].shape[0]
    # every sequence's keys and values as [sequence, kv head, position, width]
    pages = table.clamp(min=0)
    k, v = (_decode(case, state[n + "_pool"][pages], None if state[n + "_scale"] is None else state[n + "_scale"][pages])
            .float().transpose(1, 2).flatten(2, 3) for n in ("k", "v"))
    # queries as [sequence, kv head, (query head of it, draft), width], the smaller trees padded
    count = start[1:] - start[:-1]
    row = start[:-1, None] + torch.arange(most, device="cuda")
    there = torch.arange(most, device="cuda") < count[:, None]
    row = row.clamp(max=rows - 1)
    q = state["q"][row].float().view(seqs, most, kv, heads // kv, width).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(width)).unflatten(2, (heads // kv, most))
    key = torch.arange(k.shape[2], device="cuda")
    base = (length - count)[:, None, None]
    own_place = state["position"].long()[row][:, :, None]
    seen = key.expand(seqs, most, -1) < base
    if case["window"]:
        seen = seen & ((key > own_place - case["window"]) | (key < case["sinks"]))
    draft = key - base                                                       # [sequence, 1, position]
    word = state["seen"].long()[row].gather(2, (draft // 32).clamp(0, state["seen"].shape[1] - 1).expand(-1, most, -1))
    seen = seen | ((draft >= 0) & (draft < count[:, None, None]) & ((word >> (draft % 32)) & 1).bool())
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.exp_()
    total = score.sum(-1)
    out = torch.matmul(score.flatten(2, 3), v).unflatten(2, (heads // kv, most))
    out /= total.clamp(min=1e-30)[..., None]
    out = out.permute(0, 3, 1, 2, 4).flatten(2)
    result = torch.zeros_like(state["out"])
    result[row[there]] = out[there].half()
    return result


def _plain_keep(state):
    case, start = state["case"], state["start"].long()
    kept, keep, page = state["kept"].long(), state["keep"].long(), case["page"]
    row = torch.arange(keep.shape[0], device="cuda")
    b = torch.searchsorted(start, row, right=True) - 1
    i = row - start[b]
    moved = i < kept[b]
    b, i, frm = b[moved], i[moved], keep[moved]
    base = state["length"].long()[b] - (start[b + 1] - start[b])
    table = state["table"].long()
    src, dst = table[b, (base + frm) // page], table[b, (base + i) // page]
    src_slot, dst_slot = (base + frm) % page, (base + i) % page
    for pool in state["pools"]:
        pool[dst, :, dst_slot] = pool[src, :, src_slot]
    state["new_length"].copy_(state["length"] - (start[1:] - start[:-1]) + kept)
    return (state["new_length"], *state["pools"])


def _plain_select(state):
    case, logits = state["case"], state["logits"].double()
    groups, beams, vocab, n_out = case["groups"], case["beams"], case["vocab"], case["n_out"]
    most = logits.amax(1, keepdim=True)
    total = logits - most - (logits - most).exp().sum(1, keepdim=True).log() + state["score"].double()[:, None]
    total = total.view(groups, beams * vocab)
    border = torch.topk(total, n_out, 1).values[:, -1:]
    group, flat = torch.nonzero(total >= border, as_tuple=True)              # all that may be chosen, in order of beam and token
    value = total[group, flat]
    order = torch.sort(value, descending=True, stable=True).indices
    order = order[torch.sort(group[order], stable=True).indices]
    group, flat, value = group[order], flat[order], value[order]
    nth = torch.arange(group.shape[0], device="cuda") - torch.searchsorted(group, group)
    chosen = nth < n_out
    flat, value = flat[chosen].view(groups, n_out), value[chosen].view(groups, n_out)
    row = flat // vocab + beams * torch.arange(groups, device="cuda")[:, None]
    return value.float(), (flat % vocab).int(), row.int()


def _plain_reorder(state):
    case, length, source, page = state["case"], state["length"].long(), state["source"].long(), state["case"]["page"]
    n, seqs = length[source], length.shape[0]
    table = state["table"][source].clone()
    full, tail = n // page, n % page
    copied = (tail > 0) & (source != torch.arange(seqs, device="cuda"))
    b = torch.nonzero(copied).flatten()
    frm, to = state["table"].long()[source[b], full[b]], state["fresh"].long()[b]
    table[b, full[b]] = state["fresh"][b]
    inside = torch.arange(page, device="cuda") < tail[b, None]
    which, slot = torch.nonzero(inside, as_tuple=True)
    for pool in state["pools"]:
        pool[to[which], :, slot] = pool[frm[which], :, slot]
    state["new_table"].copy_(table)
    state["new_length"].copy_(n)
    return (state["new_length"], state["new_table"], *state["pools"])


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return globals()["_plain_" + kind](state)
    mil = _mil()
    if kind == "rope":
        assert mil.rope(_queue, state["call"])
        return state["q"], state["k"]
    if kind == "tree":
        assert mil.attention_tree(_queue, state["call"], state["tree"])
        return state["out"]
    if kind == "keep":
        assert mil.kv_keep(_queue, state["caches"], state["batch"], _at(state["keep"]), _at(state["kept"]), _at(state["new_length"]))
        return (state["new_length"], *state["pools"])
    if kind == "select":
        assert mil.beam_select(_queue, state["call"])
        return state["out_score"], state["out_token"], state["out_row"]
    assert mil.kv_reorder(_queue, state["caches"], state["call"])
    return (state["new_length"], state["new_table"], *state["pools"])


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rope":
        row = (case["heads"] + case["kv_heads"]) * case["width"]
        return dict(bytes=case["tokens"] * (4 * row + 4 * len(case["sections"].split(","))) + 2 * case["rot"],
                    flops=case["tokens"] * (case["heads"] + case["kv_heads"]) * 3 * case["rot"])
    if kind == "select":
        rows = case["groups"] * case["beams"]
        return dict(bytes=rows * (2 * case["vocab"] + 4) + 12 * case["groups"] * case["n_out"], flops=4 * rows * case["vocab"])
    row = case["kv_heads"] * case["width"] * 2
    if kind == "keep":
        moved = sum(1 for p in _paths(case) for i, x in enumerate(p) if x != i)
        return dict(bytes=4 * case["layers"] * moved * row + 12 * case["seqs"] + 4 * sum(map(len, _paths(case))), flops=0)
    if kind == "reorder":
        length, source = _beam_sizes(case)
        rows = sum(length[s] % case["page"] for b, s in enumerate(source) if b != s)
        pages = sum(-(-length[s] // case["page"]) for s in source)
        return dict(bytes=4 * case["layers"] * rows * row + 8 * pages + 16 * len(length), flops=0)
    row = case["kv_heads"] * {"f16": 2 * case["width"], "int8": case["width"] + 2,
                              "q4": case["width"] // 2 + case["width"] // 16}[case["cache"]]
    nodes, before = _tree_sizes(case)
    parents, depths = _tree_rows(case)
    cached = keys = 0
    for n, m, p, d in zip(nodes, before, parents, depths):
        first = [max(0, m + x - case["window"] + 1) if case["window"] else 0 for x in d]     # of each row's window
        cached += n + m - min(first) + min(min(first), case["sinks"])
        # (a window of less than the depth would leave out all earlier positions; the ancestors it leaves in)
        keys += sum(m - min(f, m) + min(f, case["sinks"], m) + x + 1 for f, x in zip(first, d))
    return dict(bytes=2 * cached * row + sum(nodes) * case["heads"] * case["width"] * 4, flops=4 * keys * case["heads"] * case["width"])


# ---- the definition in 64 bits -----------------------------------------------------------------------

def _exact_rope(case, state):
    rot, width, heads = case["rot"], case["width"], case["heads"]
    axis = state["axis"].tolist()
    x = state["qkv"].double().view(case["tokens"], -1, width)[:, :heads + case["kv_heads"]]
    out = x.clone()
    for i in range(rot // 2):
        turn = state["position"][axis[i]].double() * float(state["inv_freq"][i])
        a, b = (i, i + rot // 2) if case["split"] else (2 * i, 2 * i + 1)
        c, s = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
        out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        out[:, :, b] = x[:, :, a] * s + x[:, :, b] * c
    return out[:, :heads].flatten(1), out[:, heads:].flatten(1)


def _exact_tree(case, state):
    nodes, before = _tree_sizes(case)
    parents, depths = _tree_rows(case)
    heads, kv, width, page = case["heads"], case["kv_heads"], case["width"], case["page"]
    table, out = state["table"].tolist(), torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")

    def values(name, pages):
        stored = state[name + "_pool"][pages]
        if case["cache"] == "f16":
            return stored.double()
        scale = state[name + "_scale"][pages].double()
        if case["cache"] == "int8":
            return (stored.double() * scale[..., None]).half().double()
        both = torch.empty(*stored.shape[:-1], width, dtype=torch.float64, device="cuda")
        both[..., 0::2], both[..., 1::2] = (stored % 16).double() - 8, torch.div(stored, 16, rounding_mode="floor").double() - 8
        return (both * scale[..., torch.arange(width, device="cuda") // 32]).half().double()

    first = 0
    for b, (n, m) in enumerate(zip(nodes, before)):
        pages = torch.tensor(table[b][:-(-(n + m) // page)], device="cuda")
        k, v = (values(name, pages).permute(1, 0, 2, 3).reshape(kv, -1, width)[:, :n + m] for name in "kv")
        hidden = torch.zeros(n, n + m, dtype=torch.bool)
        for i in range(n):
            if case["window"]:
                end = min(max(m + depths[b][i] - case["window"] + 1, 0), m)
                hidden[i, min(case["sinks"], end):end] = True
            hidden[i, m:] = True
            j = i
            while j >= 0:
                hidden[i, m + j] = False
                j = parents[b][j]
        hidden = hidden.cuda()
        q = state["q"][first:first + n].double().view(n, heads, width)
        for h in range(heads):
            g = h // (heads // kv)
            s = (q[:, h] @ k[g].T / math.sqrt(width)).masked_fill(hidden, -math.inf)
            out[first:first + n, h * width:(h + 1) * width] = torch.softmax(s, 1) @ v[g]
        first += n
    return out


def _exact_keep(case, state):
    nodes, before = _tree_sizes(case)
    page, table = case["page"], state["table"].tolist()
    result = [torch.tensor([m + len(p) for m, p in zip(before, _paths(case))], dtype=torch.int32, device="cuda")]
    moves = [(table[b][(m + x) // page], (m + x) % page, table[b][(m + i) // page], (m + i) % page)
             for b, (m, p) in enumerate(zip(before, _paths(case))) for i, x in enumerate(p)]
    src, src_slot, dst, dst_slot = (torch.tensor(x, device="cuda") for x in zip(*moves))
    for pool in state["pools"]:
        new = pool.clone()
        new[dst, :, dst_slot] = pool[src, :, src_slot]
        result.append(new)
    return tuple(result)


def _exact_select(case, state):
    scores, tokens, rows = [], [], []
    for g in range(case["groups"]):
        best = []
        for r in range(g * case["beams"], (g + 1) * case["beams"]):
            x = state["logits"][r].double()
            x = x - torch.logsumexp(x, 0) + state["score"][r].double()
            some = min(4 * case["n_out"], x.shape[0])
            values = torch.topk(x, some).values
            for t in torch.nonzero(x >= values[min(case["n_out"], some) - 1]).flatten().tolist():
                best.append((-x[t].item(), r, t))
        best.sort()
        scores.append([-s for s, _, _ in best[:case["n_out"]]])
        rows.append([r for _, r, _ in best[:case["n_out"]]])
        tokens.append([t for _, _, t in best[:case["n_out"]]])
    return torch.tensor(scores, dtype=torch.float64, device="cuda"), _ints(tokens), _ints(rows)


def _exact_reorder(case, state):
    length, source = _beam_sizes(case)
    page, table, fresh = case["page"], state["table"].tolist(), state["fresh"].tolist()
    new_table, copies = [], []
    for b, s in enumerate(source):
        line = list(table[s])
        if b != s and length[s] % page:
            line[length[s] // page] = fresh[b]
            copies.append((table[s][length[s] // page], fresh[b], length[s] % page))
        new_table.append(line)
    pools = []
    for pool in state["pools"]:
        new = pool.clone()
        for frm, to, rows in copies:
            new[to, :, :rows] = pool[frm, :, :rows]
        pools.append(new)
    return (_ints([length[s] for s in source]), _ints(new_table), *pools)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
