"""Steps of several new tokens and of very long caches, as cases to time and to compare.

Beside the decode step of one new token per sequence a server runs steps whose sequences bring several: the tokens that a
drafter proposes (a tree or a chain of them) and chunks of prompts.  Such a step needs its tables, slots and positions, the
residual's addition and norm between its linear layers, and an attention that lets each new token see the cache and its own
ancestors.  And where a cache is very long, a decoded token attends to the pages that a cheap bound on their scores selects.
`run` computes each in its plain form, elementary torch operations in 32 bits (64 where near equal scores are compared), or, where
`own` is true, with the package's calls.  Head and layer sizes are the 27B-class ones of this repository's benchmark (hidden
5120, intermediate 17408, 40 query and 8 key heads of 128) or generic.
"""
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
FP8_MAX = 448.0


def _package():
    path = os.path.join(_ROOT, "hyperqwen-rtx4080s32_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gguf_hip

    return gguf_hip


def listed():
    heads = {"hq": 40, "hkv": 8, "d": 128}
    return [
        # a batch of chats, each with a small drafted tree: the step's tables, before anything else of it can run
        {"name": "tables-32-trees", "op": "tables", "b": 32, "slots": 64, "width": 256, "len": 4000, "new": 16, "tree": True,
         "page": 16},
        # a full server: many chats and chunks of prompts, long page lists
        {"name": "tables-512-chunks", "op": "tables", "b": 512, "slots": 600, "width": 2048, "len": 30000, "new": 63, "tree": False,
         "page": 16},
        # between two layers, one new token: latency alone
        {"name": "add-norm-1", "op": "norm", "t": 1, "dim": 5120, "dtype": "bf16", "weight": "bf16", "eight": False, "group": 0,
         "offset": False},
        # a batch's drafted tokens, normalized into 8 bits with a scale for each 128 columns
        {"name": "add-norm-fp8-96", "op": "norm", "t": 96, "dim": 17408, "dtype": "bf16", "weight": "fp32", "eight": True,
         "group": 128, "offset": True},
        # a chunk of prompts
        {"name": "add-norm-8191", "op": "norm", "t": 8191, "dim": 5120, "dtype": "bf16", "weight": "bf16", "eight": False, "group": 0,
         "offset": False},
        # one chat, a chain of four drafted tokens behind a short context
        {"name": "draft-1x4", "op": "tree", "b": 1, "len": 500, "new": 4, "tree": False, **heads, "page": 16, "q": "bf16",
         "kv": "bf16", "window": 0, "layout": "heads"},
        # a batch of chats, a tree of drafted tokens each
        {"name": "tree-32x16", "op": "tree", "b": 32, "len": 4000, "new": 16, "tree": True, **heads, "page": 16, "q": "bf16",
         "kv": "bf16", "window": 0, "layout": "heads"},
        # a few long documents in 8-bit pages, wide trees
        {"name": "tree-4x61-fp8", "op": "tree", "b": 4, "len": 32768, "new": 61, "tree": True, **heads, "page": 64, "q": "bf16",
         "kv": "fp8", "window": 0, "layout": "heads"},
        # wide heads under a sliding window
        {"name": "tree-24x7-window", "op": "tree", "b": 24, "len": 7999, "new": 7, "tree": True, "hq": 32, "hkv": 4, "d": 256,
         "page": 32, "q": "fp16", "kv": "fp16", "window": 4096, "layout": "tokens"},
        # the second chunk of a long prompt
        {"name": "chunk-4096", "op": "tree", "b": 1, "len": 4096, "new": 4096, "tree": False, **heads, "page": 16, "q": "bf16",
         "kv": "bf16", "window": 0, "layout": "heads"},
        # one question about a very long document: 64 of its pages
        {"name": "sparse-1x131072", "op": "sparse", "b": 1, "len": 131072, "keep": 64, **heads, "page": 64, "q": "bf16", "kv": "bf16",
         "sink": 1, "recent": 2, "layout": "heads"},
        # a batch of long chats, a quarter of their pages each at most, 8-bit pages
        {"name": "sparse-48x16000-fp8", "op": "sparse", "b": 48, "len": 16000, "keep": 125, **heads, "page": 32, "q": "bf16",
         "kv": "fp8", "sink": 1, "recent": 4, "layout": "heads"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choices(("tables", "norm", "tree", "sparse"), (2, 3, 5, 3))[0]
    if op == "tables":
        b, page, tree = _log(rng, 1, 512), rng.choice((8, 16, 16, 48, 64)), rng.random() < 0.5
        length = _log(rng, 1, 30000)
        new = _log(rng, 1, max(2, min(256 if tree else 4096, 32256 // b, 4096 if not tree else 4096 // max(1, b // 8))))
        return {"op": op, "b": b, "slots": b + rng.randint(0, 100), "width": -(-(length + new) // page) + rng.randint(0, 20), "len": length,
                "new": new, "tree": tree, "page": page}
    if op == "norm":
        dim = rng.choice((5120, 17408, 8 * _log(rng, 8, 2048), _log(rng, 64, 17408)))
        dtype, eight = rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.4
        return {"op": op, "t": _log(rng, 1, max(2, min(8191, 8191 * 5120 // dim))), "dim": dim, "dtype": dtype,
                "weight": rng.choice((dtype, dtype, "fp32")), "eight": eight,
                "group": 128 if eight and dim % 128 == 0 and rng.random() < 0.5 else 0, "offset": rng.random() < 0.3}
    hkv, d, kv = rng.choice((1, 2, 4, 8, 8)), rng.choice((64, 80, 128, 128, 256)), rng.choice(("bf16", "bf16", "fp16", "fp8"))
    group, page = rng.choice((1, 2, 3, 5, 8, 16)), rng.choice((8, 16, 16, 32, 64, 48, 128))
    case = {"op": op, "hq": hkv * group, "hkv": hkv, "d": d, "page": page, "q": "fp16" if kv == "fp16" else "bf16", "kv": kv,
            "layout": rng.choice(("heads", "tokens"))}
    if op == "tree":
        tree = rng.random() < 0.6
        new = _log(rng, 1, 256 if tree else 4096)
        b = _log(rng, 1, max(1.5, min(64, 8192 / new)))
        # as many scores, and as many keys and values, as the largest case has
        most = min(40 * 4096 * 8192 * 128 // (b * new * hkv * group * d), (3 << 26) // (b * hkv * d * 2), 65536)
        length = _log(rng, 1, max(2, most - new))
        return {**case, "b": b, "len": length, "new": new, "tree": tree, "window": rng.choice((0, 0, 0, _log(rng, 2, 8192)))}
    b = _log(rng, 1, 64)
    length = _log(rng, 1, max(2, min(131072, (1 << 29) // (2 * b * hkv * d))))
    pages = -(-length // page)
    return {**case, "b": b, "len": length, "keep": max(4, min(_log(rng, 4, 256), pages)), "sink": rng.choice((0, 1, 1, 2)),
            "recent": rng.choice((1, 1, 2))}


# ---- inputs ----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _spread(top, b, least=1):
    """b numbers: the largest, then evenly down to a quarter of it."""
    return [max(least, top - i * (3 * top // 4) // b) for i in range(b)]


def _lengths(case):
    """Keys in the cache of each sequence before the step."""
    return _spread(case["len"], case["b"])


def _counts(case):
    """New tokens of each sequence; in a batch of many the last has none."""
    n = _spread(case["new"], case["b"])
    if case["b"] >= 8:
        n[-1] = 0
    return n


def _parents(counts, seed):
    """A drafted tree for each sequence: a token's parent is one of the few before it (-1: the last token of the cache)."""
    g = torch.Generator().manual_seed(seed)
    at = torch.cat([torch.arange(n) for n in counts]) if sum(counts) else torch.zeros(0, dtype=torch.long)
    back = 1 + (torch.rand(at.shape, generator=g) ** 2 * 4).long()
    return (at - back).clamp_min(-1).to(torch.int32)


def _bits(counts, parents, words):
    """Each token's ancestors and itself, as 32-bit words."""
    rows, t = [], 0
    for n in counts:
        seen = []
        for i in range(n):
            p = int(parents[t + i])
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows += seen
        t += n
    low = [[(r >> 32 * w) & 0xFFFFFFFF for w in range(words)] for r in rows]
    return torch.tensor(low, dtype=torch.int64).reshape(len(rows), words).to(torch.int32)


def _cache(case, gen, need):
    """Pages of one layer as [pages, tokens, heads, dim], in a random order, and the tables of the sequences."""
    count, width = sum(need) + 1, max(1, max(need))
    heads_first = case["layout"] == "heads"
    shape = (count, case["hkv"], case["page"], case["d"]) if heads_first else (count, case["page"], case["hkv"], case["d"])

    def plane():
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen).to(DTYPES[case["kv"]])
        return x.transpose(1, 2) if heads_first else x

    order = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    at = torch.cumsum(torch.tensor([0] + need[:-1]), 0).to("cuda")
    cols = torch.arange(width, device="cuda")
    have = cols[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(have, order[(at[:, None] + cols[None]).clamp(max=count - 1)], -1).to(torch.int32)
    scales = (None, None)
    if case["kv"] == "fp8":
        scales = tuple(0.5 + torch.rand(case["hkv"], device="cuda", generator=gen) for _ in range(2))
    return {"k": plane(), "v": plane(), "table": table, "k_scale": scales[0], "v_scale": scales[1]}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_tables(case, gen, seed):
    counts = _counts(case)
    tokens = -(-sum(counts) // 64) * 64                      # the rows of a captured step
    lists = torch.randint(0, 1 << 20, (case["slots"], case["width"]), device="cuda", generator=gen).to(torch.int32)
    requests = torch.randperm(case["slots"], device="cuda", generator=gen)[:case["b"]].to(torch.int32)
    parents = None
    if case["tree"]:
        parents = torch.full((tokens,), -1, dtype=torch.int32)
        parents[:sum(counts)] = _parents(counts, seed)
        parents = parents.cuda()
    return {"lists": lists, "requests": requests, "lens": _ints(_lengths(case)), "counts": _ints(counts), "parents": parents,
            "tokens": tokens}


def _prepare_norm(case, gen, seed):
    x, r = (torch.empty((case["t"], case["dim"]), dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen) for _ in range(2))
    w = torch.rand(case["dim"], device="cuda", generator=gen) + (0 if case["offset"] else 0.5)
    return {"x": x, "r": r * 4, "w": w if case["weight"] == "fp32" else w.to(DTYPES[case["weight"]])}


def _prepare_tree(case, gen, seed):
    lens, counts = _lengths(case), _counts(case)
    s = _cache(case, gen, [-(-(m + n) // case["page"]) for m, n in zip(lens, counts)])
    # normalized and weighted heads: scores of a few units, as a trained layer's
    q = 1.5 * torch.randn((sum(counts), case["hq"], case["d"]), device="cuda", generator=gen)
    starts = [sum(counts[:i]) for i in range(case["b"] + 1)]
    mask = _bits(counts, _parents(counts, seed), -(-case["new"] // 32)).cuda() if case["tree"] else None
    return {**s, "q": q.to(DTYPES[case["q"]]), "lens": _ints([m + n for m, n in zip(lens, counts)]), "starts": _ints(starts), "mask": mask,
            "max": max(m + n for m, n in zip(lens, counts))}


def _as_bytes(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x   # the type has no indexed writes of its own


def _prepare_sparse(case, gen, seed):
    lens = _lengths(case)
    s = _cache(case, gen, [-(-n // case["page"]) for n in lens])
    q = 1.5 * torch.randn((case["b"], case["hq"], case["d"]), device="cuda", generator=gen)
    # the bounds that the program keeps: of all pages but those that the step's new tokens are in
    k = s["k"].float()
    bounds = torch.stack([k.amin(1), k.amax(1)], 1).to(s["k"].dtype)
    last = torch.tensor([(n - 1) // case["page"] for n in lens], device="cuda")
    _as_bytes(bounds)[s["table"].long().gather(1, last[:, None])[:, 0]] = 0
    return {**s, "q": q.to(DTYPES[case["q"]]), "lens": _ints(lens), "bounds": bounds, "max": max(lens)}


_PREPARE = {"tables": _prepare_tables, "norm": _prepare_norm, "tree": _prepare_tree, "sparse": _prepare_sparse}


def prepare(case, seed):
    return {"case": dict(case), **_PREPARE[case["op"]](case, _gen(seed), seed)}


# ---- one pass --------------------------------------------------------------------------------

def _tables(s):
    """Every sequence's row of the page lists, every token's place, and the ancestors of a drafted token by powers of its
    tree's matrix."""
    c, tokens = s["case"], s["tokens"]
    lens, counts = s["lens"].long(), s["counts"].long()
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    total = lens + counts
    lists = s["lists"][s["requests"].long()]
    cols = torch.arange(c["width"], device="cuda")
    table = torch.where(cols[None] * c["page"] < total[:, None], lists, -1)
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    live = seq < c["b"]
    at = seq.clamp_max(c["b"] - 1)
    i = t - starts[at]
    place = lens[at] + i
    page = lists[at, (place // c["page"]).clamp_max(c["width"] - 1)].long()
    slots = torch.where(live, page * c["page"] + place % c["page"], -1)
    out = {"block_table": table, "lengths": total.to(torch.int32), "starts": starts.to(torch.int32), "slots": slots,
           "sequences": torch.where(live, seq, -1).to(torch.int32)}
    if not c["tree"]:
        return {**out, "positions": torch.where(live, place, 0).to(torch.int32)}
    n, words = c["new"], -(-c["new"] // 32)
    parent = s["parents"].long()
    step = torch.zeros((c["b"], n + 1, n + 1), dtype=torch.float64, device="cuda")
    step[at, torch.where(live, i, n), torch.where(live & (parent >= 0), parent, n)] = 1
    step[:, n] = 0
    own = torch.eye(n + 1, dtype=torch.float64, device="cuda")
    seen = torch.linalg.matrix_power(step + own, n)[:, :n, :n] > 0
    depth = seen.sum(-1) - 1
    seen = torch.nn.functional.pad(seen, (0, words * 32 - n)).unflatten(-1, (words, 32))
    bits = (seen << torch.arange(32, device="cuda")).sum(-1)
    row = i.clamp_max(n - 1)
    return {**out, "positions": torch.where(live, lens[at] + depth[at, row], 0).to(torch.int32),
            "mask": torch.where(live[:, None], bits[at, row], 0).to(torch.int32)}


def _norm(s):
    c = s["case"]
    x = s["x"].float() + s["r"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (s["w"].float() + (1.0 if c["offset"] else 0.0))
    if not c["eight"]:
        return {"out": y.to(s["x"].dtype), "residual": x.to(s["r"].dtype)}
    y = y.unflatten(1, (-1, c["group"] or c["dim"]))
    scale = y.abs().amax(-1, keepdim=True) / FP8_MAX
    out = (y / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return {"out": out.flatten(1), "scale": scale[..., 0], "residual": x.to(s["r"].dtype)}


def _softmax_sum(score, live, v):
    """The sum of the values under the softmax of the scores that are live; none: zeros."""
    score = score.masked_fill(~live, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _scaled(s, name, x):
    scale = s[name + "_scale"]
    return x.float() if scale is None else x.float() * scale[None, :, None, None]


def _tree(s):
    """Scores of every key of the padded batch, masked, their softmax, and the sum of the values."""
    c = s["case"]
    b, hq, hkv, d, n = c["b"], c["hq"], c["hkv"], c["d"], c["new"]
    table = s["table"].long().clamp_min(0)
    k, v = (_scaled(s, name, s[name][table].flatten(1, 2).permute(0, 2, 1, 3)) for name in ("k", "v"))   # [b, hkv, keys, d]
    keys = k.shape[2]
    starts, lens = s["starts"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device="cuda")
    has = i[None] < count[:, None]                           # [b, n]: the new tokens there are
    row = (starts[:-1, None] + i[None]).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[row].unflatten(2, (hkv, -1)).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d) * d ** -0.5
    at = torch.arange(keys, device="cuda")
    place = at[None] - (lens - count)[:, None]               # a key's number among the new ones
    if s["mask"] is None:
        live = place[:, None] <= i[None, :, None]
    else:
        bits = ((s["mask"][:, :, None] >> torch.arange(32, device="cuda")) & 1).flatten(1).bool()[row]   # [b, n, 32 words]
        live = bits.gather(2, place.clamp(0, bits.shape[2] - 1)[:, None].expand(b, n, keys)) | (place < 0)[:, None]
    live = live & (at[None] < lens[:, None])[:, None] & has[:, :, None]
    if c["window"]:                                          # of the keys that a token sees, the last ones
        live &= live.flip(2).cumsum(2).flip(2) <= c["window"]
    live = live[:, None, :, None].expand(b, 1, n, hq // hkv, keys).flatten(2, 3)
    out = _softmax_sum(q @ k.transpose(2, 3), live, v)
    out = out.reshape(b, hkv, n, -1, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    return out[has].to(s["q"].dtype)


def _sparse(s):
    """Bounds of the pages with new keys, a bound on each page's scores, the best pages and those always taken, attention
    over them."""
    c = s["case"]
    b, hkv, d, page = c["b"], c["hkv"], c["d"], c["page"]
    lens, table = s["lens"].long(), s["table"].long()
    pages = (lens + page - 1) // page
    last = table.gather(1, (pages - 1)[:, None])[:, 0]
    k = s["k"][last].float()
    have = (torch.arange(page, device="cuda")[None] < (lens - (pages - 1) * page)[:, None])[:, :, None, None]
    lo, hi = k.masked_fill(~have, float("inf")).amin(1), k.masked_fill(~have, float("-inf")).amax(1)
    _as_bytes(s["bounds"])[last] = _as_bytes(torch.stack([lo, hi], 1).to(s["bounds"].dtype))
    near = s["bounds"].float()[table.clamp_min(0)].double()  # [b, pages, 2, hkv, d]
    q = s["q"].double().unflatten(1, (hkv, -1))
    score = (q.clamp_min(0) @ near[:, :, 1].permute(0, 2, 3, 1).contiguous()
             + q.clamp_max(0) @ near[:, :, 0].permute(0, 2, 3, 1).contiguous()).amax(2)   # [b, hkv, pages]
    at = torch.arange(table.shape[1], device="cuda")[None]
    taken = (at < c["sink"]) | (at >= (pages - c["recent"])[:, None])
    score = score.masked_fill(taken[:, None], float("inf")).masked_fill((at >= pages[:, None])[:, None], float("-inf"))
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    best = torch.where(best < pages[:, None, None], best, table.shape[1]).sort(-1).values
    some = best < table.shape[1]
    chosen = torch.where(some, table[:, None].expand(b, hkv, -1).gather(2, best.clamp_max(table.shape[1] - 1)), -1)
    short = torch.where(pages > c["keep"], lens - (pages - c["keep"]) * page, lens)
    index = chosen.clamp_min(0)
    h = torch.arange(hkv, device="cuda")[None, :, None]
    k, v = (_scaled(s, name, s[name][index, :, h].flatten(2, 3)) for name in ("k", "v"))   # [b, hkv, keys, d]
    live = (torch.arange(k.shape[2], device="cuda")[None] < short[:, None])[:, None, None]
    out = _softmax_sum(s["q"].float().unflatten(1, (hkv, -1)) * d ** -0.5 @ k.transpose(2, 3), live, v)
    if best.shape[2] < c["keep"]:
        chosen = torch.nn.functional.pad(chosen, (0, c["keep"] - best.shape[2]), value=-1)
    return {"out": out.flatten(1, 2).to(s["q"].dtype), "table": chosen.to(torch.int32), "lengths": short.to(torch.int32),
            "bounds": s["bounds"]}


_PLAIN = {"tables": _tables, "norm": _norm, "tree": _tree, "sparse": _sparse}


def _own(s):
    g, c = _package(), s["case"]
    if c["op"] == "tables":
        t = g.step_tables(s["lists"], s["requests"], s["lens"], s["counts"], s["tokens"], c["page"], parents=s["parents"],
                          tree=c["new"] if c["tree"] else 0)
        out = {"block_table": t.block_table, "lengths": t.lengths, "starts": t.starts, "slots": t.slots, "sequences": t.sequences,
               "positions": t.positions}
        return {**out, "mask": t.mask} if c["tree"] else out
    if c["op"] == "norm":
        if c["eight"]:
            out, scale, residual = g.add_rms_norm_fp8(s["x"], s["r"], s["w"], eps=1e-6, unit_offset=c["offset"], group=c["group"])
            return {"out": out, "scale": scale, "residual": residual}
        out, residual = g.add_rms_norm(s["x"], s["r"], s["w"], eps=1e-6, unit_offset=c["offset"])
        return {"out": out, "residual": residual}
    if c["op"] == "tree":
        return g.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["mask"], window=c["window"],
                                k_scale=s["k_scale"], v_scale=s["v_scale"], max_length=s["max"], max_tokens=c["new"])
    g.page_bounds(s["k"], s["table"], s["lens"], s["bounds"], count=1)
    table, lengths = g.select_pages(s["q"], s["bounds"], s["table"], s["lens"], c["keep"], c["page"], sink=c["sink"],
                                    recent=c["recent"], max_length=s["max"])
    out = g.paged_attention(s["q"], s["k"], s["v"], table, lengths, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"out": out, "table": table, "lengths": lengths, "bounds": s["bounds"]}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def work(case):
    if case["op"] == "tables":
        counts = _counts(case)
        tokens = -(-sum(counts) // 64) * 64
        pages = sum(-(-(m + n) // case["page"]) for m, n in zip(_lengths(case), counts))
        words = -(-case["new"] // 32) if case["tree"] else 0
        return {"bytes": 4 * (pages + case["b"] * (case["width"] + 6)) + tokens * (16 + 4 * words + (4 if case["tree"] else 0)), "flops": 0}
    if case["op"] == "norm":
        n = case["t"] * case["dim"]
        scales = 4 * n // (case["group"] or case["dim"]) if case["eight"] else 0
        return {"bytes": n * (6 + (1 if case["eight"] else 2)) + scales + case["dim"] * (4 if case["weight"] == "fp32" else 2), "flops": 6 * n}
    size = DTYPES[case["kv"]].itemsize
    if case["op"] == "tree":
        window = case["window"] or 1 << 40
        live = seen = tokens = 0
        for m, n in zip(_lengths(case), _counts(case)):
            tokens += n
            if n:
                seen += min(m + n, window + n - 1)
                # a tree's tokens see some of the new ones: a few, as its depth grows with the logarithm of its size at least
                live += sum(min(m + (i.bit_length() if case["tree"] else i), window) for i in range(1, n + 1))
        return {"bytes": 2 * seen * case["hkv"] * case["d"] * size + 4 * tokens * case["hq"] * case["d"], "flops": 4 * live * case["hq"] * case["d"]}
    kept = bounds = 0
    for n in _lengths(case):
        pages = -(-n // case["page"])
        bounds += pages if pages > case["keep"] else 0
        kept += n - max(0, pages - case["keep"]) * case["page"]
    return {"bytes": 2 * (bounds + kept) * case["hkv"] * case["d"] * size + 4 * case["b"] * case["hq"] * case["d"],
            "flops": 4 * (bounds + kept) * case["hq"] * case["d"]}


# ---- the same results in 64 bits, by the definitions -----------------------------------------

def _exact_norm(c, s):
    x = s["x"].double() + s["r"].double()
    y = x / ((x ** 2).sum(1, keepdim=True) / c["dim"] + 1e-6).sqrt() * (s["w"].double() + int(c["offset"]))
    if not c["eight"]:
        return {"out": y, "residual": x}
    parts = y.split(c["group"] or c["dim"], 1)
    scale = torch.stack([p.abs().max(1).values / FP8_MAX for p in parts], 1)
    return {"out": torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], 1), "scale": scale, "residual": x}


def _attend(q, k, v):
    """One head's query over its keys: [tokens, d], [keys, d]; rows of scores may hold -inf for what is not seen."""
    e = k @ q / q.shape[0] ** 0.5
    e = (e - e.max()).exp()
    return e @ v / e.sum()


def _head(s, name, rows, h):
    x = s[name][rows[0], rows[1], h].double()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"][h].double()


def _exact_tree(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, t = c["hq"] // c["hkv"], 0
    for b, (m, n) in enumerate(zip(_lengths(c), _counts(c))):
        if n == 0:
            continue
        at = torch.arange(m + n, device="cuda")
        rows = (s["table"][b].long()[at // c["page"]], at % c["page"])
        sees = torch.ones((n, m + n), dtype=torch.bool, device="cuda")
        if c["tree"]:
            words = s["mask"][t:t + n].long() & 0xFFFFFFFF
            j = torch.arange(n, device="cuda")
            sees[:, m:] = (words[:, j // 32] >> (j % 32)) % 2 == 1
        else:
            sees[:, m:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        if c["window"]:
            after = sees.sum(1, keepdim=True) - sees.cumsum(1)          # keys that a token sees behind a key
            sees &= after < c["window"]
        for h in range(c["hkv"]):
            k, v = _head(s, "k", rows, h), _head(s, "v", rows, h)
            for g in range(group):
                e = (s["q"][t:t + n, h * group + g].double() @ k.t() / c["d"] ** 0.5).masked_fill(~sees, -float("inf"))
                e = (e - e.max(1, keepdim=True).values).exp()
                out[t:t + n, h * group + g] = e @ v / e.sum(1, keepdim=True)
        t += n
    return out


def _exact_sparse(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, page = c["hq"] // c["hkv"], c["page"]
    for b, n in enumerate(_lengths(c)):
        pages = -(-n // page)
        table = s["table"][b, :pages].long()
        near = s["k"][table].double()                                    # [pages, tokens, heads, d]
        low, high = near.clone(), near
        low[-1, n - (pages - 1) * page:] = float("inf")
        high[-1, n - (pages - 1) * page:] = -float("inf")
        low, high = low.min(1).values, high.max(1).values
        for h in range(c["hkv"]):
            q = s["q"][b, h * group:(h + 1) * group].double()
            chosen = list(range(pages))
            if pages > c["keep"]:
                score = torch.maximum(q[:, None] * low[None, :, h], q[:, None] * high[None, :, h]).sum(2).max(0).values
                fixed = set(range(c["sink"])) | set(range(pages - c["recent"], pages))
                rest = [j for j in torch.argsort(score, descending=True, stable=True).tolist() if j not in fixed]
                chosen = sorted(fixed | set(rest[:c["keep"] - len(fixed)]))
            at = (torch.tensor(chosen, device="cuda")[:, None] * page + torch.arange(page, device="cuda")[None]).flatten()
            at = at[at < n]
            rows = (s["table"][b].long()[at // page], at % page)
            k, v = _head(s, "k", rows, h), _head(s, "v", rows, h)
            for g in range(group):
                out[b, h * group + g] = _attend(q[g], k, v)
    return {"out": out, "table": None, "lengths": None, "bounds": None}


def exact(case, seed):
    if case["op"] == "tables":   # whole numbers
        return None
    s = _PREPARE[case["op"]](case, _gen(seed), seed)
    return {"norm": _exact_norm, "tree": _exact_tree, "sparse": _exact_sparse}[case["op"]](case, s)
