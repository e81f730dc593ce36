"""The decode step around the GGUF linear path, as cases to time and to compare.

A server that multiplies by GGUF weights does four more things with their outputs in every decoder layer: it adds the
low-rank adapters of the requests in the batch to a projection, it normalizes and rotates the heads of queries and keys
and stores keys and values into the pages of its cache, it attends from each new token over those pages, and between
steps it copies pages (a fork of a prompt, a compaction).  `run` computes each in its plain form, elementary torch
operations in 32 bits, or, where `own` is true, with the package's call.  Head and layer sizes are the 27B-class ones
of this repository's benchmark (hidden 5120, intermediate 17408, a 7168-row qkv: 40 query and 8 key heads of 128) or
generic.
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
        # the first tokens of one chat: latency alone
        {"name": "attend-1x61", "op": "attend", "b": 1, "len": 61, **heads, "page": 16, "q": "bf16", "kv": "bf16", "window": 0,
         "layout": "heads"},
        # a batch of chats of many lengths, one of them not begun
        {"name": "attend-32x4000", "op": "attend", "b": 32, "len": 4000, **heads, "page": 16, "q": "bf16", "kv": "bf16",
         "window": 0, "layout": "heads"},
        # one question about a very long document, its cache in 8 bits
        {"name": "attend-1x131072-fp8", "op": "attend", "b": 1, "len": 131072, **heads, "page": 64, "q": "bf16", "kv": "fp8",
         "window": 0, "layout": "heads"},
        # a large batch with a sliding window and wide heads, pages that hold a token's heads side by side
        {"name": "attend-96x7999-window", "op": "attend", "b": 96, "len": 7999, "hq": 32, "hkv": 4, "d": 256, "page": 32,
         "q": "fp16", "kv": "fp16", "window": 4096, "layout": "tokens"},
        # one new token: its heads normalized, rotated and stored
        {"name": "norm-rope-1", "op": "rope", "t": 1, **heads, "rot": 128, "interleaved": False, "dtype": "bf16", "page": 16,
         "kv": "bf16", "keep_k": False, "unit_offset": False, "prefill": False},
        # a batch of new tokens, half of each head rotated in interleaved pairs, into an 8-bit cache
        {"name": "norm-rope-64-fp8", "op": "rope", "t": 64, **heads, "rot": 64, "interleaved": True, "dtype": "bf16", "page": 16,
         "kv": "fp8", "keep_k": False, "unit_offset": True, "prefill": False},
        # a chunk of prompts: the keys are also kept beside the pages
        {"name": "norm-rope-8191", "op": "rope", "t": 8191, **heads, "rot": 128, "interleaved": False, "dtype": "bf16",
         "page": 16, "kv": "bf16", "keep_k": True, "unit_offset": False, "prefill": True},
        # copy on write of a few shared pages, one for each fork of a prompt
        {"name": "copy-pages-3", "op": "copy", "planes": 32, "pages": 128, "copies": 3, "page_bytes": 32768},
        # compaction of a cache of 64 layers after many requests ended
        {"name": "copy-pages-400", "op": "copy", "planes": 128, "pages": 1024, "copies": 400, "page_bytes": 16384},
        # one chat with an adapter, beside the qkv projection
        {"name": "adapters-qkv-1", "op": "adapters", "m": 1, "k": 5120, "n": "5120,1024,1024", "rank": 16, "slots": 4, "used": 1,
         "dtype": "bf16", "prefill": False},
        # a batch of chats with many adapters (one in eight rows without any), beside gate_up
        {"name": "adapters-gate_up-48", "op": "adapters", "m": 48, "k": 5120, "n": "17408,17408", "rank": 32, "slots": 16,
         "used": 12, "dtype": "bf16", "prefill": False},
        # prompts of three requests, beside the long-K projection
        {"name": "adapters-down-4096", "op": "adapters", "m": 4096, "k": 17408, "n": "5120", "rank": 64, "slots": 8, "used": 3,
         "dtype": "bf16", "prefill": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choices(("attend", "rope", "copy", "adapters"), (4, 3, 2, 3))[0]
    if op == "attend":
        hkv = rng.choice((1, 2, 4, 8, 8))
        d = rng.choice((64, 80, 128, 128, 256))
        kv = rng.choice(("bf16", "bf16", "fp16", "fp8"))
        size = 1 if kv == "fp8" else 2
        b = _log(rng, 1, 128)
        length = _log(rng, 1, max(2, min(131072, (1 << 30) // (2 * b * hkv * d * size))))
        return {"op": op, "b": b, "len": length, "hq": hkv * rng.choice((1, 2, 3, 5, 8, 16)), "hkv": hkv, "d": d,
                "page": rng.choice((8, 16, 16, 32, 64, 48, 128)), "q": "fp16" if kv == "fp16" else "bf16", "kv": kv,
                "window": rng.choice((0, 0, 0, _log(rng, 16, 8192))), "layout": rng.choice(("heads", "tokens"))}
    if op == "rope":
        hkv = rng.choice((1, 2, 4, 8))
        d = rng.choice((64, 80, 128, 128, 256))
        hq = hkv * rng.choice((1, 2, 5, 8))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        t = _log(rng, 1, max(2, min(8191, 8191 * 48 * 128 // ((hq + hkv) * d))))
        return {"op": op, "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rng.choice((d, d, d // 2 // 16 * 16 or 16)),
                "interleaved": rng.random() < 0.3, "dtype": dtype, "page": rng.choice((8, 16, 16, 48, 64)),
                "kv": rng.choice((dtype, dtype, "fp8")), "keep_k": rng.random() < 0.3, "unit_offset": rng.random() < 0.3,
                "prefill": t > 256}
    if op == "copy":
        planes, page_bytes = rng.choice((2, 32, 64, 128)), 16 * _log(rng, 64, 2048)
        pages = max(4, min(4096, (2 << 30) // (planes * page_bytes)))
        return {"op": op, "planes": planes, "pages": pages, "copies": _log(rng, 1, max(2, pages * 2 // 5)), "page_bytes": page_bytes}
    m = _log(rng, 1, 4096)
    slots = _log(rng, 1, 32)
    k, n = rng.choice(((5120, (5120, 1024, 1024)), (5120, (17408, 17408)), (17408, (5120,)),
                       (8 * _log(rng, 64, 1024), (_log(rng, 100, 8192),)),
                       (8 * _log(rng, 64, 1024), (_log(rng, 100, 4096), _log(rng, 100, 4096)))))
    m = max(1, min(m, 4096 * 22528 // (k + 2 * sum(n))))
    return {"op": op, "m": m, "k": k, "n": ",".join(map(str, n)), "rank": rng.choice((8, 16, 16, 32, 64, 128 if m < 1024 else 64)),
            "slots": slots, "used": rng.randint(1, slots), "dtype": rng.choice(("bf16", "bf16", "fp16")), "prefill": m > 256}


# ---- inputs ----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """Tokens in the cache of each sequence: the longest, then evenly down to a quarter of it; in a batch of many the
    last has none."""
    b, top = case["b"], case["len"]
    lens = [max(1, top - i * (3 * top // 4) // b) for i in range(b)]
    if b >= 8:
        lens[-1] = 0
    return lens


def _pages(case, gen, count, kv):
    """A cache's pages of one layer, as [pages, tokens, heads, dim]."""
    shape = (count, case["hkv"], case["page"], case["d"]) if case.get("layout", "heads") == "heads" else (
        count, case["page"], case["hkv"], case["d"])
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen).to(DTYPES[kv])
    return x.transpose(1, 2) if case.get("layout", "heads") == "heads" else x


def _prepare_attend(case, gen):
    lens = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in lens]
    width = max(1, max(need))
    count = sum(need) + 1
    order = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    at = torch.cumsum(torch.tensor([0] + need[:-1]), 0).to("cuda")
    cols = torch.arange(width, device="cuda")
    have = cols[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(have, order[(at[:, None] + cols[None]).clamp(max=count - 1)], 0).to(torch.int32)
    # normalized and weighted heads: scores of a few units, as a trained layer's
    q = 1.5 * torch.randn((case["b"], case["hq"], case["d"]), device="cuda", generator=gen)
    scales = (None, None)
    if case["kv"] == "fp8":
        scales = tuple(0.5 + torch.rand(case["hkv"], device="cuda", generator=gen) for _ in range(2))
    return {"q": q.to(DTYPES[case["q"]]), "k": _pages(case, gen, count, case["kv"]), "v": _pages(case, gen, count, case["kv"]),
            "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "max": max(lens), "k_scale": scales[0],
            "v_scale": scales[1]}


def _prepare_rope(case, gen):
    t, hq, hkv, d, rot = (case[n] for n in ("t", "hq", "hkv", "d", "rot"))
    dtype = DTYPES[case["dtype"]]
    qkv = (2 * torch.randn((t, (hq + 2 * hkv) * d), device="cuda", generator=gen)).to(dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split((hq * d, hkv * d, hkv * d), 1))
    most = 32768
    angle = torch.arange(most, device="cuda")[:, None].double() / 4 * 1e6 ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)
    table = torch.cat([angle.cos(), angle.sin()], 1).float()
    if case["prefill"]:   # chunks of prompts: runs of positions
        pos = (torch.arange(t, device="cuda") + torch.randint(0, 8192, (1,), device="cuda", generator=gen)) % most
    else:
        pos = torch.randint(0, most, (t,), device="cuda", generator=gen)
    count = -(-t // case["page"]) + 2
    slots = torch.randperm(count * case["page"], device="cuda", generator=gen)[:t]
    weights = [(torch.rand(d, device="cuda", generator=gen) + (0 if case["unit_offset"] else 0.5)).to(dtype) for _ in range(2)]
    return {"q": q, "k": k, "v": v, "pos": pos, "table": table, "wq": weights[0], "wk": weights[1], "slots": slots,
            "k_pages": _pages(case, gen, count, case["kv"]), "v_pages": _pages(case, gen, count, case["kv"])}


def _prepare_copy(case, gen):
    words = case["page_bytes"] // 4
    pages = torch.empty((case["planes"], case["pages"], words), dtype=torch.int32, device="cuda").random_(generator=gen)
    order = torch.randperm(case["pages"], device="cuda", generator=gen).cpu()
    return {"pages": pages, "src": order[:case["copies"]].clone(), "dst": order[case["copies"]:2 * case["copies"]].clone()}


def _prepare_adapters(case, gen):
    m, k, rank, slots = (case[n] for n in ("m", "k", "rank", "slots"))
    n = [int(x) for x in case["n"].split(",")]
    dtype = DTYPES[case["dtype"]]
    rnd = lambda *shape: torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)  # noqa: E731
    which = torch.randperm(slots, device="cuda", generator=gen)[:case["used"]]
    if case["prefill"]:   # the prompts of a few requests, one after the other
        ids = which[torch.arange(m, device="cuda") * case["used"] // m]
    else:
        ids = which[torch.randint(0, case["used"], (m,), device="cuda", generator=gen)]
        ids[7::8] = -1
    return {"y": rnd(m, sum(n)), "x": rnd(m, k), "a": rnd(slots, len(n), rank, k) * k ** -0.5, "b": rnd(slots, sum(n), rank),
            "ids": ids.to(torch.int32), "scales": 0.25 + torch.rand(slots, device="cuda", generator=gen), "n": n}


_PREPARE = {"attend": _prepare_attend, "rope": _prepare_rope, "copy": _prepare_copy, "adapters": _prepare_adapters}


def prepare(case, seed):
    return {"case": dict(case), **_PREPARE[case["op"]](case, _gen(seed))}


# ---- one pass --------------------------------------------------------------------------------

def _attend(s):
    """Scores of every key of the padded batch, masked, their softmax, and the sum of the values."""
    c = s["case"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    table = s["table"].long()
    k, v = (s[n][table].flatten(1, 2).permute(0, 2, 1, 3).float() for n in ("k", "v"))      # [b, hkv, keys, d]
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][None, :, None, None], v * s["v_scale"][None, :, None, None]
    q = s["q"].float().reshape(b, hkv, hq // hkv, d) * d ** -0.5
    score = q @ k.transpose(2, 3)
    at = torch.arange(score.shape[-1], device=q.device)
    lens = s["lens"][:, None]
    live = at[None] < lens
    if c["window"]:
        live &= at[None] >= lens - c["window"]
    score = score.masked_fill(~live[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, hq, d).to(s["q"].dtype)


def _heads(x, weight, s):
    """RMS norm of each head and the rotation of its first `rot` dims, in 32 bits."""
    c = s["case"]
    rot = c["rot"]
    x, weight = x.float(), weight.float() + (1.0 if c["unit_offset"] else 0.0)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    cos, sin = s["table"][s["pos"]][:, None].chunk(2, -1)
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _store(pages, slots, x):
    if pages.dtype == torch.float8_e4m3fn:   # indexed writes as bytes: the type has none of its own
        x = x.float().clamp(-FP8_MAX, FP8_MAX).to(pages.dtype).view(torch.uint8)
        pages = pages.view(torch.uint8)
    page = pages.shape[1]
    pages[slots // page, slots % page] = x.to(pages.dtype)


def _rope(s):
    q, k = _heads(s["q"], s["wq"], s).to(s["q"].dtype), _heads(s["k"], s["wk"], s)
    _store(s["k_pages"], s["slots"], k)
    _store(s["v_pages"], s["slots"], s["v"])
    out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return {**out, "k": k.to(s["k"].dtype)} if s["case"]["keep_k"] else out


def _copy(s):
    s["pages"][:, s["dst"]] = s["pages"][:, s["src"]]
    return s["pages"]


def _adapters(s):
    """Each slot's products for every row, kept where the row's adapter is that slot: one product with all slots' A
    side by side, and one with all slots' B."""
    slots, parts, rank, k = s["a"].shape
    x = s["x"].float()
    h = (x @ s["a"].float().flatten(0, 2).t()).unflatten(1, (slots, parts, rank))
    mine = s["ids"][:, None] == torch.arange(slots, device=x.device)
    h = h * (mine * s["scales"])[:, :, None, None]
    start = [sum(s["n"][:i]) for i in range(parts)]
    b = s["b"].float()
    delta = [h[:, :, i].flatten(1) @ b[:, a:a + n].permute(0, 2, 1).flatten(0, 1) for i, (a, n) in enumerate(zip(start, s["n"]))]
    return (s["y"].float() + torch.cat(delta, 1)).to(s["y"].dtype)


_PLAIN = {"attend": _attend, "rope": _rope, "copy": _copy, "adapters": _adapters}


def _own(s):
    g, c = _package(), s["case"]
    if c["op"] == "attend":
        return g.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], window=c["window"], k_scale=s["k_scale"],
                                 v_scale=s["v_scale"], max_length=s["max"])
    if c["op"] == "rope":
        out_k = torch.empty_like(s["k"], memory_format=torch.contiguous_format) if c["keep_k"] else None
        q, k = g.qk_norm_rope(s["q"], s["k"], s["pos"], s["table"], s["wq"], s["wk"], eps=1e-6, unit_offset=c["unit_offset"],
                              interleaved=c["interleaved"], v=s["v"], k_pages=s["k_pages"], v_pages=s["v_pages"],
                              slots=s["slots"], out_k=out_k)
        out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        return {**out, "k": k} if c["keep_k"] else out
    if c["op"] == "copy":
        g.copy_pages(s["pages"], s["src"], s["dst"], dim=1)
        return s["pages"]
    return g.lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scales"], s["n"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def work(case):
    if case["op"] == "attend":
        live = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
        size = DTYPES[case["kv"]].itemsize
        return {"bytes": 2 * live * case["hkv"] * case["d"] * size + 4 * case["b"] * case["hq"] * case["d"],
                "flops": 4 * live * case["hq"] * case["d"]}
    if case["op"] == "rope":
        t, hq, hkv, d = (case[n] for n in ("t", "hq", "hkv", "d"))
        size = DTYPES[case["kv"]].itemsize
        return {"bytes": t * d * (4 * hq + 4 * hkv + 2 * hkv * size + (2 * hkv if case["keep_k"] else 0)) + t * 4 * case["rot"],
                "flops": 10 * t * d * (hq + hkv)}
    if case["op"] == "copy":
        return {"bytes": 2 * case["planes"] * case["copies"] * case["page_bytes"], "flops": 0}
    m, k, rank = case["m"], case["k"], case["rank"]
    n = [int(x) for x in case["n"].split(",")]
    used = min(case["used"], m)
    return {"bytes": 2 * (m * k + 2 * m * sum(n) + used * rank * (len(n) * k + sum(n))), "flops": 2 * m * rank * (len(n) * k + sum(n))}


# ---- the same results in 64 bits, by the definitions -----------------------------------------

def _exact_attend(c, s):
    out = torch.zeros((c["b"], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    group = c["hq"] // c["hkv"]
    one = torch.ones(c["hkv"], dtype=torch.float64, device="cuda")
    ks, vs = (one if s[n] is None else s[n].double() for n in ("k_scale", "v_scale"))
    for i, n in enumerate(_lengths(c)):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        page, slot = s["table"][i].long()[at // c["page"]], at % c["page"]
        for h in range(c["hkv"]):
            k, v = s["k"][page, slot, h].double() * ks[h], s["v"][page, slot, h].double() * vs[h]
            for g in range(group):
                e = (k * s["q"][i, h * group + g].double()).sum(-1) / c["d"] ** 0.5
                e = (e - e.max()).exp()
                out[i, h * group + g] = (e[:, None] * v).sum(0) / e.sum()
    return out


def _exact_heads(x, w, c, s):
    x = x.double()
    x = x / ((x ** 2).sum(-1, keepdim=True) / c["d"] + 1e-6).sqrt() * (w.double() + int(c["unit_offset"]))
    half = c["rot"] // 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    row = s["table"][s["pos"]].double()[:, None]
    turn = torch.complex(row[..., :half], row[..., half:]) * torch.complex(x[..., first], x[..., second])
    out = x.clone()
    out[..., first], out[..., second] = turn.real, turn.imag
    return out


def _exact_rope(c, s):
    q, k = _exact_heads(s["q"], s["wq"], c, s), _exact_heads(s["k"], s["wk"], c, s)
    out = {"q": q}
    for name, x in (("k", k), ("v", s["v"].double())):
        pages = s[name + "_pages"].double()
        pages[s["slots"] // c["page"], s["slots"] % c["page"]] = x.clamp(-FP8_MAX, FP8_MAX) if c["kv"] == "fp8" else x
        out[name + "_pages"] = pages
    return {**out, "k": k} if c["keep_k"] else out


def _exact_adapters(c, s):
    out = s["y"].double()
    for a in range(c["slots"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        col = 0
        for part, n in enumerate(s["n"]):
            if rows.numel():
                h = s["x"][rows].double() @ s["a"][a, part].double().t()
                out[rows, col:col + n] += s["scales"][a].double() * (h @ s["b"][a, col:col + n].double().t())
            col += n
    return out


def exact(case, seed):
    if case["op"] == "copy":   # bytes, moved
        return None
    s = _PREPARE[case["op"]](case, _gen(seed))
    return {"attend": _exact_attend, "rope": _exact_rope, "adapters": _exact_adapters}[case["op"]](case, s)
