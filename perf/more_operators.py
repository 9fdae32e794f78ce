"""Serving many sequences from one pool of pages: what is timed of it.

A layer's keys and values lie in pages of 16 to 256 tokens; a table [sequence, page] says which page of the pool holds
which part of a sequence. Four operators, each in its plain form (elementary torch operations on the pages' codes) and
as the calls that a user makes:

  store   new tokens are quantized into their pages, and read back as the fp16 values that the codes stand for
  attend  attention of a sequence's newest tokens (mostly one) over its pages, causal among them
  sparse  each KV head picks the pages whose bounds promise the largest scores for the new token, and attends those alone
  rope    rotary positions of several axes (time, height, width), a position of its own for each token and axis; rope_store
          rotates, stores the keys and values in their pages and reads them back

Page bounds: for each page and KV head, the least and the largest key of every dim, as 8-bit codes over the page's
largest magnitude, rounded outwards. With q as 8-bit codes over its group's largest magnitude, the bound of q . k is a
sum of whole numbers times that magnitude: both forms give the same pages.

Sizes: the package's own heads (24 over 4 of 256 dims, 32 over 8 of 128), contexts of up to 32k tokens, speculative
blocks of up to 8 rows, prompts of up to 32k tokens a call.
"""
import math

import numpy as np
import torch

own = False

GEOMETRIES = ((24, 4, 256), (16, 2, 256), (32, 8, 128), (24, 4, 128), (8, 8, 128), (12, 1, 256))
BITS = {"affine4": 4, "affine8": 8, "int8": 8, "fp16": 16}
MODES = tuple(BITS)
PAGES = (16, 32, 64, 128, 256)


def listed():
    g = {"hq": 24, "hkv": 4, "d": 256}
    s = {"hq": 32, "hkv": 8, "d": 128}
    return [
        # a decoding step of 33 chats: one token each, somewhere in a page
        {"name": "store_33x1", "op": "store", "mode": "affine4", "page": 16, "seqs": 33, "ctx": 4000, "new": 33, **s},
        # seven prompts of different lengths, some behind an earlier turn
        {"name": "store_7x6k", "op": "store", "mode": "affine8", "page": 64, "seqs": 7, "ctx": 3000, "new": 6001, **g},
        # a bulk prefill
        {"name": "store_5x64k", "op": "store", "mode": "int8", "page": 32, "seqs": 5, "ctx": 0, "new": 65536, **s},
        # one short conversation: latency and launches count
        {"name": "attend_1x513", "op": "attend", "mode": "affine8", "page": 16, "seqs": 1, "ctx": 513, "rows": 1, **s},
        # a batch of chats of very different lengths
        {"name": "attend_17x8k", "op": "attend", "mode": "affine4", "page": 64, "seqs": 17, "ctx": 8191, "rows": 1, **g},
        # speculative decoding over long contexts, 5 rows a sequence
        {"name": "attend_4x32k_rows5", "op": "attend", "mode": "int8", "page": 128, "seqs": 4, "ctx": 32768, "rows": 5, **g},
        # a full batch in fp16
        {"name": "attend_64x16k", "op": "attend", "mode": "fp16", "page": 32, "seqs": 64, "ctx": 16384, "rows": 1, **s},
        # one long chat of which an eighth is read
        {"name": "sparse_1x32k", "op": "sparse", "mode": "affine4", "page": 16, "seqs": 1, "ctx": 32768, "budget": 256, "sink": 1, "recent": 4, "rows": 1, **g},
        # a batch over documents
        {"name": "sparse_32x32k", "op": "sparse", "mode": "fp16", "page": 32, "seqs": 32, "ctx": 32768, "budget": 128, "sink": 1, "recent": 2, "rows": 1, **s},
        # a decoding step of 64 sequences, partial rotary, stored and read back
        {"name": "rope_store_64x1", "op": "rope_store", "mode": "affine8", "page": 64, "seqs": 64, "ctx": 2000, "new": 64, "rope": 64, "interleaved": True, **g},
        # a prompt with two images
        {"name": "rope_4k", "op": "rope", "new": 4099, "rope": 64, "interleaved": True, **g},
        # a video
        {"name": "rope_32k", "op": "rope", "new": 32768, "rope": 128, "interleaved": False, **s},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, d = rng.choice(GEOMETRIES)
    op = rng.choice(("store", "attend", "attend", "sparse", "rope", "rope_store"))
    c = {"op": op, "hq": hq, "hkv": hkv, "d": d}
    if op != "rope":
        c.update(mode=rng.choice(MODES), page=rng.choice(PAGES))
    if op in ("rope", "rope_store"):
        c.update(rope=rng.choice((32, 64, d)), interleaved=rng.random() < 0.5)
    if op in ("store", "rope_store"):
        seqs = _log(rng, 1, 100)
        c.update(seqs=seqs, ctx=rng.choice((0, _log(rng, 1, 4000))), new=max(seqs, _log(rng, 1, 32768)))
    elif op == "rope":
        c.update(new=_log(rng, 1, 32768))
    else:
        seqs = _log(rng, 1, 64)
        rows = rng.choice((1, 1, rng.randint(2, 8)))
        c.update(seqs=seqs, rows=rows, ctx=max(rows, _log(rng, 1, min(32768, 2 ** 28 // (seqs * hkv * d)))))
        if op == "sparse":
            sink, recent = rng.choice((0, 1)), rng.choice((1, 2, 4))
            c.update(sink=sink, recent=recent, budget=max(sink + recent, _log(rng, 4, 300)))
    return c


# ------------------------------------------------------------------ inputs


def _lengths(case, most, least):
    """The sequences' lengths: from the longest down to a third of it, spread by the golden ratio."""
    n = case["seqs"]
    return [max(least, int(most * (1 - 0.66 * ((0.618034 * i) % 1.0)))) for i in range(n)]


def _shares(case):
    """How `new` tokens fall to the sequences: one each at least, the rest in proportion to i + 1."""
    n, new = case["seqs"], case["new"]
    w = np.arange(1, n + 1, dtype=np.float64)
    c = 1 + np.floor((new - n) * w / w.sum()).astype(np.int64)
    c[-1] += new - c.sum()
    return c


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + case["hkv"] * 7919 + case.get("ctx", 0) * 131 + case.get("new", 0) * 17)
    return g


def _rows_of(g, n, heads, d):
    """[n, heads, d] rows, N(0, 1) with a scale of its own for each head."""
    s = torch.rand((1, heads, 1), device="cuda", generator=g) + 0.5
    return (torch.randn((n, heads, d), device="cuda", generator=g) * s).half()


def _table(g, pages, width):
    """Pages of a pool in random order, the sequences' one after another; -1 behind a sequence's last."""
    perm = torch.randperm(int(pages.sum()), device="cuda", generator=g).to(torch.int32)
    first = torch.from_numpy(np.cumsum(pages) - pages).cuda()
    at = torch.arange(width, device="cuda")
    has = at < torch.from_numpy(pages).cuda()[:, None]
    idx = torch.where(has, first[:, None] + at, 0)
    return torch.where(has, perm[idx], -1).to(torch.int32).contiguous()


def _axes_positions(case, g):
    """Positions [3, new]: text runs on all axes alike, images of 24 x 32 patches between on height and width, time in steps."""
    n = case["new"]
    i = torch.arange(n, device="cuda")
    first = torch.randint(0, 100000, (1,), device="cuda", generator=g)
    image = (i // 768) % 2 == 1
    r = i % 768
    t = torch.where(image, i - r, i)
    return (first + torch.stack([t, torch.where(image, t + r // 32, i), torch.where(image, t + r % 32, i)])).to(torch.int32)


def _sections(case):
    """Pairs of the time, height and width axes: a quarter for time, the rest shared."""
    half = case["rope"] // 2
    side = 3 * half // 8
    return (half - 2 * side, side, side)


def _inputs(case, seed):
    g = _generator(case, seed)
    op, hq, hkv, d = (case[k] for k in ("op", "hq", "hkv", "d"))
    x = {}
    if op in ("rope", "rope_store"):
        x["qkv"] = _rows_of(g, case["new"], hq + 2 * hkv, d).reshape(case["new"], -1)
        x["positions"] = _axes_positions(case, g)
    if op == "rope":
        return x
    page, b = case["page"], case["seqs"]
    if op in ("store", "rope_store"):
        counts = _shares(case)
        start = np.array(_lengths(case, case["ctx"], 0), dtype=np.int64) if case["ctx"] else np.zeros(b, np.int64)
        pages = -(-(start + counts) // page)
        x["table"] = _table(g, pages, int(pages.max()))
        x["starts"] = torch.from_numpy(start.astype(np.int32)).cuda()
        x["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
        x["n_pages"] = int(pages.sum())
        if op == "store":
            x["k"], x["v"] = _rows_of(g, case["new"], hkv, d), _rows_of(g, case["new"], hkv, d)
        return x
    length = np.array(_lengths(case, case["ctx"], case["rows"]), dtype=np.int64)
    pages = -(-length // page)
    width = int(pages.max())
    x["table"] = _table(g, pages, width)
    x["lengths"] = torch.from_numpy(length.astype(np.int32)).cuda()
    x["n_pages"] = int(pages.sum())
    # keys of neighbouring tokens have something in common, so that some pages matter more than others
    t = width * page
    v = _rows_of(g, b * t, hkv, d).reshape(b, t, hkv, d)
    k = _rows_of(g, b * t, hkv, d).reshape(b, t, hkv, d)
    common = _rows_of(g, b * (t // 16), hkv, d).reshape(b, t // 16, 1, hkv, d)
    k = (k.reshape(b, t // 16, 16, hkv, d) + common).reshape(b, t, hkv, d)
    x["k"], x["v"] = k, v
    x["q"] = (torch.randn((b, hq, case["rows"], d), device="cuda", generator=g)).half()
    return x


def _as(x, value):
    return torch.full_like(x, value)


def _quantize(x, mode):
    """Codes, scales and biases of rows [..., d]. Affine: groups of 64 dims, the edge of the larger magnitude stored without
    loss; int8: a row's largest magnitude over 127."""
    if mode == "fp16":
        return {"x": x}
    if mode == "int8":
        top = x.float().abs().amax(-1, keepdim=True)
        s = (top / _as(top, 127.0)).half()
        s = torch.where(top == 0, _as(s, 1.0), s)
        return {"codes": (x / s).float().round().clamp(-128, 127).to(torch.int8), "scales": s}
    top = 2 ** BITS[mode] - 1
    x = x.float().reshape(*x.shape[:-1], -1, 64)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    low = lo.abs() > hi.abs()
    s = ((hi - lo) / _as(hi, float(top))).clamp_min(1e-7)
    s = torch.where(low, s, -s)
    edge = torch.where(low, lo, hi)
    steps = (edge / s).round()
    b = torch.where(steps != 0, edge, _as(edge, 0.0))
    s = torch.where(steps != 0, edge / steps, s)
    return {"codes": ((x - b) / s).round().clamp(0, top).to(torch.uint8), "scales": s.half(), "biases": b.half()}


def _values(t):
    """What the codes stand for, in float32."""
    if "x" in t:
        return t["x"].float()
    if "biases" not in t:
        return t["codes"].float() * t["scales"].float()
    return (t["codes"].float() * t["scales"].float() + t["biases"].float()).flatten(-2)


def _stored(t):
    """The fp16 values that reading back gives: code times scale, then plus bias, each rounded."""
    if "x" in t:
        return t["x"]
    if "biases" not in t:
        return t["codes"].half() * t["scales"]
    return (t["codes"].half() * t["scales"] + t["biases"]).flatten(-2)


def _bounds(k, length, page):
    """Keys [b, t, heads, d] to the pages' bounds: codes of the largest and the least key of each dim, and the magnitude."""
    b, t, h, d = k.shape
    seen = (torch.arange(t, device=k.device) < length[:, None]).reshape(b, -1, page, 1, 1)
    k = k.reshape(b, -1, page, h, d)
    hi = k.masked_fill(~seen, -math.inf).amax(2).float()
    lo = k.masked_fill(~seen, math.inf).amin(2).float()
    none = ~seen.any(2)
    hi, lo = hi.masked_fill(none, 0.0), lo.masked_fill(none, 0.0)
    top = torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True)
    inv = torch.where(top > 0, _as(top, 127.0) / top.clamp_min(1e-30), _as(top, 0.0))
    return {"hi": (hi * inv).ceil().clamp(-127, 127).to(torch.int8), "lo": (lo * inv).floor().clamp(-127, 127).to(torch.int8), "top": top[..., 0]}


def _in_pool(x, table, n_pages):
    """[b, width * page, ...] rows of the sequences to [n_pages, page, ...]."""
    b, w = table.shape
    x = x.reshape(b, w, -1, *x.shape[2:])
    pool = x.new_zeros((n_pages, *x.shape[2:]))
    has = table >= 0
    pool[table[has].long()] = x[has]
    return pool


def prepare(case, seed):
    """The pages as they stand before the call: the codes, and, where the package's own calls are timed, its cache that holds them."""
    x = _inputs(case, seed)
    x["case"] = case
    op = case["op"]
    if own and op != "rope":
        import qw_amd

        x["cache"] = qw_amd.PagedKVCache(case["mode"], case["hkv"], case["d"], x["n_pages"], page_size=case["page"])
    if op in ("attend", "sparse"):
        k, v, n = x.pop("k"), x.pop("v"), x["lengths"]
        if own:
            has = torch.arange(k.shape[1], device="cuda") < n[:, None]
            offsets = torch.cat([n.new_zeros(1), n.cumsum(0, dtype=torch.int32)])
            x["cache"].update(k[has], v[has], x["table"], torch.zeros_like(n), offsets=offsets)
        else:
            if op == "sparse":
                bounds = _bounds(k, n, case["page"])
                for name, t in bounds.items():
                    x[name] = _in_pool(t, x["table"], x["n_pages"])[:, 0]
            for name, t in (("k", k), ("v", v)):
                x[name] = {part: _in_pool(y, x["table"], x["n_pages"]) for part, y in _quantize(t, case["mode"]).items()}
    return x


# ------------------------------------------------------------------ one pass


def _slots(x, case):
    """The pool's row of each new token."""
    token = torch.arange(case["new"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(x["offsets"], token, right=True) - 1
    at = x["starts"][seq] + token - x["offsets"][seq]
    return x["table"][seq, torch.div(at, case["page"], rounding_mode="floor").long()].long() * case["page"] + at % case["page"]


def _plain_store(x, case, k, v):
    slot = _slots(x, case)
    out = []
    for name, t in (("pool_k", k), ("pool_v", v)):
        new = _quantize(t, case["mode"])
        if name not in x:  # the pool is a buffer that the program keeps
            x[name] = {p: y.new_zeros((x["n_pages"] * case["page"], *y.shape[1:])) for p, y in new.items()}
        for p, y in new.items():
            x[name][p][slot] = y
        out.append(_stored({p: y[slot] for p, y in x[name].items()}))
    return tuple(out)


def _taken(parts, pages):
    """Pages [b, w] of pool parts [pages, page, heads, ...]: values [b, heads, w * page, d]."""
    t = _values({p: y[pages] for p, y in parts.items()})
    b, w, page, h, d = t.shape
    return t.permute(0, 3, 1, 2, 4).reshape(b, h, w * page, d)


def _taken_by_head(parts, pages):
    """Pages [b, heads, w], of each head its own: values [b, heads, w * page, d]."""
    head = torch.arange(pages.shape[1], device=pages.device)[:, None]
    t = _values({p: y.transpose(1, 2)[pages, head] for p, y in parts.items()})
    return t.flatten(2, 3)


def _softmax_rows(q, k, v, seen, scale):
    """q [b, hkv, g, rows, d] over k, v [b, hkv, t, d] where seen [b, 1 or hkv, rows, t]."""
    b, h, gr, rows, d = q.shape
    s = ((q.reshape(b, h, gr * rows, d) * scale) @ k.transpose(2, 3)).reshape(b, h, gr, rows, -1)
    s = s.masked_fill(~seen[:, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(b, h, gr * rows, -1) @ v).reshape(b, h, gr, rows, d)
    return (o / total.masked_fill(total == 0, 1.0)).reshape(b, h * gr, rows, d).half()


def _last_seen(x, case):
    """The last key that each row sees: [b, rows, 1]."""
    rows = case["rows"]
    return (x["lengths"][:, None] - rows + torch.arange(rows, device="cuda"))[:, :, None]


def _plain_attend(x, case):
    table = x["table"].clamp_min(0).long()
    k, v = _taken(x["k"], table), _taken(x["v"], table)
    hkv = case["hkv"]
    q = x["q"].float().reshape(case["seqs"], hkv, -1, case["rows"], case["d"])
    seen = torch.arange(k.shape[2], device=k.device) <= _last_seen(x, case)
    return _softmax_rows(q, k, v, seen[:, None], case["d"] ** -0.5)


def _plain_pick(x, case):
    b, hkv, d, page = (case[k] for k in ("seqs", "hkv", "d", "page"))
    table, n = x["table"].clamp_min(0).long(), x["lengths"]
    pages = torch.div(n + page - 1, page, rounding_mode="floor")
    q = x["q"].float().reshape(b, hkv, -1, d)
    top = q.abs().amax((2, 3), keepdim=True)
    qi = (q * (_as(top, 127.0) / top)).round()
    hi, lo = (x[p][table].float().transpose(1, 2) for p in ("hi", "lo"))  # [b, hkv, w, d]
    s = (qi.clamp_min(0) @ hi.transpose(2, 3) + qi.clamp_max(0) @ lo.transpose(2, 3)).amax(2)
    s = s * x["top"][table].transpose(1, 2)
    at = torch.arange(table.shape[1], device=s.device)
    there = at < pages[:, None]
    s = s.masked_fill(((at < case["sink"]) | (at >= pages[:, None] - case["recent"]))[:, None], math.inf)
    s = s.masked_fill(~there[:, None], -math.inf)
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :case["budget"]]
    order = torch.where(order < pages[:, None, None], order, table.shape[1]).sort(-1).values
    picked = torch.where(order < table.shape[1], order, -1).to(torch.int32)
    short = case["budget"] - picked.shape[-1]
    return torch.nn.functional.pad(picked, (0, short), value=-1) if short > 0 else picked


def _plain_sparse(x, case):
    b, hkv, d, page = (case[k] for k in ("seqs", "hkv", "d", "page"))
    picked = _plain_pick(x, case)
    at = picked.long()
    pages = x["table"].clamp_min(0).long()[:, None].expand(-1, hkv, -1).gather(2, at.clamp_min(0))
    k, v = _taken_by_head(x["k"], pages), _taken_by_head(x["v"], pages)
    key = (at[..., None] * page + torch.arange(page, device=at.device)).flatten(2)
    key = torch.where((at >= 0).repeat_interleave(page, dim=2), key, 2 ** 31)
    q = x["q"].float().reshape(b, hkv, -1, case["rows"], d)
    seen = key[:, :, None] <= _last_seen(x, case)[:, None]
    return {"out": _softmax_rows(q, k, v, seen, d ** -0.5), "picked": picked}


def _axis_of_pair(case):
    """Which axis turns each pair: runs of the sections' lengths, or the axes in turn as long as each has pairs left."""
    sec, half = _sections(case), case["rope"] // 2
    if not case["interleaved"]:
        return np.repeat(np.arange(3), sec)
    p = np.arange(half)
    return np.where((p % 3 > 0) & (p < 3 * np.array(sec)[p % 3]), p % 3, 0)


def _plain_rope(x, case):
    n, hq, hkv, d, r = (case[k] for k in ("new", "hq", "hkv", "d", "rope"))
    h = r // 2
    axis = torch.from_numpy(_axis_of_pair(case)).cuda()
    inv = 1e6 ** (-torch.arange(h, device="cuda", dtype=torch.float64) / h)
    a = x["positions"][axis].T.double() * inv  # far positions: the angle in 64 bits
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    t = x["qkv"].reshape(n, hq + 2 * hkv, d)[:, :hq + hkv]
    u, w = t[..., :h].float(), t[..., h:r].float()
    t = torch.cat([(u * c - w * s).half(), (u * s + w * c).half(), t[..., r:]], dim=-1)
    return t[:, :hq].contiguous(), t[:, hq:].contiguous()


def _plain_rope_store(x, case):
    q, k = _plain_rope(x, case)
    v = x["qkv"].reshape(case["new"], -1, case["d"])[:, case["hq"] + case["hkv"]:]
    return (q, *_plain_store(x, case, k, v))


def run(x):
    case = x["case"]
    op = case["op"]
    if not own:
        if op == "store":
            return _plain_store(x, case, x["k"], x["v"])
        return {"attend": _plain_attend, "sparse": _plain_sparse, "rope": _plain_rope, "rope_store": _plain_rope_store}[op](x, case)
    cache = x.get("cache")
    if op == "store":
        cache.update(x["k"], x["v"], x["table"], x["starts"], offsets=x["offsets"])
        return cache.gather(x["table"], x["starts"], case["new"], offsets=x["offsets"])
    if op == "attend":
        return cache.attention(x["q"], x["table"], x["lengths"], case["d"] ** -0.5)
    if op == "sparse":
        picked = cache.select_pages(x["q"], x["table"], x["lengths"], case["budget"], sink=case["sink"], recent=case["recent"])
        return {"out": cache.attention(x["q"], x["table"], x["lengths"], case["d"] ** -0.5, picked=picked), "picked": picked}
    if op == "rope":
        import qw_amd

        return qw_amd.rope_axes(x["qkv"], x["positions"], _sections(case), case["hq"], case["hkv"], case["d"], 1e6, interleaved=case["interleaved"])
    q = cache.rope_update(x["qkv"], x["positions"], _sections(case), case["hq"], 1e6, x["table"], x["starts"], offsets=x["offsets"],
                          interleaved=case["interleaved"])
    return (q, *cache.gather(x["table"], x["starts"], case["new"], offsets=x["offsets"]))


# ------------------------------------------------------------------ what a pass cannot do without


def _row_bytes(mode, d):
    """Bytes of a token's K and V rows in one head."""
    return 2 * {"affine4": d // 2 + d // 16, "affine8": d + d // 16, "int8": d + 2, "fp16": 2 * d}[mode]


def work(case):
    op, hq, hkv, d = (case[k] for k in ("op", "hq", "hkv", "d"))
    if op in ("store", "rope", "rope_store"):
        n, byte, flops = case["new"], 0, 0
        if op != "store":  # q and k of the projection in and out
            byte += 2 * n * (hq + hkv) * d * 2 + 12 * n
            flops += n * (hq + hkv) * case["rope"] * 3
        if op != "rope":  # new rows in, codes out and in again, values out
            byte += n * hkv * (4 * d + 2 * _row_bytes(case["mode"], d) + 4 * d)
            flops += n * hkv * d * 10
            byte -= 2 * n * hkv * d if op == "rope_store" else 0  # rotated keys go straight into their page
            byte -= 2 * n * hkv * d if op == "rope_store" else 0
        return {"bytes": int(byte), "flops": int(flops)}
    rows, page = case["rows"], case["page"]
    byte = flops = 0
    for n in _lengths(case, case["ctx"], rows):
        keys, pages = n, -(-n // page)
        if op == "sparse":
            keep = min(pages, case["budget"])
            keys = n if keep == pages else keep * page
            byte += hkv * (pages * (2 * d + 4) + 4 * case["budget"])
            flops += hq * rows * pages * 4 * d
        byte += hkv * keys * _row_bytes(case["mode"], d) + 4 * hq * rows * d + 4 * pages
        flops += 4 * hq * rows * d * (keys - (rows - 1) / 2)
    return {"bytes": int(byte), "flops": int(flops)}


# ------------------------------------------------------------------ in 64 bits


def _exact_codec(x, mode):
    """(values in 64 bits, the fp16 values that are read back) of rows [..., d], from the codec's definition."""
    x = x.double()
    if mode == "fp16":
        return x, x
    if mode == "int8":
        top = x.abs().max(dim=-1, keepdim=True).values
        s = (top.float() / top.float().new_full((1,), 127)).half().double()
        s[top == 0] = 1
        y = torch.clamp(torch.round((x / s).half().double()), -128, 127) * s
        return y, y.half().double()
    # (the codec's definition has steps and codes in 32 bits: ties of the fp16 values fall by them)
    top = {"affine4": 15, "affine8": 255}[mode]
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    least, most = g.min(dim=-1, keepdim=True).values, g.max(dim=-1, keepdim=True).values
    from_least = least.abs() > most.abs()
    step = torch.clamp((most - least) / most.new_full((1,), top), min=1e-7)
    step = torch.where(from_least, step, -step)
    edge = torch.where(from_least, least, most)
    whole = torch.round(edge / step)
    moved = whole != 0
    step = torch.where(moved, edge / torch.where(moved, whole, torch.ones_like(whole)), step)
    base = torch.where(moved, edge, torch.zeros_like(edge))
    code = torch.clamp(torch.round((g - base) / step), 0, top).double()
    step, base = step.half().double(), base.half().double()
    back = ((code * step).half().double() + base).half().double()
    return (code * step + base).reshape(x.shape), back.reshape(x.shape)


def _exact_turn(x, case):
    """The rotation as a product of complex numbers."""
    n, hq, hkv, d, r = (case[k] for k in ("new", "hq", "hkv", "d", "rope"))
    sec = _sections(case)
    pairs = r // 2
    axis, left = [0] * pairs, list(sec)
    for p in range(pairs):
        if case["interleaved"]:
            a = p % 3
            axis[p] = a if a and p < 3 * sec[a] else 0
        else:
            axis[p] = next(a for a in range(3) if p < sum(sec[:a + 1]))
    theta = np.array([1e6 ** (-2.0 * p / r) for p in range(pairs)])
    angle = x["positions"].cpu().numpy().astype(np.float64)[axis] * theta[:, None]
    turn = torch.from_numpy(np.exp(1j * angle.T)).cuda()[:, None]
    t = x["qkv"].double().reshape(n, hq + 2 * hkv, d)
    z = torch.complex(t[..., :pairs], t[..., pairs:r]) * turn
    t = torch.cat([z.real, z.imag, t[..., r:]], dim=-1)
    return t[:, :hq], t[:, hq:hq + hkv]


def exact(case, seed):
    x = _inputs(case, seed)
    op, hq, hkv, d = (case[k] for k in ("op", "hq", "hkv", "d"))
    if op == "rope":
        return _exact_turn(x, case)
    if op == "store":
        return tuple(_exact_codec(x[p], case["mode"])[1] for p in ("k", "v"))
    if op == "rope_store":
        q, k = _exact_turn(x, case)
        v = x["qkv"].reshape(case["new"], -1, d)[:, hq + hkv:]
        # (what is stored is the rotated key rounded to fp16)
        return q, _exact_codec(k.half(), case["mode"])[1], _exact_codec(v, case["mode"])[1]
    rows, gr, page = case["rows"], hq // hkv, case["page"]
    out = torch.zeros((case["seqs"], hq, rows, d), dtype=torch.float64, device="cuda")
    picked = torch.full((case["seqs"], hkv, case.get("budget", 0)), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(x["lengths"].tolist()):
        for h in range(hkv):
            k, v = (_exact_codec(x[p][b, :n, h], case["mode"])[0] for p in ("k", "v"))
            q = x["q"][b, h * gr:(h + 1) * gr].double()
            at = torch.arange(n, device="cuda")
            if op == "sparse":
                which = _exact_pick(x["k"][b, :n, h], x["q"][b, h * gr:(h + 1) * gr], case)
                picked[b, h, :len(which)] = which.to(torch.int32)
                at = at[torch.isin(torch.div(at, page, rounding_mode="floor"), which)]
                k, v = k[at], v[at]
            z = (q.reshape(gr * rows, d) @ k.T / math.sqrt(d)).reshape(gr, rows, -1)
            z = z.masked_fill(at > torch.arange(n - rows, n, device="cuda")[:, None], -math.inf)
            p = torch.softmax(z, dim=-1).nan_to_num(0.0)  # a row that sees none of the pages is zeros
            out[b, h * gr:(h + 1) * gr] = (p.reshape(gr * rows, -1) @ v).reshape(gr, rows, d)
    return {"out": out, "picked": picked} if op == "sparse" else out


def _exact_pick(k, q, case):
    """The picked pages of one head of one sequence, ascending: whole-number bounds, ordered by (-score, page)."""
    page, budget = case["page"], case["budget"]
    n, d = k.shape
    pages = -(-n // page)
    fill = pages * page - n
    k = k.float()
    most = torch.cat([k, k[-1:].expand(fill, d)]).reshape(pages, page, d)  # (the last key again changes no bound)
    least, most = most.min(1).values, most.max(1).values
    top = torch.maximum(least.abs(), most.abs()).max(1).values
    inv = torch.where(top > 0, _as(top, 127.0) / top, top)[:, None]
    least, most = torch.floor(least * inv).clamp(-127, 127).long(), torch.ceil(most * inv).clamp(-127, 127).long()
    q = q.float().reshape(-1, d)
    big = q.abs().max()
    q = torch.round(q * (_as(big, 127.0) / big)).long()
    total = torch.maximum(q[:, None] * most, q[:, None] * least).sum(-1).max(0).values
    score = (total.float() * top).cpu().numpy()
    fixed = [p for p in range(pages) if p < case["sink"] or p >= pages - case["recent"]]
    rest = sorted((p for p in range(pages) if case["sink"] <= p < pages - case["recent"]), key=lambda p: (-score[p], p))
    keep = (fixed + rest)[:budget] if pages > budget else range(pages)
    return torch.tensor(sorted(keep), device="cuda")
