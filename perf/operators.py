"""Serving many requests from one prompt, and keeping a cache within a budget: what is timed of it.

Three operators over a layer's KV cache, each in its plain form (elementary torch operations on the cache's packed
tensors) and as the calls that a user makes:

  shared  attention of a batch of sequences that share a long prefix: every sequence's rows see the whole prefix cache
          and their own tail, keys starts[b] .. of a cache that holds all tails side by side, causal among its last rows
  scored  attention over a cache that also gives each key the softmax weight it got, summed over rows and over the
          query heads of its KV head, added to what it had before (times a decay)
  evict   each KV head keeps its first `sink` and last `recent` keys and, of the others, those of the largest weight
          (ties to the earlier key) up to `budget`; their rows move to a cache of their own, in order

Sizes: the package's own heads (24 over 4 of 256 dims, 32 over 8 of 128), contexts of up to 128k keys, speculative
blocks of up to 16 rows, prefill chunks of 1536 rows, 4 sinks and a 512-key window.
"""
import math

import numpy as np
import torch

own = False

GEOMETRIES = ((24, 4, 256), (16, 2, 256), (32, 8, 128), (24, 4, 128), (8, 8, 128), (12, 1, 256))
BITS = {"affine4": 4, "affine8": 8, "int8": 8, "fp16": 16}
MODES = tuple(BITS)


def listed():
    g = {"hq": 24, "hkv": 4, "d": 256}
    s = {"hq": 32, "hkv": 8, "d": 128}
    return [
        # two samples of one short prompt at their third token: latency and launches count
        {"name": "shared_2x257", "op": "shared", "mode": "affine8", "tail_mode": "affine8", "prefix": 257, "seqs": 2, "tail": 3, "rows": 1, **s},
        # sixteen chats over one long system prompt, their own turns of different lengths behind it
        {"name": "shared_16x32k", "op": "shared", "mode": "affine4", "tail_mode": "affine4", "prefix": 32768, "seqs": 16, "tail": 515, "rows": 1, **g},
        # eight requests in speculative decoding, 5 rows each, tails kept in fp16
        {"name": "shared_8x16k_verify5", "op": "shared", "mode": "affine8", "tail_mode": "fp16", "prefix": 16397, "seqs": 8, "tail": 1001, "rows": 5, **g},
        # a full batch over a document
        {"name": "shared_64x64k", "op": "shared", "mode": "fp16", "tail_mode": "fp16", "prefix": 65536, "seqs": 64, "tail": 256, "rows": 1, **s},
        # one token of a fresh conversation, weights counted from its start
        {"name": "scored_1x301", "op": "scored", "mode": "affine4", "ctx": 301, "rows": 1, "decay": 1.0, **s},
        # one token of a long chat, weights accumulated with forgetting
        {"name": "scored_1x32k", "op": "scored", "mode": "affine4", "ctx": 32769, "rows": 1, "decay": 0.98, **g},
        # the last 64 rows of a prompt observe which keys matter: a fresh count
        {"name": "scored_64x16k", "op": "scored", "mode": "affine8", "ctx": 16384, "rows": 64, "decay": 0.0, **g},
        # a prefill chunk that accumulates as it goes
        {"name": "scored_1536x9k", "op": "scored", "mode": "int8", "ctx": 9728, "rows": 1536, "decay": 1.0, **g},
        # a short conversation cut to its budget
        {"name": "evict_500_256", "op": "evict", "mode": "affine8", "ctx": 500, "budget": 256, "sink": 4, "recent": 64, **s},
        # a long chat cut to an eighth
        {"name": "evict_32k_4k", "op": "evict", "mode": "affine4", "ctx": 32769, "budget": 4096, "sink": 4, "recent": 512, **g},
        # a document of which three quarters stay: keys that nothing ever looked at are among them, tied at zero
        {"name": "evict_64k_48k", "op": "evict", "mode": "fp16", "ctx": 65543, "budget": 49160, "sink": 0, "recent": 1, **g},
        # the longest context, cut to 16k
        {"name": "evict_128k_16k", "op": "evict", "mode": "affine8", "ctx": 131072, "budget": 16387, "sink": 4, "recent": 512, **g},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, d = rng.choice(GEOMETRIES)
    op = rng.choice(("shared", "scored", "evict"))
    c = {"op": op, "mode": rng.choice(MODES), "hq": hq, "hkv": hkv, "d": d}
    if op == "shared":
        rows = rng.choice((1, 1, rng.randint(2, 16)))
        seqs = _log(rng, 1, max(1, 96 // rows))
        tail = max(rows, _log(rng, 1, 1200))
        c.update(tail_mode=rng.choice((c["mode"], c["mode"], rng.choice(MODES))), seqs=seqs, rows=rows, tail=tail,
                 prefix=_log(rng, 1, min(65536, 2500000 // (seqs * rows))))
    elif op == "scored":
        rows = rng.choice((1, 1, _log(rng, 2, 1024)))
        c.update(rows=rows, ctx=max(rows, _log(rng, 16, min(131072, 8000000 // rows))), decay=rng.choice((0.0, 1.0, 0.95)))
    else:
        ctx = _log(rng, 64, 131072)
        sink, recent = rng.choice((0, 4)), rng.choice((1, 32, 512))
        c.update(ctx=ctx, sink=sink, recent=recent, budget=max(sink + recent, _log(rng, 16, min(ctx, 49152))))
    return c


# ------------------------------------------------------------------ inputs


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + case["hkv"] * 7919 + case.get("ctx", 0) * 131 + case.get("prefix", 0) * 17)
    return g


def _values(g, heads, n, d):
    """[heads, n, d] rows, N(0, 1) with a scale of its own for each head."""
    s = torch.rand((heads, 1, 1), device="cuda", generator=g) * 1.0 + 0.5
    return (torch.randn((heads, n, d), device="cuda", generator=g) * s).half()


def _pack(x, bits):
    """Groups of 64 dims to codes with a scale and a bias, 32-bit words with the lowest dim in the lowest bits."""
    h, n, d = x.shape
    x = x.float().reshape(h, n, d // 64, 64)
    lo, hi, top = x.amin(-1), x.amax(-1), 2 ** bits - 1
    scales = ((hi - lo) / top).half().clamp_min(2.0 ** -14)
    codes = ((x - lo.half().float()[..., None]) / scales.float()[..., None]).round().clamp(0, top).to(torch.int32)
    shifts = torch.arange(0, 32, bits, device="cuda", dtype=torch.int32)
    words = (codes.reshape(h, n, d * bits // 32, 32 // bits) << shifts).sum(-1).to(torch.int32)
    return words, scales, lo.half()


def _tensors(g, mode, heads, n, d):
    """A cache's rows as it stores them, by the names of its snapshot."""
    k, v = _values(g, heads, n, d), _values(g, heads, n, d)
    if mode == "fp16":
        return {"keys": k, "values": v}
    if mode == "int8":
        t = {}
        for name, scale, x in (("keys", "key_scales", k), ("values", "val_scales", v)):
            t[scale] = (x.float().abs().amax(-1, keepdim=True) / 127).half()
            t[name] = (x.float() / t[scale].float()).round().clamp(-127, 127).to(torch.int8)
        return t
    t = {}
    t["k_codes"], t["k_scales"], t["k_biases"] = _pack(k, BITS[mode])
    t["v_codes"], t["v_scales"], t["v_biases"] = _pack(v, BITS[mode])
    return t


def _inputs(case, seed):
    g = _generator(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = {}
    if case["op"] == "shared":
        b, rows = case["seqs"], case["rows"]
        x["prefix"] = _tensors(g, case["mode"], hkv, case["prefix"], d)
        x["tails"] = _tensors(g, case["tail_mode"], b * hkv, case["tail"], d)
        # a sequence's own part: anything from its newest rows to the whole tail; the first has all of it
        u = torch.rand((b,), device="cuda", generator=g)
        u[0] = 0
        x["starts"] = (u * (case["tail"] - rows + 1)).floor().clamp(0, case["tail"] - rows).to(torch.int32)
        x["q"] = (2 * torch.randn((b, hq, rows, d), device="cuda", generator=g)).half()
        return x
    x["cache"] = _tensors(g, case["mode"], hkv, case["ctx"], d)
    # what earlier steps left: a few keys with most of it, three in ten never looked at
    w = torch.exp(2 * torch.randn((hkv, case["ctx"]), device="cuda", generator=g))
    x["weights"] = w * (torch.rand((hkv, case["ctx"]), device="cuda", generator=g) > 0.3)
    if case["op"] == "scored":
        x["q"] = (2 * torch.randn((1, hq, case["rows"], d), device="cuda", generator=g)).half()
    return x


def prepare(case, seed):
    """The packed rows, and, where the package's own calls are timed, the caches that hold them."""
    x = _inputs(case, seed)
    x["case"] = case
    if own:
        import qw_amd

        def cache(tensors, mode, heads, n):
            c = qw_amd.KVCache(mode, heads, case["d"], capacity=n)
            c.restore_snapshot(tensors)
            return c

        if case["op"] == "shared":
            x["prefix"] = cache(x["prefix"], case["mode"], case["hkv"], case["prefix"])
            x["tails"] = cache(x["tails"], case["tail_mode"], case["seqs"] * case["hkv"], case["tail"])
        else:
            x["cache"] = cache(x["cache"], case["mode"], case["hkv"], case["ctx"])
        if case["op"] == "evict":
            x["into"] = qw_amd.KVCache(case["mode"], case["hkv"], case["d"], capacity=min(case["ctx"], case["budget"]))
    return x


# ------------------------------------------------------------------ one pass


def _unpack(words, scales, biases, d):
    """The fp16 values that the codes stand for: f16(f16(code * scale) + bias), in float32."""
    bits = words.shape[-1] * 32 // d
    shifts = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    codes = (words[..., None] >> shifts) & (2 ** bits - 1)
    codes = codes.reshape(*words.shape[:2], d // 64, 64).half()
    return (codes * scales[..., None] + biases[..., None]).float().reshape(*words.shape[:2], d)


def _rows(t, d):
    if "k_codes" in t:
        return tuple(_unpack(t[f"{p}_codes"], t[f"{p}_scales"], t[f"{p}_biases"], d) for p in "kv")
    if "key_scales" in t:
        return (t["keys"].half() * t["key_scales"]).float(), (t["values"].half() * t["val_scales"]).float()
    return t["keys"].float(), t["values"].float()


def _plain_shared(x, case):
    b, rows, hq, hkv, d, n = (case[k] for k in ("seqs", "rows", "hq", "hkv", "d", "tail"))
    gr = hq // hkv
    pk, pv = _rows(x["prefix"], d)
    tk, tv = _rows(x["tails"], d)
    q = x["q"].float().reshape(b, hkv, gr * rows, d) * d ** -0.5
    qp = q.transpose(0, 1).reshape(hkv, b * gr * rows, d)
    s = (qp @ pk.transpose(1, 2)).reshape(hkv, b, gr * rows, -1).transpose(0, 1)
    t = (q.reshape(b * hkv, gr * rows, d) @ tk.transpose(1, 2)).reshape(b, hkv, gr, rows, n)
    key = torch.arange(n, device=t.device)
    seen = (key >= x["starts"][:, None, None]) & (key <= torch.arange(n - rows, n, device=t.device)[:, None])
    t = t.masked_fill(~seen[:, None, None], -math.inf).reshape(b, hkv, gr * rows, n)
    m = torch.maximum(s.amax(-1, keepdim=True), t.amax(-1, keepdim=True))
    s, t = torch.exp(s - m), torch.exp(t - m)
    total = s.sum(-1, keepdim=True) + t.sum(-1, keepdim=True)
    o = (s.transpose(0, 1).reshape(hkv, b * gr * rows, -1) @ pv).reshape(hkv, b, gr * rows, d).transpose(0, 1)
    o = o + (t.reshape(b * hkv, gr * rows, n) @ tv).reshape(b, hkv, gr * rows, d)
    return (o / total).reshape(b, hq, rows, d).half()


def _plain_scored(x, case):
    rows, hq, hkv, d, n = (case[k] for k in ("rows", "hq", "hkv", "d", "ctx"))
    k, v = _rows(x["cache"], d)
    q = x["q"].float().reshape(hkv, hq // hkv * rows, d) * d ** -0.5
    s = (q @ k.transpose(1, 2)).reshape(hkv, hq // hkv, rows, n)
    if rows > 1:
        seen = torch.arange(n, device=s.device) <= torch.arange(n - rows, n, device=s.device)[:, None]
        s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(hkv, -1, n)
    w = p.sum(1)
    if case["decay"]:
        w = w + case["decay"] * x["weights"]
    return {"out": (p @ v).reshape(1, hq, rows, d).half(), "weights": w}


def _plain_evict(x, case):
    n, budget, sink, recent = (case[k] for k in ("ctx", "budget", "sink", "recent"))
    w = x["weights"]
    rank = w.clone()
    rank[:, :sink] = math.inf
    rank[:, max(0, n - recent):] = math.inf
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices
    kept = order[:, :min(n, budget)].sort(dim=1).values
    out = {k: t.gather(1, kept[:, :, None].expand(-1, -1, t.shape[2])) for k, t in x["cache"].items()}
    out["kept"] = kept.to(torch.int32)
    out["weights"] = w.gather(1, kept)
    return out


def run(x):
    case = x["case"]
    scale = case["d"] ** -0.5
    if not own:
        return {"shared": _plain_shared, "scored": _plain_scored, "evict": _plain_evict}[case["op"]](x, case)
    if case["op"] == "shared":
        return x["prefix"].shared_attention(x["q"], x["tails"], scale, starts=x["starts"])
    if case["op"] == "scored":
        weights = x["weights"] if case["decay"] else None
        out, w = x["cache"].attention_scored(x["q"], scale, weights=weights, decay=case["decay"], causal=True)
        return {"out": out, "weights": w}
    kept, w = x["cache"].evict(x["weights"], case["budget"], sink=case["sink"], recent=case["recent"], into=x["into"])
    return {**x["into"].snapshot_tensors(), "kept": kept, "weights": w}


# ------------------------------------------------------------------ what a pass cannot do without


def _row_bytes(mode, d):
    """Bytes of a key's K and V rows in one head."""
    return 2 * {"affine4": d // 2 + d // 16, "affine8": d + d // 16, "int8": d + 2, "fp16": 2 * d}[mode]


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "shared":
        b, rows, prefix, tail = case["seqs"], case["rows"], case["prefix"], case["tail"]
        own_keys = 1 + (tail - rows) / 2 + (rows - 1) / 2  # the sequences' parts are spread evenly
        read = hkv * (prefix * _row_bytes(case["mode"], d) + b * (own_keys + (rows - 1) / 2) * _row_bytes(case["tail_mode"], d))
        return {"bytes": int(read + 4 * b * hq * rows * d), "flops": int(4 * b * hq * rows * d * (prefix + own_keys))}
    n = case["ctx"]
    if case["op"] == "scored":
        rows = case["rows"]
        counts = 4 * hkv * n * (2 if case["decay"] else 1)
        return {"bytes": int(hkv * n * _row_bytes(case["mode"], d) + 4 * hq * rows * d + counts),
                "flops": int(4 * hq * rows * d * (n - (rows - 1) / 2))}
    keep = min(n, case["budget"])
    return {"bytes": int(4 * hkv * n + hkv * keep * (2 * _row_bytes(case["mode"], d) + 8)), "flops": int(hkv * n)}


# ------------------------------------------------------------------ in 64 bits


def _exact_rows(t, d):
    """A cache's values, decoded on their own: the two fp16 roundings are part of what the codes mean."""
    def codes(words):
        bits = words.shape[-1] * 32 // d
        w = words.to(torch.int64) & 0xFFFFFFFF
        return torch.stack([(w >> s) & ((1 << bits) - 1) for s in range(0, 32, bits)], dim=-1).reshape(*words.shape[:2], d)

    if "k_codes" in t:
        out = []
        for p in ("k", "v"):
            s = t[f"{p}_scales"].double().repeat_interleave(64, dim=2)
            z = t[f"{p}_biases"].double().repeat_interleave(64, dim=2)
            out.append(((codes(t[f"{p}_codes"]).double() * s).half().double() + z).half().double())
        return out
    if "key_scales" in t:
        return [(t[a].double() * t[c].double()).half().double() for a, c in (("keys", "key_scales"), ("values", "val_scales"))]
    return [t["keys"].double(), t["values"].double()]


def _head(tensors, h):
    return {k: t[h:h + 1] for k, t in tensors.items()}


def exact(case, seed):
    x = _inputs(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    gr = hq // hkv
    if case["op"] == "evict":
        return _exact_evict(x, case)
    rows = case["rows"]
    if case["op"] == "shared":
        b, n = case["seqs"], case["tail"]
        out = torch.empty((b, hq, rows, d), dtype=torch.float64, device="cuda")
        starts = x["starts"].tolist()
        for h in range(hkv):
            pk, pv = (t[0] for t in _exact_rows(_head(x["prefix"], h), d))
            for s in range(b):
                tk, tv = (t[0] for t in _exact_rows(_head(x["tails"], s * hkv + h), d))
                for r in range(rows):
                    keys = torch.cat([pk, tk[starts[s]:n - rows + r + 1]])
                    z = x["q"][s, h * gr:(h + 1) * gr, r].double() @ keys.T / math.sqrt(d)
                    out[s, h * gr:(h + 1) * gr, r] = torch.softmax(z, dim=-1) @ torch.cat([pv, tv[starts[s]:n - rows + r + 1]])
        return out
    n = case["ctx"]
    out = torch.empty((1, hq, rows, d), dtype=torch.float64, device="cuda")
    weights = case["decay"] * x["weights"].double() if case["decay"] else torch.zeros((hkv, n), dtype=torch.float64, device="cuda")
    limit = torch.arange(n - rows, n, device="cuda")[:, None]
    for j in range(hq):
        if j % gr == 0:
            k, v = (t[0] for t in _exact_rows(_head(x["cache"], j // gr), d))
        z = x["q"][0, j].double() @ k.T / math.sqrt(d)
        p = torch.softmax(z.masked_fill(torch.arange(n, device="cuda") > limit, -math.inf), dim=-1)
        out[0, j] = p @ v
        weights[j // gr] += p.sum(0)
    return {"out": out, "weights": weights}


def _exact_evict(x, case):
    n, budget, sink, recent = (case[k] for k in ("ctx", "budget", "sink", "recent"))
    w = x["weights"].double().cpu().numpy()
    kept = []
    for h in range(case["hkv"]):
        t = np.arange(n)
        fixed = (t < sink) | (t >= n - recent)
        order = np.lexsort((t, -w[h], ~fixed))  # the protected first, then by weight, then by position
        kept.append(np.sort(order[:min(n, budget)]))
    kept = torch.from_numpy(np.stack(kept)).cuda()
    rows = torch.arange(case["hkv"], device="cuda")[:, None]
    out = {k: t[rows, kept] for k, t in x["cache"].items()}
    out["kept"] = kept.to(torch.int32)
    out["weights"] = x["weights"].double()[rows, kept]
    return out
