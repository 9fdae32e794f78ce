"""The pages that a head reads (qw_paged_select) against whole-number bounds and a sort on the host, exact; and the
calls of a decoding layer one after another: rotate, store, select, attend."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import MODES, Sequences, dev, ints, queries, rows, side_stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def bounds(k, ps):
    """[T, hkv, D] fp16 keys to (hi codes, lo codes, top) of each page and head."""
    pages = -(-len(k) // ps)
    hi = np.stack([k[p * ps:(p + 1) * ps].max(0) for p in range(pages)]).astype(np.float32)
    lo = np.stack([k[p * ps:(p + 1) * ps].min(0) for p in range(pages)]).astype(np.float32)
    return coded(hi, lo)


def coded(hi, lo):
    top = np.maximum(np.abs(hi), np.abs(lo)).max(-1).astype(np.float32)
    inv = np.where(top > 0, np.float32(127) / np.where(top > 0, top, np.float32(1)), np.float32(0)).astype(np.float32)[..., None]
    return (np.clip(np.ceil(hi * inv), -127, 127).astype(np.int64), np.clip(np.floor(lo * inv), -127, 127).astype(np.int64), top)


def scores_of(bound, q):
    """[pages, D] bounds of one head and its rows q [R, D]."""
    hi, lo, top = bound
    q = q.astype(np.float32)
    big = np.abs(q).max()
    c = np.rint(q * (np.float32(127) / big)).astype(np.int64) if big > 0 else np.zeros(q.shape, np.int64)
    total = (np.maximum(c, 0) @ hi.T + np.minimum(c, 0) @ lo.T).max(0)
    return total.astype(np.float32) * top


def ranked(score, budget, sink, recent):
    n = len(score)
    if n <= budget:
        return np.arange(n)
    at = np.arange(n)
    fixed = (at < sink) | (at >= n - recent)
    order = np.lexsort((at, -score.astype(np.float64), ~fixed))
    return np.sort(order[:budget])


def check_picked(picked, s, q, budget, sink, recent, lengths=None, bound=None):
    picked, q = picked.cpu().numpy(), q.cpu().numpy()
    B, hq, L, D = q.shape
    gr = hq // s.hkv
    for b in range(B):
        n = s.lengths[b] if lengths is None else lengths[b]
        for h in range(s.hkv):
            want = np.full(budget, -1)
            if n > 0:
                x = bounds(s.k[b][:, h:h + 1], s.ps) if bound is None else bound[b][h]
                x = tuple(y[:-(-n // s.ps)] for y in x)
                hi, lo, top = (y.reshape(len(y), -1) for y in x)
                w = ranked(scores_of((hi, lo, top[:, 0]), q[b, h * gr:(h + 1) * gr].reshape(-1, D)), budget, sink, recent)
                want[:len(w)] = w
            assert np.array_equal(picked[b, h], want), (b, h, picked[b, h], want)


CASES = [
    # hq, hkv, D, page, rows, lengths, budget, sink, recent
    (8, 2, 128, 16, 1, [1, 0, 16, 17, 500], 4, 1, 1),
    (24, 4, 256, 16, 1, [3000, 1601], 30, 1, 2),
    (32, 8, 128, 32, 1, [2000, 4095], 17, 0, 1),
    (24, 4, 256, 64, 5, [1300, 6000], 9, 2, 3),      # thirty rows: two tiles
    (4, 1, 128, 16, 1, [40000], 100, 0, 0),          # 2500 pages
    (16, 1, 128, 16, 2, [20000, 31], 1, 0, 0),       # one page; two row tiles
    (8, 2, 128, 256, 1, [2560, 100], 10, 4, 6),      # all pages, and nothing left to choose
    (2, 2, 256, 16, 1, [1700], 106, 1, 1),           # all but one
]


@pytest.mark.parametrize("hq,hkv,D,ps,L,lengths,budget,sink,recent", CASES)
@pytest.mark.parametrize("mode", ["affine4", "fp16"])
def test_select(mode, hq, hkv, D, ps, L, lengths, budget, sink, recent):
    print(f"case {mode} {hq}/{hkv} D={D} ps={ps} L={L} {lengths} budget={budget}", flush=True)
    r = rng(sum(lengths) + budget)
    s = Sequences(r, mode, hkv, D, ps, lengths, width=-(-max(lengths) // ps) + 3)
    q = queries(r, len(lengths), hq, L, D)
    args = (q, ints(s.table), ints(lengths), budget)
    picked = s.cache.select_pages(*args, sink=sink, recent=recent)
    check_picked(picked, s, q, budget, sink, recent)
    assert torch.equal(picked, s.cache.select_pages(*args, sink=sink, recent=recent))
    out = s.cache.attention(q, ints(s.table), ints(lengths), D ** -0.5, picked=picked)
    if sum(lengths) < 10000:
        s.check(out, q, D ** -0.5, picked=picked.cpu().numpy())


@pytest.mark.parametrize("pages,budget", [(9000, 500), (65536, 2000), (65536, 65535)])
def test_select_of_very_many_pages(pages, budget):
    """A table whose columns name the same few pages over and over: whole runs of equal scores."""
    import qw_amd

    r = rng(pages)
    ps, D = 16, 128
    few = 37
    cache = qw_amd.PagedKVCache("affine8", 1, D, few, page_size=ps)
    k = rows(r, few * ps, 1, D)
    cache.update(dev(k), dev(k), ints([np.arange(few)]), ints([0]))
    table = r.integers(0, few, (1, pages))
    q = queries(r, 1, 4, 1, D)
    picked = cache.select_pages(q, ints(table), ints([pages * ps]), budget, sink=3, recent=2)
    hi, lo, top = (y.reshape(few, -1) for y in bounds(k, ps))
    score = scores_of((hi, lo, top[:, 0]), q[0, :, 0].cpu().numpy())[table[0]]
    assert np.array_equal(picked[0, 0].cpu().numpy(), ranked(score, budget, 3, 2))


@pytest.mark.parametrize("kind", ["same", "zero", "negative", "few", "missing"])
def test_select_of_odd_scores(kind):
    """Ties of all pages, keys of zeros, scores below zero, pages that the table does not name."""
    import qw_amd

    r = rng(3)
    ps, D, n = 32, 128, 40 * 32
    cache = qw_amd.PagedKVCache("int8", 2, D, 41, page_size=ps)
    k = rows(r, n, 2, D)
    if kind == "same":
        k[:] = k[:1]
    elif kind == "zero":
        k[:] = 0
    elif kind == "negative":
        k = -np.abs(k)
    elif kind == "few":
        k = np.sign(k).astype(np.float16) * r.integers(1, 3, (n // ps, 1, 1)).repeat(ps, 0).astype(np.float16)
    table = np.arange(40)[None].copy()
    cache.update(dev(k), dev(k), ints(table), ints([0]))
    q = torch.abs(queries(r, 1, 4, 1, D)) if kind == "negative" else queries(r, 1, 4, 1, D)
    if kind == "missing":
        table[0, ::3] = [-1, 41] * 7
    picked = cache.select_pages(q, ints(table), ints([n]), 30, sink=0, recent=1).cpu().numpy()
    for h in range(2):
        hi, lo, top = (y.reshape(40, -1) for y in bounds(k[:, h:h + 1], ps))
        score = scores_of((hi, lo, top[:, 0]), q[0, 2 * h:2 * h + 2, 0].cpu().numpy())
        if kind == "missing":
            score[::3] = -np.inf
        assert np.array_equal(picked[0, h], ranked(score, 30, 0, 1))
    zeros = cache.select_pages(torch.zeros_like(q), ints(np.arange(40)[None]), ints([n]), 5).cpu().numpy()
    assert np.array_equal(zeros, np.tile(np.arange(5), (1, 2, 1)))


@pytest.mark.parametrize("mode", MODES)
def test_bounds_follow_the_writes(mode):
    """Bounds hold every key since slot 0 was written: they grow with appends and rewrites, and start anew with it."""
    import qw_amd

    r = rng(4)
    ps, D = 16, 128
    cache = qw_amd.PagedKVCache(mode, 1, D, 6, page_size=ps)
    table = ints([np.arange(6)])
    state = [None] * 6
    q = queries(r, 1, 2, 1, D)

    def write(at, n, sigma):
        k = rows(r, n, 1, D, sigma)
        cache.update(dev(k), dev(k), table, ints([at]))
        for p in range(6):
            new = k[max(p * ps - at, 0):max((p + 1) * ps - at, 0), 0]
            if len(new) == 0:
                continue
            hi, lo = new.max(0).astype(np.float32), new.min(0).astype(np.float32)
            if at > p * ps and state[p] is not None:
                hi, lo = np.maximum(hi, state[p][0]), np.minimum(lo, state[p][1])
            state[p] = (hi, lo)

    write(0, 96, 1.0)
    for at, n, sigma in ((17, 3, 2.0), (40, 1, 5.0), (63, 2, 3.0), (80, 16, 0.5), (32, 5, 0.1), (95, 1, 4.0), (0, 20, 0.7)):
        write(at, n, sigma)
        hi, lo, top = coded(np.stack([x[0] for x in state]), np.stack([x[1] for x in state]))
        score = scores_of((hi, lo, top), q[0, :, 0].cpu().numpy())
        for budget in (1, 2, 4):
            picked = cache.select_pages(q, table, ints([96]), budget).cpu().numpy()
            assert np.array_equal(picked[0, 0], ranked(score, budget, 0, 0)), (at, budget)


def test_select_refusals():
    import qw_amd

    r = rng(50)
    s = Sequences(r, "fp16", 2, 128, 16, [40])
    q = queries(r, 1, 4, 1, 128)
    t, n = ints(s.table), ints([40])
    for budget, sink, recent in ((0, 0, 0), (3, 2, 2), (3, -1, 0), (3, 0, -1), (2 ** 40, 0, 0), (-1, 0, 0)):
        with pytest.raises(qw_amd.QwError):
            s.cache.select_pages(q, t, n, budget, sink=sink, recent=recent)
    with pytest.raises(qw_amd.QwError):
        s.cache.select_pages(q, t.repeat(1, 30000), n, 3)
    assert torch.all(s.cache.select_pages(q, t[:, :0], n, 3) == -1)
    z = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    assert s.cache.select_pages(q[:0], z, z[:, 0].contiguous(), 3).shape == (0, 2, 3)


@pytest.mark.parametrize("mode", MODES)
def test_a_layer_step_after_step(mode):
    """Three sequences decode: rotate and store the new token, pick pages, attend them, against the same by parts."""
    import qw_amd

    r = rng(60)
    hq, hkv, D, ps, B = 8, 2, 128, 16, 3
    lengths = [100, 7, 250]
    s = Sequences(r, mode, hkv, D, ps, lengths, width=20)
    table = s.table.copy()
    spare = [p for p in range(s.n_pages) if p not in table]
    sections = (8, 12, 12)
    for step in range(12):
        qkv = dev(r.standard_normal((B, (hq + 2 * hkv) * D)).astype(np.float16))
        pos = ints(np.array([lengths, [n + 3 for n in lengths], [2 * n for n in lengths]]))
        for b in range(B):
            if lengths[b] % ps == 0 and table[b, lengths[b] // ps] < 0:
                table[b, lengths[b] // ps] = spare.pop()
        q1, k1 = qw_amd.rope_axes(qkv, pos, sections, hq, hkv, D, 1e4, interleaved=True)
        q = s.cache.rope_update(qkv, pos, sections, hq, 1e4, ints(table), ints(lengths), interleaved=True)
        assert torch.equal(q, q1)
        v1 = qkv.view(B, hq + 2 * hkv, D)[:, hq + hkv:]
        for b in range(B):
            s.k[b] = np.concatenate([s.k[b], k1[b:b + 1].cpu().numpy()])
            s.v[b] = np.concatenate([s.v[b], v1[b:b + 1].cpu().numpy()])
            lengths[b] += 1
        s.lengths = list(lengths)
        s.table = table
        qq = q.view(B, 1, hq, D).transpose(1, 2)
        picked = s.cache.select_pages(qq, ints(table), ints(lengths), 5, sink=1, recent=1)
        check_picked(picked, s, qq, 5, 1, 1)
        out = s.cache.attention(qq, ints(table), ints(lengths), 0.09, picked=picked)
        s.check(out, qq, 0.09, picked=picked.cpu().numpy())


@pytest.mark.parametrize("mode", ["affine4", "fp16"])
def test_a_step_in_a_graph(mode):
    """A step captured once serves growing sequences: lengths, tables and tokens are read at each replay."""
    import qw_amd

    r = rng(61)
    hq, hkv, D, ps, B = 8, 2, 128, 16, 2
    lengths = [300, 90]
    s = Sequences(r, mode, hkv, D, ps, lengths, width=24)
    table, pos, n, starts = ints(s.table), ints(np.zeros((3, B))), ints(lengths), ints(lengths)
    qkv = dev(r.standard_normal((B, (hq + 2 * hkv) * D)).astype(np.float16))

    def step(cache):
        q = cache.rope_update(qkv, pos, (8, 12, 12), hq, 1e4, table, starts)
        q = q.view(B, 1, hq, D).transpose(1, 2)
        picked = cache.select_pages(q, table, n, 6, sink=1, recent=1)
        return picked, cache.attention(q, table, n, 0.09, picked=picked), cache.attention(q, table, n, 0.09)

    spare = [p for p in range(s.n_pages) if p not in s.table]
    s.table[0, 19], s.table[1, 6] = spare[:2]
    table.copy_(ints(s.table))
    stream = side_stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        n.add_(1)
        step(s.cache)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = step(s.cache)
    for turn in range(4):
        qkv.copy_(dev(r.standard_normal(qkv.shape).astype(np.float16)))
        pos.add_(7)
        g.replay()
        torch.cuda.synchronize()
        want = step(s.cache)  # the same tokens again, eagerly: a slot may be written again
        for x, y in zip(got, want):
            assert torch.equal(x, y), turn
        starts.add_(1)
        n.add_(1)
        _ = (qkv.float() * 2).sum().item()


def test_two_streams_and_threads():
    """Calls of two host threads on streams of their own over one pool's pages give what they give alone."""
    import threading

    r = rng(62)
    s = Sequences(r, "affine8", 2, 256, 32, [700, 1500])
    args = []
    for b in range(2):
        q = queries(r, 1, 12, 1, 256)
        t, n = ints(s.table[b:b + 1]), ints([s.lengths[b]])
        args.append((q, t, n, s.cache.select_pages(q, t, n, 9, recent=1), s.cache.attention(q, t, n, 1 / 16)))
    torch.cuda.synchronize()
    wrong, streams = [], [side_stream(2), side_stream(3)]

    def work(b):
        q, t, n, picked, out = args[b]
        stream = streams[b]
        with torch.cuda.stream(stream):
            for _ in range(30):
                p = s.cache.select_pages(q, t, n, 9, recent=1)
                o = s.cache.attention(q, t, n, 1 / 16)
                stream.synchronize()
                if not (torch.equal(p, picked) and torch.equal(o, out)):
                    wrong.append(b)

    threads = [threading.Thread(target=work, args=(b,)) for b in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
