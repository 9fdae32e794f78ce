"""Pages of a pool (qw_paged_*): what is written and read back against a cache of one sequence, bit for bit, and
attention over pages against 64-bit softmax attention on the codes' unrounded values.

The bar of an attention output, from the kernel's roundings (u = 2^-11, half a step of fp16; e = 2^-24), with code
values c s + b, A = sum p (|c s| + |b|) and L = sum e^(s - max s):
  a weight, or a weight times a key's scale, is rounded to fp16 once, at most u of itself or, below fp16's normal
  numbers, half its step 2^-25; the kernel holds weights at 2^11 at its reference, which lies at most 4 (log2) below
  the largest score: as a share of the row's largest weight 2^-25 / 2^11, times a code (255 at most) where it was
  multiplied by a scale: 2^-28 of the scale's unit for every key;
  the output is rounded, u of itself; a score's sums in fp32, at most g = (D + 40) e |scale| sum |q| H, which
  scales a weight by 1 + g and the row's sum alike, and the output's at most (n / 32 + 40) e sum p H, with H the
  magnitudes that are summed: |c s| + |b|, and of int8, whose codes are held 128 above their value and lose
  that again in fp32, |c s| + 256 s:
  |error| <= (u + 2 g) A + (n / 32 + 40) e sum p H + u |out| + 2^-25 + sum over keys of 2^-28 max(1, |s|) / L."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U, E = 2.0 ** -11, 2.0 ** -24
MODES = ["fp16", "affine8", "affine4", "int8"]


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def ints(x):
    return dev(np.asarray(x, dtype=np.int32))


def make_table(r, pages, width, n_pages, bad=-1):
    """Pages in random order; `bad` behind each sequence's last."""
    perm = r.permutation(n_pages)
    t = np.full((len(pages), width), bad, dtype=np.int32)
    at = 0
    for b, n in enumerate(pages):
        t[b, :n] = perm[at:at + n]
        at += n
    return t


def codes_of(words, bits, d):
    w = words.cpu().numpy().view(np.uint32)
    c = np.stack([(w >> s) & ((1 << bits) - 1) for s in range(0, 32, bits)], -1)
    return c.reshape(*w.shape[:-1], d)


def unrounded(mode, k, hkv, D):
    """[T, hkv, D] fp16 rows as one sequence's cache holds them: values, magnitudes A and H in 64 bits, [hkv, T, D] each."""
    import qw_amd

    c = qw_amd.KVCache(mode, hkv, D)
    x = dev(k.transpose(1, 0, 2))
    c.update(x, x)
    t = c.snapshot_tensors()
    if mode == "fp16":
        y = t["keys"].double().cpu().numpy()
        return y, np.abs(y), np.abs(y)
    if mode == "int8":
        s = t["key_scales"].double().cpu().numpy()
        y = t["keys"].double().cpu().numpy() * s
        return y, np.abs(y), np.abs(y) + 256 * s
    s, b = (np.repeat(t[n].double().cpu().numpy(), 64, -1) for n in ("k_scales", "k_biases"))
    y = codes_of(t["k_codes"], c.bits, D) * s
    return y + b, np.abs(y) + np.abs(b), np.abs(y) + np.abs(b)


def stored(mode, k, v, hkv, D):
    """What a cache of one sequence gives back of [T, hkv, D] rows."""
    import qw_amd

    c = qw_amd.KVCache(mode, hkv, D)
    c.update(dev(k.transpose(1, 0, 2)), dev(v.transpose(1, 0, 2)))
    return tuple(x[0].cpu().numpy().transpose(1, 0, 2) for x in c.dequantize())


def rows(r, n, hkv, D, sigma=1.0):
    return (sigma * r.standard_normal((n, hkv, D))).astype(np.float16)


def side_stream(i=0):
    """A stream of torch's, which hands its 32 out in turn. A workspace that a graph holds stays its stream's: a whole turn
    leaves the tests behind this one the streams that they had. The same for the same i."""
    return sorted((torch.cuda.Stream() for _ in range(32)), key=lambda s: s.cuda_stream)[i]


class Sequences:
    """Random sequences of the given lengths in a pool, with a spare page of NaN-free rubbish."""

    def __init__(self, r, mode, hkv, D, ps, lengths, sigma=1.0, width=None, bad=-1):
        import qw_amd

        self.mode, self.hkv, self.D, self.ps, self.lengths = mode, hkv, D, ps, list(lengths)
        pages = [-(-n // ps) for n in lengths]
        self.n_pages = sum(pages) + 3
        self.width = max(pages + [1]) if width is None else width
        self.table = make_table(r, pages, self.width, self.n_pages, bad)
        self.cache = qw_amd.PagedKVCache(mode, hkv, D, self.n_pages, page_size=ps)
        self.k = [rows(r, n, hkv, D, sigma) for n in lengths]
        self.v = [rows(r, n, hkv, D, sigma) for n in lengths]
        n = sum(lengths)
        if n:
            offsets = np.concatenate([[0], np.cumsum(lengths)])
            self.cache.update(dev(np.concatenate(self.k)), dev(np.concatenate(self.v)), ints(self.table),
                              ints([0] * len(lengths)), offsets=ints(offsets))

    def check(self, out, q, scale, lengths=None, picked=None):
        out, q = out.double().cpu().numpy(), q.double().cpu().numpy()
        B, hq, L, D = q.shape
        worst = 0.0
        for b in range(B):
            n = self.lengths[b] if lengths is None else min(max(lengths[b], 0), self.lengths[b])
            if n:
                k, v = (unrounded(self.mode, x[b], self.hkv, D) for x in (self.k, self.v))
            for j in range(hq):
                h = j // (hq // self.hkv)
                for i in range(L):
                    at = np.arange(max(n - L + i + 1, 0))
                    if picked is not None:
                        at = at[np.isin(at // self.ps, picked[b, h])]
                    if len(at) == 0:
                        assert np.all(out[b, j, i] == 0), (b, j, i)
                        continue
                    kk, kh, vv, va, vh = k[0][h, at], k[2][h, at], v[0][h, at], v[1][h, at], v[2][h, at]
                    s = (kk @ q[b, j, i]) * scale
                    p = np.exp(s - s.max())
                    total = p.sum()
                    ref = p @ vv / total
                    g = (D + 40) * E * abs(scale) * (kh @ np.abs(q[b, j, i])).max()
                    sv = np.abs(va).max()
                    bar = (U + 2 * g) * (p @ va) / total + (len(at) / 32 + 40) * E * (p @ vh) / total + U * np.abs(ref) + 2.0 ** -25 + len(at) * 2.0 ** -28 * max(1.0, sv) / total
                    err = np.abs(out[b, j, i] - ref) / bar
                    assert np.isfinite(out[b, j, i]).all() and err.max() <= 1.0, (b, j, i, err.max())
                    worst = max(worst, err.max())
        print(f"worst error {worst:.2f} of the bar", flush=True)


def queries(r, B, hq, L, D, sigma=2.0):
    return dev((sigma * r.standard_normal((B, hq, L, D))).astype(np.float16))


# ------------------------------------------------------------------ store


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hkv,D,ps", [(4, 256, 16), (2, 128, 16), (3, 128, 64), (1, 256, 256), (8, 128, 32), (2, 256, 128)])
def test_rows_come_back_as_a_cache_gives_them(mode, hkv, D, ps):
    """Ragged sequences written in pieces that begin and end inside pages and inside blocks of 8."""
    import qw_amd

    print(f"case {mode} hkv={hkv} D={D} ps={ps}", flush=True)
    r = rng(ps + D + hkv)
    lengths = [1, 7, 8, ps, ps + 1, 2 * ps - 1, 3 * ps + 5]
    pages = [-(-n // ps) for n in lengths]
    n_pages = sum(pages) + 2
    table = ints(make_table(r, pages, max(pages) + 1, n_pages))
    cache = qw_amd.PagedKVCache(mode, hkv, D, n_pages, page_size=ps)
    k, v = ([rows(r, n, hkv, D) for n in lengths] for _ in range(2))
    done = np.zeros(len(lengths), dtype=int)
    while (done < lengths).any():
        step = np.minimum(r.integers(0, ps + 3, len(lengths)), np.array(lengths) - done)
        if step.sum() == 0:
            continue
        offsets = np.concatenate([[0], np.cumsum(step)])
        kn, vn = (np.concatenate([x[b][done[b]:done[b] + step[b]] for b in range(len(lengths))]) for x in (k, v))
        cache.update(dev(kn), dev(vn), table, ints(done), offsets=ints(offsets))
        done += step
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    gk, gv = cache.gather(table, ints([0] * len(lengths)), int(offsets[-1]), offsets=ints(offsets))
    for b, n in enumerate(lengths):
        want = stored(mode, k[b], v[b], hkv, D)
        for got, ref in zip((gk, gv), want):
            assert np.array_equal(got[offsets[b]:offsets[b + 1]].cpu().numpy().view(np.uint16), ref.view(np.uint16)), (b, n)
    # a middle part of each, equal counts
    starts = [max(0, n - 5) for n in lengths]
    gk, gv = cache.gather(table, ints(starts), 5 * len(lengths))
    for b, n in enumerate(lengths):
        want = stored(mode, k[b], v[b], hkv, D)
        m = min(5, n)
        assert np.array_equal(gk[5 * b:5 * b + m].cpu().numpy(), want[0][-m:]) and np.array_equal(gv[5 * b:5 * b + m].cpu().numpy(), want[1][-m:])


@pytest.mark.parametrize("mode", MODES)
def test_slots_of_no_token_stay(mode):
    """A write of one slot leaves its page's other slots, and every other page, as they were; a rewrite replaces."""
    import qw_amd

    r = rng(7)
    hkv, D, ps = 2, 128, 32
    cache = qw_amd.PagedKVCache(mode, hkv, D, 4, page_size=ps)
    all_pages = ints([[0, 1, 2, 3]])
    k, v = rows(r, 4 * ps, hkv, D), rows(r, 4 * ps, hkv, D)
    cache.update(dev(k), dev(v), all_pages, ints([0]))
    for at, n in ((37, 1), (40, 8), (63, 2), (95, 1)):
        kn, vn = rows(r, n, hkv, D), rows(r, n, hkv, D)
        cache.update(dev(kn), dev(vn), all_pages, ints([at]))
        k[at:at + n], v[at:at + n] = kn, vn
        got = cache.gather(all_pages, ints([0]), 4 * ps)
        for x, y in zip(got, stored(mode, k, v, hkv, D)):
            assert np.array_equal(x.cpu().numpy().view(np.uint16), y.view(np.uint16)), (at, n)


@pytest.mark.parametrize("mode", ["affine4", "fp16"])
def test_places_outside_the_pool(mode):
    """Tokens of no page are dropped and read as zeros; tokens behind the table too; rows of no sequence stay."""
    import qw_amd

    r = rng(8)
    hkv, D, ps = 2, 256, 16
    cache = qw_amd.PagedKVCache(mode, hkv, D, 3, page_size=ps)
    k, v = rows(r, 80, hkv, D), rows(r, 80, hkv, D)
    table = ints([[0, 3, 1, -5]])  # pages 3 and -5 are none
    cache.update(dev(k), dev(v), table, ints([0]))
    gk, gv = cache.gather(table, ints([0]), 80)
    wk, wv = stored(mode, k, v, hkv, D)
    for got, want in ((gk, wk), (gv, wv)):
        want = want.copy()
        want[16:32] = 0
        want[48:] = 0
        assert np.array_equal(got.cpu().numpy(), want)
    other = cache.gather(ints([[2]]), ints([0]), 16)
    assert all(torch.all(x == 0) for x in other)
    # no tokens, and a sequence of none between others
    cache.update(dev(k[:0]), dev(v[:0]), table, ints([0]))
    two = ints([[2], [1], [0]])
    cache.update(dev(k[:3]), dev(v[:3]), two, ints([0, 4, 1]), offsets=ints([0, 2, 2, 3]))
    got = cache.gather(two, ints([0, 4, 1]), 3, offsets=ints([0, 2, 2, 3]))
    assert np.array_equal(got[0].cpu().numpy(), stored(mode, k[:3], v[:3], hkv, D)[0])


def test_strided_rows_and_tables():
    """Rows inside a projection, a table inside a larger one."""
    import qw_amd

    r = rng(9)
    hq, hkv, D, ps, n = 4, 2, 128, 16, 40
    qkv = dev(r.standard_normal((n, (hq + 2 * hkv) * D)).astype(np.float16))
    x = qkv.view(n, hq + 2 * hkv, D)
    k, v = x[:, hq:hq + hkv], x[:, hq + hkv:]
    big = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    big[:, 2:4] = ints([[3, 0], [2, 1]])
    for table in (big[:, 2:4], big[:, 2:4].t().contiguous().t()):
        cache = qw_amd.PagedKVCache("affine8", hkv, D, 4, page_size=ps)
        cache.update(k, v, table, ints([0, 0]))
        got = cache.gather(table, ints([0, 0]), n)
        want = stored("affine8", k.cpu().numpy(), v.cpu().numpy(), hkv, D)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
        q = queries(r, 2, hq, 1, D)
        strided = torch.empty((2, 1, hq, D), dtype=torch.float16, device="cuda").transpose(1, 2)
        strided.copy_(q)
        lengths = ints([20, 20])
        assert torch.equal(cache.attention(q, table, lengths, 0.1), cache.attention(strided, table, lengths, 0.1))


# ------------------------------------------------------------------ attention

CASES = [
    # hq, hkv, D, page, rows, lengths
    (8, 2, 128, 16, 1, [1]),
    (24, 4, 256, 16, 1, [0, 1, 15, 16, 17, 300]),
    (24, 4, 256, 64, 1, [127, 128, 129, 5, 700]),
    (32, 8, 128, 32, 1, [1000, 33, 2049]),
    (8, 8, 128, 128, 1, [513, 128]),
    (4, 2, 256, 256, 1, [255, 257, 1000]),
    (24, 4, 256, 32, 5, [200, 5, 3, 0, 64]),          # two row tiles; fewer keys than rows
    (12, 1, 256, 16, 3, [400, 37]),                   # three row tiles
    (16, 1, 128, 64, 1, [65, 640]),                   # a whole row tile
    (16, 2, 128, 16, 8, [90, 1200]),
    (2, 2, 128, 16, 17, [100, 9]),                    # seventeen rows
]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hq,hkv,D,ps,L,lengths", CASES)
def test_attention(mode, hq, hkv, D, ps, L, lengths):
    print(f"case {mode} {hq}/{hkv} D={D} ps={ps} L={L} {lengths}", flush=True)
    r = rng(sum(lengths) + D + L)
    s = Sequences(r, mode, hkv, D, ps, lengths, width=max(-(-max(lengths) // ps), 1) + 2)
    q = queries(r, len(lengths), hq, L, D)
    out = s.cache.attention(q, ints(s.table), ints(lengths), D ** -0.5)
    s.check(out, q, D ** -0.5)
    # fewer keys than the pages hold, and lengths past the table or below 0
    odd = [max(n - 3 - i, -1) for i, n in enumerate(lengths)]
    out = s.cache.attention(q, ints(s.table), ints(odd), D ** -0.5)
    s.check(out, q, D ** -0.5, lengths=odd)


@pytest.mark.parametrize("mode", MODES)
def test_attention_long_and_many(mode):
    """Pieces of one sequence from many workers, and many sequences in one worker's run."""
    r = rng(21)
    s = Sequences(r, mode, 1, 128, 16, [20011])
    q = queries(r, 1, 4, 1, 128)
    s.check(s.cache.attention(q, ints(s.table), ints([20011]), 0.09), q, 0.09)
    lengths = [int(x) for x in r.integers(0, 60, 300)]
    s = Sequences(r, mode, 1, 128, 16, lengths)
    q = queries(r, 300, 2, 1, 128)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.09), q, 0.09)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("sigma,scale", [(100.0, 1e-4), (1e-3, 90.0), (1.0, 0.0), (1.0, -0.06), (8.0, 0.3), (2000.0, 1e-6)])
def test_attention_of_odd_ranges(mode, sigma, scale):
    """Values whose scales pass 1 (P gives way) or lie far below it, peaked and flat softmaxes, scores of both signs."""
    r = rng(int(sigma) + 5)
    lengths = [130, 400]
    s = Sequences(r, mode, 2, 256, 16, lengths, sigma=sigma)
    # one page's values are larger than the others', late in the sequence
    big = rows(r, 16, 2, 256, min(50 * sigma, 8000.0))
    s.cache.update(dev(s.k[1][352:368]), dev(big), ints(s.table[1:]), ints([352]))
    s.v[1][352:368] = big
    q = queries(r, 2, 8, 1, 256)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), scale), q, scale)


@pytest.mark.parametrize("mode", MODES)
def test_what_stands_behind_the_end_takes_no_part(mode):
    """NaN and infinities in slots behind a sequence's end and in pages of others."""
    r = rng(31)
    ps, D = 32, 128
    s = Sequences(r, mode, 2, D, ps, [70, 33])
    rubbish = np.full((26, 2, D), np.nan, dtype=np.float16)
    rubbish[::2] = np.inf
    q = queries(r, 2, 8, 1, D)
    want = s.cache.attention(q, ints(s.table), ints([70, 33]), 0.1)
    s.cache.update(dev(rubbish), dev(rubbish), ints(s.table[:1]), ints([70]))
    s.cache.update(dev(rubbish), dev(rubbish), ints(s.table[1:]), ints([33]))
    out = s.cache.attention(q, ints(s.table), ints([70, 33]), 0.1)
    s.check(out, q, 0.1)
    if mode in ("fp16",):
        assert torch.equal(out, want)


@pytest.mark.parametrize("mode", ["affine4", "fp16"])
@pytest.mark.parametrize("ps", [16, 64])
def test_missing_pages_are_skipped(mode, ps):
    r = rng(33)
    s = Sequences(r, mode, 2, 128, ps, [6 * ps, 3 * ps + 1], bad=2 ** 30)
    table = s.table.copy()
    table[0, 2] = -1
    table[1, 0] = s.n_pages
    q = queries(r, 2, 8, 1, 128)
    out = s.cache.attention(q, ints(table), ints(s.lengths), 0.1)
    picked = np.full((2, 2, 5), -1)
    picked[0, :] = [0, 1, 3, 4, 5]
    picked[1, :, :3] = [1, 2, 3]
    s.check(out, q, 0.1, picked=picked)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("ps,L", [(16, 1), (64, 1), (16, 6)])
def test_attention_over_picked_pages(mode, ps, L):
    """Lists of each head its own, shorter and longer than its pages, with entries that name none, in any order."""
    r = rng(40 + ps + L)
    hkv, D = 2, 256
    lengths = [20 * ps - 3, 5 * ps + 1, 2, 0]
    s = Sequences(r, mode, hkv, D, ps, lengths)
    n = 7
    picked = np.full((4, hkv, n), -1, dtype=np.int32)
    for b, length in enumerate(lengths):
        pages = -(-length // ps)
        for h in range(hkv):
            m = min(n, pages)
            picked[b, h, :m] = r.permutation(pages)[:m]
    picked[0, 1, 3] = -1
    picked[0, 1, 5] = s.width + 7
    q = queries(r, 4, 6, L, D)
    out = s.cache.attention(q, ints(s.table), ints(lengths), 1 / 16, picked=ints(picked))
    s.check(out, q, 1 / 16, picked=picked)


def test_refusals():
    import qw_amd

    r = rng(50)
    s = Sequences(r, "affine8", 2, 128, 16, [40])
    q = queries(r, 1, 4, 1, 128)
    t, n = ints(s.table), ints([40])
    k = dev(s.k[0])
    bad = [
        lambda: s.cache.attention(q, t, n, float("nan")),
        lambda: s.cache.attention(q, t, n, 2.0 ** 41),
        lambda: s.cache.attention(q[:, :3], t, n, 0.1),
        lambda: s.cache.attention(q.float(), t, n, 0.1),
        lambda: s.cache.attention(q, t.long(), n, 0.1),
        lambda: s.cache.attention(q, t.cpu(), n, 0.1),
        lambda: s.cache.attention(q, t, n[:0], 0.1),
        lambda: s.cache.attention(q, t, n, 0.1, picked=torch.zeros((1, 2, 0), dtype=torch.int32, device="cuda")),
        lambda: s.cache.attention(q, t, n, 0.1, picked=torch.zeros((1, 4, 2), dtype=torch.int32, device="cuda")),
        lambda: s.cache.attention(q.expand(1, 4, 1, 128).repeat(2, 1, 1, 1), t, n, 0.1),
        lambda: s.cache.attention(torch.zeros((1, 4, 9000, 128), dtype=torch.float16, device="cuda"), t, n, 0.1),
        lambda: s.cache.update(k, k[:3], t, ints([0])),
        lambda: s.cache.update(k[:, :1], k[:, :1], t, ints([0])),
        lambda: s.cache.update(k[:3], k[:3], t.repeat(2, 1), ints([0, 0])),
        lambda: s.cache.update(k, k, t, ints([0]), offsets=ints([0])),
        lambda: s.cache.update(k, k, t[:, :0], ints([0])),
        lambda: s.cache.gather(t, ints([0]), -1),
        lambda: qw_amd.PagedKVCache("turbo4", 2, 128, 4),
        lambda: qw_amd.PagedKVCache("fp16", 2, 64, 4),
        lambda: qw_amd.PagedKVCache("fp16", 2, 128, 4, page_size=48),
        lambda: qw_amd.PagedKVCache("affine4", 2, 128, 4, group_size=32),
        lambda: qw_amd.PagedKVCache("fp16", 2, 128, 0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((qw_amd.QwError, RuntimeError)):
            f()
            print("not refused:", i)
    closed = qw_amd.PagedKVCache("fp16", 2, 128, 4)
    closed.close()
    with pytest.raises(qw_amd.QwError):
        closed.attention(q, t, n, 0.1)
    assert s.cache.nbytes() > 0
    # nothing to do
    e = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    z = torch.zeros((0,), dtype=torch.int32, device="cuda")
    assert s.cache.attention(q[:0], e, z, 0.1).shape == (0, 4, 1, 128)
    s.cache.update(k[:0], k[:0], e, z)
    assert torch.all(s.cache.attention(q, t[:, :0], n, 0.1) == 0)  # a table without columns


@pytest.mark.parametrize("mode", MODES)
def test_odd_rows_are_stored_as_a_cache_stores_them(mode):
    """Zeros, constants, the smallest and the largest numbers, one number among zeros, negative rows."""
    import qw_amd

    r = rng(70)
    hkv, D, ps = 2, 128, 16
    x = rows(r, 40, hkv, D)
    x[0] = 0
    x[1] = 1.5
    x[2] = 2.0 ** -24
    x[3] = r.integers(0, 9, x[3].shape) * 2.0 ** -24
    x[4] = 65504
    x[5] = 65504 * np.sign(r.standard_normal(x[5].shape))
    x[6] = 0
    x[6, :, 77] = -3e-5
    x[7] = -np.abs(x[7])
    x[8] = np.abs(x[8]) * 1e-6
    x[9, :, :64] = 0
    x[10] = np.float16(2.0 ** -14) * (1 + r.integers(0, 3, x[10].shape))
    x[11:30] = (r.standard_normal((19, hkv, D)) * 10.0 ** r.uniform(-6, 4, (19, 1, 1))).astype(np.float16)
    y = x[::-1].copy()
    cache = qw_amd.PagedKVCache(mode, hkv, D, 3, page_size=ps)
    t = ints([[2, 0, 1]])
    cache.update(dev(x), dev(y), t, ints([0]))
    got = cache.gather(t, ints([0]), 40)
    for a, b in zip(got, stored(mode, x, y, hkv, D)):
        assert np.array_equal(a.cpu().numpy().view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("mode", ["affine8", "fp16"])
@pytest.mark.parametrize("hq,hkv,n_seq,most,L", [(2, 2, 64, 700, 1), (2, 2, 65, 400, 1), (32, 32, 40, 300, 1), (16, 2, 3, 900, 9), (3, 1, 70, 120, 1)])
def test_attention_of_ragged_batches(mode, hq, hkv, n_seq, most, L):
    """Batches at the line of the lane-held plan, with sequences without keys among them; rows in many tiles; short ones."""
    r = rng(n_seq + most)
    lengths = [int(x) for x in r.integers(0, most, n_seq)]
    lengths[::7] = [0] * len(lengths[::7])
    lengths[-1] = most
    s = Sequences(r, mode, hkv, 128, 16, lengths)
    q = queries(r, n_seq, hq, L, 128)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.09), q, 0.09)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("D", [128, 256])
def test_short_sequences_stay_whole(mode, D):
    """Around the lengths up to which no sequence is cut."""
    r = rng(D)
    for lengths in ([5, 0, 128], [129, 256, 0], [384, 385, 1], [512, 100], [513], [640, 0], [641]):
        s = Sequences(r, mode, 2, D, 16, lengths)
        q = queries(r, len(lengths), 8, 1, D)
        s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.09), q, 0.09)


@pytest.mark.parametrize("mode", ["fp16", "affine8"])
def test_a_pool_past_32_bits(mode):
    """Pages whose bytes, and whose rows, lie past 2^32 in the pool's planes."""
    import qw_amd

    r = rng(71)
    hkv, D, ps = 8, 256, 256
    n_pages = 4300 if mode == "fp16" else 8500  # 1 MB, or half of it, a page in each plane
    cache = qw_amd.PagedKVCache(mode, hkv, D, n_pages, page_size=ps)
    small = qw_amd.PagedKVCache(mode, hkv, D, 3, page_size=ps)
    k, v = rows(r, 700, hkv, D), rows(r, 700, hkv, D)
    far, near, zero = ints([[n_pages - 1, n_pages - 3, n_pages - 2]]), ints([[0, 2, 1]]), ints([0])
    q, n = queries(r, 1, 16, 1, D), ints([700])
    for c, t in ((cache, far), (small, near)):
        c.update(dev(k), dev(v), t, zero)
    for x, y in zip(cache.gather(far, zero, 700), small.gather(near, zero, 700)):
        assert torch.equal(x, y)
    assert torch.equal(cache.attention(q, far, n, 1 / 16), small.attention(q, near, n, 1 / 16))
    assert torch.equal(cache.select_pages(q, far, n, 2), small.select_pages(q, near, n, 2))
    assert all(torch.all(x == 0) for x in cache.gather(ints([[0, 1]]), zero, 512))


def test_stream_per_thread_is_refused():
    """One handle for a stream a thread: the calls that keep a workspace of their stream name it as unsupported."""
    import qw_amd

    r = rng(72)
    s = Sequences(r, "fp16", 2, 128, 16, [40])
    q, out = queries(r, 1, 4, 1, 128), torch.empty((1, 4, 1, 128), dtype=torch.float16, device="cuda")
    t, n = ints(s.table), ints([40])
    picked = ints(np.zeros((1, 2, 3)))
    args = (s.cache._h, q.data_ptr(), 512, 128, 128, 1, 4, 1, n.data_ptr(), t.data_ptr(), 3, 3)
    assert qw_amd.lib().qw_paged_attention(*args, None, 0, 0.1, out.data_ptr(), 2) == 2
    assert qw_amd.lib().qw_paged_select(*args, 2, 0, 0, picked.data_ptr(), 2) == 2


def test_first_use_inside_a_capture():
    """A call that has to make its workspace is refused while its stream is captured, and the capture goes on."""
    import qw_amd

    r = rng(73)
    s = Sequences(r, "affine4", 2, 128, 16, [3000])
    q, t, n = queries(r, 1, 8, 1, 128), ints(s.table), ints([3000])
    want = s.cache.attention(q, t, n, 0.1)
    stream = side_stream(1)
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    refused = False
    x = torch.zeros(8, device="cuda")
    with torch.cuda.graph(g, stream=stream):
        try:
            s.cache.attention(q, t, n, 0.1)
        except qw_amd.QwError as e:
            refused = e.status == 5
        x.add_(1)
    g.replay()
    torch.cuda.synchronize()
    assert refused and torch.all(x == 1)
    assert torch.equal(s.cache.attention(q, t, n, 0.1), want)


@pytest.mark.parametrize("mode,hq,hkv,n_seq", [("int8", 4, 2, 130), ("affine4", 2, 2, 300), ("fp16", 40, 2, 65)])
def test_many_sequences_of_which_few_are_long(mode, hq, hkv, n_seq):
    """More than a wave's lanes: runs that end in a long sequence, begin with one, or hold many, empty ones among them."""
    r = rng(n_seq)
    lengths = [int(x) for x in r.integers(0, 40, n_seq)]
    lengths[3], lengths[64], lengths[n_seq - 1] = 5000, 2611, 1500
    lengths[4:20] = [0] * 16
    lengths[5] = 256
    s = Sequences(r, mode, hkv, 128, 16, lengths)
    q = queries(r, n_seq, hq, 1, 128)
    out = s.cache.attention(q, ints(s.table), ints(lengths), 0.09)
    s.check(out, q, 0.09)
    assert torch.equal(s.cache.attention(q, ints(s.table), ints(lengths), 0.09), out)
    none = s.cache.attention(q, ints(s.table), ints([0] * n_seq), 0.09)
    assert torch.all(none == 0)
    none = s.cache.attention(q, ints(s.table)[:, :0], ints(lengths), 0.09)
    assert torch.all(none == 0)


@pytest.mark.parametrize("n_seq", [65, 127, 200, 1000])
def test_stores_of_many_sequences(n_seq):
    """More sequences than a wave's lanes, most of them with no token."""
    import qw_amd

    r = rng(n_seq)
    hkv, D, ps = 2, 128, 16
    n = [int(x) if r.random() < 0.3 else 0 for x in r.integers(1, 25, n_seq)]
    n[-1] = 17
    starts = [int(x) for x in r.integers(0, 20, n_seq)]
    width = 3
    cache = qw_amd.PagedKVCache("affine8", hkv, D, n_seq * width, page_size=ps)
    table = ints(r.permutation(n_seq * width).reshape(n_seq, width))
    k, v = rows(r, sum(n), hkv, D), rows(r, sum(n), hkv, D)
    offsets = ints(np.concatenate([[0], np.cumsum(n)]))
    cache.update(dev(k), dev(v), table, ints(starts), offsets)
    got = cache.gather(table, ints(starts), sum(n), offsets)
    for a, b in zip(got, stored("affine8", k, v, hkv, D)):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("mode", MODES)
def test_values_of_one_sign(mode):
    """Values of 0 and more: a V group's middle lies far from many of them. Its weights' rounding meets a code's distance from
    the middle, at most c0 scale <= 1.004 * the group's largest value / 2 * 2, and the middle itself twice (the weights'
    rounding and its own): 3.02 U of the group's largest value for each key, and the result's rounding."""
    r = rng(90)
    D, n = 128, 300
    s = Sequences(r, mode, 1, D, 16, [n])
    v = np.maximum(rows(r, n, 1, D), 0)
    v[:, :, 5] = 0
    s.cache.update(dev(s.k[0]), dev(v), ints(s.table), ints([0]))
    s.v = [v]
    q = queries(r, 1, 4, 1, D)
    out = s.cache.attention(q, ints(s.table), ints([n]), 0.09).double().cpu().numpy()
    k, vv = unrounded(mode, s.k[0], 1, D), unrounded(mode, v, 1, D)
    big = np.repeat(np.abs(v[:, 0]).astype(np.float64).reshape(n, D // 64, 64).max(2), 64, axis=1)
    for j in range(4):
        x = q[0, j, 0].double().cpu().numpy()
        sc = (k[0][0] @ x) * 0.09
        p = np.exp(sc - sc.max())
        g = (D + 40) * E * 0.09 * (k[2][0] @ np.abs(x)).max()
        ref = p @ vv[0][0] / p.sum()
        bar = (3.02 * U + 2 * g + 60 * E) * (p @ big) / p.sum() + U * np.abs(ref) + 2.0 ** -25 + n * 2.0 ** -28 / p.sum()
        assert (np.abs(out[0, j, 0] - ref) <= bar).all()


@pytest.mark.parametrize("mode,D,n_seq,most", [("affine8", 128, 300, 1024), ("affine4", 256, 270, 640), ("fp16", 128, 129, 1100)])
def test_more_sequences_than_workers(mode, D, n_seq, most):
    """A worker's several sequences, one behind the other, whole (up to 8 rounds) or in runs."""
    r = rng(n_seq + D)
    lengths = [int(x) for x in r.integers(0, 60, n_seq)]
    lengths[0], lengths[128], lengths[n_seq - 1] = most, most - 3, 129
    lengths[7:11] = [0] * 4
    s = Sequences(r, mode, 4, D, 16, lengths)
    q = queries(r, n_seq, 4, 1, D)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.07), q, 0.07)


@pytest.mark.parametrize("mode", ["int8", "affine4"])
def test_a_page_named_twice_counts_twice(mode):
    """In a list of pages and in the table, as the same keys stored twice would."""
    r = rng(91)
    hkv, D, ps, scale = 2, 128, 16, 0.09
    s = Sequences(r, mode, hkv, D, ps, [6 * ps])
    q = queries(r, 1, 4, 1, D)
    twice = np.array([[1, 4, 1, 0, 1]] * hkv)[None]
    table = ints(np.concatenate([s.table[:, :6], s.table[:, twice[0, 0]]], axis=1))  # the same columns, once more
    out = s.cache.attention(q, ints(s.table), ints([6 * ps]), scale, picked=ints(twice))
    # (unmasked: every key of the first 6 pages is before the end)
    keys = np.concatenate([np.arange(ps) + ps * p for p in twice[0, 0]])
    again = Sequences(r, mode, hkv, D, ps, [5 * ps])
    again.k[0], again.v[0] = s.k[0][keys], s.v[0][keys]
    again.check(out, q, scale)
    out = s.cache.attention(q, table, ints([11 * ps]), scale)
    both = Sequences(r, mode, hkv, D, ps, [11 * ps])
    both.k[0], both.v[0] = np.concatenate([s.k[0], s.k[0][keys]]), np.concatenate([s.v[0], s.v[0][keys]])
    both.check(out, q, scale)


@pytest.mark.parametrize("mode,D,L", [("affine4", 256, 90), ("fp16", 128, 260), ("int8", 256, 33)])
def test_many_rows(mode, D, L):
    """Row tiles over many workgroups, tiles that end in a head, rows before a sequence's first key."""
    r = rng(L)
    lengths = [L + 70, L, 100 if L > 100 else 20]
    s = Sequences(r, mode, 1, D, 32, lengths)
    q = queries(r, 3, 3, L, D)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.07), q, 0.07)


@pytest.mark.parametrize("mode,D", [("affine4", 256), ("int8", 128), ("fp16", 256), ("affine8", 128)])
@pytest.mark.parametrize("L", [1, 5])
def test_tables_of_more_than_the_caches_hold(mode, D, L):
    """Tables whose width allows for more keys than the caches hold, of sequences that have few."""
    r = rng(D + L)
    lengths = [900, 0, 33, 260]
    s = Sequences(r, mode, 8, D, 16, lengths, width=20000)
    q = queries(r, 4, 32, L, D)
    s.check(s.cache.attention(q, ints(s.table), ints(lengths), 0.07), q, 0.07)


def test_whole_calls_need_no_workspace():
    """Short tables: a first call inside a capture, replayed as the sequences grow."""
    r = rng(74)
    s = Sequences(r, "affine8", 2, 128, 16, [100, 0, 77])
    q, t, n = queries(r, 3, 8, 1, 128), ints(s.table), ints([100, 0, 77])
    torch.cuda.synchronize()
    stream = side_stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = s.cache.attention(q, t, n, 0.1)
    for lengths in ([100, 0, 77], [3, 0, 0], [64, 0, 76]):
        n.copy_(ints(lengths))
        g.replay()
        torch.cuda.synchronize()
        s.check(out, q, 0.1, lengths=lengths)
        assert torch.equal(out, s.cache.attention(q, t, n, 0.1))
