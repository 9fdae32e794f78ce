"""Attention of a batch over a shared prefix and its tails (qw_kv_shared_attention) against 64-bit
softmax attention on the caches' own dequantized rows.

The bar of an output, from the kernel's roundings (u = 2^-11, half a step of fp16; e = 2^-24): each weight
rounded to fp16, at most u of itself or, below fp16's normal numbers, 2^-25 of the row's largest; the output
rounded, u of itself; a score's D products and sums in fp32, at most g = (D + 8) e scale sum |q_d k_d| off, which
scales a weight by 1 + g and the row's sum alike. With A = sum p |v|:
  |error| <= (u + 2 g) A + u |out| + 2^-25 sum |v| / L,   L = sum e^(s - max s)."""
import numpy as np
import pytest

import oracle
from conftest import rng

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U, E = 2.0 ** -11, 2.0 ** -24


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def rows_of(cache):
    """A cache's K and V as the fetch gives them, [H, T, D] in 64 bits."""
    if cache is None or cache.offset == 0:
        return None
    return tuple(x[0].double().cpu().numpy() for x in cache.dequantize())


def attend(q, k, v, scale):
    """One row's 64-bit output, its error bar, its weights and the scores' bar g."""
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    total = p.sum()
    w = p / total
    out = w @ v
    g = (q.size + 8) * E * abs(scale) * (np.abs(k) @ np.abs(q)).max()
    bar = (U + 2 * g) * (w @ np.abs(v)) + U * np.abs(out) + 2.0 ** -25 * np.abs(v).sum(0) / total + 2.0 ** -25
    return out, bar, w, g


def check_shared(out, q, prefix, tails, starts, scale, only=None):
    out, q = out.double().cpu().numpy(), q.double().cpu().numpy()
    B, hq, L, D = q.shape
    pre, tail = rows_of(prefix), rows_of(tails)
    hkv = prefix.n_kv_heads
    T = 0 if tail is None else tail[0].shape[1]
    worst = 0.0
    for b in range(B) if only is None else only:
        lo = 0 if starts is None else min(max(int(starts[b]), 0), T)
        for j in range(hq):
            h = j // (hq // hkv)
            for r in range(L):
                parts = [(pre[0][h], pre[1][h])] if pre else []
                if tail:
                    t = (b * hkv + h, slice(lo, T - L + r + 1))
                    parts.append((tail[0][t], tail[1][t]))
                k, v = (np.concatenate([p[i] for p in parts]) for i in range(2))
                if len(k) == 0:
                    assert np.all(out[b, j, r] == 0), (b, j, r)
                    continue
                ref, bar, _, _ = attend(q[b, j, r], k, v, scale)
                err = np.abs(out[b, j, r] - ref) / bar
                assert err.max() <= 1.0, (b, j, r, err.max())
                worst = max(worst, err.max())
    print(f"worst error {worst:.2f} of the bar", flush=True)


def filled(mode, heads, D, n, r, sigma=1.0):
    import qw_amd

    c = qw_amd.KVCache(mode, heads, D)
    if n:
        k, v = ((sigma * r.standard_normal((heads, n, D))).astype(np.float16) for _ in range(2))
        c.update(dev(k), dev(v))
    return c


def queries(r, B, hq, L, D):
    return dev((2 * r.standard_normal((B, hq, L, D))).astype(np.float16))


CASES = [
    # prefix mode, tail mode, hq, hkv, D, sequences, rows, prefix, tail
    ("affine4", "affine4", 24, 4, 256, 3, 1, 700, 37),
    ("affine8", "affine8", 24, 4, 256, 2, 5, 65, 64),       # one key into a tile; a whole tile
    ("int8", "int8", 8, 2, 128, 4, 2, 127, 129),
    ("fp16", "fp16", 16, 2, 256, 5, 3, 300, 70),            # 120 rows a head
    ("affine8", "fp16", 24, 4, 128, 7, 4, 513, 33),         # 168 rows: two query tiles; two launches
    ("affine4", "int8", 12, 1, 256, 2, 16, 1000, 16),       # 384 rows; a tail of the newest rows alone
    ("fp16", "affine4", 4, 4, 128, 1, 1, 1, 1),             # one key each, one row a head
    ("int8", "affine8", 32, 8, 128, 20, 1, 2050, 5),        # one width, two codes
    ("affine4", "affine4", 32, 8, 128, 33, 1, 129, 300),
    ("fp16", "fp16", 8, 8, 128, 2, 40, 4000, 41),
]


@pytest.mark.parametrize("pm,tm,hq,hkv,D,B,L,P,T", CASES)
def test_shared_matches_64_bits(pm, tm, hq, hkv, D, B, L, P, T):
    print(f"case {pm} {tm} hq={hq} hkv={hkv} D={D} B={B} L={L} P={P} T={T}", flush=True)
    r = rng(P + T + B + L)
    prefix, tails = filled(pm, hkv, D, P, r), filled(tm, B * hkv, D, T, r)
    q = queries(r, B, hq, L, D)
    starts = r.integers(0, T - L + 1, B).astype(np.int32)
    starts[0] = 0
    out = prefix.shared_attention(q, tails, D ** -0.5, starts=dev(starts))
    check_shared(out, q, prefix, tails, starts, D ** -0.5)
    assert torch.equal(out, prefix.shared_attention(q, tails, D ** -0.5, starts=dev(starts)))
    if T == L or P < 3:
        check_shared(prefix.shared_attention(q, tails, -0.11), q, prefix, tails, None, -0.11)


@pytest.mark.parametrize("mode", ["affine4", "fp16"])
def test_shared_without_prefix_or_tails(mode):
    r = rng(5)
    q = queries(r, 3, 8, 2, 128)
    prefix, tails = filled(mode, 2, 128, 200, r), filled(mode, 6, 128, 90, r)
    empty, none = filled(mode, 2, 128, 0, r), filled(mode, 6, 128, 0, r)
    check_shared(prefix.shared_attention(q, None, 0.09), q, prefix, None, None, 0.09)
    check_shared(prefix.shared_attention(q, none, 0.09), q, prefix, none, None, 0.09)
    # a sequence with nothing of its own, one that starts at its newest row (its first row sees nothing)
    # and starts outside the tail
    starts = np.array([90, 89, -5], np.int32)
    check_shared(empty.shared_attention(q, tails, 0.09, starts=dev(starts)), q, empty, tails, starts, 0.09)
    starts = np.array([2 ** 31 - 1, 88, 17], np.int32)
    check_shared(prefix.shared_attention(q, tails, 0.09, starts=dev(starts)), q, prefix, tails, starts, 0.09)


def test_shared_rows_stay_apart():
    """What a sequence does not see - rows below its start, rows behind the cache's offset, the other
    sequences' tails - may hold anything."""
    r = rng(11)
    prefix, tails = filled("fp16", 2, 128, 130, r), filled("fp16", 6, 128, 0, r)
    k, v = (r.standard_normal((6, 100, 128)).astype(np.float16) for _ in range(2))
    for x, bad in ((k, np.nan), (v, np.inf)):
        x[2:4, :40] = bad   # sequence 1: padding below its start
        x[4:6, 50] = bad    # sequence 2: a key that it sees itself
        x[:, 95:] = bad     # trimmed again
    tails.update(dev(k), dev(v))
    tails.trim(5)
    q = queries(r, 3, 8, 3, 128)
    starts = np.array([0, 40, 3], np.int32)
    out = prefix.shared_attention(q, tails, 0.09, starts=dev(starts))
    assert torch.isnan(out[2]).any()
    check_shared(out, q, prefix, tails, starts, 0.09, only=(0, 1))


@pytest.mark.parametrize("mode", ["affine4", "affine8", "int8", "fp16"])
def test_shared_update_appends_first(mode):
    r = rng(3)
    prefix, a = filled(mode, 2, 256, 320, r), filled(mode, 8, 256, 255, r)
    b = filled(mode, 8, 256, 255, rng(3))
    b.restore_snapshot(a.snapshot_tensors())
    starts = dev(np.array([0, 100, 200, 255], np.int32))
    for L in (1, 4):
        q = queries(r, 4, 12, L, 256)
        k, v = (dev(r.standard_normal((4, 2, L, 256)).astype(np.float16)) for _ in range(2))
        out = prefix.update_and_shared_attention(q, a, k, v, 0.0625, starts=starts)
        b.update(k.reshape(8, L, 256), v.reshape(8, L, 256))
        assert a.offset == b.offset and prefix.offset == 320
        assert torch.equal(out, prefix.shared_attention(q, b, 0.0625, starts=starts))
        for x, y in zip(a.snapshot_tensors().values(), b.snapshot_tensors().values()):
            assert torch.equal(x, y)
        check_shared(out, q, prefix, a, starts.cpu().numpy(), 0.0625)


def test_shared_streams_views_and_graph():
    """Another stream, q off any vector alignment, strided starts, and a captured call replayed with the
    program's own work between."""
    r = rng(9)
    prefix, tails = filled("affine8", 4, 128, 900, r), filled("affine8", 12, 128, 60, r)
    q = queries(r, 3, 16, 2, 128)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    starts = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    starts[:, 0] = torch.tensor([0, 30, 58])
    want = prefix.shared_attention(q, tails, 0.1, starts=starts[:, 0])
    assert torch.equal(want, prefix.shared_attention(odd, tails, 0.1, starts=starts[:, 0]))
    check_shared(want, q, prefix, tails, [0, 30, 58], 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(want, prefix.shared_attention(q, tails, 0.1, starts=starts[:, 0]))
        st = starts[:, 0].contiguous()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = prefix.shared_attention(q, tails, 0.1, starts=st)
    for i in range(4):
        q.copy_(queries(r, 3, 16, 2, 128))
        st.fill_(7 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, prefix.shared_attention(q, tails, 0.1, starts=st))


def turbo4_rows(cache):
    """A Turbo4 cache's rows in their rotated bases, [H, T, D] in 64 bits, and its tables."""
    tab = oracle.turbo4_tables(cache.head_dim, cache.turbo_seed)
    snap = {n: x.cpu().numpy() for n, x in cache.snapshot_tensors().items()}
    k = oracle.turbo4_expand_rotated(snap["k_packed"], snap["k_rescale"][..., 0], tab)
    v = oracle.turbo4_expand_rotated(snap["v_packed"], snap["v_rescale"][..., 0], tab)
    return k.astype(np.float64), v.astype(np.float64), tab


def turbo4_close(out, ref):
    """The bar of the other Turbo4 attention tests: 2e-3 absolute, 1e-3 relative L2 (q and the rotated
    output are rounded to fp16 between the rotations)."""
    err = np.abs(out - ref)
    assert err.max() <= 2e-3 and np.linalg.norm(out - ref) <= 1e-3 * np.linalg.norm(ref), (err.max(), np.linalg.norm(out - ref) / np.linalg.norm(ref))


@pytest.mark.parametrize("hq,hkv,D,B,L,P,T", [(24, 4, 256, 3, 1, 700, 37), (8, 2, 128, 4, 2, 127, 129), (24, 4, 128, 6, 5, 1030, 60),
                                              (12, 1, 256, 1, 1, 64, 1), (16, 2, 256, 5, 4, 300, 70)])
def test_shared_turbo4(hq, hkv, D, B, L, P, T):
    r = rng(P + T)
    prefix, tails = filled("turbo4", hkv, D, P, r), filled("turbo4", B * hkv, D, T, r)
    q = queries(r, B, hq, L, D)
    starts = r.integers(0, T - L + 1, B).astype(np.int32)
    out = prefix.shared_attention(q, tails, D ** -0.5, starts=dev(starts)).double().cpu().numpy()
    pk, pv, tab = turbo4_rows(prefix)
    tk, tv, _ = turbo4_rows(tails)
    q = oracle.turbo4_rotate(q.double().cpu().numpy(), tab["k_s1"], tab["k_s2"]).astype(np.float16).astype(np.float64)
    ref = np.zeros_like(out)
    for b in range(B):
        for j in range(hq):
            h = j // (hq // hkv)
            for i in range(L):
                t = (b * hkv + h, slice(starts[b], T - L + i + 1))
                k, v = np.concatenate([pk[h], tk[t]]), np.concatenate([pv[h], tv[t]])
                ref[b, j, i] = attend(q[b, j, i], k, v, D ** -0.5)[0]
    turbo4_close(out, oracle.turbo4_rotate(ref, tab["v_s2"], tab["v_s1"]))


def test_shared_long_offsets():
    """Rows behind element 2^31 of a plane."""
    import qw_amd

    heads, n, D = 160, 53000, 256  # 2.2e9 halves of K
    tails = qw_amd.KVCache("fp16", heads, D, capacity=n)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((heads, n, D), dtype=torch.float16, device="cuda").normal_(generator=g)
    tails.update(x, x)
    prefix = filled("fp16", 2, D, 40, rng(1))
    q = queries(rng(2), 80, 4, 1, D)
    starts = np.full(80, n - 900, np.int32)
    out = prefix.shared_attention(q, tails, 0.0625, starts=dev(starts))
    pre = rows_of(prefix)
    for h in range(2):
        t = x[158 + h, n - 900:].double().cpu().numpy()
        k, v = (np.concatenate([p[h], t]) for p in pre)
        for j in (2 * h, 2 * h + 1):
            ref, bar, _, _ = attend(q[79, j, 0].double().cpu().numpy(), k, v, 0.0625)
            assert np.all(np.abs(out[79, j, 0].double().cpu().numpy() - ref) <= bar)


def test_shared_refusals():
    import qw_amd

    r = rng(1)
    prefix, tails = filled("fp16", 2, 128, 20, r), filled("fp16", 6, 128, 3, r)
    q = queries(r, 3, 8, 1, 128)
    kv = dev(np.zeros((3, 2, 1, 128), np.float16))

    def refused(status, f, *a, **k):
        with pytest.raises(qw_amd.QwError) as e:
            f(*a, **k)
        assert e.value.status == status, e.value

    call, upd = prefix.shared_attention, prefix.update_and_shared_attention
    refused(1, call, q[0], tails, 0.1)                                    # no batch dimension
    refused(1, call, q.float(), tails, 0.1)
    refused(1, call, q[:2], tails, 0.1)                                   # 2 sequences, 6 heads of tails
    refused(1, call, q[:, :7], tails, 0.1)                                # 7 query heads over 2
    refused(1, call, q, tails, float("inf"))
    refused(1, call, q, prefix, 0.1)
    refused(1, call, queries(r, 3, 8, 4, 128), tails, 0.1)                # 4 rows, 3 tail rows
    refused(1, call, q, tails, 0.1, starts=torch.zeros(3, device="cuda"))
    refused(1, call, q, tails, 0.1, starts=torch.zeros(3, dtype=torch.int32))
    refused(1, call, q, tails, 0.1, starts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused(1, upd, q, None, kv, kv, 0.1)
    refused(1, upd, q, tails, kv, kv[:, :1], 0.1)
    refused(1, filled("fp16", 2, 128, 0, r).shared_attention, q, None, 0.1)
    one = filled("fp16", 1, 128, 5, r)
    refused(1, one.shared_attention, q[:1, :1], one, 0.1)                 # the prefix as its own tail
    refused(1, prefix.shared_attention, queries(r, 3, 8, 1, 256), filled("fp16", 6, 256, 3, r), 0.1)
    refused(2, prefix.shared_attention, q, filled("turbo4", 6, 128, 3, r), 0.1)
    refused(2, filled("turbo4", 2, 128, 20, r).shared_attention, q, filled("affine4", 6, 128, 3, r), 0.1)
    other = qw_amd.KVCache("turbo4", 6, 128, turbo_seed=7)
    refused(2, filled("turbo4", 2, 128, 20, r).shared_attention, q, other, 0.1)
    closed = filled("fp16", 6, 128, 3, r)
    closed.close()
    refused(1, call, q, closed, 0.1)
    assert tails.offset == 3 and prefix.offset == 20


@pytest.mark.parametrize("n_rows", [1 << 24, 1 << 26])
def test_too_many_rows_refused(n_rows):
    """More rows than a launch's threads cover: refused on the host, by the declared sizes alone."""
    import qw_amd

    prefix = filled("fp16", 1, 128, 20, rng(3))
    x, w = torch.zeros(128, dtype=torch.float16, device="cuda"), torch.zeros((1, 20), device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    lib, q = qw_amd.lib(), x.data_ptr()
    assert lib.qw_kv_shared_attention(prefix._h, None, 1, None, q, 1, n_rows, 0.1, q, st) == 2
    assert lib.qw_kv_attention_scored(prefix._h, q, 1, n_rows, 0.1, 0, None, 0, 0, 0.0, w.data_ptr(), 20, q, st) in (1, 2)
    torch.cuda.synchronize()
    assert prefix.offset == 20 and not w.any()


@pytest.mark.parametrize("hq,hkv,D,B,L,P,T", [(8, 2, 128, 2, 1, 700, 300), (12, 2, 256, 1, 2, 2500, 130), (16, 1, 128, 1, 1, 1, 33)])
def test_shared_turbo4_few_rows(hq, hkv, D, B, L, P, T):
    """At most 16 rows of a head in both caches."""
    test_shared_turbo4(hq, hkv, D, B, L, P, T)
