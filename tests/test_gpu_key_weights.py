"""Attention that counts the keys' softmax weights (qw_kv_attention_scored) against 64 bits.

The bar of a weight's sum W over n rows (e = 2^-24): each weight is off by at most 2 g of itself, g the scores'
bar of test_gpu_shared.attend (its scores and its row's maximum and sum are formed from the same products), and a
few roundings of its own (the exponential's, 2 e; the quotient's, the split sums', the products': under 16 e); the
n weights are added in fp32 in any order, n e at most; decay * weights adds a product and a sum, 2 e."""
import numpy as np
import pytest

import oracle
from conftest import rng
from test_gpu_shared import E, attend, dev, filled, queries, rows_of, turbo4_close, turbo4_rows

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def check_scored(out, weights, q, cache, scale, causal, before=None, decay=1.0):
    q = q.double().cpu().numpy()[0]
    out, weights = out.double().cpu().numpy()[0], weights.double().cpu().numpy()
    k, v = rows_of(cache)
    hq, L, D = q.shape
    hkv, T, _ = k.shape
    ref = np.zeros((hkv, T))
    bar = np.zeros((hkv, T))
    for j in range(hq):
        h = j // (hq // hkv)
        for r in range(L):
            n = T - L + r + 1 if causal else T
            o, ob, w, g = attend(q[j, r], k[h, :n], v[h, :n], scale)
            assert np.all(np.abs(out[j, r] - o) <= ob), (j, r)
            ref[h, :n] += w
            bar[h, :n] += (2 * g + (16 + hq // hkv * L) * E) * w
    bar += 2.0 ** -126
    if before is not None and decay:
        b = np.zeros((hkv, T))
        m = min(T, before.shape[1])
        b[:, :m] = before.double().cpu().numpy()[:, :m]
        ref += np.float64(np.float32(decay)) * b
        bar += 2 * E * (np.abs(decay * b) + ref)
    assert weights.shape == ref.shape
    err = np.abs(weights - ref) / bar
    print(f"worst error {err.max():.2f} of the bar", flush=True)
    assert err.max() <= 1.0, np.unravel_index(err.argmax(), err.shape)


CASES = [
    # mode, hq, hkv, D, rows, keys, causal
    ("affine4", 24, 4, 256, 1, 1, True),
    ("affine8", 24, 4, 256, 1, 700, True),
    ("int8", 8, 2, 128, 1, 129, False),
    ("fp16", 16, 2, 256, 3, 65, True),
    ("affine4", 32, 8, 128, 5, 1000, True),
    ("affine8", 12, 1, 256, 33, 640, True),     # 396 rows
    ("fp16", 8, 8, 128, 130, 130, True),        # a prompt's first rows: row r sees r + 1 keys
    ("int8", 24, 4, 256, 24, 300, False),
    ("affine4", 4, 4, 128, 1, 4097, False),
    ("affine4", 16, 1, 256, 140, 333, True),    # 2240 rows: key tiles laid out once
    ("affine8", 32, 2, 256, 130, 130, True),
    ("int8", 16, 1, 128, 257, 500, False),      # 4112 rows
]


@pytest.mark.parametrize("mode,hq,hkv,D,L,T,causal", CASES)
def test_scored_matches_64_bits(mode, hq, hkv, D, L, T, causal):
    print(f"case {mode} hq={hq} hkv={hkv} D={D} L={L} T={T} causal={causal}", flush=True)
    r = rng(T + L + D)
    cache = filled(mode, hkv, D, T, r)
    q = queries(r, 1, hq, L, D)
    out, w = cache.attention_scored(q, D ** -0.5, causal=causal)
    check_scored(out, w, q, cache, D ** -0.5, causal)
    again = cache.attention_scored(q, D ** -0.5, causal=causal)
    assert torch.equal(out, again[0]) and torch.equal(w, again[1])
    # added to earlier counts of fewer keys (a strided view of a longer array), and in place
    store = torch.rand((hkv, T + 9), device="cuda")
    early = store[:, :max(1, T - 3)]
    out, w = cache.attention_scored(q, D ** -0.5, weights=early, decay=0.75, causal=causal)
    check_scored(out, w, q, cache, D ** -0.5, causal, early, 0.75)
    before = store.clone()
    out, w = cache.attention_scored(q, D ** -0.5, weights=store, causal=causal, weights_out=store)
    assert w.data_ptr() == store.data_ptr() and torch.equal(store[:, T:], before[:, T:])
    check_scored(out, w, q, cache, D ** -0.5, causal, before[:, :T], 1.0)


@pytest.mark.parametrize("L", [1, 9, 40])
def test_scored_negative_and_zero_scale(L):
    r = rng(L)
    cache = filled("affine4", 2, 128, 200, r)
    q = queries(r, 1, 8, L, 128)
    for scale in (-0.08, 0.0):
        out, w = cache.attention_scored(q, scale, causal=True)
        check_scored(out, w, q, cache, scale, True)


@pytest.mark.parametrize("hq,hkv,D,L,T", [(24, 4, 256, 1, 700), (8, 2, 128, 3, 129), (24, 4, 128, 30, 300), (12, 1, 256, 20, 64)])
def test_scored_turbo4(hq, hkv, D, L, T):
    r = rng(T + L)
    cache = filled("turbo4", hkv, D, T, r)
    q = queries(r, 1, hq, L, D)
    before = torch.rand((hkv, T), device="cuda")
    out, w = cache.attention_scored(q, D ** -0.5, weights=before, decay=0.5, causal=True)
    k, v, tab = turbo4_rows(cache)
    q = oracle.turbo4_rotate(q.double().cpu().numpy()[0], tab["k_s1"], tab["k_s2"]).astype(np.float16).astype(np.float64)
    ref, wr = np.zeros(out.shape[1:]), 0.5 * before.double().cpu().numpy()
    for j in range(hq):
        h = j // (hq // hkv)
        for i in range(L):
            n = T - L + i + 1
            ref[j, i], _, p, _ = attend(q[j, i], k[h, :n], v[h, :n], D ** -0.5)
            wr[h, :n] += p
    turbo4_close(out.double().cpu().numpy()[0], oracle.turbo4_rotate(ref, tab["v_s2"], tab["v_s1"]))
    # a rotated q that rounds the other way moves a score by a step of fp16: 2^-10 of sum |q k| scale at most
    assert np.allclose(w.double().cpu().numpy(), wr, rtol=2e-2, atol=1e-6)


def test_scored_decay_zero_reads_nothing():
    r = rng(2)
    cache = filled("affine8", 2, 128, 77, r)
    q = queries(r, 1, 8, 2, 128)
    bad = torch.full((2, 77), float("nan"), device="cuda")
    out, w = cache.attention_scored(q, 0.1, weights=bad, decay=0.0, causal=True, weights_out=bad)
    check_scored(out, w, q, cache, 0.1, True)


@pytest.mark.parametrize("mode", ["affine4", "affine8", "int8", "fp16"])
def test_scored_steps_of_decoding(mode):
    """Tokens appended one by one, the counts carried along; the last keys' are new each time."""
    r = rng(8)
    cache = filled(mode, 2, 128, 30, r)
    want = filled(mode, 2, 128, 0, r)
    want.restore_snapshot(cache.snapshot_tensors())
    w = w2 = None
    for _ in range(5):
        q = queries(r, 1, 8, 1, 128)
        k, v = (dev(r.standard_normal((1, 2, 1, 128)).astype(np.float16)) for _ in range(2))
        out, w = cache.update_and_attention_scored(q, k, v, 0.09, weights=w, decay=0.5, causal=True)
        want.update(k, v)
        out2, w2 = want.attention_scored(q, 0.09, weights=w2, decay=0.5, causal=True)
        assert w.shape == (2, cache.offset) and torch.equal(out, out2) and torch.equal(w, w2)
    # each of the 4 heads of a group adds 1 a step
    total = 4 * sum(0.5 ** i for i in range(5))
    assert torch.allclose(w.sum(1), torch.full((2,), total, device="cuda"), rtol=1e-5)


def test_scored_ignores_what_rows_do_not_see():
    """Rows behind the offset, and a later row's key to the count of the rows before it."""
    r = rng(4)
    k, v = (r.standard_normal((2, 70, 128)).astype(np.float16) for _ in range(2))
    k[:, 60:], v[:, 60:] = np.nan, np.inf
    cache = filled("fp16", 2, 128, 0, r)
    cache.update(dev(k), dev(v))
    cache.trim(10)
    q = queries(r, 1, 4, 3, 128)
    out, w = cache.attention_scored(q, 0.09, causal=True)
    check_scored(out, w, q, cache, 0.09, True)


def test_scored_graph_and_streams():
    r = rng(6)
    cache = filled("affine4", 4, 256, 2000, r)
    q = queries(r, 1, 24, 1, 256)
    w = torch.rand((4, 2000), device="cuda")
    acc, side = w.clone(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attention_scored(q, 0.0625, weights=w, causal=True)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, _ = cache.attention_scored(q, 0.0625, weights=acc, decay=0.9, causal=True, weights_out=acc)
    for _ in range(4):
        q.copy_(queries(r, 1, 24, 1, 256))
        graph.replay()
        torch.cuda.synchronize()
        out2, w = cache.attention_scored(q, 0.0625, weights=w, decay=0.9, causal=True)
        assert torch.equal(out, out2) and torch.equal(acc, w)


def test_scored_views_off_alignment():
    """q off any vector alignment, one row and many."""
    r = rng(13)
    cache = filled("affine8", 2, 128, 700, r)
    for L in (1, 40):
        q = queries(r, 1, 8, L, 128)
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
        odd.copy_(q)
        out, w = cache.attention_scored(q, 0.09, causal=True)
        out2, w2 = cache.attention_scored(odd, 0.09, causal=True)
        assert torch.equal(out, out2) and torch.equal(w, w2)


def test_refused_in_a_capture_before_the_append():
    """A call that needs memory in a captured stream appends nothing."""
    import qw_amd

    r = rng(14)
    cache = filled("fp16", 2, 128, 250, r)
    prefix = filled("fp16", 1, 128, 30, r)
    q, kv = queries(r, 1, 8, 1, 128), dev(r.standard_normal((1, 2, 1, 128)).astype(np.float16))
    qb, kvb = queries(r, 2, 4, 9, 128), dev(r.standard_normal((2, 1, 9, 128)).astype(np.float16))
    torch.cuda.synchronize()
    for call in (lambda: cache.update_and_attention_scored(q, kv, kv, 0.1),
                 lambda: prefix.update_and_shared_attention(qb, cache, kvb, kvb, 0.1)):
        with pytest.raises(qw_amd.QwError) as e:
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
                call()
        assert e.value.status == 5 and cache.offset == 250
    out, w = cache.update_and_attention_scored(q, kv, kv, 0.1, causal=True)
    check_scored(out, w, q, cache, 0.1, True)


def test_scored_refusals():
    import qw_amd

    r = rng(1)
    cache = filled("fp16", 2, 128, 20, r)
    q = queries(r, 1, 8, 1, 128)
    w = torch.zeros((2, 20), device="cuda")

    def refused(status, f, *a, **k):
        with pytest.raises(qw_amd.QwError) as e:
            f(*a, **k)
        assert e.value.status == status, e.value

    call = cache.attention_scored
    refused(1, call, q[:, :7], 0.1)
    refused(1, call, queries(r, 1, 8, 1, 256), 0.1)
    refused(1, call, queries(r, 1, 8, 21, 128), 0.1, causal=True)
    refused(1, call, q, float("nan"))
    refused(1, call, q, 0.1, weights=w, decay=-1.0)
    refused(1, call, q, 0.1, weights=w.double())
    refused(1, call, q, 0.1, weights=w[:1])
    refused(1, call, q, 0.1, weights=w.cpu())
    refused(1, call, q, 0.1, weights_out=w[:, :19])
    refused(1, call, q, 0.1, weights_out=torch.zeros((20, 2), device="cuda").t())
    buf = torch.zeros((2, 44), device="cuda")
    refused(1, call, q, 0.1, weights=buf[:, :20], weights_out=buf[:, 5:25])  # shifted overlap
    refused(1, filled("fp16", 2, 128, 0, r).attention_scored, q, 0.1)
    kv = dev(np.zeros((1, 2, 1, 128), np.float16))
    refused(1, cache.update_and_attention_scored, q, kv, kv[:, :1], 0.1)
    assert cache.offset == 20


@pytest.mark.parametrize("hq,hkv,D,L,T", [(24, 4, 256, 1, 5000), (8, 2, 128, 1, 1), (32, 2, 256, 1, 33), (8, 2, 128, 4, 1500)])
def test_scored_turbo4_few_rows(hq, hkv, D, L, T):
    """Up to 16 rows a KV head: several key splits, a single key, a chunk's first key, causal limits inside one."""
    test_scored_turbo4(hq, hkv, D, L, T)


def test_scored_turbo4_steps_of_decoding():
    """Tokens appended by the call itself; the same bits as an append before it."""
    r = rng(9)
    cache, want = filled("turbo4", 2, 128, 30, r), filled("turbo4", 2, 128, 0, r)
    want.restore_snapshot(cache.snapshot_tensors())
    w = w2 = None
    for _ in range(4):
        q = queries(r, 1, 8, 1, 128)
        k, v = (dev(r.standard_normal((1, 2, 1, 128)).astype(np.float16)) for _ in range(2))
        out, w = cache.update_and_attention_scored(q, k, v, 0.09, weights=w, decay=0.5, causal=True)
        want.update(k, v)
        out2, w2 = want.attention_scored(q, 0.09, weights=w2, decay=0.5, causal=True)
        assert w.shape == (2, cache.offset) and torch.equal(out, out2) and torch.equal(w, w2)
