"""Eviction by key weights (qw_kv_evict) against a sort on the host: the kept positions, their weights and
every stored code, all exact."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_key_weights import check_scored
from test_gpu_shared import check_shared, dev, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def keep(w, T, budget, sink, recent):
    out = []
    for row in w[:, :T].astype(np.float64):
        t = np.arange(T)
        fixed = (t < sink) | (t >= T - recent)
        rank = np.where(np.isnan(row), -np.inf, row)
        order = np.lexsort((t, -rank, np.isnan(row), ~fixed))
        out.append(np.sort(order[:min(T, budget)]))
    return np.stack(out)


def check_evict(cache, into, w, budget, sink, recent):
    T = cache.offset
    before = {n: x.clone() for n, x in cache.snapshot_tensors().items()}
    want = keep(w.cpu().numpy(), T, budget, sink, recent)
    kept, wo = cache.evict(w, budget, sink=sink, recent=recent, into=into)
    dst = cache if into is None else into
    assert dst.offset == want.shape[1] == min(T, budget)
    assert cache.offset == (T if into is not None and into is not cache else dst.offset)
    assert np.array_equal(kept.cpu().numpy(), want)
    rows = np.arange(want.shape[0])[:, None]
    got, ref = wo.cpu().numpy(), w.cpu().numpy()[rows, want]
    assert np.array_equal(got.view(np.uint32), ref.view(np.uint32))
    after = dst.snapshot_tensors()
    for name, x in before.items():
        picked = x.cpu().numpy()[rows, want]
        have = after[name].cpu().numpy()
        assert np.array_equal(have.view(np.uint8), np.ascontiguousarray(picked).view(np.uint8)), name
    return kept, wo


def weights(r, hkv, T, kind):
    w = np.exp(2 * r.standard_normal((hkv, T))).astype(np.float32)
    if kind == "ties":  # few values, zeros of both signs among them
        w = r.integers(-1, 3, (hkv, T)).astype(np.float32)
        w[w == -1] = -0.0
    elif kind == "odd":
        w *= r.choice([-1.0, 1.0], (hkv, T)).astype(np.float32)
        w[r.random((hkv, T)) < 0.1] = np.nan
        w[r.random((hkv, T)) < 0.05] = np.inf
        w[r.random((hkv, T)) < 0.05] = -np.inf
        w[r.random((hkv, T)) < 0.05] = 1e-42
    elif kind == "same":
        w[:] = 0.25
    return w


CASES = [
    # hkv, D, T, budget, sink, recent, weights
    (4, 256, 1, 1, 0, 0, "log"),
    (4, 256, 9, 8, 4, 4, "log"),         # nothing left to choose
    (2, 128, 300, 300, 4, 32, "log"),    # everything stays
    (2, 128, 300, 1000, 4, 700, "odd"),  # recent beyond the cache
    (8, 128, 1000, 129, 4, 64, "log"),
    (4, 256, 777, 500, 0, 1, "ties"),
    (3, 128, 2049, 1024, 1, 0, "odd"),
    (1, 256, 5000, 17, 0, 0, "same"),
    (4, 128, 4097, 4096, 0, 4096, "log"),  # one key goes
    (2, 256, 70001, 9001, 4, 512, "ties"),
]


@pytest.mark.parametrize("mode", ["affine4", "affine8", "int8", "fp16", "turbo4"])
@pytest.mark.parametrize("hkv,D,T,budget,sink,recent,kind", CASES)
def test_evict_matches_a_sort(mode, hkv, D, T, budget, sink, recent, kind):
    import qw_amd

    print(f"case {mode} hkv={hkv} D={D} T={T} budget={budget} sink={sink} recent={recent} {kind}", flush=True)
    r = rng(T + budget)
    cache = filled(mode, hkv, D, T, r)
    w = dev(weights(r, hkv, T + 5, kind))  # a longer array than the cache
    into = qw_amd.KVCache(mode, hkv, D)    # grows to the budget
    kept, wo = check_evict(cache, into, w, budget, sink, recent)
    # once more into a cache that holds other rows, then in place
    check_evict(cache, into, w[:, :T].flip(1).contiguous(), max(1, budget // 2), min(sink, budget // 4), 0)
    kept2, wo2 = check_evict(cache, None, w, budget, sink, recent)
    assert torch.equal(kept, kept2) and torch.equal(wo.view(torch.int32), wo2.view(torch.int32))


def test_evict_keeps_the_dequantization_of_its_source():
    """Scales outside the range of the short dequantization go with their rows."""
    import qw_amd

    r = rng(3)
    cache = filled("affine4", 2, 128, 100, r, sigma=4000.0)
    into = qw_amd.KVCache("affine4", 2, 128)
    w = torch.rand((2, 100), device="cuda")
    kept, _ = cache.evict(w, 40, into=into)
    k, v = cache.dequantize()
    k2, v2 = into.dequantize()
    idx = kept.long()[None, :, :, None].expand(1, 2, 40, 128)
    assert torch.equal(k.gather(2, idx), k2) and torch.equal(v.gather(2, idx), v2)
    q = queries(r, 1, 8, 1, 128)
    fresh = qw_amd.KVCache("affine4", 2, 128)
    fresh.restore_snapshot(into.snapshot_tensors())
    assert torch.equal(into.attention(q, 1e-4), fresh.attention(q, 1e-4))


def test_evict_graph():
    """A step with an eviction in place, captured: the graph reads the same 600 rows at every replay."""
    import qw_amd

    r = rng(5)
    full = filled("affine8", 2, 128, 600, r)
    into = qw_amd.KVCache("affine8", 2, 128, capacity=512)
    w = dev(weights(r, 2, 600, "log"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        full.evict(w, 300, sink=4, recent=32, into=into)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept, wo = full.evict(w, 300, sink=4, recent=32, into=into)
    for i in range(3):
        w.copy_(dev(weights(r, 2, 600, ("log", "ties", "odd")[i])))
        graph.replay()
        torch.cuda.synchronize()
        got = {n: x.clone() for n, x in into.snapshot_tensors().items()}
        kept2, wo2 = full.evict(w, 300, sink=4, recent=32, into=into)
        assert torch.equal(kept, kept2) and torch.equal(wo.view(torch.int32), wo2.view(torch.int32))
        for n, x in into.snapshot_tensors().items():
            assert torch.equal(x, got[n])


def test_evict_refusals():
    import qw_amd

    r = rng(1)
    cache = filled("affine8", 2, 128, 20, r)
    w = torch.rand((2, 20), device="cuda")

    def refused(status, f, *a, **k):
        with pytest.raises(qw_amd.QwError) as e:
            f(*a, **k)
        assert e.value.status == status, e.value

    refused(1, cache.evict, w, 0)
    refused(1, cache.evict, w, -3)
    refused(1, cache.evict, w, 10, sink=6, recent=5)
    refused(1, cache.evict, w, 10, sink=-1)
    refused(1, cache.evict, w, 10, recent=-1)
    refused(1, cache.evict, w[:, :19], 10)
    refused(1, cache.evict, w.half(), 10)
    refused(1, cache.evict, w, 10, into=qw_amd.KVCache("affine4", 2, 128))
    refused(1, cache.evict, w, 10, into=qw_amd.KVCache("affine8", 4, 128))
    refused(1, cache.evict, w, 10, into=qw_amd.KVCache("affine8", 2, 256))
    refused(1, filled("turbo4", 2, 128, 20, r).evict, w, 10, into=qw_amd.KVCache("turbo4", 2, 128, turbo_seed=5))
    closed = qw_amd.KVCache("affine8", 2, 128)
    closed.close()
    refused(1, cache.evict, w, 10, into=closed)
    refused(1, cache.evict, w, 2 ** 40, sink=2 ** 31, recent=1)
    assert cache.offset == 20
    empty = qw_amd.KVCache("affine8", 2, 128)
    kept, wo = empty.evict(w, 10)
    assert kept.shape == wo.shape == (2, 0) and empty.offset == 0


@pytest.mark.parametrize("mode", ["affine4", "fp16"])
def test_prompt_observed_cut_and_shared(mode):
    """The three together: a prompt goes in by chunks that count weights, is cut to a budget, and a batch of
    sequences decodes over what is left."""
    import qw_amd

    r = rng(12)
    hq, hkv, D, B = 12, 2, 128, 3
    prompt = qw_amd.KVCache(mode, hkv, D)
    w = None
    for L in (200, 133, 64):
        q = queries(r, 1, hq, L, D)
        k, v = (dev(r.standard_normal((hkv, L, D)).astype(np.float16)) for _ in range(2))
        prev = w
        out, w = prompt.update_and_attention_scored(q, k, v, D ** -0.5, weights=w, causal=True)
    check_scored(out, w, q, prompt, D ** -0.5, True, prev, 1.0)
    kept, w = check_evict(prompt, None, w, 150, 4, 32)
    assert prompt.offset == 150
    tails = qw_amd.KVCache(mode, B * hkv, D)
    starts = dev(np.array([0, 2, 3], np.int32))
    for step in range(4):
        q = queries(r, B, hq, 1, D)
        k, v = (dev(r.standard_normal((B, hkv, 1, D)).astype(np.float16)) for _ in range(2))
        out = prompt.update_and_shared_attention(q, tails, k, v, D ** -0.5, starts=starts)
        check_shared(out, q, prompt, tails, starts.cpu().numpy(), D ** -0.5)
