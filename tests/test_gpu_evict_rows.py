"""What stands behind the last kept row after an eviction, and evictions in place in captured graphs.

A cache's rows past its offset have to dequantize to finite values: the attention kernels give them weight 0, and
0 x NaN is NaN."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_evict import check_evict, weights
from test_gpu_shared import dev, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

MODES = ["affine4", "affine8", "int8", "fp16", "turbo4"]


def stage_nan(D):
    """Leaves NaN in the stream's staging area: rows of a cache that holds nothing else move through it."""
    import qw_amd

    c = qw_amd.KVCache("fp16", 4, D)
    x = torch.full((4, 2048, D), float("nan"), dtype=torch.float16, device="cuda")
    c.update(x, x)
    c.evict(torch.ones((4, 2048), device="cuda"), 2047)


def same_as_fresh(cache, r, hq):
    """The cache's attention is that of a new cache with the same rows, bit for bit, and finite."""
    import qw_amd

    fresh = qw_amd.KVCache(cache.mode, cache.n_kv_heads, cache.head_dim)
    fresh.restore_snapshot(cache.snapshot_tensors())
    for L in (1, 4, 24):
        q = queries(r, 1, hq, min(L, cache.offset), cache.head_dim)
        for causal in (False, True):
            out = cache.attention(q, 0.07, causal=causal)
            assert torch.isfinite(out).all(), (L, causal)
            assert torch.equal(out, fresh.attention(q, 0.07, causal=causal)), (L, causal)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("D,T,budget", [(128, 300, 13), (256, 90, 57), (256, 2100, 1030), (128, 70, 65)])
def test_rows_behind_the_last_are_finite(mode, D, T, budget):
    r = rng(T + budget)
    cache = filled(mode, 2, D, T, r)
    w = dev(weights(r, 2, T, "log"))
    stage_nan(D)
    check_evict(cache, None, w, budget, 2, 3)
    same_as_fresh(cache, r, 8)
    # and again, to another remainder, behind another cache's rows of another layout
    stage_nan(D)
    check_evict(cache, None, w[:, :budget].contiguous(), budget - 6, 0, 0)
    same_as_fresh(cache, r, 8)
    # rows appended behind them, into the middle of a block
    k, v = (dev(r.standard_normal((2, 3, D)).astype(np.float16)) for _ in range(2))
    cache.update(k, v)
    same_as_fresh(cache, r, 8)


@pytest.mark.parametrize("mode", MODES)
def test_rows_behind_the_last_in_another_cache(mode):
    """The destination held rows of NaN at the end of its last block before."""
    import qw_amd

    r = rng(4)
    cache, into = filled(mode, 2, 128, 100, r), qw_amd.KVCache(mode, 2, 128)
    x = np.ones((2, 24, 128), np.float16)
    if mode == "fp16":
        x[:, 21:] = np.nan
    into.update(dev(x), dev(x))
    check_evict(cache, into, dev(weights(r, 2, 100, "log")), 21, 2, 3)
    same_as_fresh(into, r, 8)


@pytest.mark.parametrize("mode", ["affine8", "fp16", "turbo4"])
@pytest.mark.parametrize("T,n", [(600, 301), (17000, 5003)])
def test_evict_in_place_captured(mode, T, n):
    """An eviction in place in a graph: each replay moves the rows that the cache then holds, by the weights that
    it then finds, as an eager call does."""
    import qw_amd

    r = rng(T)
    cache, twin = filled(mode, 2, 128, T, r), qw_amd.KVCache(mode, 2, 128, capacity=T)
    full = {k: x.clone() for k, x in cache.snapshot_tensors().items()}
    w = dev(weights(r, 2, T, "log"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.evict(w, n, sink=4, recent=32)  # sizes the stream's workspaces
        cache.restore_snapshot(full)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept, wo = cache.evict(w, n, sink=4, recent=32)
    assert cache.offset == n
    for i in range(3):
        w.copy_(dev(weights(r, 2, T, ("log", "ties", "odd")[i])))
        cache.restore_snapshot(full)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        cache.trim(T - n)
        twin.restore_snapshot(full)
        kept2, wo2 = twin.evict(w, n, sink=4, recent=32)
        assert torch.equal(kept, kept2) and torch.equal(wo.view(torch.int32), wo2.view(torch.int32))
        got, want = cache.snapshot_tensors(), twin.snapshot_tensors()
        for name in want:
            assert torch.equal(got[name].view(torch.uint8), want[name].view(torch.uint8)), name
        same_as_fresh(cache, r, 8)


def poisoned(mode, D, T, bad, r):
    """A cache of T rows of which those in `bad` are NaN, and weights that are NaN for them."""
    import qw_amd

    cache = qw_amd.KVCache(mode, 2, D)
    k, v = (r.standard_normal((2, T, D)).astype(np.float16) for _ in range(2))
    k[:, bad] = v[:, bad] = np.nan
    cache.update(dev(k), dev(v))
    w = weights(r, 2, T, "log")
    w[:, bad] = np.nan
    return cache, dev(w)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("D,T,n", [(128, 400, 300), (256, 300, 257), (128, 1000, 513), (256, 900, 64)])
def test_evicted_rows_of_nan_are_gone(mode, D, T, n):
    """Rows of NaN weight go first. What an eviction leaves behind the new end, in place or in a cache that held other
    rows before, takes no part in the cache's attention."""
    import qw_amd

    r = rng(T + n)
    bad = np.concatenate([np.arange(3, T - n, 7), np.arange(n, min(T, n + 40), 5)])
    cache, w = poisoned(mode, D, T, bad[:T - n], r)
    into, _ = poisoned(mode, D, n + 200, np.arange(n, n + 200), r)
    cache.evict(w, n, into=into)
    same_as_fresh(into, r, 8)
    cache.evict(w, n)
    assert cache.offset == n
    same_as_fresh(cache, r, 8)
