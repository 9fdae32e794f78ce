"""Calls over pages that need no workspace make none, and take their tensors as they lie."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import MODES, Sequences, dev, ints, queries, side_stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def captured(f, stream):
    """f's outputs and its graph, from a first call inside a capture."""
    torch.cuda.synchronize()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = f()
    return out, g


@pytest.mark.parametrize("mode,lengths", [("affine8", [1300, 0, 300]), ("fp16", [40, 1100]), ("int8", [0, 2100] + [5, 260, 0, 17] * 17)])
def test_rows_that_fill_the_card_need_no_workspace(mode, lengths):
    """8192 rows of a KV head: a workgroup for each 32 takes all sequences, and nothing is cut."""
    r = rng(sum(lengths))
    s = Sequences(r, mode, 1, 128, 16, lengths)
    B = len(lengths)
    q, t, n = dev((2 * r.standard_normal((1, 32, 256, 128))).astype(np.float16)).expand(B, -1, -1, -1), ints(s.table), ints(lengths)
    out, g = captured(lambda: s.cache.attention(q, t, n, 0.09), side_stream(4))
    for less in (0, 3):
        now = [max(x - less, 0) for x in lengths]
        n.copy_(ints(now))
        g.replay()
        torch.cuda.synchronize()
        s.check(out[:, 31:], q[:, 31:], 0.09, lengths=now)
        assert torch.equal(out, s.cache.attention(q, t, n, 0.09))


def in_a_large_pool(r, mode, hkv, D, ps, lengths, width, nbytes):
    """Sequences whose pages lie anywhere in a pool of more than nbytes bytes of codes."""
    import qw_amd

    s = Sequences(r, mode, hkv, D, ps, lengths)
    s.cache.close()
    s.n_pages = int(nbytes // (2 * ps * hkv * D * s.cache.bits // 8)) + 2
    at = s.table >= 0
    s.table = np.pad(s.table, ((0, 0), (0, width - s.width)), constant_values=-1)
    s.width = width
    named = int(at.sum())
    s.table[:, :at.shape[1]][at] = np.concatenate([[s.n_pages - 1, 0], 1 + r.permutation(s.n_pages - 2)[:named - 2]])
    s.cache = qw_amd.PagedKVCache(mode, hkv, D, s.n_pages, page_size=ps)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    s.cache.update(dev(np.concatenate(s.k)), dev(np.concatenate(s.v)), ints(s.table), ints([0] * len(lengths)), offsets=ints(offsets))
    return s


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n_seq,L,picks", [(3, 1, 0), (3, 3, 0), (70, 1, 0), (3, 1, 9), (70, 2, 9)])
def test_keys_past_the_caches(mode, D, n_seq, L, picks):
    """Tables and pools of more than the caches hold, on both sides of 64 sequences, of one and two row tiles, over all pages
    and over picked ones."""
    r = rng(D + n_seq + L + picks)
    hkv, ps = 2, 16
    lengths = [0, 33, 700] if n_seq == 3 else [int(x) for x in r.integers(0, 90, n_seq)]
    lengths[1], lengths[n_seq - 1] = 150, 1700
    s = in_a_large_pool(r, mode, hkv, D, ps, lengths, 40000, 300 * 2 ** 20)
    hq = 8 * hkv if L > 2 else 4 * hkv
    q, t, n = queries(r, n_seq, hq, L, D), ints(s.table), ints(lengths)
    picked = None
    if picks:
        picked = np.full((n_seq, hkv, 20000), -1, dtype=np.int32)  # (as many as make a list's keys more than the caches hold)
        for b, length in enumerate(lengths):
            for h in range(hkv):
                some = r.permutation(-(-length // ps))[:picks]
                picked[b, h, :len(some)] = some
    out = s.cache.attention(q, t, n, 0.08, picked=None if picked is None else ints(picked))
    s.check(out, q, 0.08, picked=picked)


@pytest.mark.parametrize("mode", MODES)
def test_a_pool_named_over_and_over(mode):
    """More keys than the pool holds, by a wide table that names its pages again and again, and sequences that share them."""
    r = rng(81)
    s = Sequences(r, mode, 8, 128, 16, [160])
    table = np.full((5, 20000), -1)
    table[:, :900] = s.table[0, np.arange(900) % 10]
    lengths = [14400, 160, 1, 0, 333]
    q = queries(r, 5, 16, 1, 128)
    out = s.cache.attention(q, ints(table), ints(lengths), 0.1)
    again = Sequences(r, mode, 8, 128, 16, [1])
    again.lengths = lengths
    again.k, again.v = ([np.tile(x[0], (90, 1, 1))[:m] for m in lengths] for x in (s.k, s.v))
    again.check(out, q, 0.1)


@pytest.mark.parametrize("counts", [[1] * 5, [40, 0, 7]])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_projections_at_any_offset(counts, off):
    """A projection that begins inside a flat buffer, 2, 4 or 8 bytes off 16, one token a sequence and more."""
    import qw_amd

    r = rng(82 + off)
    hq, hkv, D, n, B = 4, 2, 128, sum(counts), len(counts)
    row = (hq + 2 * hkv) * D
    flat = dev(r.standard_normal(n * row + off).astype(np.float16))
    qkv = flat[off:].view(n, row)
    pos, starts = ints(r.integers(0, 9000, (3, n))), ints([3] * B)
    offsets = ints(np.concatenate([[0], np.cumsum(counts)]))
    table = ints(r.permutation(4 * B).reshape(B, 4))
    q0, k0 = qw_amd.rope_axes(qkv.clone(), pos, (8, 4, 4), hq, hkv, D, 1e4)
    for x, y in zip(qw_amd.rope_axes(qkv, pos, (8, 4, 4), hq, hkv, D, 1e4), (q0, k0)):
        assert torch.equal(x, y)
    a, b = (qw_amd.PagedKVCache("affine8", hkv, D, 4 * B, page_size=16) for _ in range(2))
    assert torch.equal(a.rope_update(qkv, pos, (8, 4, 4), hq, 1e4, table, starts, offsets=offsets), q0)
    b.update(k0, qkv.view(n, -1, D)[:, hq + hkv:], table, starts, offsets)
    for x, y in zip(a.gather(table, starts, n, offsets), b.gather(table, starts, n, offsets)):
        assert torch.equal(x, y)


def test_stream_per_thread_where_no_workspace_is_kept():
    """A token a sequence rotates in the launch that stores it, on any stream; more pass through a workspace of their stream."""
    import qw_amd

    r = rng(83)
    hq, hkv, D = 4, 2, 128
    a, b = (qw_amd.PagedKVCache("fp16", hkv, D, 6, page_size=16) for _ in range(2))
    qkv = dev(r.standard_normal((3, (hq + 2 * hkv) * D)).astype(np.float16))
    pos, starts, table = ints(r.integers(0, 9000, (1, 3))), ints([0, 5, 17]), ints([[0, 1], [2, 3], [4, 5]])
    want = a.rope_update(qkv, pos, (64,), hq, 1e4, table, starts)
    q = torch.zeros_like(want)
    torch.cuda.synchronize()

    def call(n_seq):
        return qw_amd.lib().qw_paged_rope_update(b._h, qkv.data_ptr(), hq, D, 0, 1e4, 1.0, pos.data_ptr(), 3, 1, bytes(64),
                                                 q.data_ptr(), 3, n_seq, None, starts.data_ptr(), table.data_ptr(), 2, 2, 2)

    assert call(1) == 2 and b"hipStreamPerThread" in qw_amd.lib().qw_last_error()
    assert torch.all(q == 0)
    assert call(3) == 0
    torch.cuda.synchronize()
    assert torch.equal(q, want)
    for x, y in zip(a.gather(table, starts, 3), b.gather(table, starts, 3)):
        assert torch.equal(x, y)


def test_a_refused_pool_leaves_a_capture_alone():
    """A pool that is refused by its arguments is refused before any device call: one that waits for the device ends a capture."""
    import qw_amd

    x = torch.zeros(8, device="cuda")

    def refused():
        for args in (("fp16", 2, 64, 4), ("fp16", 2, 128, 0), ("turbo4", 2, 128, 4)):
            with pytest.raises(qw_amd.QwError):
                qw_amd.PagedKVCache(*args)
        x.add_(1)

    _, g = captured(refused, side_stream(6))
    g.replay()
    torch.cuda.synchronize()
    assert torch.all(x == 1)
