"""Sizes and values at the ends of what the shared, scored and evicting calls take."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_key_weights import check_scored
from test_gpu_shared import attend, check_shared, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INT_MAX = 2 ** 31 - 1


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("n_seq,n_rows,group", [(INT_MAX, INT_MAX, 1), (INT_MAX, INT_MAX, 4), (INT_MAX, INT_MAX, 6), (INT_MAX, INT_MAX, 8),
                                                (2 ** 30, 2 ** 30, 8), (2 ** 24, 1, 1), (1, 2 ** 24 - 1, 2), (INT_MAX, 1, INT_MAX)])
def test_row_counts_whose_product_wraps(n_seq, n_rows, group):
    """Refused on the host, by the declared sizes alone: (2^31 - 1)^2 * 4 is -2^34 + 4 in 64 bits."""
    import qw_amd

    prefix = filled("fp16", 1, 128, 20, rng(3))
    x = torch.zeros(128, dtype=torch.float16, device="cuda")
    call = qw_amd.lib().qw_kv_shared_attention
    assert call(prefix._h, None, n_seq, None, x.data_ptr(), group, n_rows, 0.1, x.data_ptr(), stream()) in (1, 2)
    torch.cuda.synchronize()
    assert prefix.offset == 20 and not x.any()


def test_too_many_turbo4_rows_refused():
    """2^26 query rows over a Turbo4 cache, fewer than 2^24 a KV head: the rotations' launches have a wave a row, and
    2^32 threads are one too many. Refused on the host, by the declared sizes, before workspaces and the append."""
    import qw_amd

    cache, tails = filled("turbo4", 8, 128, 20, rng(3)), filled("turbo4", 8, 128, 5, rng(4))
    x, w = torch.zeros(128, dtype=torch.float16, device="cuda"), torch.zeros((8, 20), device="cuda")
    lib, q, n = qw_amd.lib(), x.data_ptr(), 1 << 23
    free = torch.cuda.mem_get_info()[0]
    assert lib.qw_kv_shared_attention(cache._h, None, 1, None, q, 8, n, 0.1, q, stream()) == 2
    assert lib.qw_kv_attention_scored(cache._h, q, 8, n, 0.1, 0, None, 0, 0, 0.0, w.data_ptr(), 20, q, stream()) == 2
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] >= free - (64 << 20) and cache.offset == 20 and not w.any()


def test_images_of_a_batch_stay_within_their_bound():
    """A batch of prompts without a prefix: what the key tiles' images may take (2^29 halves of K) counts every
    sequence's heads. 64 sequences of 70000 keys would take 2.4 GB for them."""
    import qw_amd

    B, T, L, hq = 64, 70000, 512, 8
    prefix, tails = filled("affine4", 1, 128, 0, rng(1)), qw_amd.KVCache("affine4", B, 128, capacity=T)
    g = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(7):
        x = torch.empty((2, B, T // 7, 128), dtype=torch.float16, device="cuda").normal_(generator=g)
        tails.update(x[0], x[1])
    q = queries(rng(3), B, hq, L, 128)
    qw_amd.release_workspaces()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    out = prefix.shared_attention(q, tails, 0.09)
    torch.cuda.synchronize()
    taken = free - torch.cuda.mem_get_info()[0]
    print(f"taken {taken / 1e9:.2f} GB", flush=True)
    assert taken < 1.5e9
    k, v = (x[0, B - 1].double().cpu().numpy() for x in tails.dequantize())
    for j, i in ((0, 0), (5, 300), (7, L - 1)):
        n = T - L + i + 1
        ref, bar, _, _ = attend(q[B - 1, j, i].double().cpu().numpy(), k[:n], v[:n], 0.09)
        assert np.all(np.abs(out[B - 1, j, i].double().cpu().numpy() - ref) <= bar), (j, i)
    qw_amd.release_workspaces()


def test_one_head_takes_weights_of_any_row_stride():
    """With one KV head a row's stride means nothing: the transpose of an [n, 1] tensor is as good as any."""
    r = rng(6)
    cache, q = filled("fp16", 1, 128, 50, r), queries(r, 1, 4, 2, 128)
    plain = torch.rand((1, 50), device="cuda")
    column = torch.empty((50, 1), device="cuda").copy_(plain.t()).t()
    assert column.stride() == (1, 1)
    want = cache.attention_scored(q, 0.09, weights=plain, causal=True)
    for w in (column, plain.as_strided((1, 50), (7, 1))):
        got = cache.attention_scored(q, 0.09, weights=w, causal=True, weights_out=torch.zeros((50, 1), device="cuda").t())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(cache.evict(plain, 20, into=filled("fp16", 1, 128, 0, r)), cache.evict(column, 20, into=filled("fp16", 1, 128, 0, r))):
        assert torch.equal(a, b)
    # in place through two views of one array, one of them shorter
    got = cache.attention_scored(q, 0.09, weights=column, causal=True, weights_out=column.as_strided((1, 50), (50, 1)))
    assert torch.equal(got[1], want[1]) and torch.equal(column, want[1])
    early = plain.clone()
    want = cache.attention_scored(q, 0.09, weights=early[:, :40], causal=True)
    got = cache.attention_scored(q, 0.09, weights=early[:, :40], causal=True, weights_out=early)
    assert torch.equal(got[1], want[1]) and torch.equal(early, want[1])
    # one key: its own stride means nothing either
    one = filled("fp16", 2, 128, 1, r)
    q, grid = queries(r, 1, 4, 1, 128), torch.zeros((2, 60), device="cuda")
    one.attention_scored(q, 0.09, weights_out=grid[:, 5::30][:, :1])
    assert torch.equal(grid[:, 5], torch.full((2,), 2.0, device="cuda")) and not grid[:, 6:].any()


@pytest.mark.parametrize("L", [1, 40])
@pytest.mark.parametrize("scale", [3e38, -3e38, 1e-38])
def test_scales_at_the_ends_of_fp32(L, scale):
    """Scores of 0 stay 0 under the largest scale (times log2 e it passes fp32): a mean of the keys seen."""
    r = rng(7)
    cache, prefix = filled("affine4", 2, 128, 90, r), filled("affine4", 1, 128, 33, r)
    q = torch.zeros((1, 8, L, 128), dtype=torch.float16, device="cuda")
    out, w = cache.attention_scored(q, scale, causal=True)
    check_scored(out, w, q, cache, scale, True)
    q = torch.zeros((2, 4, L, 128), dtype=torch.float16, device="cuda")
    check_shared(prefix.shared_attention(q, cache, scale), q, prefix, cache, None, scale)


def test_evict_counts_beyond_an_int_are_not_wrapped():
    """-2^32 + 3 is not 3: negative counts are refused whatever their size, and large ones are large."""
    import qw_amd

    cache, w = filled("affine8", 2, 128, 20, rng(8)), torch.rand((2, 20), device="cuda")
    for a in ({"budget": 10, "sink": -2 ** 32 + 3}, {"budget": 10, "recent": -2 ** 32}, {"budget": -2 ** 32 + 5},
              {"budget": 10, "sink": 2 ** 32}, {"budget": 2 ** 31 - 1, "sink": 2 ** 40}):
        with pytest.raises(qw_amd.QwError) as e:
            cache.evict(w, **a)
        assert e.value.status == 1 and cache.offset == 20, a
    kept, _ = cache.evict(w, 2 ** 40, sink=2 ** 30, recent=2 ** 30 - 1)
    assert kept.shape == (2, 20) and cache.offset == 20
