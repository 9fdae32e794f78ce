"""Rotary positions of several axes (qw_rope_axes) against the rotation in 64 bits.

The bar: the angle is reduced in 64 bits and its cosine and sine are taken in fp32 of an fp32 angle, at most 2^-22 off
(the angle's rounding, pi 2^-24, and the functions'); a product and a fused sum, three roundings of 2^-24; the result is
rounded to fp16, half a step 2^-11 of itself or 2^-25:  |error| <= 2^-11 |r| + 2^-25 + 2^-21 (|x1| + |x2|)."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import dev, ints, stored

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def axis_of(sections, interleaved):
    out = []
    for p in range(sum(sections)):
        if interleaved:
            a = p % len(sections)
            out.append(a if p < len(sections) * sections[a] else 0)
        else:
            out.append(next(a for a in range(len(sections)) if p < sum(sections[:a + 1])))
    return np.array(out)


def turned(x, positions, sections, base, scale, interleaved, traditional):
    """[n, heads, D] rows in 64 bits, and the bar."""
    half = sum(sections)
    axis = axis_of(sections, interleaved)
    theta = np.float64(np.float32(scale)) * np.float64(np.float32(base)) ** (-np.arange(half) / half)
    angle = (positions.astype(np.float64)[axis] * theta[:, None]).T[:, None]
    x = x.astype(np.float64)
    y, bar = x.copy(), np.zeros_like(x)
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if traditional else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., one], x[..., two]
    y[..., one] = a * np.cos(angle) - b * np.sin(angle)
    y[..., two] = a * np.sin(angle) + b * np.cos(angle)
    for z in (one, two):
        bar[..., z] = 2.0 ** -11 * np.abs(y[..., z]) + 2.0 ** -25 + 2.0 ** -21 * (np.abs(a) + np.abs(b))
    return y, bar


CASES = [
    # n, hq, hkv, D, sections, interleaved, traditional, scale, positions up to
    (1, 24, 4, 256, (11, 11, 10), True, False, 1.0, 100),
    (7, 8, 2, 128, (16, 24, 24), False, False, 1.0, 5000),
    (1030, 4, 1, 128, (8, 4, 4), True, True, 1.0, 40000),
    (5000, 2, 2, 256, (64, 32, 32), True, False, 0.25, 2 ** 31 - 1),
    (33, 3, 1, 128, (1, 0, 2), False, False, 1.0, 10 ** 6),       # three pairs: dim by dim
    (9, 2, 1, 34, (5,), False, True, -2.0, 1000),                 # a head of 34 dims, one axis
    (600, 1, 1, 512, (100, 100, 56), False, False, 1.0, 10 ** 6),
    (12, 5, 3, 80, (2, 2, 2, 2), True, False, 1.0, 300),
]


@pytest.mark.parametrize("n,hq,hkv,D,sections,interleaved,traditional,scale,far", CASES)
def test_rope_axes(n, hq, hkv, D, sections, interleaved, traditional, scale, far):
    import qw_amd

    r = rng(n + D)
    qkv = r.standard_normal((n, hq + 2 * hkv, D)).astype(np.float16)
    pos = r.integers(0, far, (len(sections), n), dtype=np.int64).astype(np.int32)
    pos[:, 0] = [-far // 2, far, 0, 1][:len(sections)] if far < 2 ** 31 - 1 else far
    q, k = qw_amd.rope_axes(dev(qkv.reshape(n, -1)), ints(pos), sections, hq, hkv, D, 1e6, scale, interleaved, traditional)
    want, bar = turned(qkv[:, :hq + hkv], pos, sections, 1e6, scale, interleaved, traditional)
    got = np.concatenate([q.cpu().numpy(), k.cpu().numpy()], 1).astype(np.float64)
    assert (np.abs(got - want) <= bar).all(), np.max(np.abs(got - want) - bar)


def test_one_axis_is_the_plain_rotation():
    """All axes alike: qw_fused_rope_qk_append's rotation, which forms its angles in fp32."""
    import qw_amd

    r = rng(5)
    n, hq, hkv, D = 50, 4, 2, 128
    qkv = dev(r.standard_normal((n, (hq + 2 * hkv) * D)).astype(np.float16))
    pos = torch.arange(n, dtype=torch.int32, device="cuda").expand(3, n)
    q, k = qw_amd.rope_axes(qkv, pos, (16, 24, 24), hq, hkv, D, 1e4)
    q1, k1, _ = qw_amd.fused_rope_qk_append(qkv[None], hq, hkv, D, 128, 1e4, dest_layout=1)
    # an angle below 50 is off by at most 50 * 4 * 2^-24 there: less than 2^-16 of the pair's magnitude (below 2^3); then
    # both round to fp16, a step of 2^-8 apart at most
    assert (q.float() - q1[0].transpose(0, 1).float()).abs().max() <= 2.0 ** -13 + 2.0 ** -8
    assert (k.float() - k1[0].float()).abs().max() <= 2.0 ** -13 + 2.0 ** -8


@pytest.mark.parametrize("mode", ["affine8", "fp16", "int8", "affine4"])
def test_rotated_rows_in_their_pages(mode):
    import qw_amd

    r = rng(6)
    hq, hkv, D, ps = 4, 2, 128, 32
    counts = [1, 70, 0, 33]
    n = sum(counts)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    starts = [31, 5, 9, 0]
    cache = qw_amd.PagedKVCache(mode, hkv, D, 12, page_size=ps)
    table = ints(r.permutation(12).reshape(4, 3))
    big = dev(r.standard_normal((n, 2 * (hq + 2 * hkv) * D)).astype(np.float16))
    qkv = big[:, (hq + 2 * hkv) * D:]
    pos = ints(r.integers(0, 9000, (3, n)))
    q = cache.rope_update(qkv, pos, (8, 4, 4), hq, 1e4, table, ints(starts), offsets=ints(offsets), interleaved=True)
    q1, k1 = qw_amd.rope_axes(qkv.contiguous(), pos, (8, 4, 4), hq, hkv, D, 1e4, interleaved=True)
    assert torch.equal(q, q1)
    v = qkv.reshape(n, -1, D)[:, hq + hkv:].cpu().numpy()
    got = cache.gather(table, ints(starts), n, offsets=ints(offsets))
    for b in range(4):
        at = slice(offsets[b], offsets[b + 1])
        if counts[b]:
            for x, y in zip(got, stored(mode, k1[at].cpu().numpy(), v[at], hkv, D)):
                assert np.array_equal(x[at].cpu().numpy(), y)
    assert cache.rope_update(qkv[:0], pos[:, :0], (8, 4, 4), hq, 1e4, table, ints(starts), offsets=ints([0] * 5)).shape == (0, hq, D)


def test_rope_axes_refusals():
    import qw_amd

    x = torch.zeros((4, 8 * 64), dtype=torch.float16, device="cuda")
    pos = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    ok = dict(n_q_heads=4, n_kv_heads=2, head_dim=64, rope_base=1e4)
    qw_amd.rope_axes(x, pos, (8, 12, 12), **ok)
    for args, kw in (
        ((x, pos, (8, 12, 13)), ok),                      # more dims than a head has
        ((x, pos, (0, 0, 0)), ok),
        ((x, pos, (8, -1, 9)), ok),
        ((x, pos[:2], (8, 12, 12)), ok),
        ((x, pos.long(), (8, 12, 12)), ok),
        ((x.float(), pos, (8, 12, 12)), ok),
        ((x, pos, (8, 12, 12)), dict(ok, n_q_heads=5)),
        ((x, pos, (8, 12, 12)), dict(ok, rope_base=0.0)),
        ((x, pos, (8, 12, 12)), dict(ok, rope_base=float("nan"))),
        ((x, pos, (8, 12, 12)), dict(ok, rope_scale=float("inf"))),
    ):
        with pytest.raises(qw_amd.QwError):
            qw_amd.rope_axes(*args, **kw)
    assert qw_amd.rope_axes(x[:0], pos[:, :0], (8, 12, 12), **ok)[0].shape == (0, 4, 64)


@pytest.mark.parametrize("mode,hq,hkv,D,sections,interleaved,traditional", [
    ("fp16", 24, 4, 256, (16, 24, 24), False, False), ("affine8", 9, 3, 128, (8, 4, 4), True, True), ("int8", 2, 2, 256, (128,), False, False),
    ("affine4", 20, 2, 128, (3, 2, 2), True, False), ("affine8", 8, 8, 256, (2, 2), False, True), ("int8", 3, 1, 128, (64,), False, True)])
@pytest.mark.parametrize("counts", [[1] * 9, [3, 0, 0, 9] + [0] * 9, [1, 0, 5, 30], [3000, 1], [1] * 256, [1] * 257])
def test_rotated_on_their_way(mode, hq, hkv, D, sections, interleaved, traditional, counts):
    """Few tokens rotate in the launch that stores them, many before it: both as rope_axes and update give them, with tokens
    that have no page among them."""
    import qw_amd

    r = rng(sum(counts) + D)
    n, B, ps = sum(counts), len(counts), 16
    starts = [int(x) for x in r.integers(0, 40, B)]
    width = -(-(max(counts) + 40) // ps)
    table = r.permutation(B * width).reshape(B, width)
    table[B - 1, starts[B - 1] // ps] = -1
    table = ints(table)
    offsets = None if counts == [1] * B else ints(np.concatenate([[0], np.cumsum(counts)]))
    qkv = dev(r.standard_normal((n, (hq + 2 * hkv) * D)).astype(np.float16))
    pos = ints(r.integers(0, 100000, (len(sections), n)))
    a, b = (qw_amd.PagedKVCache(mode, hkv, D, B * width, page_size=ps) for _ in range(2))
    args = dict(interleaved=interleaved, traditional=traditional)
    q = a.rope_update(qkv, pos, sections, hq, 1e6, table, ints(starts), offsets=offsets, **args)
    q1, k1 = qw_amd.rope_axes(qkv, pos, sections, hq, hkv, D, 1e6, **args)
    b.update(k1, qkv.view(n, -1, D)[:, hq + hkv:], table, ints(starts), offsets)
    assert torch.equal(q, q1)
    for x, y in zip(a.gather(table, ints(starts), n, offsets), b.gather(table, ints(starts), n, offsets)):
        assert torch.equal(x, y)
