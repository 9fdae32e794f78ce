"""Shared and scored attention in the forms that sizes and stored scales choose: fp16 caches under few rows, several
32-key chunks a wave, several query tiles without and with laid-out key tiles, six row tiles of a computing wave each,
and scales outside the range of the short dequantization. Against 64 bits at the bars of test_gpu_shared and
test_gpu_key_weights."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_key_weights import check_scored
from test_gpu_shared import check_shared, dev, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SHARED = [
    # prefix mode, tail mode, hq, hkv, D, sequences, rows, prefix, tail
    ("fp16", "fp16", 16, 2, 256, 1, 1, 5000, 40),       # 8 rows a head
    ("fp16", "fp16", 8, 2, 256, 2, 2, 2100, 300),       # 16 and 8
    ("fp16", "fp16", 16, 8, 256, 1, 1, 16500, 3),       # splits of some 512 keys: two chunks a wave
    ("fp16", "fp16", 32, 8, 128, 1, 2, 33000, 70),      # of some 1024
    ("affine4", "affine4", 16, 8, 256, 1, 1, 16500, 3),
    ("int8", "affine8", 8, 8, 128, 3, 1, 33000, 2),
    ("turbo4", "turbo4", 8, 8, 128, 1, 1, 33000, 2),
    ("affine4", "affine8", 8, 2, 128, 20, 16, 500, 60),  # 1280 rows: five query tiles
    ("fp16", "fp16", 8, 2, 128, 9, 8, 700, 300),         # 288: two
    ("affine8", "affine8", 12, 2, 128, 3, 100, 90, 130),  # tails of 600 rows: three
    ("fp16", "fp16", 4, 1, 256, 5, 33, 200, 40),         # D = 256: 660 rows and tails of 132
    ("affine4", "affine4", 24, 4, 256, 16, 1, 700, 40),  # 96 rows: six row tiles
    ("fp16", "fp16", 24, 4, 256, 16, 1, 700, 40),
    ("affine8", "int8", 24, 4, 256, 15, 1, 300, 9),      # 90, the last one partly filled
    ("int8", "int8", 20, 4, 256, 15, 1, 300, 9),         # 75: five
    ("turbo4", "turbo4", 24, 4, 256, 16, 1, 700, 40),
]


@pytest.mark.parametrize("pm,tm,hq,hkv,D,B,L,P,T", SHARED)
def test_shared_forms(pm, tm, hq, hkv, D, B, L, P, T):
    print(f"case {pm} {tm} hq={hq} hkv={hkv} D={D} B={B} L={L} P={P} T={T}", flush=True)
    if pm == "turbo4":
        from test_gpu_shared import test_shared_turbo4

        return test_shared_turbo4(hq, hkv, D, B, L, P, T)
    r = rng(P + T + B + L)
    prefix, tails = filled(pm, hkv, D, P, r), filled(tm, B * hkv, D, T, r)
    q = queries(r, B, hq, L, D)
    starts = r.integers(0, T - L + 1, B).astype(np.int32)
    out = prefix.shared_attention(q, tails, D ** -0.5, starts=dev(starts))
    check_shared(out, q, prefix, tails, starts, D ** -0.5, only=range(0, B, max(1, B * hq * L // 1500)))
    assert torch.equal(out, prefix.shared_attention(q, tails, D ** -0.5, starts=dev(starts)))


@pytest.mark.parametrize("mode,hq,hkv,D,L", [("affine4", 16, 1, 256, 125), ("affine8", 16, 1, 128, 242), ("int8", 32, 2, 256, 121)])
def test_batch_of_prompts_over_images(mode, hq, hkv, D, L):
    """No prefix and no starts, 16 query tiles a sequence: each sequence's key tiles laid out once."""
    r = rng(L)
    prefix, tails = filled(mode, hkv, D, 0, r), filled(mode, 3 * hkv, D, L + 70, r)
    q = queries(r, 3, hq, L, D)
    check_shared(prefix.shared_attention(q, tails, D ** -0.5), q, prefix, tails, None, D ** -0.5, only=(0, 2))


SCORED = [
    # mode, hq, hkv, D, rows, keys, causal
    ("fp16", 16, 2, 256, 1, 5000, True),
    ("fp16", 16, 8, 256, 1, 16500, True),       # two chunks a wave
    ("fp16", 16, 4, 256, 4, 700, False),
    ("fp16", 32, 8, 128, 2, 33000, True),
    ("affine4", 16, 8, 256, 2, 16500, True),
    ("affine8", 8, 8, 128, 1, 33000, False),
    ("affine8", 8, 2, 128, 100, 900, True),     # 400 rows: two query tiles
    ("fp16", 16, 2, 128, 60, 1300, True),       # 480
    ("affine4", 24, 4, 256, 16, 2000, True),    # 96: six row tiles
    ("fp16", 24, 4, 256, 15, 2000, True),
    ("affine4", 24, 4, 256, 128, 130, True),    # 768 rows, nearly as many as keys
]


@pytest.mark.parametrize("mode,hq,hkv,D,L,T,causal", SCORED)
def test_scored_forms(mode, hq, hkv, D, L, T, causal):
    print(f"case {mode} hq={hq} hkv={hkv} D={D} L={L} T={T} causal={causal}", flush=True)
    r = rng(T + L + D)
    cache, q = filled(mode, hkv, D, T, r), queries(r, 1, hq, L, D)
    before = torch.rand((hkv, T), device="cuda")
    out, w = cache.attention_scored(q, D ** -0.5, weights=before, decay=0.5, causal=causal)
    check_scored(out, w, q, cache, D ** -0.5, causal, before, 0.5)
    again = cache.attention_scored(q, D ** -0.5, weights=before, decay=0.5, causal=causal)
    assert torch.equal(out, again[0]) and torch.equal(w, again[1])


@pytest.mark.parametrize("mode", ["affine4", "affine8"])
@pytest.mark.parametrize("sigma", [4000.0, 1e-3])
@pytest.mark.parametrize("hq,hkv,D,L,T", [
    (24, 4, 256, 1, 700), (8, 2, 128, 4, 300),      # few rows
    (24, 4, 256, 20, 300), (16, 2, 128, 40, 500),   # many
    (16, 1, 256, 125, 260), (16, 1, 128, 250, 260),  # laid-out key tiles
])
def test_scales_outside_the_short_dequantization(mode, sigma, hq, hkv, D, L, T):
    """Scales from 64 on, and 4-bit ones below 2^-10, take the long dequantization in the whole cache."""
    print(f"case {mode} sigma={sigma} hq={hq} hkv={hkv} D={D} L={L} T={T}", flush=True)
    r = rng(T + L)
    scale = float(np.float32(D ** -0.5 / sigma))
    cache, q = filled(mode, hkv, D, T, r, sigma=sigma), queries(r, 1, hq, L, D)
    scales = cache.snapshot_tensors()["k_scales"].float().abs()
    assert bool((scales >= 64).any()) == (sigma == 4000.0) and bool((scales < 2.0 ** -10).any()) == (sigma == 1e-3)
    out, w = cache.attention_scored(q, scale, causal=True)
    check_scored(out, w, q, cache, scale, True)
    # as the prefix of a batch, before tails in the short range; and as the tails
    ones = filled(mode, 2 * hkv, D, 20, r, sigma=1.0)
    L = min(L, 20)
    q = queries(r, 2, hq, L, D)
    starts = np.array([0, 20 - L], np.int32)
    check_shared(cache.shared_attention(q, ones, scale, starts=dev(starts)), q, cache, ones, starts, scale)
    if hkv % 2 == 0:
        short = filled(mode, hkv // 2, D, 100, r)
        q = queries(r, 2, hq // 2, L, D)
        check_shared(short.shared_attention(q, cache, scale), q, short, cache, None, scale)
