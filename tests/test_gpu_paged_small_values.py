"""Attention over pages of 4- and 8-bit codes whose V steps are small: a weight times its key's step keeps its bits.

Long runs of keys go to one wave by a table that names the same few pages over and over, and by many KV heads. The bar, with
u = 2^-11, e = 2^-24, codes c of step s and base b, c0 the middle of the codes (int8: none), m = b + c0 s:
  a weight times a step is rounded to fp16 and meets c - c0 (int8's codes are whole numbers beside 0: 128 above themselves in
  the kernel, less 128), a weight alone meets m, which is rounded once too: u (|c - c0| s + 2 |m|) of each key's weight;
  below fp16's normal numbers half a step, 2^-25: the row's largest weight stands at 2^10 or more, steps are lifted to
  the largest one's power of two, but by 2^15 at most, and no more than leaves |m| below 2^15:
  2^-35 (128 max(s, 2^-15) + 2 |m|) of the row's largest weight for every key;
  sums in fp32 as in test_gpu_paged.py: a score g = (D + 40) e |scale| sum |q| H, twice, the output (n / 32 + 40) e sum p H;
  the output's rounding, u of itself or 2^-25."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import E, U, codes_of, dev, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def held(mode, x, D):
    """[T, D] fp16 rows of a head as one sequence's cache holds them, in 64 bits: values, H, |c - c0| s, steps, |m|."""
    import qw_amd

    c = qw_amd.KVCache(mode, 1, D)
    c.update(dev(x[None]), dev(x[None]))
    t = c.snapshot_tensors()
    if mode == "int8":
        s = t["key_scales"].double().cpu().numpy()
        y = (t["keys"].double().cpu().numpy() * s)[0]
        s = np.broadcast_to(s[0], y.shape)
        return y, np.abs(y) + 256 * s, np.abs(y), s, np.zeros_like(y)
    s, b = (np.repeat(t[n].double().cpu().numpy(), 64, -1)[0] for n in ("k_scales", "k_biases"))
    code, c0 = codes_of(t["k_codes"], c.bits, D)[0], 2.0 ** (c.bits - 1)
    return code * s + b, np.abs(code * s) + np.abs(b), np.abs((code - c0) * s), np.abs(s), np.abs(b + c0 * s)


CASES = [
    # D, heads, pages named, the first key's lead over the others' scores, V's size, its shift, the size of page 1's other keys
    (128, 1024, 64, 14.2, 1e-3, 0.0, 0.0),
    (256, 512, 40, 13.0, 1e-3, 0.0, 0.0),
    (128, 1024, 30, 12.0, 3e-5, 0.0, 0.0),
    (128, 1024, 30, 15.0, 1e-6, 0.0, 0.0),
    (256, 512, 20, 9.0, 1.0, 0.0, 0.0),
    (128, 1024, 30, 13.0, 1e-3, 0.5, 0.0),      # bases far above the steps
    (128, 1024, 30, 13.0, 0.05, 3e4, 0.0),
    (128, 1024, 64, 14.2, 1e-3, 0.0, 0.3),      # (int8's step of a key of zeros is 1, and its score's bar as wide)
    (256, 512, 40, 13.0, 3e-4, 0.0, 0.3),
    (128, 1024, 30, 13.0, 300.0, 0.0, 0.3),
]


@pytest.mark.parametrize("mode", ["affine8", "affine4", "int8"])
@pytest.mark.parametrize("D,hkv,named,lead,size,shift,rest", CASES)
@pytest.mark.parametrize("late", [False, True])
def test_weights_times_small_steps(mode, D, hkv, named, lead, size, shift, rest, late):
    import qw_amd

    print(f"case {mode} D={D} lead={lead} size={size} shift={shift} rest={rest} late={late}", flush=True)
    r = rng(named + D)
    ps, n = 256, 256 * named
    cache = qw_amd.PagedKVCache(mode, hkv, D, 3, page_size=ps)
    k, v = np.zeros((2 * ps, D), np.float16), np.zeros((2 * ps, D), np.float16)
    if rest:
        k[ps:] = (rest / D * r.standard_normal((ps, D))).astype(np.float16)
    k[ps] = lead / D  # page 1's first key; page 0's have scores near 0
    k[:ps] = (0.3 / D * r.standard_normal((ps, D))).astype(np.float16)
    v[:ps] = (size * (np.where(np.arange(D) % 3, 1.0, -0.5) + 0.2 * r.standard_normal((ps, D))) + shift).astype(np.float16)
    v[ps:] = (0.1 * size * r.standard_normal((ps, D))).astype(np.float16)
    cache.update(*(dev(x)[:, None].expand(-1, hkv, -1) for x in (k, v)), ints([[0, 1]]), ints([0]))
    pages = np.zeros(named, int)
    pages[-1 if late else 0] = 1
    q = torch.ones((1, hkv, 1, D), dtype=torch.float16, device="cuda")
    out = cache.attention(q, ints([pages]), ints([n]), 1.0)
    assert torch.equal(out, out[:, :1].expand_as(out))

    at = (ps * pages[:, None] + np.arange(ps)).reshape(-1)
    kv, kh, *_ = held(mode, k, D)
    vv, vh, vc, vs, vm = held(mode, v, D)
    s = kv.sum(1)[at]
    p = np.exp(s - s.max())
    p, total = p / p.sum(), p.sum()
    ref = p @ vv[at]
    g = (D + 40) * E * kh.sum(1).max()
    bar = p @ (U * (vc + 2 * vm))[at] + (2 * g + (n / 32 + 40) * E) * (p @ vh[at]) + U * np.abs(ref) + 2.0 ** -25
    bar += n * 2.0 ** -35 * (128 * max(vs.max(), 2.0 ** -15) + 2 * vm.max()) / total
    err = np.abs(out[0, 0, 0].double().cpu().numpy() - ref) / bar
    print(f"worst error {err.max():.3f} of the bar", flush=True)
    assert err.max() <= 1.0
