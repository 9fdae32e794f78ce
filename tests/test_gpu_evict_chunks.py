"""Eviction's select by chunks of keys (caches of more than 16384), every digit of the weights at work: kept
positions, weights and rows exact, against a sort on the host."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_evict import check_evict, weights
from test_gpu_shared import dev, filled

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def near(r, hkv, T, bits):
    """Weights that share all but their lowest `bits` bits, ties among them."""
    low = r.integers(0, 1 << bits, (hkv, T)).astype(np.uint32)
    return (np.uint32(0x3F8A5000) + low).view(np.float32)


CASES = [
    # hkv, T, budget, sink, recent, weights
    (4, 16385, 4000, 4, 512, "log"),
    (2, 20481, 20000, 0, 1, "log"),
    (3, 40000, 700, 0, 0, "odd"),
    (2, 33000, 30000, 4, 32, "odd"),        # the cut among the negative ones
    (2, 33000, 32900, 0, 0, "odd"),         # and among the NaN
    (2, 20000, 5000, 4, 32, "same"),
    (4, 30000, 9000, 4, 512, "near10"),     # the third digit alone decides
    (4, 30000, 9000, 4, 512, "near6"),      # with some 450 ties a value
    (2, 50000, 20000, 100, 9000, "near20"),  # the second and third
    (2, 20000, 600, 88, 512, "log"),        # sinks and recent keys are all of it
    (2, 20000, 20000, 4, 32, "log"),        # everything stays
    (2, 20000, 30000, 4, 19999, "odd"),
    (1, 17000, 16999, 0, 0, "near10"),      # one key goes
    (2, 20000, 9000, 5000, 4000, "same"),   # sinks past a chunk, nothing else
    (2, 30000, 12001, 5000, 7000, "near10"),  # one key of the middle
    (2, 25000, 1, 0, 0, "near10"),
]


@pytest.mark.parametrize("hkv,T,budget,sink,recent,kind", CASES)
def test_chunked_select(hkv, T, budget, sink, recent, kind):
    import qw_amd

    print(f"case hkv={hkv} T={T} budget={budget} sink={sink} recent={recent} {kind}", flush=True)
    r = rng(T + budget)
    cache = filled("affine4", hkv, 128, T, r)
    w = near(r, hkv, T, int(kind[4:])) if kind.startswith("near") else weights(r, hkv, T, kind)
    into = qw_amd.KVCache("affine4", hkv, 128)
    kept, wo = check_evict(cache, into, dev(w), budget, sink, recent)
    kept2, wo2 = check_evict(cache, None, dev(w), budget, sink, recent)
    assert torch.equal(kept, kept2) and torch.equal(wo.view(torch.int32), wo2.view(torch.int32))


@pytest.mark.parametrize("T,budget,kind", [(1000, 300, "near10"), (3000, 900, "near6"), (16000, 5000, "near20"), (16384, 16000, "odd"),
                                           (9000, 4000, "log")])
def test_select_of_one_workgroup_a_head(T, budget, kind):
    test_chunked_select(2, T, budget, 4, 32, kind)
