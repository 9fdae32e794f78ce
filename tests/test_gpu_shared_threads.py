"""The shared, scored and evicting calls from several host threads, each on a stream of its own, over one prefix: every
result is the one that the calls give alone."""
import threading

import numpy as np
import pytest

from conftest import rng
from test_gpu_evict import weights
from test_gpu_shared import dev, filled, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def step(prefix, seed, mode):
    """One request: a batch over the prefix, a scored chunk and a cut in place; all that they return and leave."""
    r = rng(seed)
    tails, own = filled(mode, 6, 128, 40 + seed, r), filled(mode, 2, 128, 700 + 13 * seed, r)
    out = []
    for L in (1, 7):
        q = queries(r, 3, 8, L, 128)
        k, v = (dev(r.standard_normal((3, 2, L, 128)).astype(np.float16)) for _ in range(2))
        out.append(prefix.update_and_shared_attention(q, tails, k, v, 0.09, starts=dev(np.array([0, 9, 30], np.int32))))
        q = queries(r, 1, 8, 5 * L, 128)
        out += own.attention_scored(q, 0.09, weights=dev(weights(r, 2, own.offset, "log")), causal=True)
    out += own.evict(out[-1], 300 + seed, sink=4, recent=32)
    out += list(own.snapshot_tensors().values())
    out.append(own.attention(queries(r, 1, 8, 2, 128), 0.09, causal=True))
    return out


@pytest.mark.parametrize("mode", ["affine4", "fp16", "turbo4"])
def test_threads_and_streams(mode):
    prefix = filled(mode, 2, 128, 1500, rng(77))
    want = [step(prefix, s, mode) for s in range(4)]
    torch.cuda.synchronize()
    got, errors = [[] for _ in range(4)], []

    def work(s):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(3):
                    got[s].append(step(prefix, s, mode))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for s in range(4):
        for again in got[s]:
            assert len(again) == len(want[s]) and all(torch.equal(a, b) for a, b in zip(again, want[s])), s
