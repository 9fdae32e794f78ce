"""Page selection over some thousand columns: scores in the registers of sixteen waves, with whole runs of equal ones."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_paged import dev, ints, queries, rows
from test_gpu_paged_select import bounds, ranked, scores_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("columns,few,budget,sink,recent", [
    (2049, 1, 1000, 3, 2),       # one page: all scores equal
    (4096, 5, 700, 0, 0),        # some eight hundred of each
    (4100, 5, 4099, 7, 0),       # all but one
    (8192, 37, 1, 0, 0),         # one of some two hundred equal ones
    (8192, 3, 5000, 64, 100),    # whole runs, and a part of one
    (8191, 900, 2000, 1, 1),     # about nine of each
    (6000, 37, 66, 64, 2),       # nothing left to choose
])
@pytest.mark.parametrize("missing", [False, True])
def test_equal_scores_over_many_waves(columns, few, budget, sink, recent, missing):
    import qw_amd

    r = rng(columns + budget)
    ps, D, hkv = 16, 128, 2
    cache = qw_amd.PagedKVCache("affine8", hkv, D, few, page_size=ps)
    k = rows(r, few * ps, hkv, D)
    cache.update(dev(k), dev(k), ints([np.arange(few)]), ints([0]))
    table = r.integers(0, few, (2, columns + 3))
    if missing:
        table[:, 5::7] = [[-1], [few]]
    q = queries(r, 2, 6, 1, D)
    lengths = [columns * ps, columns * ps - 5 * ps - 3]
    picked = cache.select_pages(q, ints(table), ints(lengths), budget, sink=sink, recent=recent).cpu().numpy()
    for b in range(2):
        n = -(-lengths[b] // ps)
        for h in range(hkv):
            hi, lo, top = (y.reshape(few, -1) for y in bounds(k[:, h:h + 1], ps))
            score = scores_of((hi, lo, top[:, 0]), q[b, 3 * h:3 * h + 3, 0].cpu().numpy())
            score = np.append(score, -np.inf)[np.where((table[b, :n] < 0) | (table[b, :n] >= few), few, table[b, :n])]
            want = np.full(budget, -1)
            w = ranked(score, budget, sink, recent)
            want[:len(w)] = w
            assert np.array_equal(picked[b, h], want), (b, h)
